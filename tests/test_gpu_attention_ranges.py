"""Attention over the 4-bit cache where magnitudes differ: between groups of dimensions, between keys, between queries
and scale.  References, tolerances' terms (u = 2^-24, A, W) and helpers are those of test_gpu_attention; here a result is
held to the magnitudes of its own group of dimensions (dimension d is of group d mod D/32), not to the head's largest."""
import math

import pytest
import torch

from test_gpu_attention import TYPES, U, close, fill, gen, half_step, ints, offsets, randn, ref_attention, ref_prompt, stored, tiny, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A(cuda_lib):
    from exl3_b200 import attention

    return attention


def check_groups(got, q, cache, slots, lens, scale=None):
    """check_attend with W and max |v| of each group by itself."""
    rows, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    share, G = heads // cache.kv_heads, dim // 32
    kv, vv = (values(*stored(c, s)) for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
    for r, (slot, n) in enumerate(zip(slots, lens)):
        for h in range(heads):
            for j in range(G):
                want, a, w, top = ref_attention(q[r, h:h + 1], kv[slot, h // share, :n], vv[slot, h // share, :n, j::G], n, scale)
                tol = (64 * a + 64) * U * top + half_step(got.dtype) * want.abs() + tiny(got.dtype)
                if got.dtype != torch.float32:
                    tol = tol + 2.0 ** -11 * w
                close(got[r, h:h + 1, j::G], want, tol, (r, h, n, j))


# a cluster to a row, shares (few and many parts), a CTA to a row
PATHS = [dict(rows=1, max_len=1024), dict(rows=2, max_len=8192), dict(rows=100, max_len=4160), dict(rows=257, max_len=1024)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (8, 1, 128), (8, 1, 64), (3, 1, 64)])
@pytest.mark.parametrize("path", PATHS, ids=lambda p: f"{p['rows']}x{p['max_len']}")
def test_small_groups_beside_large_ones(A, dtype, heads, kv, dim, path):
    """Value scales of one group up to 2^32 times those of another, from the first key on and from a later one on."""
    g = gen(dim + heads)
    G, n = dim // 32, 1000
    cache = A.Kv4Cache(2, kv, path["max_len"], dim)
    fill(cache, g)
    low, high = (0.02, 1e4) if dtype == torch.float16 else (1e-5, 6e4)
    size = torch.full((G,), low, device="cuda")
    size[1], size[-1] = high, (high if G == 2 else 1.0)
    for slot in range(2):
        x = torch.rand(cache.v_scales[slot].shape, generator=g, device="cuda") * 0.5 + 0.5
        big = torch.ones(path["max_len"], dtype=torch.bool, device="cuda") if slot == 0 else \
            torch.arange(path["max_len"], device="cuda") == 700
        cache.v_scales[slot] = torch.where(big[None, :, None], x * size, x * low).half()
    rows = path["rows"]
    q = randn(g, rows, heads, dim).to(dtype)
    slots = [r % 2 for r in range(rows)]
    got = cache.attend(q, ints(slots), ints([n - 1] * rows), ints([0, 1]))
    some = [r for r in range(rows) if r < 2 or r >= rows - 2]
    check_groups(got[some], q[some], cache, [slots[r] for r in some], [n] * len(some))


def one_hot(rows, heads, dim, size, dtype):
    q = torch.zeros((rows, heads, dim), device="cuda")
    q[:, torch.arange(heads), torch.arange(heads) * 5 % dim] = size
    return q.to(dtype)


@pytest.mark.parametrize("dtype,size,key", [
    (torch.float32, 2.0 ** 10, 2.0 ** -3), (torch.float32, 2.0 ** 24, 2.0 ** -3), (torch.float32, 2.0 ** 40, 2.0 ** -3),
    (torch.float32, 2.0 ** 100, 2.0 ** 3), (torch.bfloat16, 2.0 ** 26, 2.0 ** -3), (torch.bfloat16, 2.0 ** 90, 1.0),
    (torch.float16, 2.0 ** 15, 2.0 ** 15)])
@pytest.mark.parametrize("heads,dim", [(4, 128), (8, 128), (8, 64)])
@pytest.mark.parametrize("max_len", [1024, 8192])
def test_attend_scores_of_any_size(A, dtype, size, key, heads, dim, max_len):
    """Scores are exact (one product of powers of two and a code), so that the term in A falls away: the keys of the
    largest score share the result, however large it is."""
    g = gen(heads + dim)
    cache = A.Kv4Cache(1, 1, max_len, dim)
    fill(cache, g)
    cache.k_scales.fill_(key)
    q = one_hot(3, heads, dim, size, dtype)
    lens = [1, 77, 1000]
    got = cache.attend(q, ints([0] * 3), ints([n - 1 for n in lens]), ints([0]), scale=1.0)
    k, v = (values(*stored(c[0, 0], s[0, 0])) for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
    for r, n in enumerate(lens):
        want, _, w, top = ref_attention(q[r], k[:n], v[:n], n, 1.0)
        tol = 64 * U * top + half_step(dtype) * want.abs() + tiny(dtype)
        close(got[r], want, tol if dtype == torch.float32 else tol + 2.0 ** -11 * w, (r, n))


@pytest.mark.parametrize("dtype,size,key", [
    (torch.float16, 2.0 ** 15, 2.0 ** 4), (torch.float16, 2.0 ** 15, 2.0 ** 7), (torch.float16, 2.0 ** 15, 2.0 ** 8),
    (torch.bfloat16, 2.0 ** 20, 2.0 ** 3), (torch.bfloat16, 2.0 ** 40, 2.0 ** -17),
    (torch.float16, 2.0 ** 15, 2.0 ** 12), (torch.bfloat16, 2.0 ** 60, 2.0 ** 40)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("past", [0, 3000])
def test_prompt_large_scores(A, dtype, size, key, dim, past):
    """The same for prompts, whole and with their keys divided among CTAs, up to the documented 2^26; a row whose
    largest score is beyond that becomes NaN."""
    g = gen(dim + past)
    n = 300
    q = one_hot(n, 4, dim, size, dtype)
    k = (torch.randint(-7, 8, (n + past, 1, dim), generator=g, device="cuda") * key).to(dtype)
    k[0] = 7 * key                                          # the largest score is 7 size key for every row
    v = randn(g, n + past, 1, dim).to(dtype)
    got = A.prompt_attention(q, k, v, ints([0, n]), ints([0, n + past]), scale=1.0)
    if 7 * size * key > 2.0 ** 27:
        assert bool(got.isnan().all())
        return
    for h in range(4):
        want, _, w, _ = ref_attention(q[:, h], k[:, 0], v[:, 0], past, 1.0)
        tol = (1.5 * half_step(dtype) + 64 * U) * w + half_step(dtype) * want.abs() + 8 * tiny(dtype)
        close(got[:, h], want, tol, h)


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("past", [1000, 6000])
def test_prompt_scores_far_below_the_others(A, dtype, past):
    """Scores of -2^29 before ordinary ones: they have no weight, as in 64 bits."""
    g = gen(past)
    n, early = 40, past // 2
    q = randn(g, n, 4, 64).to(dtype)
    q[..., 0] = 2.0 ** 15
    k, v = randn(g, n + past, 1, 64).to(dtype), randn(g, n + past, 1, 64).to(dtype)
    k[..., 0] = 0
    k[:early, 0, 0] = -2.0 ** 14
    got = A.prompt_attention(q, k, v, ints([0, n]), ints([0, n + past]), scale=1.0)
    for h in range(4):
        # the score's term in A is that of the keys that have weight: q and k without dimension 0
        want, _, w, _ = ref_attention(q[:, h], k[early:, 0], v[early:, 0], past - early, 1.0)
        _, a, _, _ = ref_attention(q[:, h, 1:], k[early:, 0, 1:], v[early:, 0], past - early, 1.0)
        tol = (1.5 * half_step(dtype) + (64 * a + 64) * U) * w + half_step(dtype) * want.abs() + 8 * tiny(dtype)
        close(got[:, h], want, tol, h)


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("value", [-math.inf, math.inf, math.nan])
def test_prompt_queries_not_finite(A, dtype, value):
    """A query whose every score is -inf has no softmax: NaN, as with +inf and NaN; the other rows keep their results (to
    the tolerance: when the reference of a row's weights moves is decided for a warp's rows together)."""
    g = gen(51)
    n = 400
    q = randn(g, n, 4, 64).to(dtype)
    k, v = randn(g, n, 1, 64).to(dtype), randn(g, n, 1, 64).to(dtype)
    k[:, 0, 3] = k[:, 0, 3].abs() + 0.5
    bad = q.clone()
    rows = [0, 5, 127, 128, 300, 399]
    bad[rows, 2, 3] = value
    got = A.prompt_attention(bad, k, v, ints([0, n]), ints([0, n]))
    assert bool(got[rows, 2].isnan().all())
    want, tol = ref_prompt(q, k, v, [n], [(0, n)], 64 ** -0.5)
    got[rows, 2] = want[rows, 2].to(dtype)
    close(got, want, tol + half_step(dtype) * want.abs() + 8 * tiny(dtype))


@pytest.mark.parametrize("dtype,size,scale", [
    (torch.float32, 1e-25, 1e25), (torch.float32, 1e-30, 1e30), (torch.float32, 1e-36, 1e30), (torch.bfloat16, 1e-30, 1e30),
    (torch.float32, 1e20, 1e-20), (torch.bfloat16, 1e30, 1e-30), (torch.float16, 2.0 ** -18, 2.0 ** 18)])
@pytest.mark.parametrize("max_len", [512, 8192])
def test_attend_small_queries_and_large_scales(A, dtype, size, scale, max_len):
    g = gen(52)
    cache = A.Kv4Cache(2, 2, max_len, 128)
    fill(cache, g)
    cache.k_scales.mul_(4)
    q = (randn(g, 2, 8, 128) * size).to(dtype)
    lens = [500, 65]
    check_groups(cache.attend(q, ints([0, 1]), ints([n - 1 for n in lens]), ints([1, 0]), scale=scale), q, cache, [1, 0], lens, scale)


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (8, 2, 64)])
@pytest.mark.parametrize("max_len", [1024, 8192])
def test_attend_f32_rows_keep_their_digits(A, heads, kv, dim, max_len):
    """f32 rows as pairs of halves: small elements of a query beside a large one where the keys make up for it, and
    values 2^-21 of those of a key whose weight is below 2^-40; held to W instead of the largest value."""
    g = gen(dim)
    G, n = dim // 32, 900
    cache = A.Kv4Cache(1, kv, max_len, dim)
    fill(cache, g)
    cache.k_scales[..., 0], cache.k_scales[..., 1:] = 2.0 ** -10, 2.0 ** 10
    q = randn(g, 1, heads, dim)
    q[..., [d for d in range(dim) if d % G]] *= 2.0 ** -20
    scale = 2.0 ** 10 / dim ** 0.5
    check_groups(cache.attend(q, ints([0]), ints([n - 1]), ints([0]), scale=scale), q, cache, [0], [n], scale)

    cache.k_scales.fill_(2.0 ** -3)
    cache.v_scales.copy_(torch.rand(cache.v_scales.shape, generator=g, device="cuda") * 0.01 + 0.02)
    for at in (0, 500):
        c = A.Kv4Cache.from_tensors(*(t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)))
        c.v_scales[:, :, at] = 6e4
        c.k_codes[:, :, at] = 0x11                          # -7 everywhere
        q = torch.full((1, heads, dim), 0.5, device="cuda") + 0.1 * randn(g, 1, heads, dim)
        got = c.attend(q, ints([0]), ints([n - 1]), ints([0]), scale=1.0)
        for h in range(heads):
            k, v = (values(*stored(a[0, h // (heads // kv)], b[0, h // (heads // kv)]))[:n] for a, b in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)))
            want, a, w, _ = ref_attention(q[0, h:h + 1], k, v, n, 1.0)
            close(got[0, h:h + 1], want, (64 * a + 64) * U * w + half_step(torch.float32) * want.abs(), (at, h))


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1e-31, 1e-20])
def test_smallest_scales(A, dtype, scale):
    """All visible keys alike; rows that see nothing are zero as ever."""
    g = gen(53)
    q, k, v = randn(g, 200, 4, 64).to(dtype), randn(g, 3000, 1, 64).to(dtype), randn(g, 3000, 1, 64).to(dtype)
    for lens, spans in (([200], [(0, 3000)]), ([150, 50], [(0, 10), (10, 300)])):
        begin, end = zip(*spans)
        got = A.prompt_attention(q, k, v, offsets(lens), kv_begin=ints(begin), kv_end=ints(end), scale=scale)
        want, tol = ref_prompt(q, k, v, lens, spans, scale)
        close(got, want, tol + half_step(dtype) * want.abs() + 8 * tiny(dtype))
    cache = A.Kv4Cache(1, 1, 700, 64)
    fill(cache, g)
    check_groups(cache.attend(q[:3], ints([0] * 3), ints([0, 99, 650]), ints([0]), scale=scale), q[:3], cache, [0] * 3, [1, 100, 651], scale)

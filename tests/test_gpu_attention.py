"""The attention operators (exl3_b200.attention) against plain 64-bit forms.

Tolerances, with u = 2^-24 (half a step of f32) and e = half a step of the output's type:
  qk_norm_rope  norm: sum of D squares, rsqrt and three products, at most 10 u; cosine and sine: reduced
                angle below pi, 2 u, the function 2 u, the factor 1 u; product and fma 2 u.  Per element
                20 u (|a| + |b|) factor over its pair, and e |result|.
  cache         exact: codes and scales are defined by comparisons that floating point can decide.
  attend        score error of at most 32 u A, A = scale max_k sum |q k| (sums of D products and the group
                scales); it moves a weight by at most twice that; sums of a few thousand weights and
                products 64 u.  (64 A + 64) u max|v|, and e |result|.  Rows of a 16-bit type have each weight
                times its value scale rounded to a half: result = sum_k w_k (c_k - 8) with w_k off by at most
                2^-11 w_k (the offset is taken off the rounded weights), which sums to at most 2^-11 W,
                W = sum p |v|, and 2^-25 of the largest scale where w_k is below the normal halves (the
                largest scale seen is at 2^13 there, far above).
  prompt        weights rounded to the 16-bit type, half a step of each: e_in W, W = sum p |v|, half as
                much again for what the exponential and its argument are off; the score as above.
                1.5 e_in W + (64 A + 64) u W, and e |result|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def A(cuda_lib):
    from exl3_b200 import attention

    return attention


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):  # half a step of the type's subnormals
    return torch.finfo(t).tiny * torch.finfo(t).eps


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def offsets(lens):
    o = [0]
    for n in lens:
        o.append(o[-1] + n)
    return ints(o)


def close(got, want, tol, where=""):
    got, want = got.double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol))
    assert not bool(bad.any()), (where, int(bad.sum()), float((got - want).abs()[bad].max()))


# -- norm and rotary positions ----------------------------------------------------------------------

def ref_rope(x, w, pos, inv_freq, eps, interleaved, factor):
    """64-bit result and the sum |a| + |b| over each dimension's pair."""
    y = x.double()
    if w is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    r = 2 * len(inv_freq) if inv_freq is not None else 0
    out, size = y.clone(), y.abs()
    if r:
        th = (pos.double()[:, None] * inv_freq.double())[:, None]
        c, s = th.cos() * factor, th.sin() * factor
        one = torch.arange(r // 2, device=x.device) * (2 if interleaved else 1)
        two = one + (1 if interleaved else r // 2)
        out[..., one] = y[..., one] * c - y[..., two] * s
        out[..., two] = y[..., two] * c + y[..., one] * s
        size[..., one] = size[..., two] = (y[..., one].abs() + y[..., two].abs()) * factor
    return out, size


def check_rope(got, x, w, pos, inv_freq, eps, interleaved, factor):
    want, size = ref_rope(x, w, pos, inv_freq, eps, interleaved, factor)
    close(got, want, 20 * U * size + half_step(got.dtype) * want.abs() + tiny(got.dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,rotary,interleaved,rows,heads,kv", [
    (128, 128, False, 1, 16, 4), (128, 64, True, 77, 16, 4), (128, 32, False, 5, 12, 4), (64, 64, True, 33, 8, 8),
    (64, 16, False, 3, 10, 2), (128, 0, False, 9, 3, 1), (64, 64, False, 513, 1, 1)])
def test_rope(A, dtype, dim, rotary, interleaved, rows, heads, kv):
    g = gen(rows)
    qkv = (randn(g, rows, heads + 2 * kv, dim) * 2).to(dtype)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv]  # strided rows of one projection
    qw, kw = 1 + 0.1 * randn(g, dim), 1 + 0.1 * randn(g, dim)
    pos = torch.randint(0, 2_000_000, (rows,), generator=g, device="cuda").to(torch.int32)
    freq, factor = None, 1.0
    if rotary:
        f, factor = A.rope_frequencies(rotary, 1e6, 8.0 if rotary > 16 else 1.0, 32768)
        freq = torch.from_numpy(f).cuda()
    qo, ko = A.qk_norm_rope(q, k, pos, freq, qw, kw, eps=1e-6, interleaved=interleaved, attention_factor=factor)
    assert qo.dtype == ko.dtype == dtype
    check_rope(qo, q, qw, pos, freq, 1e-6, interleaved, factor)
    check_rope(ko, k, kw, pos, freq, 1e-6, interleaved, factor)


def test_rope_without_weights_in_place_and_mixed_types(A):
    g = gen(3)
    q, k = randn(g, 21, 6, 128), randn(g, 21, 2, 128)
    pos = ints([-1 if i % 5 == 4 else i * 1000 for i in range(21)])
    live = pos >= 0
    freq = torch.from_numpy(A.rope_frequencies(64)[0]).cuda()
    q16 = torch.full((21, 6, 128), 7.0, dtype=torch.float16, device="cuda")
    q0, k0 = q.clone(), k.clone()
    _, ko = A.qk_norm_rope(q, k, pos, freq, None, None, q_out=q16, k_out=k)
    assert ko is k
    check_rope(q16[live], q0[live], None, pos[live], freq, 0, False, 1.0)
    check_rope(k[live], k0[live], None, pos[live], freq, 0, False, 1.0)
    assert bool((q16[~live] == 7).all()) and torch.equal(k[~live], k0[~live])  # rows without a position: as they were
    only, none = A.qk_norm_rope(q0, None, pos.clamp(min=0), freq, k0[0, 0].contiguous(), out_dtype=torch.bfloat16)
    assert none is None
    check_rope(only, q0, k0[0, 0], pos.clamp(min=0), freq, 1e-6, False, 1.0)
    empty, _ = A.qk_norm_rope(q[:0], k[:0], pos[:0], freq)
    assert empty.shape == (0, 6, 128)


def test_rope_rows_of_zeros_and_not_finite(A):
    q = torch.zeros((3, 2, 64), device="cuda")
    q[1, 0, 5], q[2, 1, 7] = math.inf, math.nan
    w = torch.ones(64, device="cuda")
    out, _ = A.qk_norm_rope(q, None, ints([0, 1, 2]), torch.from_numpy(A.rope_frequencies(64)[0]).cuda(), w)
    assert bool((out[0] == 0).all()) and bool((out[1, 1] == 0).all()) and bool((out[2, 0] == 0).all())
    assert bool(out[1, 0, 5].isnan()) and bool(out[2, 1].isnan().all())


# -- the cache ------------------------------------------------------------------------------------------

def ref_quantise(x):
    """(code - 8 per dimension, scale per group [.., G] as f64) of rows [.., D], from the definition."""
    x = x.double()
    G = x.shape[-1] // 32
    xg = x.unflatten(-1, (32, G))
    top = xg.abs().amax(-2)
    s = (top.clamp(max=7 * 65504) / 7).half()
    s = torch.where((s.double() * 7 < top) & (s < 65504), (s.view(torch.int16) + 1).view(torch.float16), s)
    s = torch.where(top.isfinite(), s.double(), torch.nan)
    code = torch.where(s.unsqueeze(-2) > 0, torch.round(xg / s.unsqueeze(-2)), 0.0).clamp(-7, 7)
    return code.flatten(-2), s


def values(code, s):
    return (code.unflatten(-1, (32, s.shape[-1])) * s.unsqueeze(-2)).flatten(-2)


def stored(codes, scales):
    """(code - 8 [.., D], scale [.., G]) of a cache's memory."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double() - 8
    return c, scales.double()


def fill(cache, g, garbage=True):
    """Random codes and scales everywhere; with garbage, some scales not finite (set only where no test looks)."""
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device="cuda", dtype=torch.uint8))
        scales.copy_(torch.rand(scales.shape, generator=g, device="cuda") * 0.2 + 0.01)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,kv,rows", [(128, 4, 37), (64, 3, 130), (128, 1, 1)])
def test_append_then_read(A, dtype, dim, kv, rows):
    g = gen(dim + rows)
    cache = A.Kv4Cache(3, kv, 150, dim)
    assert cache.max_len == 192
    fill(cache, g)
    before = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    kvs = (randn(g, rows, 2 * kv, dim) * torch.logspace(-4, 3, rows, device="cuda")[:, None, None]).to(dtype)
    k, v = kvs[:, :kv], kvs[:, kv:]
    seq_slot = ints([2, 0])
    n0 = rows // 3
    lens = [n0, rows - n0]
    row_seq = ints([0] * n0 + [1] * (rows - n0))
    pos = list(range(n0)) + list(range(rows - n0))
    cache.append(k, v, row_seq, ints(pos), seq_slot)
    touched = torch.zeros((3, 192), dtype=torch.bool, device="cuda")
    touched[2, :n0] = touched[0, :rows - n0] = True
    at = (seq_slot.long()[row_seq.long()], slice(None), torch.tensor(pos, device="cuda"))
    for x, codes, scales, c0, s0 in ((k, cache.k_codes, cache.k_scales, *before[:2]),
                                     (v, cache.v_codes, cache.v_scales, *before[2:])):
        want_c, want_s = ref_quantise(x)
        got_c, got_s = stored(codes[at], scales[at])
        assert torch.equal(got_s, want_s) and torch.equal(got_c, want_c)
        keep = ~touched[:, None, :].expand(3, kv, 192)
        assert torch.equal(codes[keep], c0[keep]) and torch.equal(scales[keep], s0[keep])
    for out_type in TYPES:
        ko, vo = cache.read(seq_slot, offsets(lens), rows, dtype=out_type)
        assert torch.equal(ko, values(*ref_quantise(k)).to(out_type))
        assert torch.equal(vo, values(*ref_quantise(v)).to(out_type))


def test_append_edges(A):
    """Ties, saturated, zero, subnormal and not finite groups; rows that are skipped."""
    cache = A.Kv4Cache(1, 1, 64, 64)
    x = torch.zeros((8, 1, 64), device="cuda")
    x[0, 0, 0::2] = torch.tensor([3.5, 7, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5] * 4, device="cuda") * 0.25  # s = 0.25
    x[0, 0, 1::2] = torch.nextafter(x[0, 0, 0::2], torch.tensor(-1e9, device="cuda"))
    x[1, 0, 3], x[1, 0, 0] = 1e30, 458528.0
    x[2, 0, 4], x[2, 0, 5] = math.nan, 3.0
    x[3, 0, 6], x[3, 0, 7] = -math.inf, -3.0
    x[4, 0, 0], x[4, 0, 1] = 1e-42, 3e-7
    x[5, 0] = 1.0
    seq = ints([0, 0, 0, 0, 0, 0, 1, -1])
    pos = ints([0, 1, 2, 3, 63, 64, 5, 6])  # row 5: past the end; rows 6 and 7: no such sequence
    before = cache.k_codes.clone()
    cache.append(x, x, seq, pos, ints([0]))
    want_c, want_s = ref_quantise(x)
    for i, p in ((0, 0), (1, 1), (2, 2), (3, 3), (4, 63)):
        c, s = stored(cache.k_codes[0, 0, p], cache.k_scales[0, 0, p])
        assert torch.equal(s.nan_to_num(-1), want_s[i, 0].nan_to_num(-1)), i
        assert torch.equal(torch.where(s.isnan().repeat(32), 0.0, c), torch.where(s.isnan().repeat(32), 0.0, want_c[i, 0])), i
    assert torch.equal(cache.k_codes[0, 0, 4:63], before[0, 0, 4:63])
    k, _ = cache.read(ints([0]), ints([0, 4]), 4, dtype=torch.float32)
    assert bool(k[2, 0, 0::2].isnan().all()) and bool((k[2, 0, 1::2] == values(want_c, want_s)[2, 0, 1::2]).all())
    assert float(k[1, 0, 3]) == 7 * 65504.0


def test_read_rows_outside_the_cache(A):
    g = gen(5)
    cache = A.Kv4Cache(2, 2, 64, 128)
    fill(cache, g)
    k = torch.full((140, 2, 128), 5.0, device="cuda")
    v = k.clone()
    # sequence 0: 66 positions of a slot of 64; 1: empty; 2: no such slot; 3: three rows; the rest: left alone
    cache.read(ints([1, 0, 2, 0]), ints([0, 66, 66, 68, 71]), 140, k_out=k, v_out=v)
    c, s = stored(cache.k_codes, cache.k_scales)
    want = values(c, s).transpose(1, 2)
    assert torch.equal(k[:64], want[1].float()) and torch.equal(k[68:71], want[0, :3].float())
    assert bool((k[64:68] == 0).all()) and bool((v[64:68] == 0).all())
    assert bool((k[71:] == 5).all()) and bool((v[71:] == 5).all())


# -- attention ------------------------------------------------------------------------------------------

def ref_attention(q, k, v, first, scale):
    """One head in 64 bits: query i of q [n, D] sees keys 0 .. first + i.  (out, A, W, max |v|)."""
    n, m = len(q), len(k)
    q, k, v = q.double(), k.double(), v.double()
    seen = torch.arange(m, device=q.device) <= first + torch.arange(n, device=q.device)[:, None]
    s = torch.where(seen, q @ k.t() * scale, -torch.inf)
    size = torch.where(seen, q.abs() @ k.abs().t() * scale, 0.0)
    p = torch.where(seen.any(-1, keepdim=True), torch.softmax(s, -1), 0.0)
    a = size.amax(-1, keepdim=True) if m else torch.zeros(n, 1, device=q.device, dtype=torch.float64)
    return p @ v, a, p @ v.abs(), (v.abs().max() if m else torch.zeros((), device=q.device))


def check_attend(got, q, cache, slots, lens, scale=None):
    rows, heads, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    share = heads // cache.kv_heads
    kv, vv = (values(*stored(c, s)) for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
    for r, (slot, n) in enumerate(zip(slots, lens)):
        for h in range(heads):
            want, a, w, top = ref_attention(q[r, h:h + 1], kv[slot, h // share, :n], vv[slot, h // share, :n], n, scale)
            tol = (64 * a + 64) * U * top + half_step(got.dtype) * want.abs() + tiny(got.dtype)
            if got.dtype != torch.float32:
                tol = tol + 2.0 ** -11 * w
            close(got[r, h:h + 1], want, tol, (r, h, n))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim,lens", [
    (16, 4, 128, [1]), (16, 4, 128, [767]), (16, 4, 128, [1, 2, 63, 64, 65, 1000, 2049, 31]), (32, 4, 64, [5, 300, 128]),
    (8, 8, 128, [129, 15]), (12, 4, 128, [70, 200]), (10, 2, 64, [257]), (1, 1, 64, [3, 1]), (64, 2, 128, [100, 17])])
def test_attend(A, dtype, heads, kv, dim, lens):
    g = gen(heads + len(lens))
    n = len(lens)
    cache = A.Kv4Cache(n + 1, kv, max(lens) + 7, dim)
    fill(cache, g)
    slots = [(i * 5 + 1) % (n + 1) if (n + 1) % 5 else n - i for i in range(n)]
    for i, m in zip(slots, lens):  # what lies past the last visible position must not matter
        for s in (cache.k_scales, cache.v_scales):
            s[i, :, m:] = math.nan
            s[i, :, m + 1::2] = math.inf
    qkv = (randn(g, n, heads + 2, dim) * 1.5).to(dtype)
    q = qkv[:, :heads]
    got = cache.attend(q, ints(list(range(n))), ints([m - 1 for m in lens]), ints(slots))
    clean = A.Kv4Cache.from_tensors(cache.k_codes, cache.k_scales.nan_to_num(0, 0, 0), cache.v_codes,
                                    cache.v_scales.nan_to_num(0, 0, 0))
    check_attend(got, q, clean, slots, lens)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim,lens", [
    (16, 4, 128, [767]), (16, 4, 128, [1, 2, 63, 64, 65, 1000, 2049, 31]), (32, 4, 64, [5, 300, 128]), (8, 8, 128, [129, 15]),
    (10, 2, 64, [257, 4097]), (64, 2, 128, [100, 5000])])
def test_attend_in_a_long_cache(A, dtype, heads, kv, dim, lens):
    """Short contexts in a cache for long ones: the rows' tiles are cut into shares, not dealt to clusters."""
    g = gen(heads + len(lens) + 1)
    n = len(lens)
    cache = A.Kv4Cache(n, kv, 5120, dim)
    fill(cache, g)
    q = randn(g, n, heads, dim).to(dtype)
    got = cache.attend(q, ints(list(range(n))), ints([m - 1 for m in lens]), ints(list(range(n))[::-1]))
    check_attend(got, q, cache, list(range(n))[::-1], lens)


@pytest.mark.parametrize("n", [1, 64, 65, 449, 512, 513, 577, 4033, 4096])
def test_attend_at_the_edges_of_a_clusters_shares(A, n):
    g = gen(n)
    cache = A.Kv4Cache(2, 2, 4096, 64)
    fill(cache, g)
    q = randn(g, 3, 8, 64)
    # the last row sees nothing: its cluster has nothing to join
    got = cache.attend(q, ints([0, 1, 0]), ints([n - 1, 4095, -1]), ints([1, 0]))
    check_attend(got[:2], q[:2], cache, [1, 0], [n, 4096])
    assert bool((got[2] == 0).all())


def test_attend_long_and_many_rows(A):
    """A context long enough to be split many ways, and more rows than the GPU has places."""
    g = gen(11)
    cache = A.Kv4Cache(2, 2, 20000, 128)
    fill(cache, g)
    q = randn(g, 1, 8, 128)
    check_attend(cache.attend(q, ints([0]), ints([19990]), ints([1])), q, cache, [1], [19991])
    lens = [int(x) for x in torch.randint(1, 400, (150,), generator=g, device="cuda")]
    q = randn(g, 150, 8, 128).half()
    got = cache.attend(q, ints([i % 2 for i in range(150)]), ints([m - 1 for m in lens]), ints([1, 0]))
    check_attend(got, q, cache, [1 - i % 2 for i in range(150)], lens)


def test_attend_as_many_rows_as_are_cut_into_shares(A):
    g = gen(22)
    cache = A.Kv4Cache(256, 1, 128, 128)
    fill(cache, g)
    lens = [int(x) for x in torch.randint(1, 129, (256,), generator=g, device="cuda")]
    q = randn(g, 256, 2, 128)
    order = torch.randperm(256, generator=g, device="cuda").to(torch.int32)
    got = cache.attend(q, ints(list(range(256))), ints([n - 1 for n in lens]), order)
    check_attend(got, q, cache, order.tolist(), lens)


def test_attend_more_rows_than_are_cut_into_shares(A):
    """Above 256 rows a CTA takes a row whole; rows of no position and of no sequence among them."""
    g = gen(21)
    cache = A.Kv4Cache(3, 2, 256, 64)
    fill(cache, g)
    lens = [int(x) for x in torch.randint(0, 256, (300,), generator=g, device="cuda")]
    q = randn(g, 300, 6, 64).bfloat16()
    out = torch.full((300, 6, 64), 7.0, device="cuda").bfloat16()
    seq = [i % 4 - (1 if i % 50 == 49 else 0) * 8 for i in range(300)]  # 3: no such slot; negative: no sequence
    cache.attend(q, ints(seq), ints([n - 1 for n in lens]), ints([2, 0, 1, 9]), out=out)
    dead = [i for i in range(300) if seq[i] < 0]
    zero = [i for i in range(300) if seq[i] == 3 or (seq[i] >= 0 and lens[i] == 0)]
    live = [i for i in range(300) if i not in dead and i not in zero]
    assert bool((out[dead] == 7).all()) and bool((out[zero] == 0).all())
    check_attend(out[live], q[live], cache, [[2, 0, 1][seq[i]] for i in live], [lens[i] for i in live])


def test_attend_rows_that_see_nothing(A):
    g = gen(6)
    cache = A.Kv4Cache(2, 4, 128, 128)
    fill(cache, g)
    q = randn(g, 6, 16, 128)
    out = torch.full((6, 16, 128), 9.0, device="cuda")
    # row 0: no position; 1: ordinary; 2: no such slot; 3 and 4: no such sequence; 5: past the end, the whole slot
    cache.attend(q, ints([0, 1, 2, -1, 3, 1]), ints([-1, 40, 3, 3, 3, 1000]), ints([0, 1, 7]), out=out)
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all())
    assert bool((out[3] == 9).all()) and bool((out[4] == 9).all())
    check_attend(out[[1, 5]], q[[1, 5]], cache, [1, 1], [41, 128])


def test_attend_extreme_values(A):
    """Scores of hundreds, scales from the smallest to the largest half, queries of any size."""
    g = gen(8)
    cache = A.Kv4Cache(1, 2, 128, 128)
    fill(cache, g)
    cache.k_scales.mul_(8)
    q = randn(g, 3, 8, 128) * torch.tensor([20.0, 1e-6, 1e-30], device="cuda")[:, None, None]
    check_attend(cache.attend(q, ints([0, 0, 0]), ints([99, 99, 99]), ints([0])), q, cache, [0] * 3, [100] * 3)
    cache.v_scales.copy_(torch.logspace(-7, 4.5, 128, device="cuda")[None, None, :, None].expand_as(cache.v_scales))
    cache.k_scales.copy_(torch.rand(cache.k_scales.shape, generator=g, device="cuda") * 0.1)
    q = randn(g, 1, 8, 128)
    for n in (1, 10, 40, 128):  # early positions: the smallest values
        check_attend(cache.attend(q, ints([0]), ints([n - 1]), ints([0])), q, cache, [0], [n])
    cache.v_scales.copy_(cache.v_scales.flip(2))
    for n in (1, 40, 128):
        check_attend(cache.attend(q, ints([0]), ints([n - 1]), ints([0])), q, cache, [0], [n])
    cache.k_scales[0, 0, 3] = math.nan  # a visible NaN reaches its own head group and no other
    out = cache.attend(q, ints([0]), ints([9]), ints([0]))
    assert bool(out[0, :4].isnan().all()) and bool(out[0, 4:].isfinite().all())
    q[0, 5, 0] = math.nan
    out = cache.attend(q, ints([0]), ints([2]), ints([0]))
    assert bool(out[0, 5].isnan().all()) and bool(out[0, :5].isfinite().all()) and bool(out[0, 6:].isfinite().all())


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("dim,value", [(128, math.nan), (64, math.inf)])
def test_attend_a_group_of_values_not_finite(A, dtype, dim, value):
    """A NaN among the visible values reaches the dimensions of its group; the others are as exact as ever."""
    g = gen(23)
    cache = A.Kv4Cache(1, 2, 256, dim)
    fill(cache, g)
    G = dim // 32
    cache.v_scales[0, 0, 5, 1] = value
    q = randn(g, 3, 8, dim).to(dtype)
    clean = A.Kv4Cache.from_tensors(cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales.nan_to_num(0, 0, 0))
    at = (ints([0, 0, 0]), ints([199, 6, 4]), ints([0]))
    got, want = cache.attend(q, *at), clean.attend(q, *at)
    d = torch.arange(dim, device="cuda") % G == 1
    # row 2 does not see position 5; heads 4 .. 7 read the other K/V head
    assert not bool(got[:2, :4][..., d].isfinite().any())
    got[:2, :4] = torch.where(d, want[:2, :4], got[:2, :4])
    check_attend(got, q, clean, [0, 0, 0], [200, 7, 5])


def ref_prompt(q, k, v, q_lens, kv_spans, scale):
    outs, tols = [], []
    heads, share = q.shape[1], q.shape[1] // k.shape[1]
    e_in, at = half_step(q.dtype), 0
    for n, (b, e) in zip(q_lens, kv_spans):
        for h in range(heads):
            want, a, w, _ = ref_attention(q[at:at + n, h], k[b:e, h // share], v[b:e, h // share], e - b - n, scale)
            outs.append(want)
            tols.append(1.5 * e_in * w + (64 * a + 64) * U * w)
        at += n
    def pack(parts):
        return torch.cat([torch.stack(parts[i * heads:(i + 1) * heads], 1) for i in range(len(q_lens))])
    return pack(outs), pack(tols)


def check_prompt(got, q, k, v, q_lens, kv_spans, scale=None):
    want, tol = ref_prompt(q, k, v, q_lens, kv_spans, q.shape[2] ** -0.5 if scale is None else scale)
    close(got[:len(want)], want, tol + half_step(got.dtype) * want.abs() + tiny(q.dtype) * 8, q_lens)


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("heads,kv,dim,q_lens,past", [
    (16, 4, 128, [1], 0), (16, 4, 128, [37], 0), (16, 4, 128, [128, 1, 0, 65, 200], 0), (16, 4, 128, [512, 1, 64], 300),
    (32, 4, 64, [130, 7], 0), (8, 8, 128, [257, 128], 0), (8, 8, 64, [300], 77), (12, 4, 128, [100, 31], 5),
    (10, 2, 64, [66], 129), (1, 1, 128, [700], 0), (64, 2, 128, [50], 0), (6, 2, 128, [129], 1000), (7, 1, 64, [40], 0)])
def test_prompt(A, dtype, heads, kv, dim, q_lens, past):
    g = gen(heads + dim + len(q_lens))
    rows, kv_lens = sum(q_lens), [n + past if n else 0 for n in q_lens]
    q = (randn(g, rows, heads, dim) * 1.5).to(dtype)
    k, v = (randn(g, sum(kv_lens), kv, dim).to(dtype) for _ in range(2))
    ko = offsets(kv_lens).tolist()
    got = A.prompt_attention(q, k, v, offsets(q_lens), ints(ko))
    check_prompt(got, q, k, v, q_lens, list(zip(ko, ko[1:])))
    got = A.prompt_attention(q, k, v, offsets(q_lens), ints(ko), out=torch.empty_like(q, dtype=torch.float32), scale=0.05)
    check_prompt(got, q, k, v, q_lens, list(zip(ko, ko[1:])), 0.05)


def test_prompt_rows_that_see_nothing_and_rows_behind(A):
    """More queries than keys, no keys at all, and rows behind the last sequence."""
    g = gen(9)
    q = randn(g, 300, 8, 128).half()
    k, v = randn(g, 90, 2, 128).half(), randn(g, 90, 2, 128).half()
    out = torch.full((300, 8, 128), 3.0, device="cuda").half()
    q_lens, spans = [140, 10, 70], [(0, 5), (5, 5), (5, 90)]
    A.prompt_attention(q, k, v, offsets(q_lens), kv_begin=ints([0, 5, 5]), kv_end=ints([5, 5, 90]), out=out)
    check_prompt(out, q, k, v, q_lens, spans)
    assert bool((out[:135] == 0).all()) and bool((out[140:150] == 0).all()) and bool((out[220:] == 3).all())
    none = A.prompt_attention(q, k[:0], v[:0], ints([0, 300]), ints([0, 0]))
    assert bool((none == 0).all())


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_prompt_not_finite_where_masked(A, value):
    """Keys and values that a query does not see never reach it; what it sees does."""
    g = gen(10)
    n = 200
    q = randn(g, n, 4, 128).half()
    k, v = randn(g, n + 100, 1, 128).half(), randn(g, n + 100, 1, 128).half()
    clean = A.prompt_attention(q, k, v, ints([0, n]), ints([0, n]))
    k2, v2 = k.clone(), v.clone()
    k2[n:], v2[n:] = value, value                   # behind the sequence
    v2[150, 0, 7] = value                           # one channel of a later value
    k2[170] = math.nan                              # a later key
    got = A.prompt_attention(q, k2, v2, ints([0, n]), ints([0, n]))
    assert torch.equal(got[:150], clean[:150])
    keep = [d for d in range(128) if d != 7]
    assert torch.equal(got[150:170][..., keep], clean[150:170][..., keep])
    seven = got[150:170, :, 7]
    assert bool(seven.isnan().all()) if math.isnan(value) else bool((seven == value).all())
    assert bool(got[170:].isnan().all())


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("heads,kv,dim,q_lens,past", [
    (16, 4, 128, [1], 20000), (16, 4, 128, [130], 5001), (8, 2, 64, [3, 100, 1], 2500), (2, 2, 128, [300, 17], 1900),
    (16, 4, 128, [512], 1500)])
def test_prompt_keys_divided_among_ctas(A, dtype, heads, kv, dim, q_lens, past):
    """Few query rows behind long starts: the keys of a block are shared and the parts joined; without scratch
    a block keeps its keys."""
    g = gen(past + heads)
    rows, kv_lens = sum(q_lens), [n + past * (i + 1) // len(q_lens) for i, n in enumerate(q_lens)]
    assert A.prompt_scratch_bytes(rows, len(q_lens), sum(kv_lens), heads, kv, dim) > 0
    q = (randn(g, rows, heads, dim) * 1.5).to(dtype)
    k, v = (randn(g, sum(kv_lens), kv, dim).to(dtype) for _ in range(2))
    ko = offsets(kv_lens)
    spans = list(zip(ko.tolist(), ko.tolist()[1:]))
    out = torch.full((rows + 3, heads, dim), 5.0, device="cuda").to(dtype)
    padded = torch.cat((q, q.new_zeros(3, heads, dim)))
    A.prompt_attention(padded, k, v, offsets(q_lens), ko, out=out)
    check_prompt(out, q, k, v, q_lens, spans)
    assert bool((out[rows:] == 5).all())
    whole = A.prompt_attention(q, k, v, offsets(q_lens), ko, scratch=torch.empty(0, dtype=torch.uint8, device="cuda"))
    check_prompt(whole, q, k, v, q_lens, spans)


def test_prompt_divided_keys_not_finite(A):
    """The same rules for what is seen and what is not when a block's keys are shared."""
    g = gen(31)
    n, m = 100, 4000
    q = randn(g, n, 4, 128).bfloat16()
    k, v = randn(g, m, 1, 128).bfloat16(), randn(g, m, 1, 128).bfloat16()
    v[m - 40, 0, 3] = math.inf      # seen by the last 40 rows
    v[m - 20, 0, 3] = -math.inf     # and this by the last 20
    v[100, 0, 9] = math.nan         # seen by all, far from the end
    clean = v.clone()
    clean[m - 40, 0, 3] = clean[m - 20, 0, 3] = clean[100, 0, 9] = 0
    got = A.prompt_attention(q, k, v, ints([0, n]), ints([0, m]))
    want = A.prompt_attention(q, k, clean, ints([0, n]), ints([0, m]))
    keep = [d for d in range(128) if d not in (3, 9)]
    assert torch.equal(got[..., keep], want[..., keep]) and bool(got[..., 9].isnan().all())
    assert torch.equal(got[:60, :, 3], want[:60, :, 3])
    assert bool((got[61:80, :, 3] == math.inf).all()) and bool(got[81:, :, 3].isnan().all())
    none = A.prompt_attention(q, k[:30], v[:30], ints([0, n]), ints([0, 30]))
    assert bool((none[:70] == 0).all())


def test_prompt_long_flat_tail(A):
    """One strong key before 20000 weak ones, each 2^-26 of it: together they move the result, and no part of
    them is lost to the 16-bit weights."""
    n = 20001
    k = torch.zeros((n, 1, 64), device="cuda").half()
    k[0, 0, 0] = 8.0
    v = torch.zeros((n, 1, 64), device="cuda").half()
    v[0], v[1:] = 1.0, 16384.0
    q = torch.zeros((n, 1, 64), device="cuda").half()
    q[:, :, 0] = 1.0
    scale = 26 * math.log(2) / 8
    got = A.prompt_attention(q=q[-200:], k=k, v=v, q_offsets=ints([0, 200]), kv_offsets=ints([0, n]), scale=scale,
                             out=torch.empty((200, 1, 64), device="cuda"))
    check_prompt(got, q[-200:], k, v, [200], [(0, n)], scale)


def test_prompt_many_sequences_and_rows_before_the_first(A):
    """More sequences than a warp has lanes, empty ones among them; rows before the first one are left alone."""
    g = gen(17)
    lens = [(i * 7) % 40 for i in range(75)]
    q_offs = torch.tensor([9] + lens, device="cuda").cumsum(0).to(torch.int32)
    rows = int(q_offs[-1])
    kv_lens = [n + (i % 3) * 50 if n else 0 for i, n in enumerate(lens)]
    ko = offsets(kv_lens)
    q = randn(g, rows, 8, 64).half()
    k, v = randn(g, sum(kv_lens), 2, 64).half(), randn(g, sum(kv_lens), 2, 64).half()
    out = torch.full((rows, 8, 64), 4.0, device="cuda").half()
    A.prompt_attention(q, k, v, q_offs, ko, out=out)
    assert bool((out[:9] == 4).all())
    check_prompt(out[9:], q[9:], k, v, lens, list(zip(ko.tolist(), ko.tolist()[1:])))


def test_captured_read_and_prompt_with_other_lengths(A):
    """A captured step replayed for other lengths of the same capacity: offsets are read on the device."""
    g = gen(18)
    cache = A.Kv4Cache(3, 2, 320, 128)
    fill(cache, g)
    cap_q, cap_kv = 200, 900
    q = randn(g, cap_q, 8, 128).half()
    slots, q_offs, kv_offs = ints([2, 0, 1]), ints([0, 10, 20, 30]), ints([0, 10, 20, 30])
    k, v = (torch.zeros((cap_kv, 2, 128), device="cuda").half() for _ in range(2))
    out = torch.zeros((cap_q, 8, 128), device="cuda").half()
    stream = torch.cuda.Stream()

    def step():
        cache.read(slots, kv_offs, cap_kv, k_out=k, v_out=v)
        A.prompt_attention(q, k, v, q_offs, kv_offs, out=out)

    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for lens, kv_lens in (([1, 150, 3], [300, 200, 3]), ([0, 0, 200], [0, 0, 320]), ([66, 65, 64], [66, 320, 100])):
        q_offs.copy_(offsets(lens))
        kv_offs.copy_(offsets(kv_lens))
        graph.replay()
        o = offsets(kv_lens).tolist()
        check_prompt(out, q, k, v, lens, list(zip(o, o[1:])))


def test_prompt_in_a_slot_cache_and_strided(A):
    """Keys in fp16 slots [slots][kv][max_len][D], queries as columns of a packed projection."""
    g = gen(12)
    slots, kv, max_len, dim, heads = 3, 4, 160, 128, 16
    kc, vc = randn(g, slots, kv, max_len, dim).half(), randn(g, slots, kv, max_len, dim).half()
    rows = slots * kv * max_len - (kv - 1) * max_len
    kview, vview = (t.as_strided((rows, kv, dim), (dim, max_len * dim, 1)) for t in (kc, vc))
    q_lens, lens, order = [70, 1, 30], [150, 97, 30], [2, 0, 1]
    proj = randn(g, 101, heads + 2 * kv, dim).half()
    q = proj[:, :heads]
    begin = [s * kv * max_len for s in order]
    out = torch.zeros((101, heads + 1, dim), device="cuda")[:, :heads]
    A.prompt_attention(q, kview, vview, offsets(q_lens), kv_begin=ints(begin),
                       kv_end=ints([b + n for b, n in zip(begin, lens)]), out=out)
    check_prompt(out, q, kview, vview, q_lens, [(b, b + n) for b, n in zip(begin, lens)])


def test_layer_in_4_bits(A):
    """The operators together, as a layer runs them: a ragged prefill step through norm, cache, read and
    prompt attention, then captured decode steps through norm, cache and attend, replayed at later
    positions.  Both forms are held to 64-bit attention over what the cache holds."""
    g = gen(13)
    heads, kv, dim, max_len = 16, 4, 128, 256
    cache = A.Kv4Cache(4, kv, max_len, dim)
    freq = torch.from_numpy(A.rope_frequencies(dim, 1e7)[0]).cuda()
    qw, kw = 1 + 0.1 * randn(g, dim), 1 + 0.1 * randn(g, dim)
    lens, slots = [100, 1, 63], [3, 0, 2]
    total = sum(lens)
    seq_slot, kv_offs = ints(slots), offsets(lens)
    row_seq = ints([s for s, n in enumerate(lens) for _ in range(n)])
    row_pos = ints([i for n in lens for i in range(n)])
    qkv = randn(g, total, heads + 2 * kv, dim)
    q16 = torch.empty((total, heads, dim), dtype=torch.float16, device="cuda")
    q16, k32 = A.qk_norm_rope(qkv[:, :heads], qkv[:, heads:heads + kv], row_pos, freq, qw, kw, q_out=q16)
    cache.append(k32, qkv[:, heads + kv:], row_seq, row_pos, seq_slot)
    k, v = cache.read(seq_slot, kv_offs, total)
    out = A.prompt_attention(q16, k, v, kv_offs, kv_offs)
    o = kv_offs.tolist()
    check_prompt(out, q16, k, v, lens, list(zip(o, o[1:])))

    one, new = ints([0, 1, 2]), torch.empty((3, heads + 2 * kv, dim), device="cuda")
    pos = ints(lens)
    result = torch.empty((3, heads, dim), device="cuda")
    qs = torch.empty((3, heads, dim), device="cuda")

    def step():
        _, kr = A.qk_norm_rope(new[:, :heads], new[:, heads:heads + kv], pos, freq, qw, kw, q_out=qs)
        cache.append(kr, new[:, heads + kv:], one, pos, seq_slot)
        cache.attend(qs, one, pos, seq_slot, out=result)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    new.copy_(randn(g, 3, heads + 2 * kv, dim))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for t in range(3):
        new.copy_(randn(g, 3, heads + 2 * kv, dim))
        pos.copy_(ints([n + t for n in lens]))
        graph.replay()
        check_attend(result, qs, cache, slots, [n + t + 1 for n in lens])


@pytest.mark.parametrize("dtype", TYPES)
def test_native_and_python_calls_agree(A, dtype):
    """The native module and the Python functions, which take the calls that it leaves, launch the same."""
    g = gen(31)
    qkv = randn(g, 6, 16, 64).to(dtype)
    q, k, v = qkv[:, :8], qkv[:, 8:12], qkv[:, 12:]
    pos, seq, slots = ints([3, 4, 5, 0, 1, 2]), ints([0, 0, 0, 1, 1, 1]), ints([1, 0])
    inv, w = torch.tensor(A.rope_frequencies(32)[0], device="cuda"), randn(g, 64)
    caches = [A.Kv4Cache(2, 4, 64, 64) for _ in range(2)]
    got = []
    for cache, form in zip(caches, (lambda f: f, lambda f: f.__wrapped__)):
        r = list(form(A.qk_norm_rope)(q, k, pos, inv, w, None, eps=1e-5, interleaved=True, attention_factor=1.5,
                                      out_dtype=torch.float32))
        r += form(A.qk_norm_rope)(q, k, pos, q_out=torch.empty_like(q), k_weight=w)
        assert form(A.Kv4Cache.append)(cache, k, v, seq, pos, slots) is None
        r += form(A.Kv4Cache.read)(cache, slots, ints([0, 6, 9]), 9, dtype)
        out = torch.zeros(6, 8, 64, device="cuda", dtype=dtype)
        same = form(A.Kv4Cache.attend)(cache, q, seq, pos, slots, 0.2, out=out)
        assert same is out
        r += [out, form(A.Kv4Cache.attend)(cache, q, seq, pos, slots, scratch=torch.empty(1 << 20, dtype=torch.uint8, device="cuda"))]
        if dtype != torch.float32:
            kw = dict(kv_begin=ints([0, 3]), kv_end=ints([3, 6]))
            r += [form(A.prompt_attention)(q, k, v, ints([0, 3, 6]), **kw),
                  form(A.prompt_attention)(q, k, v, ints([0, 3, 6]), ints([0, 3, 6]), scale=1, out=torch.empty(6, 8, 64, device="cuda"))]
        r += [cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales]
        got.append(r)
    for a, b in zip(*got):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_cache_past_32_bits(A):
    """Slots whose codes begin beyond 4 GiB, rows at the end of a million positions; all the others are zeros."""
    g = gen(41)
    length, n = 1 << 20, 70
    cache = A.Kv4Cache(9, 8, length, 128)
    k, v = randn(g, n, 8, 128), randn(g, n, 8, 128)
    slots = ints([8, 7])
    cache.append(k, v, ints([0] * n), torch.arange(length - n, length, device="cuda").to(torch.int32), slots)
    cache.append(k, v, ints([1] * n), torch.arange(n, device="cuda").to(torch.int32), slots)
    kq, vq = (values(*stored(c[8, :, -n:], s[8, :, -n:])) for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
    k1, v1 = cache.read(ints([7]), offsets([n + 3]), n + 3, torch.float32)
    assert torch.equal(k1[:n], kq.transpose(0, 1).float()) and torch.equal(v1[:n], vq.transpose(0, 1).float())
    assert not bool(k1[n:].any()) and not bool(v1[n:].any())
    q = randn(g, 2, 8, 128) * 8
    got = cache.attend(q, ints([0, 1]), ints([length - 1, n - 1]), slots)
    s = torch.einsum("rhd,hnd->rhn", q.double(), kq) * 128 ** -0.5
    rest = torch.tensor([length - n, 0], dtype=torch.float64, device="cuda")[:, None, None]  # scores of zero
    top = s.amax(-1, keepdim=True).clamp_min(0)
    e = (s - top).exp()
    want = torch.einsum("rhn,hnd->rhd", e / (e.sum(-1, keepdim=True) + rest * (-top).exp()), vq)
    size = torch.einsum("rhd,hnd->rhn", q.double().abs(), kq.abs()).amax(-1, keepdim=True) * 128 ** -0.5
    close(got, want, (64 * size + 64) * U * vq.abs().max())


def test_rows_past_32_bits(A):
    """Rows 2^27 elements apart: queries, keys, values and outputs as columns of one buffer of 5.4 billion elements."""
    g = gen(42)
    n, stride = 40, 1 << 27
    flat = torch.empty(n * stride, dtype=torch.float16, device="cuda")

    def columns(at, heads):
        return flat.as_strided((n, heads, 64), (stride, 64, 1), at)

    q, k, v, out = columns(0, 8), columns(512, 2), columns(640, 2), columns(1024, 8)
    for t in (q, k, v):
        t.copy_(randn(g, *t.shape))
    pos = torch.arange(n, device="cuda").to(torch.int32)
    A.prompt_attention(q, k, v, offsets([n]), offsets([n]), out=out)
    check_prompt(out, q, k, v, [n], [(0, n)])
    inv = torch.tensor(A.rope_frequencies(64)[0], device="cuda")
    A.qk_norm_rope(q, k, pos, inv, q_out=out, k_out=columns(2048, 2))
    check_rope(out, q, None, pos, inv, 1e-6, False, 1.0)
    check_rope(columns(2048, 2), k, None, pos, inv, 1e-6, False, 1.0)
    cache = A.Kv4Cache(1, 2, n, 64)
    cache.append(k, v, pos * 0, pos, ints([0]))
    cache.read(ints([0]), offsets([n]), n, k_out=columns(4096, 2), v_out=columns(4224, 2))
    kq, vq = (values(*stored(c[0, :, :n], s[0, :, :n])) for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
    assert torch.equal(columns(4096, 2), kq.transpose(0, 1).half()) and torch.equal(columns(4224, 2), vq.transpose(0, 1).half())
    cache.attend(q, pos * 0, pos, ints([0]), out=out)
    check_attend(out, q, cache, [0] * n, list(range(1, n + 1)))


def test_calls_on_two_streams_at_once(A):
    """Calls that overlap on two streams, given as arguments, leave each other's results alone."""
    g = gen(14)
    cache = A.Kv4Cache(2, 4, 4096, 128)
    fill(cache, g)
    q = [randn(g, 2, 16, 128) for _ in range(2)]
    seqs, slots = ints([0, 1]), ints([0, 1])
    pos = [ints([4000, 77]), ints([3, 2500])]
    want = [cache.attend(q[i], seqs, pos[i], slots) for i in range(2)]
    qp, kp = randn(g, 600, 4, 128).half(), randn(g, 600, 2, 128).half()
    offs = ints([0, 200, 600])
    want_p = A.prompt_attention(qp, kp, kp, offs, offs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            got[i].append((cache.attend(q[i], seqs, pos[i], slots, stream=s),
                           A.prompt_attention(qp, kp, kp, offs, offs, stream=s)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, p in got[i]:
            assert torch.equal(a, want[i]) and torch.equal(p, want_p)

"""Attention over the 4-bit cache on each of its ways: a cluster of CTAs to a row, the rows' tiles in equal shares (joined by
many threads to a row, or by few), and a CTA to a row.  Rows that see nothing or belong to nothing between ordinary ones,
cached positions that are not finite, and calls that run at the same time with scratch of their own.  Tolerances are those
of test_gpu_attention."""
import math

import pytest
import torch

from test_gpu_attention import TYPES, check_attend, check_prompt, fill, gen, ints, offsets, randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def A(cuda_lib):
    from exl3_b200 import attention

    return attention


# (rows, max_len) with 4 K/V heads: clusters; shares, more than 8 to a row; shares, fewer; a long cache's; whole rows
PATHS = [(6, 1024), (6, 8192), (40, 1024), (40, 8192), (300, 1024)]
path = pytest.mark.parametrize("rows,max_len", PATHS, ids=[f"{r}x{m}" for r, m in PATHS])


def split(rows, max_len, ys=4):
    """The way that a call takes, by the sizes that the operator decides by (kept here to hold the list above to it)."""
    if rows > 256:
        return "whole"
    if max_len <= 4096 and rows * ys * 8 <= 3 * 148:
        return "clusters"
    return "many shares" if 3 * 148 // ys > 8 * rows else "few shares"


def test_the_list_covers_every_way():
    assert [split(*p) for p in PATHS] == ["clusters", "many shares", "few shares", "few shares", "whole"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim", [(16, 128), (32, 64)])
@path
def test_rows_of_every_kind(A, dtype, heads, dim, rows, max_len):
    """Ordinary rows, rows of no position, of no slot and of no sequence in turn; what lies behind the last visible
    position is not finite."""
    g = gen(rows + dim)
    cache = A.Kv4Cache(3, 4, max_len, dim)
    fill(cache, g)
    q = randn(g, rows, heads, dim).to(dtype)
    lens = [1 + int(x) for x in torch.randint(0, max_len - 1, (rows,), generator=g, device="cuda")]
    lens[0], slot = max_len, [r % 3 for r in range(rows)]
    most = [max(n for n, s in zip(lens, slot) if s == k) for k in range(3)]
    for k in range(3):
        for s in (cache.k_scales, cache.v_scales):
            s[k, :, most[k]:] = math.nan
            s[k, :, most[k] + 1::2] = math.inf
    pos, seq = [n - 1 for n in lens], list(slot)
    none, nowhere, nobody = range(1, rows, 7), range(3, rows, 7), range(5, rows, 7)
    for r in none:
        pos[r] = -1
    for r in nowhere:
        seq[r] = 3 + r % 2
    for r in nobody:
        seq[r] = -1 if r % 2 else 5
    out = torch.full((rows + 2, heads, dim), 9.0, device="cuda").to(dtype)
    cache.attend(q, ints(seq), ints(pos), ints([0, 1, 2, 7, -1]), out=out[:rows])
    assert bool((out[[*none, *nowhere]] == 0).all())
    assert bool((out[[*nobody, rows, rows + 1]] == 9).all())
    live = [r for r in range(rows) if r not in none and r not in nowhere and r not in nobody]
    clean = A.Kv4Cache.from_tensors(cache.k_codes, cache.k_scales.nan_to_num(0, 0, 0), cache.v_codes,
                                    cache.v_scales.nan_to_num(0, 0, 0))
    if rows > 60:
        live = live[:10] + live[-10:]
    check_attend(out[live], q[live], clean, [slot[r] for r in live], [lens[r] for r in live])


@path
def test_no_row_sees_anything(A, rows, max_len):
    cache = A.Kv4Cache(1, 4, max_len, 128)
    out = torch.full((rows, 16, 128), 9.0, device="cuda")
    seq = [r % 3 for r in range(rows)]
    cache.attend(torch.zeros_like(out), ints(seq), ints([-1] * rows), ints([0, 5]), out=out)
    dead = [r for r in range(rows) if seq[r] == 2]
    assert bool((out[dead] == 9).all()) and bool((out[[r for r in range(rows) if seq[r] != 2]] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@path
def test_positions_not_finite(A, dtype, rows, max_len):
    """A key that is not finite makes its head's rows NaN, a value that is not its group of dimensions; rows that do
    not see them, the other heads and the other groups are as exact as ever."""
    g = gen(rows)
    cache = A.Kv4Cache(2, 4, max_len, 128)
    fill(cache, g)
    at = max_len - 70
    cache.k_scales[0, 1, at, 2] = math.nan
    cache.v_scales[0, 2, at, 1] = math.nan
    cache.v_scales[0, 3, at, 3] = math.inf                  # none that append() writes: inf or NaN
    clean = A.Kv4Cache.from_tensors(cache.k_codes, cache.k_scales.nan_to_num(0, 0, 0), cache.v_codes,
                                    cache.v_scales.nan_to_num(0, 0, 0))
    q = randn(g, rows, 16, 128).to(dtype)
    lens = [(max_len, at, at + 1, max_len)[r % 4] for r in range(rows)]
    slots = [0 if r % 4 < 3 else 1 for r in range(rows)]
    got = cache.attend(q, ints(slots), ints([n - 1 for n in lens]), ints([0, 1]))
    want = clean.attend(q, ints(slots), ints([n - 1 for n in lens]), ints([0, 1]))
    d = torch.arange(128, device="cuda") % 4
    hit = [r for r in range(rows) if r % 4 in (0, 2)]
    assert bool(got[hit, 4:8].isnan().all())
    got[hit, 4:8] = want[hit, 4:8]
    for h, group in ((8, 1), (12, 3)):
        x = got[hit, h:h + 4]
        assert not bool(x[..., d == group].isfinite().any())
        got[hit, h:h + 4] = torch.where(d == group, want[hit, h:h + 4], x)
    some = [r for r in range(rows) if r < 8 or r >= rows - 4]
    check_attend(got[some], q[some], clean, [slots[r] for r in some], [lens[r] for r in some])


@path
def test_extreme_values(A, rows, max_len):
    """Queries of any size; value scales from the smallest to the largest half, ascending and descending."""
    g = gen(rows + 1)
    cache = A.Kv4Cache(1, 4, max_len, 128)
    fill(cache, g)
    q = randn(g, rows, 16, 128) * torch.tensor([20.0, 1e-6, 1e-30] * rows, device="cuda")[:rows, None, None]
    seq, some = ints([0] * rows), [r for r in range(rows) if r < 4 or r >= rows - 2]

    def check(lens):
        got = cache.attend(q, seq, ints([n - 1 for n in lens]), ints([0]))
        check_attend(got[some], q[some], cache, [0] * len(some), [lens[r] for r in some])

    check([max_len - r for r in range(rows)])
    cache.v_scales.copy_(torch.logspace(-7, 4.5, max_len, device="cuda")[None, None, :, None].expand_as(cache.v_scales))
    q = randn(g, rows, 16, 128)
    check([1 + r * (max_len - 1) // rows for r in range(rows)])
    cache.v_scales.copy_(cache.v_scales.flip(2))
    check([1 + r * (max_len - 1) // rows for r in range(rows)])


def big_calls(A, g):
    """A call of each operator that fills scratch and joins it: arguments and the results of a first run."""
    cache = A.Kv4Cache(2, 4, 8192, 128)
    fill(cache, g)
    seqs, slots = ints([0, 1]), ints([0, 1])
    q = [randn(g, 2, 16, 128) for _ in range(2)]
    pos = [ints([8000, 77]), ints([3, 5500])]
    assert split(2, 8192) == "many shares" and cache.scratch_bytes(2, 16) > 0
    offs, kv_offs = ints([0, 20, 60]), ints([0, 2500, 6000])
    qp = [randn(g, 60, 4, 128).half() for _ in range(2)]
    kp, vp = randn(g, 6000, 2, 128).half(), randn(g, 6000, 2, 128).half()
    assert A.prompt_scratch_bytes(60, 2, 6000, 4, 2, 128) > 0

    def run(i, **kw):
        return cache.attend(q[i], seqs, pos[i], slots, **kw), A.prompt_attention(qp[i], kp, vp, offs, kv_offs, **kw)

    want = [run(i) for i in range(2)]
    check_attend(want[0][0], q[0], cache, [0, 1], [8001, 78])
    check_prompt(want[1][1], qp[1], kp, vp, [20, 40], [(0, 2500), (2500, 6000)])
    torch.cuda.synchronize()
    return run, want


def test_calls_at_once_have_scratch_of_their_own(A):
    run, want = big_calls(A, gen(61))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            got[i].append(run(i, stream=s))
    torch.cuda.synchronize()
    for i in range(2):
        for a, p in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(p, want[i][1])


def test_captured_calls_replayed_at_once(A):
    """Two graphs of such calls, replayed over and over on two streams."""
    run, want = big_calls(A, gen(62))
    graphs, got = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            got.append(run(i))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                for t in got[i]:
                    t.zero_()
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])


def test_one_scratch_for_calls_after_one_another(A):
    """Scratch that the caller keeps, with contents of any kind, for calls of the same and of fewer rows."""
    g = gen(63)
    cache = A.Kv4Cache(3, 4, 8192, 128)
    fill(cache, g)
    scratch = torch.full((max(cache.scratch_bytes(r, 16) for r in (1, 3, 40)),), 0xff, dtype=torch.uint8, device="cuda")
    for rows in (40, 3, 1, 40):
        q = randn(g, rows, 16, 128)
        lens = [1 + int(x) for x in torch.randint(0, 8000, (rows,), generator=g, device="cuda")]
        got = cache.attend(q, ints([r % 3 for r in range(rows)]), ints([n - 1 for n in lens]), ints([2, 0, 1]), scratch=scratch)
        some = list(range(rows))[:4]
        check_attend(got[some], q[some], cache, [(2, 0, 1)[r % 3] for r in some], [lens[r] for r in some])
    q, k, v = randn(g, 30, 4, 64).half(), randn(g, 5000, 2, 64).half(), randn(g, 5000, 2, 64).half()
    need = A.prompt_scratch_bytes(30, 1, 5000, 4, 2, 64)
    assert need > 0
    scratch = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    for n in (5000, 31, 1600):
        got = A.prompt_attention(q, k, v, ints([0, 30]), offsets([n]), scratch=scratch)
        check_prompt(got, q, k, v, [30], [(0, n)])

"""The hybrid decoder with its K/V cache in 4 bits (HybridEngine(kv_bits=4)): what a step leaves in the cache is
the quantised keys and values of its own projections, the layer's output is 64-bit attention over what the cache
holds (tolerances of test_gpu_attention.py), prefill chunks and decode steps alike, and captured, multi-step and
eager decoding give the same tokens."""
import numpy as np
import pytest
import torch

from test_gpu_attention import U, close, half_step, ref_attention, ref_quantise, stored, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine(cuda_lib):
    from exl3_b200.hybrid import HybridConfig, HybridEngine, synthetic_weights

    cfg = HybridConfig(layers=2, ffn=1024, vocab=2048, full_every=2)  # the last layer is full attention
    return HybridEngine(synthetic_weights(cfg, seed=5), device=0, slots=3, max_len=200, max_rows=96, kv_bits=4)


def step(eng, rows_of, slots, tokens):
    """One step: rows_of[s] = (first position, rows) of sequence s; returns after the forward pass."""
    offs, seq, pos = [0], [], []
    for s, (p, n) in enumerate(rows_of):
        seq += [s] * n
        pos += list(range(p, p + n))
        offs.append(offs[-1] + n)
    eng.meta.fill(tokens, seq, pos, offs, slots, [o - 1 for o in offs[1:]])
    eng.meta.upload(None)
    eng.forward(offs[-1], len(slots), len(slots))
    return seq, pos


@pytest.mark.parametrize("rows_of", [[(0, 70)], [(70, 1), (0, 25), (0, 3)], [(71, 1), (25, 1), (3, 1)], [(72, 4)]])
def test_steps_against_64_bit_attention(engine, rows_of):
    """The steps run one after another on the same slots: a prompt, decode and prefill rows mixed, a decode step,
    and a short chunk (the fused path of at most 8 rows)."""
    eng, cfg = engine, engine.cfg
    rng = np.random.default_rng(len(rows_of) + rows_of[0][0])
    slots = [2, 0, 1][:len(rows_of)]
    total = sum(n for _, n in rows_of)
    for (p, _), slot in zip(rows_of, slots):
        if p == 0:
            eng.reset_slot(slot)
    seq, pos = step(eng, rows_of, slots, rng.integers(0, cfg.vocab, total))
    D, KV, hd = cfg.heads * cfg.head_dim, eng.KV, cfg.head_dim
    qkv = eng.proj.view(-1)[:eng.max_rows * (D + 2 * KV)].view(eng.max_rows, D + 2 * KV)[:total]
    cache = eng.kv4[0]
    for rows, codes, scales in ((eng.k32[:total], cache.k_codes, cache.k_scales),
                                (qkv[:, D + KV:].unflatten(1, (-1, hd)), cache.v_codes, cache.v_scales)):
        want_c, want_s = ref_quantise(rows)
        at = (torch.tensor([slots[s] for s in seq]).cuda(), slice(None), torch.tensor(pos).cuda())
        got_c, got_s = stored(codes[at], scales[at])
        assert torch.equal(got_c, want_c) and torch.equal(got_s, want_s)
    decode = all(n == 1 for _, n in rows_of)
    q = eng.q[:total].unflatten(1, (-1, hd)) if decode else eng.q16[:total]
    mix = eng.mix[:total].unflatten(1, (-1, hd))
    kc, vc = (values(*stored(c, s)) for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
    if not decode:
        kc, vc = kc.half(), vc.half()  # as read back
    r, share = 0, cfg.heads // cfg.kv_heads
    for s, (p, n) in enumerate(rows_of):
        for h in range(cfg.heads):
            k, v = kc[slots[s], h // share, :p + n], vc[slots[s], h // share, :p + n]
            want, a, w, top = ref_attention(q[r:r + n, h], k, v, p, hd ** -0.5)
            tol = (64 * a + 64) * U * (top if decode else w)
            if not decode:
                tol = tol + 1.5 * half_step(torch.float16) * w
            close(mix[r:r + n, h], want, tol + U * want.abs(), (s, h))
        r += n


def test_captured_and_multi_step_decoding_give_the_eager_tokens(engine):
    from exl3_b200.hybrid import Request, run_requests

    prompt = np.random.default_rng(3).integers(0, engine.cfg.vocab, 50).astype(np.int32)
    got = []
    for multi in (False, True):
        rq = Request(prompt.copy(), max_new=24)
        run_requests(engine, [rq], chunk=32, multi_step=multi, graphs={})
        got.append(rq.generated)
    eager = []
    engine.reset_slot(0)
    step(engine, [(0, 32)], [0], prompt[:32])
    step(engine, [(32, 18)], [0], prompt[32:])
    for p in range(50, 74):
        eager.append(int(engine.out_tokens[0]))
        step(engine, [(p, 1)], [0], [eager[-1]])
    assert got[0] == got[1] == eager


def test_captured_prompt_step_at_other_positions(engine):
    """A prompt chunk captured at the start of a context and replayed further on."""
    eng = engine
    prompt = np.random.default_rng(4).integers(0, eng.cfg.vocab, 60).astype(np.int32)

    def upload(p):
        eng.meta.fill(prompt[p:p + 20], [0] * 20, list(range(p, p + 20)), [0, 20], [1], [19])
        eng.meta.upload(None)

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    eng.reset_slot(1)
    want = []
    for p in (0, 20, 40):
        upload(p)
        torch.cuda.synchronize()
        eng.forward(20, 1, 1, stream=stream)
        torch.cuda.synchronize()
        want.append(eng.mix[:20].clone())
    eng.reset_slot(1)
    upload(0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        eng.forward(20, 1, 1, stream=stream)
    for p, w in zip((0, 20, 40), want):
        upload(p)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eng.mix[:20], w)


def test_continuous_admission(engine):
    """More requests than slots, prefill chunks between decode rows."""
    from exl3_b200.hybrid import Request, run_requests

    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, engine.cfg.vocab, n).astype(np.int32) for n in (20, 33, 12, 27)]
    reqs = [Request(p, max_new=8) for p in prompts]
    run_requests(engine, reqs, chunk=16)
    assert all(len(r.generated) == 8 for r in reqs)


def test_kv_bits_is_checked(cuda_lib):
    from exl3_b200.hybrid import HybridConfig, HybridEngine, synthetic_weights

    with pytest.raises(ValueError, match="kv_bits"):
        HybridEngine(synthetic_weights(HybridConfig(layers=1, ffn=128, vocab=128)), kv_bits=8)

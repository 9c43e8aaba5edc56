"""The attention operators' refusals and host helpers (no GPU): every declared symbol is exported, bad
arguments are refused before any launch, and the rotary frequencies follow their formulas."""
import ctypes
import math
import re
from pathlib import Path

import numpy as np
import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
INVALID = 1


@pytest.fixture(scope="module")
def L():
    from exl3_b200 import attention

    return attention._lib()


def test_declared_symbols_are_exported(L):
    names = set(re.findall(r"\b(exl3cu_\w+)\s*\(", (ROOT / "include" / "exl3cu_attn.h").read_text()))
    names = {n for n in names if not n.endswith("_bytes()")}
    assert len(names) >= 6
    for n in names:
        assert hasattr(L, n), n


P, Z = 4096, None  # an aligned address that is never read: every call below is refused first


def cache(**kw):
    from exl3_b200.attention import _Cache

    f = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, n_slots=2, kv_heads=4, max_len=128, head_dim=128)
    f.update(kw)
    return ctypes.pointer(_Cache(*f.values()))


BAD_CACHES = [dict(k_codes=None), dict(v_scales=P + 8), dict(max_len=100), dict(max_len=0), dict(head_dim=96),
              dict(n_slots=0), dict(kv_heads=0)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches_are_refused(L, kw):
    c = cache(**kw)
    assert L.exl3cu_kv4_append(c, P, 512, P, 512, 0, 1, P, P, P, 1, Z) == INVALID
    assert L.exl3cu_kv4_read(c, P, P, 1, 1, P, 512, P, 512, 0, Z) == INVALID
    assert L.exl3cu_kv4_attn(c, P, 2048, 0, 1, 16, P, P, P, 1, 1.0, P, 2048, P, 1 << 30, Z) == INVALID
    assert b"cache" in L.exl3cu_last_error()
    assert L.exl3cu_kv4_append(None, P, 512, P, 512, 0, 1, P, P, P, 1, Z) == INVALID


ROPE = dict(q=P, qs=2048, k=P, ks=512, dtype=0, rows=3, heads=16, kv=4, dim=128, pos=P, qw=P, kw=P, eps=1e-6, freq=P,
            rotary=128, inter=0, factor=1.0, qo=P, qos=2048, qot=0, ko=P, kos=512, kot=0, stream=Z)


@pytest.mark.parametrize("kw", [
    dict(dim=96), dict(dim=256), dict(dtype=2), dict(qot=3), dict(kot=9), dict(rows=-1), dict(heads=0), dict(kv=-1),
    dict(rotary=130), dict(rotary=24), dict(rotary=-16), dict(freq=None), dict(q=None), dict(q=P + 4), dict(k=None),
    dict(qs=2047), dict(qs=2046), dict(qs=2050), dict(ks=511), dict(pos=None), dict(qo=P + 8), dict(kos=500),
    dict(heads=2000)])
def test_bad_rope_arguments_are_refused(L, kw):
    assert L.exl3cu_qk_norm_rope(*{**ROPE, **kw}.values()) == INVALID
    assert b"qk_norm_rope" in L.exl3cu_last_error()


def test_bad_cache_operands_are_refused(L):
    c = cache()
    for a in ((None, 512, P, 512, 0), (P, 511, P, 512, 0), (P, 512, P + 2, 512, 1), (P, 512, P, 514, 0),
              (P, 512, P, 512, 2)):
        assert L.exl3cu_kv4_append(c, *a, 1, P, P, P, 1, Z) == INVALID
        assert L.exl3cu_kv4_read(c, P, P, 1, 1, *a, Z) == INVALID
    assert L.exl3cu_kv4_append(c, P, 512, P, 512, 0, -1, P, P, P, 1, Z) == INVALID
    assert L.exl3cu_kv4_append(c, P, 512, P, 512, 0, 1, None, P, P, 1, Z) == INVALID
    assert L.exl3cu_kv4_read(c, P, None, 1, 1, P, 512, P, 512, 0, Z) == INVALID
    assert L.exl3cu_kv4_read(c, P, P, -1, 1, P, 512, P, 512, 0, Z) == INVALID


ATTN = dict(q=P, qs=2048, dtype=0, rows=1, heads=16, seq=P, pos=P, slot=P, n_seq=1, scale=1.0, out=P, os=2048,
            scratch=P, bytes=1 << 30, stream=Z)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(q=P + 4), dict(qs=2047), dict(dtype=3), dict(rows=-1), dict(rows=70000), dict(heads=18),
    dict(heads=0), dict(heads=2048), dict(scale=0.0), dict(scale=math.inf), dict(scratch=None), dict(scratch=P + 4), dict(bytes=1000), dict(seq=None), dict(pos=None), dict(slot=None), dict(n_seq=-1), dict(out=None),
    dict(os=1024)])
def test_bad_attend_arguments_are_refused(L, kw):
    assert L.exl3cu_kv4_attn(cache(), *{**ATTN, **kw}.values()) == INVALID
    assert b"kv4_attn" in L.exl3cu_last_error()


PROMPT = dict(q=P, qs=2048, k=P, krs=512, khs=128, v=P, vrs=512, vhs=128, kv_rows=10, dtype=1, heads=16, kv=4, dim=128,
              qo=P, b=P, e=P, n=1, rows=10, scale=1.0, out=P, os=2048, ot=1, scratch=P, bytes=1 << 40, stream=Z)


@pytest.mark.parametrize("kw", [
    dict(dtype=0), dict(dtype=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(ot=4), dict(dim=80), dict(heads=15), dict(kv=0), dict(heads=2048, qs=1 << 20),
    dict(n=-1), dict(rows=-1), dict(kv_rows=-1), dict(q=None), dict(q=P + 2), dict(qs=2044), dict(qs=1024), dict(k=None),
    dict(krs=100), dict(krs=132), dict(khs=64), dict(vhs=129), dict(v=P + 8), dict(qo=None), dict(b=None), dict(e=None),
    dict(out=None), dict(os=2040), dict(krs=1 << 40), dict(kv_rows=10000, bytes=1000), dict(kv_rows=10000, scratch=P + 8)])
def test_bad_prompt_arguments_are_refused(L, kw):
    assert L.exl3cu_prompt_attn(*{**PROMPT, **kw}.values()) == INVALID
    assert b"prompt_attn" in L.exl3cu_last_error()


def test_empty_calls_do_nothing(L):
    """No rows or no sequences: success without a launch (there is no GPU here)."""
    assert L.exl3cu_qk_norm_rope(*{**ROPE, "rows": 0}.values()) == 0
    assert L.exl3cu_kv4_append(cache(), P, 512, P, 512, 0, 0, P, P, P, 1, Z) == 0
    assert L.exl3cu_kv4_read(cache(), P, P, 0, 5, P, 512, P, 512, 0, Z) == 0
    assert L.exl3cu_kv4_attn(cache(), *{**ATTN, "rows": 0}.values()) == 0
    assert L.exl3cu_prompt_attn(*{**PROMPT, "rows": 0}.values()) == 0


def test_python_refusals():
    from exl3_b200 import attention as A

    q, pos = torch.zeros(2, 4, 64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        A.qk_norm_rope(q, None, pos)
    with pytest.raises(ValueError):
        A.qk_norm_rope(q[0], None, pos)
    with pytest.raises((TypeError, ValueError)):
        A.prompt_attention(q, q, q, pos, pos)
    with pytest.raises(ValueError):
        A.Kv4Cache(1, 1, 64, 96)
    with pytest.raises(ValueError):
        A.Kv4Cache.from_tensors(*(torch.zeros(1, 1, 64, 32, dtype=torch.uint8),) * 4)
    for bad in ((0,), (7,), (64, 1e4, 0.5)):
        with pytest.raises(ValueError):
            A.rope_frequencies(*bad)


def test_rope_frequencies():
    from exl3_b200.attention import rope_frequencies

    f, a = rope_frequencies(128, 1e4)
    assert a == 1.0 and f.dtype == np.float32 and len(f) == 64 and f[0] == 1.0
    assert np.allclose(f, 1e4 ** (-np.arange(64) / 64.0), rtol=1e-7)
    lin, a = rope_frequencies(64, 1e4, 4.0)
    assert a == 1.0 and np.allclose(lin, rope_frequencies(64, 1e4)[0] / 4, rtol=1e-6)
    y, a = rope_frequencies(128, 1e4, 16.0, 4096)
    assert a == pytest.approx(0.1 * math.log(16) + 1)
    turns = 4096 * f.astype(np.float64) / (2 * math.pi)
    assert np.all(y[turns > 40] == f[turns > 40])                       # fast ones stay
    assert np.allclose(y[turns < 0.8], f[turns < 0.8] / 16, rtol=1e-6)  # slow ones are divided
    assert np.all(np.diff(y) < 0)


BY_WORDS = [
    (0, "PiPiiiiiiPPPfPiifPiiPiiP", ROPE, [dict(dim=96), dict(dtype=2), dict(kot=9), dict(kv=-1), dict(rotary=24), dict(ks=511),
                                          dict(pos=None), dict(kos=500), dict(heads=2000)]),
    (4, "PiPiiPiiiiiiiPPPiifPiiPiP", PROMPT, [dict(dtype=0), dict(ot=4), dict(scale=-1.0), dict(kv_rows=-1), dict(khs=64),
                                           dict(e=None), dict(out=None), dict(krs=1 << 40)])]


@pytest.mark.parametrize("which,kinds,args,bad", BY_WORDS)
def test_calls_by_words_are_the_calls(L, which, kinds, args, bad):
    """Every word reaches the parameter of its place: what is refused is refused with the call's own text."""
    import struct

    fn = (L.exl3cu_qk_norm_rope, None, None, None, L.exl3cu_prompt_attn)[which]
    for kw in bad + [dict(rows=0)]:
        values = {**args, **kw}.values()
        want, text = fn(*values), L.exl3cu_last_error()
        words = b"".join(struct.pack("=d" if k == "f" else "=q", v or 0) for k, v in zip(kinds, values, strict=True))
        assert L.exl3cu_attn_words(which, words) == want == (INVALID if kw != dict(rows=0) else 0)
        assert L.exl3cu_last_error() == text
    assert L.exl3cu_attn_words(which, None) == INVALID and L.exl3cu_attn_words(9, b"") == INVALID


def test_native_calls_leave_what_is_not_ordinary():
    """Wrong types, unknown or doubled keywords, tensors without a GPU: all left to the Python functions."""
    from exl3_b200 import attention

    mod, t = attention._native(), torch.zeros(2, 4, 64)
    for name in ("qk_norm_rope", "append", "read", "attend", "prompt_attention"):
        call = getattr(mod, name)
        for args, kw in (((), {}), ((t, t, t), {}), ((t,) * 12, {}), ((None, 1, "x"), {}), ((t, t), {"q": t}),
                         ((t, t), {"nothing": 1}), ((t, t, t, t, t), {}), ((t, t, t, t), {"scale": "x"})):
            assert call(*args, **kw) is NotImplemented, (name, len(args), kw)


def test_stream_of_another_device_is_refused():
    from types import SimpleNamespace

    from exl3_b200 import attention

    q = SimpleNamespace(get_device=lambda: 0)
    s = SimpleNamespace(cuda_stream=0, device=torch.device("cuda", 1))
    with pytest.raises(ValueError, match="stream"):
        attention.qk_norm_rope(q, None, None, stream=s)
    with pytest.raises(TypeError):
        attention.qk_norm_rope()
    with pytest.raises(ValueError, match="CUDA device"):
        attention.qk_norm_rope(torch.zeros(1, 1, 64), None, None)

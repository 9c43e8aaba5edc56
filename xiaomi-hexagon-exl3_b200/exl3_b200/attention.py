"""Attention operators of any head geometry (include/exl3cu_attn.h), torch-facing.

One attention layer of a decoder that keeps its K/V cache in 4 bits:

    q, k = qk_norm_rope(q, k, positions, inv_freq, q_weight, k_weight)   per-head RMSNorm + rotary positions
    cache.append(k, v, row_seq, row_pos, seq_slot)                       quantised as they are written
    decode steps:  out = cache.attend(q, row_seq, row_pos, seq_slot)     single rows over the cache in 4 bits
    prompt steps:  k, v = cache.read(seq_slot, kv_offsets, total_rows)   back to 16 bits as packed rows
                   out = prompt_attention(q, k, v, q_offsets, kv_offsets)   causal, on the tensor cores

Rows follow the ragged packer's conventions (ops.pack_ragged): row r belongs to step sequence
row_seq[r] at position row_pos[r]; sequence s uses cache slot seq_slot[s].  q, k and v are
[rows, heads, head_dim] tensors (float32, float16 or bfloat16; head_dim 64 or 128) whose last two
dimensions are contiguous or are made so; rows may be strided, e.g. the q, k and v columns of one
packed projection.  Index tensors are int32.  Calls run on the tensors' device, on its current
stream or the one given as the keyword `stream`, and can be captured in a CUDA graph.  Invalid
arguments raise ValueError, TypeError or Exl3InvalidArgument (a ValueError).
"""
from __future__ import annotations

import contextlib
import ctypes
import functools

import numpy as np
import torch

from ._lib import check, lib

BF16 = 4
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: BF16}
_I, _F, _S, _P = ctypes.c_int, ctypes.c_float, ctypes.c_size_t, ctypes.c_void_p


class _Cache(ctypes.Structure):
    _fields_ = [("k_codes", _P), ("k_scales", _P), ("v_codes", _P), ("v_scales", _P), ("n_slots", _I),
                ("kv_heads", _I), ("max_len", _I), ("head_dim", _I)]


_L = None


def _lib():
    global _L
    if _L is None:
        L = lib()
        C = ctypes.POINTER(_Cache)
        L.exl3cu_qk_norm_rope.argtypes = [_P, _S, _P, _S, _I, _I, _I, _I, _I, _P, _P, _P, _F, _P, _I, _I, _F, _P, _S,
                                          _I, _P, _S, _I, _P]
        L.exl3cu_kv4_append.argtypes = [C, _P, _S, _P, _S, _I, _I, _P, _P, _P, _I, _P]
        L.exl3cu_kv4_read.argtypes = [C, _P, _P, _I, _I, _P, _S, _P, _S, _I, _P]
        L.exl3cu_kv4_attn_scratch_bytes.restype = _S
        L.exl3cu_kv4_attn_scratch_bytes.argtypes = [C, _I, _I]
        L.exl3cu_kv4_attn.argtypes = [C, _P, _S, _I, _I, _I, _P, _P, _P, _I, _F, _P, _S, _P, _S, _P]
        L.exl3cu_prompt_attn.argtypes = [_P, _S, _P, _S, _S, _P, _S, _S, _I, _I, _I, _I, _I, _P, _P, _P, _I, _I, _F,
                                         _P, _S, _I, _P]
        for name in ("exl3cu_qk_norm_rope", "exl3cu_kv4_append", "exl3cu_kv4_read", "exl3cu_kv4_attn",
                     "exl3cu_prompt_attn"):
            getattr(L, name).restype = _I
        _L = L
    return _L


_HERE = contextlib.nullcontext()


def _on(device):
    """Context in which `device` is the current one."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _on_stream(call):
    """A call with stream=s runs as if s were the current stream: what it copies and allocates on the way
    is ordered with what it launches, and its memory belongs to s."""

    @functools.wraps(call)
    def wrapper(*args, stream=None, **kw):
        if stream is None:
            return call(*args, **kw)
        if not hasattr(stream, "cuda_stream"):
            stream = torch.cuda.ExternalStream(int(stream))
        with torch.cuda.stream(stream):
            return call(*args, **kw)

    return wrapper


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _heads(name, t, device=None, dtype=None):
    """`t` as [rows, heads, head_dim] with contiguous heads and 16-byte aligned rows; its row stride."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [rows, heads, head_dim]")
    if t.dtype not in _DTYPES or (dtype is not None and t.dtype != dtype):
        raise TypeError(f"{name} must be float32, float16 or bfloat16, and q, k and v of one type")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} must be on the CUDA device of the other operands")
    rows, heads, dim = t.shape
    s = t.stride()
    if (s[2] != 1 or (s[1] != dim and heads != 1) or (rows > 1 and s[0] < heads * dim)
            or (rows > 1 and s[0] * t.element_size() % 16) or t.data_ptr() % 16):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        s = t.stride()
    return t, (s[0] if rows > 1 else heads * dim)


def _into(name, t, rows, heads, dim, device, dtypes):
    """A caller's output: [rows, heads, dim] with contiguous heads, never copied; its row stride."""
    if tuple(t.shape) != (rows, heads, dim) or t.device != device:
        raise ValueError(f"{name} must be [{rows}, {heads}, {dim}] on {device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has an unsupported type {t.dtype}")
    s = t.stride()
    if rows and (s[2] != 1 or (s[1] != dim and heads != 1) or (rows > 1 and s[0] < heads * dim)):
        raise ValueError(f"{name} must have contiguous heads and rows that do not overlap")
    return s[0] if rows > 1 else heads * dim


def _index(name, t, count, device):
    if t.dtype != torch.int32 or t.dim() != 1 or t.device != device:
        raise ValueError(f"{name} must be a 1-D int32 tensor on {device}")
    if count is not None and t.shape[0] != count:
        raise ValueError(f"{name} must have {count} entries")
    if t.shape[0] > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _f32(name, t, count, device):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != count or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of {count} on {device}")
    return t.data_ptr()


def rope_frequencies(rotary_dim: int, theta: float = 1e4, factor: float = 1.0, original_len: int = 0,
                     fast: float = 32.0, slow: float = 1.0):
    """(inv_freq float32 [rotary_dim / 2], attention_factor) of the rotary embedding: theta^(-2i / rotary_dim).
    With a factor > 1 scaled for contexts `factor` times as long: divided by it where original_len is 0
    (linear interpolation), else by parts (YaRN, Peng et al. 2023): frequencies that turn more than `fast`
    times within original_len stay, those that turn less than `slow` times are divided, a ramp lies between,
    and the attention factor is 0.1 ln(factor) + 1."""
    if rotary_dim <= 0 or rotary_dim % 2 or factor < 1.0:
        raise ValueError("rotary_dim must be even and positive, factor at least 1")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    f = float(theta) ** (-2.0 * i / rotary_dim)
    if factor == 1.0:
        return f.astype(np.float32), 1.0
    if not original_len:
        return (f / factor).astype(np.float32), 1.0

    def dim_of(turns):  # the index whose frequency turns so often within original_len
        return rotary_dim * np.log(original_len / (turns * 2 * np.pi)) / (2 * np.log(theta))

    low, high = max(np.floor(dim_of(fast)), 0), min(np.ceil(dim_of(slow)), rotary_dim // 2 - 1)
    ramp = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
    return (f / factor * ramp + f * (1 - ramp)).astype(np.float32), float(0.1 * np.log(factor) + 1.0)


@_on_stream
def qk_norm_rope(q, k, positions, inv_freq=None, q_weight=None, k_weight=None, *, eps: float = 1e-6,
                 interleaved: bool = False, attention_factor: float = 1.0, q_out=None, k_out=None, out_dtype=None):
    """Per-head RMSNorm (where weights are given) and rotary embedding of q [rows, heads, D] and k
    [rows, kv_heads, D] (or None) in one pass (exl3cu_qk_norm_rope); returns (q, k).

    positions: int32 [rows]; rows of a negative position are not written.  inv_freq: float32
    [rotary_dim / 2] (rope_frequencies), or None for no rotation.  q_out / k_out may be q / k
    themselves, or of another of the three types; out_dtype is the type of outputs allocated here."""
    L = _lib()
    dev = q.device
    q, qs = _heads("q", q)
    rows, heads, dim = q.shape
    if k is not None:
        k, ks = _heads("k", k, dev, q.dtype)
        if k.shape[0] != rows or k.shape[2] != dim:
            raise ValueError("k must have q's rows and head_dim")
        kv = k.shape[1]
    else:
        kv, ks = 0, 0
    pos = _index("positions", positions, rows, dev)
    rotary = 0 if inv_freq is None else 2 * inv_freq.shape[0]
    freq = _f32("inv_freq", inv_freq, rotary // 2, dev)
    qw, kw = _f32("q_weight", q_weight, dim, dev), _f32("k_weight", k_weight, dim, dev)
    if q_out is None:
        q_out = torch.empty((rows, heads, dim), dtype=out_dtype or q.dtype, device=dev)
    qos = _into("q_out", q_out, rows, heads, dim, dev, _DTYPES)
    if kv and k_out is None:
        k_out = torch.empty((rows, kv, dim), dtype=out_dtype or q.dtype, device=dev)
    kos = _into("k_out", k_out, rows, kv, dim, dev, _DTYPES) if kv else 0
    with _on(dev):
        check(L.exl3cu_qk_norm_rope(q.data_ptr(), qs, k.data_ptr() if kv else None, ks, _DTYPES[q.dtype], rows, heads,
                                    kv, dim, pos, qw, kw, eps, freq, rotary, int(interleaved), attention_factor,
                                    q_out.data_ptr(), qos, _DTYPES[q_out.dtype], k_out.data_ptr() if kv else None, kos,
                                    _DTYPES[k_out.dtype] if kv else 0, _stream(dev)))
    return q_out, k_out


class Kv4Cache:
    """K/V cache in 4 bits for `slots` sequences of up to `max_len` positions (rounded up to a multiple
    of 64) on one GPU.  Layout: exl3cu_kv4_cache (include/exl3cu_attn.h); 4.5 bits a value."""

    def __init__(self, slots: int, kv_heads: int, max_len: int, head_dim: int = 128, device: int | str = 0):
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if min(slots, kv_heads, max_len) <= 0 or head_dim not in (64, 128):
            raise ValueError("slots, kv_heads and max_len must be positive, head_dim 64 or 128")
        shape = (slots, kv_heads, -(-max_len // 64) * 64)
        codes = [torch.zeros(shape + (head_dim // 2,), dtype=torch.uint8, device=dev) for _ in range(2)]
        scales = [torch.zeros(shape + (head_dim // 32,), dtype=torch.float16, device=dev) for _ in range(2)]
        self._bind(codes[0], scales[0], codes[1], scales[1])

    @classmethod
    def from_tensors(cls, k_codes, k_scales, v_codes, v_scales) -> "Kv4Cache":
        """A cache in the caller's memory: codes uint8 [slots, kv_heads, max_len, head_dim / 2], scales
        float16 [slots, kv_heads, max_len, head_dim / 32], contiguous, max_len a multiple of 64."""
        c = cls.__new__(cls)
        c._bind(k_codes, k_scales, v_codes, v_scales)
        return c

    def _bind(self, k_codes, k_scales, v_codes, v_scales):
        if k_codes.dim() != 4:
            raise ValueError("codes must be [slots, kv_heads, max_len, head_dim / 2]")
        slots, kv, max_len, half = k_codes.shape
        for name, t, dtype, width in (("k_codes", k_codes, torch.uint8, half), ("k_scales", k_scales, torch.float16, half // 16),
                                      ("v_codes", v_codes, torch.uint8, half), ("v_scales", v_scales, torch.float16, half // 16)):
            if tuple(t.shape) != (slots, kv, max_len, width) or t.dtype != dtype or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dtype} [{slots}, {kv}, {max_len}, {width}]")
            if not t.is_cuda or t.device != k_codes.device or t.data_ptr() % 16:
                raise ValueError(f"{name} must be 16-byte aligned memory of one CUDA device")
        if half not in (32, 64) or max_len % 64 or min(slots, kv, max_len) <= 0:
            raise ValueError("head_dim must be 64 or 128 and max_len a positive multiple of 64")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.device, self.slots, self.kv_heads, self.max_len, self.head_dim = k_codes.device, slots, kv, max_len, 2 * half
        self._c = _Cache(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), slots, kv,
                         max_len, 2 * half)
        self._ref = ctypes.pointer(self._c)

    @_on_stream
    def append(self, k, v, row_seq, row_pos, seq_slot) -> None:
        """Quantise rows k, v [rows, kv_heads, D] into (seq_slot[row_seq], row_pos) (exl3cu_kv4_append).
        Rows outside the cache (a position, slot or sequence out of range) are skipped."""
        L = _lib()
        dev = self.device
        k, ks = _heads("k", k, dev)
        v, vs = _heads("v", v, dev, k.dtype)
        rows = k.shape[0]
        if tuple(k.shape[1:]) != (self.kv_heads, self.head_dim) or v.shape != k.shape:
            raise ValueError(f"k and v must be [rows, {self.kv_heads}, {self.head_dim}]")
        with _on(dev):
            check(L.exl3cu_kv4_append(self._ref, k.data_ptr(), ks, v.data_ptr(), vs, _DTYPES[k.dtype], rows,
                                      _index("row_seq", row_seq, rows, dev), _index("row_pos", row_pos, rows, dev),
                                      _index("seq_slot", seq_slot, None, dev), seq_slot.shape[0], _stream(dev)))

    @_on_stream
    def read(self, seq_slot, kv_offsets, total_rows: int, dtype=torch.float16, k_out=None, v_out=None):
        """Positions 0 .. kv_offsets[s+1] - kv_offsets[s] of each sequence's slot as packed rows
        [total_rows, kv_heads, D] of `dtype` (exl3cu_kv4_read); returns (k, v).  Rows from kv_offsets[-1]
        on are left as they were (undefined where allocated here)."""
        L = _lib()
        dev = self.device
        n = seq_slot.shape[0]
        if k_out is None or v_out is None:
            if dtype not in _DTYPES:
                raise TypeError("dtype must be float32, float16 or bfloat16")
            shape = (total_rows, self.kv_heads, self.head_dim)
            if k_out is None:
                k_out = torch.empty(shape, dtype=dtype if v_out is None else v_out.dtype, device=dev)
            if v_out is None:
                v_out = torch.empty(shape, dtype=k_out.dtype, device=dev)
        ks = _into("k_out", k_out, total_rows, self.kv_heads, self.head_dim, dev, _DTYPES)
        vs = _into("v_out", v_out, total_rows, self.kv_heads, self.head_dim, dev, (k_out.dtype,))
        with _on(dev):
            check(L.exl3cu_kv4_read(self._ref, _index("seq_slot", seq_slot, None, dev),
                                    _index("kv_offsets", kv_offsets, n + 1, dev), n, total_rows, k_out.data_ptr(), ks,
                                    v_out.data_ptr(), vs, _DTYPES[k_out.dtype], _stream(dev)))
        return k_out, v_out

    def scratch_bytes(self, rows: int, heads: int) -> int:
        """Scratch that attend() needs for `rows` rows of `heads` query heads."""
        with _on(self.device):
            return _lib().exl3cu_kv4_attn_scratch_bytes(self._ref, rows, heads)

    @_on_stream
    def attend(self, q, row_seq, row_pos, seq_slot, scale: float | None = None, out=None, scratch=None):
        """Attention of rows q [rows, heads, D] over positions 0 .. row_pos of their slots
        (exl3cu_kv4_attn); scale defaults to 1/sqrt(D).  scratch: a uint8 tensor of scratch_bytes() that
        no other call uses at the same time; allocated per call when not given."""
        L = _lib()
        dev = self.device
        q, qs = _heads("q", q, dev)
        rows, heads, dim = q.shape
        if dim != self.head_dim or heads % self.kv_heads:
            raise ValueError(f"q must be [rows, a multiple of {self.kv_heads}, {self.head_dim}]")
        if out is None:
            out = torch.empty((rows, heads, dim), dtype=q.dtype, device=dev)
        os_ = _into("out", out, rows, heads, dim, dev, (q.dtype,))
        with _on(dev):
            if scratch is None:
                need = L.exl3cu_kv4_attn_scratch_bytes(self._ref, rows, heads)
                if need:
                    scratch = torch.empty(need, dtype=torch.uint8, device=dev)
            elif scratch.device != dev or not scratch.is_contiguous():
                raise ValueError(f"scratch must be contiguous memory of {dev}")
            check(L.exl3cu_kv4_attn(self._ref, q.data_ptr(), qs, _DTYPES[q.dtype], rows, heads,
                                    _index("row_seq", row_seq, rows, dev), _index("row_pos", row_pos, rows, dev),
                                    _index("seq_slot", seq_slot, None, dev), seq_slot.shape[0],
                                    dim ** -0.5 if scale is None else scale, out.data_ptr(), os_,
                                    scratch.data_ptr() if scratch is not None else None,
                                    scratch.numel() * scratch.element_size() if scratch is not None else 0,
                                    _stream(dev)))
        return out


def _kv(name, t, device, dtype, shape):
    """k or v [rows, kv_heads, D] with any row and head strides that are multiples of 16 bytes."""
    if t.dim() != 3 or t.shape[2] != shape[2] or (shape[1] and t.shape[1] != shape[1]):
        raise ValueError(f"{name} must be [rows, kv_heads, head_dim], k and v alike")
    if t.dtype != dtype or t.device != device:
        raise TypeError(f"{name} must have q's type and device")
    rs, hs, ds = t.stride()
    dim = t.shape[2]
    rs, hs = rs if t.shape[0] > 1 else t.shape[1] * dim, hs if t.shape[1] > 1 else dim
    if ds != 1 or rs % 8 or hs % 8 or rs < dim or hs < dim or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        rs, hs = t.shape[1] * dim, dim
    return t, rs, hs


@_on_stream
def prompt_attention(q, k, v, q_offsets, kv_offsets=None, *, kv_begin=None, kv_end=None, scale: float | None = None,
                     out=None):
    """Causal attention of packed sequences (exl3cu_prompt_attn): q [q_rows, heads, D], k and v
    [kv_rows, kv_heads, D], float16 or bfloat16; sequence s has query rows q_offsets[s] .. q_offsets[s+1]
    and key rows kv_offsets[s] .. kv_offsets[s+1] (or kv_begin[s] .. kv_end[s], for rows that lie in a
    slot cache).  Its last query sees all of its keys, the one before all but the last, and so on; a query
    that sees none becomes zero.  out may be float32 or of q's type; query rows outside every sequence are
    left as they were (undefined where out is allocated here)."""
    L = _lib()
    dev = q.device
    if q.dtype == torch.float32:
        raise TypeError("q, k and v must be float16 or bfloat16")
    q, qs = _heads("q", q)
    rows, heads, dim = q.shape
    k, krs, khs = _kv("k", k, dev, q.dtype, (0, 0, dim))
    v, vrs, vhs = _kv("v", v, dev, q.dtype, k.shape)
    if v.shape[0] != k.shape[0]:
        raise ValueError("k and v must have the same rows")
    if kv_offsets is not None:
        if kv_begin is not None or kv_end is not None:
            raise ValueError("give kv_offsets, or kv_begin and kv_end")
        n = kv_offsets.shape[0] - 1
        begin = _index("kv_offsets", kv_offsets, None, dev)
        end = begin + 4
    else:
        if kv_begin is None or kv_end is None:
            raise ValueError("give kv_offsets, or kv_begin and kv_end")
        n = kv_begin.shape[0]
        begin, end = _index("kv_begin", kv_begin, None, dev), _index("kv_end", kv_end, n, dev)
    if out is None:
        out = torch.empty((rows, heads, dim), dtype=q.dtype, device=dev)
    os_ = _into("out", out, rows, heads, dim, dev, (q.dtype, torch.float32))
    with _on(dev):
        check(L.exl3cu_prompt_attn(q.data_ptr(), qs, k.data_ptr(), krs, khs, v.data_ptr(), vrs, vhs, k.shape[0],
                                   _DTYPES[q.dtype], heads, k.shape[1], dim,
                                   _index("q_offsets", q_offsets, n + 1, dev), begin, end, n, rows,
                                   dim ** -0.5 if scale is None else scale, out.data_ptr(), os_, _DTYPES[out.dtype],
                                   _stream(dev)))
    return out


__all__ = ["Kv4Cache", "qk_norm_rope", "prompt_attention", "rope_frequencies"]

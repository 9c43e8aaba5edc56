"""Attention operators for any number of heads (include/exl3cu_attn.h), torch-facing.

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
packed projection.  Sums and softmax statistics are held in 32 bits; the weights of a softmax meet the values
rounded to q's type (prompt_attention) or to 11 bits (attend with rows of 16 bits).  Index tensors are contiguous int32.  Calls run on the tensors' device, on its current
stream or the one given as the keyword `stream`, and can be captured in a CUDA graph.  Invalid
arguments raise ValueError, TypeError or Exl3InvalidArgument (a ValueError).
"""
from __future__ import annotations

import ctypes
import functools
import importlib.machinery
import importlib.util
import struct
import sysconfig

import numpy as np
import torch

from ._lib import TORCH_LIB_PATH, check, lib

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
                                         _P, _S, _I, _P, _S, _P]
        L.exl3cu_prompt_attn_scratch_bytes.restype = _S
        L.exl3cu_prompt_attn_scratch_bytes.argtypes = [_I] * 6
        for name in ("exl3cu_qk_norm_rope", "exl3cu_kv4_append", "exl3cu_kv4_read", "exl3cu_kv4_attn",
                     "exl3cu_prompt_attn"):
            getattr(L, name).restype = _I
        L.exl3cu_attn_words.restype = _I
        L.exl3cu_attn_words.argtypes = [_I, ctypes.c_char_p]
        _L = L
    return _L


@functools.lru_cache(maxsize=None)
def _native():
    """csrc/exl3cu_attn_torch.cpp: the calls below in ordinary form (NotImplemented for any other)."""
    L = _lib()
    if not TORCH_LIB_PATH.exists():
        raise ImportError(f"{TORCH_LIB_PATH} is not built; run xiaomi-hexagon-exl3_b200/build.py (with a torch for CUDA)")
    loader = importlib.machinery.ExtensionFileLoader("exl3cu_torch", str(TORCH_LIB_PATH))
    mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("exl3cu_torch", loader))
    again = "run xiaomi-hexagon-exl3_b200/build.py"
    here = f"{sysconfig.get_config_var('SOABI')} {torch.__version__}"
    try:
        loader.exec_module(mod)
    except ImportError as e:
        raise ImportError(f"{TORCH_LIB_PATH} does not load into {here}; {again}") from e
    if getattr(mod, "built_for", None) != here:
        raise ImportError(f"{TORCH_LIB_PATH} was built for {getattr(mod, 'built_for', 'another torch')}, this is {here}; {again}")
    mod.bind(*(ctypes.cast(getattr(L, "exl3cu_" + n), _P).value
               for n in ("qk_norm_rope", "kv4_append", "kv4_read", "kv4_attn_scratch_bytes", "kv4_attn",
                         "prompt_attn_scratch_bytes", "prompt_attn")))
    return mod


def _call(which, types):
    """A call by exl3cu_attn_words: arguments of the given kinds (P: address or None, i: integer, f: float) are
    packed into words, which takes ctypes a fraction of the time that converting them one by one does."""
    pack = struct.Struct("=" + "".join("d" if t == "f" else "q" for t in types)).pack
    entry = None

    def call(*args):
        nonlocal entry
        if entry is None:
            entry = _lib().exl3cu_attn_words
        try:
            words = pack(*args)
        except (struct.error, OverflowError) as e:
            raise TypeError(f"a number is expected: {e}") from None
        status = entry(which, words)
        if status:
            check(status)

    return call


_rope_call = _call(0, "PiPiiiiiiPPPfPiifPiiPiiP")
_append_call = _call(1, "PPiPiiiPPPiP")
_read_call = _call(2, "PPPiiPiPiiP")
_attn_call = _call(3, "PPiiiiPPPifPiPiP")
_prompt_call = _call(4, "PiPiiPiiiiiiiPPPiifPiiPiP")


@functools.lru_cache(maxsize=4096)
def prompt_scratch_bytes(q_rows: int, n_seq: int, kv_rows: int, heads: int, kv_heads: int, head_dim: int) -> int:
    """Scratch with which prompt_attention divides the keys of few query rows over the GPU (0: it would not)."""
    return _lib().exl3cu_prompt_attn_scratch_bytes(q_rows, n_seq, kv_rows, heads, kv_heads, head_dim)


_current_device = torch.cuda.current_device
if hasattr(torch._C, "_cuda_getDevice"):  # the same without the check that CUDA is initialised: a CUDA tensor exists
    _current_device = torch._C._cuda_getDevice
_i32, _f32t, _packed = torch.int32, torch.float32, torch.contiguous_format


def _op(call):
    """An operator's entry.  Calls in ordinary form (the current device, no copies to make) are carried out by the
    native module; the Python function copies or refuses, and does the others.  It runs on the device of its first
    tensor argument (or of the cache that it is a method of), whatever the current one is.  With stream=s it runs as
    if s were the current stream: what it copies and allocates on the way is ordered with what it launches, and its
    memory belongs to s."""
    fast = None

    @functools.wraps(call)
    def wrapper(*args, stream=None, **kw):
        nonlocal fast
        if stream is None:
            if fast is None:
                fast = getattr(_native(), call.__name__)
            result = fast(*args, **kw)
            if result is not NotImplemented:
                if result.__class__ is int:
                    check(result)
                return result
        first = args[0] if args else kw.get("q")
        if first is None:
            return call(*args, **kw)  # names the missing argument
        if not hasattr(first, "get_device"):
            raise TypeError(f"{call.__name__} takes tensors, not {type(first).__name__}")
        index = first.get_device()
        if index < 0:
            raise ValueError("operands must be on a CUDA device")
        if stream is not None:
            if not hasattr(stream, "cuda_stream"):
                stream = torch.cuda.ExternalStream(int(stream), device=index)
            if stream.device.index != index:
                raise ValueError("stream must be of the operands' device")
            with torch.cuda.stream(stream):
                return wrapper(*args, **kw)
        if _current_device() != index:
            with torch.cuda.device(index):
                return call(*args, **kw)
        return call(*args, **kw)

    return wrapper


def _stream(index):
    return torch.cuda.current_stream(index).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):  # the same handle without a Stream object around it
    _stream = torch._C._cuda_getCurrentRawStream


def _tensor(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, not {type(t).__name__}")
    return t


def _count(name, t):
    """Entries of a tensor of one dimension."""
    if _tensor(name, t).dim() != 1:
        raise ValueError(f"{name} must have one dimension")
    return t.shape[0]


def _heads(name, t, index, dtype):
    """`t` as [rows, heads, head_dim] with contiguous heads and 16-byte aligned rows: the tensor (a copy where
    that is needed, to be kept until the launch), its address and its row stride."""
    _tensor(name, t)
    if t.dtype is not dtype or t.dim() != 3 or t.get_device() != index:
        if t.dim() != 3:
            raise ValueError(f"{name} must be [rows, heads, head_dim]")
        if t.get_device() != index:
            raise ValueError(f"{name} must be on the CUDA device of the other operands")
        raise TypeError(f"{name} must be of the other operands' type")
    rows, heads, dim = t.shape
    s0, s1, s2 = t.stride()
    ptr, width = t.data_ptr(), heads * dim
    if rows <= 1:
        s0 = width
    if s2 != 1 or (s1 != dim and heads != 1) or s0 < width or s0 * t.element_size() % 16 or ptr % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        ptr, s0 = t.data_ptr(), width
    return t, ptr, s0


def _into(name, t, rows, heads, dim, index, dtypes):
    """A caller's output: [rows, heads, dim] with contiguous heads, never copied; its row stride."""
    if _tensor(name, t).shape != (rows, heads, dim) or t.get_device() != index:
        raise ValueError(f"{name} must be [{rows}, {heads}, {dim}] on the device of the other operands")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has an unsupported type {t.dtype}")
    s0, s1, s2 = t.stride()
    if rows <= 1:
        s0 = heads * dim
    if rows and (s2 != 1 or (s1 != dim and heads != 1) or s0 < heads * dim):
        raise ValueError(f"{name} must have contiguous heads and rows that do not overlap")
    return s0


def _index(name, t, count, index):
    """Address of a contiguous int32 tensor of `count` entries."""
    if _tensor(name, t).dtype is not _i32 or t.get_device() != index or t.shape != (count,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {count} on the device of the other operands")
    return t.data_ptr()


def _f32(name, t, count, index):
    if t is None:
        return 0
    if _tensor(name, t).dtype is not _f32t or t.get_device() != index or t.shape != (count,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of {count} on the device of the other operands")
    return t.data_ptr()


def _known(name, dtype):
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16")
    return code


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

    low, high = max(np.floor(dim_of(fast)), 0), min(np.ceil(dim_of(slow)), rotary_dim - 1)
    ramp = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
    return (f / factor * ramp + f * (1 - ramp)).astype(np.float32), float(0.1 * np.log(factor) + 1.0)


@_op
def qk_norm_rope(q, k, positions, inv_freq=None, q_weight=None, k_weight=None, *, eps: float = 1e-6,
                 interleaved: bool = False, attention_factor: float = 1.0, q_out=None, k_out=None, out_dtype=None):
    """Per-head RMSNorm (where weights are given) and rotary embedding of q [rows, heads, D] and k
    [rows, kv_heads, D] (or None) in one pass (exl3cu_qk_norm_rope); returns (q, k).

    positions: int32 [rows]; rows of a negative position are not written.  inv_freq: float32
    [rotary_dim / 2] (rope_frequencies), or None for no rotation.  q_out / k_out may be q / k
    themselves, or of another of the three types; out_dtype is the type of outputs allocated here."""
    index, dtype = _tensor("q", q).get_device(), q.dtype
    code = _known("q", dtype)
    q, qp, qs = _heads("q", q, index, dtype)
    rows, heads, dim = q.shape
    kv, kp, ks, kop, kos, kcode = 0, 0, 0, 0, 0, 0
    if k is not None:
        k, kp, ks = _heads("k", k, index, dtype)
        kv = k.shape[1]
        if k.shape != (rows, kv, dim):
            raise ValueError("k must have q's rows and head_dim")
    rotary = 0 if inv_freq is None else 2 * _count("inv_freq", inv_freq)
    if q_out is None:
        q_out = torch.empty_like(q, dtype=out_dtype, memory_format=_packed)
        qos = heads * dim
        qcode = _known("out_dtype", q_out.dtype)
    else:
        qos = _into("q_out", q_out, rows, heads, dim, index, _DTYPES)
        qcode = _DTYPES[q_out.dtype]
    if kv:
        if k_out is None:
            k_out = torch.empty_like(k, dtype=out_dtype, memory_format=_packed)
            kos = kv * dim
        else:
            kos = _into("k_out", k_out, rows, kv, dim, index, _DTYPES)
        kop, kcode = k_out.data_ptr(), _known("k_out", k_out.dtype)
    _rope_call(qp, qs, kp, ks, code, rows, heads, kv, dim,
               _index("positions", positions, rows, index), _f32("q_weight", q_weight, dim, index),
               _f32("k_weight", k_weight, dim, index), eps,
               _f32("inv_freq", inv_freq, rotary // 2, index), rotary, bool(interleaved),
               attention_factor, q_out.data_ptr(), qos, qcode, kop, kos, kcode, _stream(index))
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
        self._at = ctypes.addressof(self._c)
        self._index = k_codes.get_device()
        self._scratch = {}  # attend()'s scratch bytes by (rows, heads): a function of the cache's shape

    def get_device(self) -> int:
        """Index of the cache's CUDA device."""
        return self._index

    @_op
    def append(self, k, v, row_seq, row_pos, seq_slot) -> None:
        """Quantise rows k, v [rows, kv_heads, D] into (seq_slot[row_seq], row_pos) (exl3cu_kv4_append).
        Rows outside the cache (a position, slot or sequence out of range) are skipped."""
        index, dtype = self._index, _tensor("k", k).dtype
        code = _known("k", dtype)
        k, kp, ks = _heads("k", k, index, dtype)
        v, vp, vs = _heads("v", v, index, dtype)
        rows, n = k.shape[0], _count("seq_slot", seq_slot)
        if k.shape != (rows, self.kv_heads, self.head_dim) or v.shape != k.shape:
            raise ValueError(f"k and v must be [rows, {self.kv_heads}, {self.head_dim}]")
        _append_call(self._at, kp, ks, vp, vs, code, rows, _index("row_seq", row_seq, rows, index),
                     _index("row_pos", row_pos, rows, index),
                     _index("seq_slot", seq_slot, n, index), n, _stream(index))

    @_op
    def read(self, seq_slot, kv_offsets, total_rows: int, dtype=torch.float16, k_out=None, v_out=None):
        """Positions 0 .. kv_offsets[s+1] - kv_offsets[s] of each sequence's slot as packed rows
        [total_rows, kv_heads, D] of `dtype` (exl3cu_kv4_read); returns (k, v).  Rows from kv_offsets[-1]
        on are left as they were (undefined where allocated here)."""
        index, n = self._index, _count("seq_slot", seq_slot)
        if total_rows < 0:
            raise ValueError("total_rows must not be negative")
        if k_out is None or v_out is None:
            for t in (k_out, v_out):
                dtype = dtype if t is None else _tensor("k_out, v_out", t).dtype
            _known("dtype", dtype)
            shape = (total_rows, self.kv_heads, self.head_dim)
            k_out = torch.empty(shape, dtype=dtype, device=self.device) if k_out is None else k_out
            v_out = torch.empty(shape, dtype=dtype, device=self.device) if v_out is None else v_out
        ks = _into("k_out", k_out, total_rows, self.kv_heads, self.head_dim, index, _DTYPES)
        vs = _into("v_out", v_out, total_rows, self.kv_heads, self.head_dim, index, (k_out.dtype,))
        _read_call(self._at, _index("seq_slot", seq_slot, n, index),
                   _index("kv_offsets", kv_offsets, n + 1, index), n, total_rows,
                   k_out.data_ptr(), ks, v_out.data_ptr(), vs, _DTYPES[k_out.dtype],
                   _stream(index))
        return k_out, v_out

    def scratch_bytes(self, rows: int, heads: int) -> int:
        """Scratch that attend() needs for `rows` rows of `heads` query heads."""
        key = (rows, heads)
        need = self._scratch.get(key)
        if need is None:
            need = self._scratch[key] = _lib().exl3cu_kv4_attn_scratch_bytes(self._ref, rows, heads)
        return need

    @_op
    def attend(self, q, row_seq, row_pos, seq_slot, scale: float | None = None, out=None, scratch=None):
        """Attention of rows q [rows, heads, D] over positions 0 .. row_pos of their slots
        (exl3cu_kv4_attn); scale defaults to 1/sqrt(D).  scratch: a uint8 tensor of scratch_bytes() that
        no other call uses at the same time; allocated per call when not given."""
        index, dtype = self._index, _tensor("q", q).dtype
        code = _known("q", dtype)
        q, qp, qs = _heads("q", q, index, dtype)
        rows, heads, dim = q.shape
        n = _count("seq_slot", seq_slot)
        if dim != self.head_dim or heads % self.kv_heads:
            raise ValueError(f"q must be [rows, a multiple of {self.kv_heads}, {self.head_dim}]")
        if out is None:
            out, os_ = torch.empty_like(q, memory_format=_packed), heads * dim
        else:
            os_ = _into("out", out, rows, heads, dim, index, (dtype,))
        if scratch is None:
            need = self._scratch.get((rows, heads))
            if need is None:
                need = self.scratch_bytes(rows, heads)
            if need:
                scratch = self.k_codes.new_empty(need)
            held = need
        else:
            held = _tensor("scratch", scratch).numel() * scratch.element_size()
            if scratch.get_device() != index or not scratch.is_contiguous():
                raise ValueError("scratch must be contiguous memory of the cache's device")
        _attn_call(self._at, qp, qs, code, rows, heads, _index("row_seq", row_seq, rows, index),
                   _index("row_pos", row_pos, rows, index),
                   _index("seq_slot", seq_slot, n, index), n,
                   dim ** -0.5 if scale is None else scale, out.data_ptr(), os_,
                   scratch.data_ptr() if held else 0, held, _stream(index))
        return out


def _kv(name, t, index, dtype, dim):
    """k or v [rows, kv_heads, D] with any row and head strides that are multiples of 16 bytes: the tensor (or
    its copy), address, row and head strides."""
    if _tensor(name, t).dim() != 3 or t.shape[2] != dim:
        raise ValueError(f"{name} must be [rows, kv_heads, {dim}]")
    if t.dtype is not dtype or t.get_device() != index:
        raise TypeError(f"{name} must have q's type and device")
    rows, heads, _ = t.shape
    rs, hs, ds = t.stride()
    ptr = t.data_ptr()
    if rows <= 1:
        rs = heads * dim
    if heads <= 1:
        hs = dim
    if ds != 1 or rs % 8 or hs % 8 or rs < dim or hs < dim or ptr % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        ptr, rs, hs = t.data_ptr(), heads * dim, dim
    return t, ptr, rs, hs


@_op
def prompt_attention(q, k, v, q_offsets, kv_offsets=None, *, kv_begin=None, kv_end=None, scale: float | None = None,
                     out=None, scratch=None):
    """Causal attention of packed sequences (exl3cu_prompt_attn): q [q_rows, heads, D], k and v
    [kv_rows, kv_heads, D], float16 or bfloat16; sequence s has query rows q_offsets[s] .. q_offsets[s+1]
    and key rows kv_offsets[s] .. kv_offsets[s+1] (or kv_begin[s] .. kv_end[s], for rows that lie in a
    slot cache).  Its last query sees all of its keys, the one before all but the last, and so on; a query
    that sees none becomes zero, one whose largest score is beyond 2^26 in size may become NaN.  out may be
    float32 or of q's type; query rows outside every sequence are left as they were (undefined where out is
    allocated here).  scratch: a uint8 tensor of prompt_scratch_bytes() that no other call uses at the same
    time; allocated per call when not given."""
    index, dtype = _tensor("q", q).get_device(), q.dtype
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise TypeError("q, k and v must be float16 or bfloat16")
    q, qp, qs = _heads("q", q, index, dtype)
    rows, heads, dim = q.shape
    k, kp, krs, khs = _kv("k", k, index, dtype, dim)
    v, vp, vrs, vhs = _kv("v", v, index, dtype, dim)
    if v.shape != k.shape:
        raise ValueError("k and v must have the same shape")
    if kv_offsets is not None:
        if kv_begin is not None or kv_end is not None:
            raise ValueError("give kv_offsets, or kv_begin and kv_end")
        n = _count("q_offsets", q_offsets) - 1
        begin = _index("kv_offsets", kv_offsets, n + 1, index)
        end = begin + 4
    else:
        if kv_begin is None or kv_end is None:
            raise ValueError("give kv_offsets, or kv_begin and kv_end")
        n = _count("kv_begin", kv_begin)
        begin, end = _index("kv_begin", kv_begin, n, index), _index("kv_end", kv_end, n, index)
    if out is None:
        out, os_ = torch.empty_like(q, memory_format=_packed), heads * dim
    else:
        os_ = _into("out", out, rows, heads, dim, index, (dtype, torch.float32))
    kv_rows, kv = k.shape[0], k.shape[1]
    if scratch is None:
        held = prompt_scratch_bytes(rows, n, kv_rows, heads, kv, dim)
    else:
        held = _tensor("scratch", scratch).numel() * scratch.element_size()
    if scratch is None:
        if held:
            scratch = torch.empty(held, dtype=torch.uint8, device=q.device)
    elif scratch.get_device() != index or not scratch.is_contiguous():
        raise ValueError("scratch must be contiguous memory of q's device")
    _prompt_call(qp, qs, kp, krs, khs, vp, vrs, vhs, kv_rows, _DTYPES[dtype], heads,
                 kv, dim, _index("q_offsets", q_offsets, n + 1, index), begin, end, n,
                 rows, dim ** -0.5 if scale is None else scale, out.data_ptr(), os_,
                 _DTYPES[out.dtype], scratch.data_ptr() if held else 0, held, _stream(index))
    return out


__all__ = ["Kv4Cache", "qk_norm_rope", "prompt_attention", "prompt_scratch_bytes", "rope_frequencies"]

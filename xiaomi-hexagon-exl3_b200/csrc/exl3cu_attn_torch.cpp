// Calls of the attention operators (exl3cu_attn.h) with torch tensors, for exl3_b200/attention.py.
//
// A call of few rows takes the GPU 2 to 8 us, and checking its arguments, allocating its outputs and converting its
// arguments in Python takes 8 to 10 (without the launch).  These functions do the same for calls in ordinary form:
// tensors of the current device whose layout needs no copy, and whose shapes and types agree.  They return
// NotImplemented for anything else, refusals and empty calls included, which attention.py then handles; a status (an
// int) where the operator refuses; and otherwise what the operator returns.  One launch with its outputs 5 us.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstdint>
#include <type_traits>

#include "exl3cu.h"
#include "exl3cu_attn.h"

namespace {

// The entries of libexl3cu.so that the package has loaded, set by bind().
struct {
    decltype(&exl3cu_qk_norm_rope) rope;
    decltype(&exl3cu_kv4_append) append;
    decltype(&exl3cu_kv4_read) read;
    decltype(&exl3cu_kv4_attn_scratch_bytes) attn_scratch;
    decltype(&exl3cu_kv4_attn) attn;
    decltype(&exl3cu_prompt_attn_scratch_bytes) prompt_scratch;
    decltype(&exl3cu_prompt_attn) prompt;
} entry;

struct Unusual {};  // thrown for a call that is left to attention.py

void require(bool usual) {
    if (!usual) throw Unusual{};
}

// ---- arguments -----------------------------------------------------------------------------------------------

constexpr int kMost = 16;  // parameters of a call

struct Signature {
    int count, positional;  // the rest by keyword only
    const char * text[kMost];
    PyObject * name[kMost];  // interned
};

void parse(const Signature & s, PyObject * const * args, Py_ssize_t n, PyObject * kwnames, PyObject ** out) {
    require(n <= s.positional);
    for (int i = 0; i < s.count; ++i) out[i] = i < n ? args[i] : nullptr;
    const Py_ssize_t named = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
    for (Py_ssize_t j = 0; j < named; ++j) {
        PyObject * key = PyTuple_GET_ITEM(kwnames, j);
        int i = 0;
        while (i < s.count && s.name[i] != key) ++i;
        require(i < s.count && !out[i]);
        out[i] = args[n + j];
    }
    for (int i = 0; i < s.count; ++i)
        if (out[i] == Py_None) out[i] = nullptr;
}

const at::Tensor & tensor(PyObject * o) {
    require(o && THPVariable_Check(o));
    return THPVariable_Unpack(o);
}

float number(PyObject * o, double otherwise) {
    if (!o) return float(otherwise);
    require(PyFloat_CheckExact(o) || PyLong_CheckExact(o));
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Unusual{};
    }
    return float(v);
}

int dtype_of(at::ScalarType t) {
    if (t == at::kFloat) return EXL3CU_F32;
    if (t == at::kHalf) return EXL3CU_F16;
    require(t == at::kBFloat16);
    return EXL3CU_BF16;
}

int count(int64_t n) {
    require(n > 0 && n <= INT_MAX);
    return int(n);
}

void on(const at::Tensor & t, int device) { require(t.is_cuda() && t.get_device() == device); }

bool aligned(const void * p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Contiguous int32 or f32 of n entries.
template <typename P> const P * list(const at::Tensor & t, int64_t n, int device) {
    on(t, device);
    require(t.scalar_type() == (std::is_same_v<P, float> ? at::kFloat : at::kInt) && t.dim() == 1 && t.size(0) == n &&
            t.is_contiguous());
    return static_cast<const P *>(t.const_data_ptr());
}

// [rows, heads, dim] with contiguous heads and 16-byte aligned rows that do not overlap.
struct Rows {
    void * p;
    size_t stride;
    int rows, heads, dim;
    Rows(const at::Tensor & t, int device) {
        on(t, device);
        require(t.dim() == 3);
        rows = count(t.size(0));
        heads = count(t.size(1));
        dim = count(t.size(2));
        const int64_t width = int64_t(heads) * dim, s0 = rows == 1 ? width : t.stride(0);
        p = const_cast<void *>(t.const_data_ptr());
        require((t.stride(2) == 1) && (heads == 1 || t.stride(1) == dim) && s0 >= width &&
                s0 * int64_t(t.element_size()) % 16 == 0 && aligned(p));
        stride = size_t(s0);
    }
};

// [rows, heads, dim] with strides of rows and heads of their own, multiples of 16 bytes; 16-bit values.
struct Keys {
    const void * p;
    size_t row_stride, head_stride;
    Keys(const at::Tensor & t, int device, int dim) {
        on(t, device);
        require(t.dim() == 3 && t.size(2) == dim && t.stride(2) == 1);
        const int64_t rs = count(t.size(0)) == 1 ? t.size(1) * dim : t.stride(0), hs = count(t.size(1)) == 1 ? dim : t.stride(1);
        p = t.const_data_ptr();
        require(rs % 8 == 0 && hs % 8 == 0 && rs >= dim && hs >= dim && aligned(p));
        row_stride = size_t(rs);
        head_stride = size_t(hs);
    }
};

at::Tensor empty(const at::Tensor & like, at::ScalarType type) { return at::empty(like.sizes(), like.options().dtype(type)); }

at::ScalarType type_of(PyObject * o, at::ScalarType otherwise) {
    if (!o) return otherwise;
    require(THPDtype_Check(o));
    return reinterpret_cast<THPDtype *>(o)->scalar_type;
}

// A caller's output of the given shape, or a new one.
at::Tensor output(PyObject * given, const at::Tensor & like, at::ScalarType type) {
    if (!given) return empty(like, type);
    const at::Tensor & t = tensor(given);
    require(t.sizes() == like.sizes());
    return t;
}

// The tensor's device, which is the current one.
int current_device_of(const at::Tensor & t) {
    require(t.is_cuda() && t.get_device() == c10::cuda::current_device());
    return t.get_device();
}

// Calls f(stream) without the interpreter's lock.
template <typename F> int unlocked(int device, F && f) {
    void * const stream = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device)).stream();
    PyThreadState * state = PyEval_SaveThread();
    const int status = f(stream);
    PyEval_RestoreThread(state);
    return status;
}

PyObject * pair(const at::Tensor & a, const at::Tensor & b) {
    PyObject * x = THPVariable_Wrap(a), * y = x ? THPVariable_Wrap(b) : nullptr, * both = y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return both;
}

// An entry: no C++ exception leaves it.  What is thrown on the way (an allocation that failed, a tensor without
// memory) is left to attention.py, which meets it again and reports it as torch does.
template <typename F> PyObject * guarded(F && f) {
    try {
        return f();
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NOTIMPLEMENTED;
    }
}

// The structure behind a Kv4Cache and its device.
struct Cache {
    const exl3cu_kv4_cache * c;
    int device;
    explicit Cache(PyObject * self) {
        static PyObject * const at = PyUnicode_InternFromString("_at"), * const index = PyUnicode_InternFromString("_index");
        require(self);
        c = reinterpret_cast<const exl3cu_kv4_cache *>(integer(self, at));
        device = int(integer(self, index));
        require(c && device == c10::cuda::current_device());
    }
    static long long integer(PyObject * self, PyObject * name) {
        PyObject * o = PyObject_GetAttr(self, name);
        if (!o) {
            PyErr_Clear();
            throw Unusual{};
        }
        const long long v = PyLong_AsLongLong(o);
        Py_DECREF(o);
        if (v == -1 && PyErr_Occurred()) {
            PyErr_Clear();
            throw Unusual{};
        }
        return v;
    }
};

// ---- calls -----------------------------------------------------------------------------------------------------

Signature rope_sig{12, 6, {"q", "k", "positions", "inv_freq", "q_weight", "k_weight", "eps", "interleaved", "attention_factor", "q_out", "k_out", "out_dtype"}, {}};

PyObject * rope(PyObject *, PyObject * const * args, Py_ssize_t n, PyObject * kwnames) {
    return guarded([&]() -> PyObject * {
        PyObject * a[kMost];
        parse(rope_sig, args, n, kwnames, a);
        const at::Tensor & q = tensor(a[0]), & k = tensor(a[1]);
        const int device = current_device_of(q);
        const Rows rq(q, device), rk(k, device);
        require(k.scalar_type() == q.scalar_type() && rk.rows == rq.rows && rk.dim == rq.dim);
        const int code = dtype_of(q.scalar_type());
        const auto * pos = list<int32_t>(tensor(a[2]), rq.rows, device);
        int rotary = 0;
        const float * freq = nullptr;
        if (a[3]) {
            const at::Tensor & f = tensor(a[3]);
            require(f.dim() == 1 && f.size(0) <= rq.dim);
            rotary = 2 * int(f.size(0));
            freq = list<float>(f, f.size(0), device);
        }
        const float * qw = a[4] ? list<float>(tensor(a[4]), rq.dim, device) : nullptr;
        const float * kw = a[5] ? list<float>(tensor(a[5]), rq.dim, device) : nullptr;
        const float eps = number(a[6], 1e-6), factor = number(a[8], 1.0);
        require(!a[7] || PyBool_Check(a[7]));
        const at::ScalarType type = type_of(a[11], q.scalar_type());
        at::Tensor qo = output(a[9], q, type), ko = output(a[10], k, type);
        const Rows oq(qo, device), ok(ko, device);
        const int qt = dtype_of(qo.scalar_type()), kt = dtype_of(ko.scalar_type());
        const int status = unlocked(device, [&](void * stream) {
            return entry.rope(rq.p, rq.stride, rk.p, rk.stride, code, rq.rows, rq.heads, rk.heads, rq.dim, pos, qw, kw, eps, freq,
                              rotary, a[7] == Py_True, factor, oq.p, oq.stride, qt, ok.p, ok.stride, kt, stream);
        });
        if (status) return PyLong_FromLong(status);
        return pair(qo, ko);
    });
}

Signature append_sig{6, 6, {"self", "k", "v", "row_seq", "row_pos", "seq_slot"}, {}};

PyObject * append(PyObject *, PyObject * const * args, Py_ssize_t n, PyObject * kwnames) {
    return guarded([&]() -> PyObject * {
        PyObject * a[kMost];
        parse(append_sig, args, n, kwnames, a);
        const Cache cache(a[0]);
        const at::Tensor & k = tensor(a[1]), & v = tensor(a[2]), & slot = tensor(a[5]);
        const Rows rk(k, cache.device), rv(v, cache.device);
        require(k.scalar_type() == v.scalar_type() && v.sizes() == k.sizes() && rk.heads == cache.c->kv_heads &&
                rk.dim == cache.c->head_dim && slot.dim() == 1);
        const int code = dtype_of(k.scalar_type()), n_seq = count(slot.size(0));
        const auto * seq = list<int32_t>(tensor(a[3]), rk.rows, cache.device);
        const auto * pos = list<int32_t>(tensor(a[4]), rk.rows, cache.device);
        const auto * slots = list<int32_t>(slot, n_seq, cache.device);
        const int status = unlocked(cache.device, [&](void * stream) {
            return entry.append(cache.c, rk.p, rk.stride, rv.p, rv.stride, code, rk.rows, seq, pos, slots, n_seq,
                                stream);
        });
        if (status) return PyLong_FromLong(status);
        Py_RETURN_NONE;
    });
}

Signature read_sig{7, 7, {"self", "seq_slot", "kv_offsets", "total_rows", "dtype", "k_out", "v_out"}, {}};

PyObject * read(PyObject *, PyObject * const * args, Py_ssize_t n, PyObject * kwnames) {
    return guarded([&]() -> PyObject * {
        PyObject * a[kMost];
        parse(read_sig, args, n, kwnames, a);
        const Cache cache(a[0]);
        const at::Tensor & slot = tensor(a[1]);
        require(slot.dim() == 1 && a[3] && PyLong_CheckExact(a[3]) && !a[5] == !a[6]);
        const int n_seq = count(slot.size(0));
        const auto * slots = list<int32_t>(slot, n_seq, cache.device);
        const auto * offsets = list<int32_t>(tensor(a[2]), int64_t(n_seq) + 1, cache.device);
        int over = 0;
        const long long given = PyLong_AsLongLongAndOverflow(a[3], &over);
        require(!over);
        const int rows = count(given);
        at::Tensor k, v;
        if (a[5]) {
            k = tensor(a[5]);
            v = tensor(a[6]);
        } else {
            const at::ScalarType type = type_of(a[4], at::kHalf);
            (void)dtype_of(type);
            k = at::empty({rows, cache.c->kv_heads, cache.c->head_dim}, slot.options().dtype(type));
            v = at::empty_like(k);
        }
        const Rows rk(k, cache.device), rv(v, cache.device);
        require(rk.rows == rows && rk.heads == cache.c->kv_heads && rk.dim == cache.c->head_dim && v.sizes() == k.sizes() &&
                v.scalar_type() == k.scalar_type());
        const int code = dtype_of(k.scalar_type());
        const int status = unlocked(cache.device, [&](void * stream) {
            return entry.read(cache.c, slots, offsets, n_seq, rows, rk.p, rk.stride, rv.p, rv.stride, code, stream);
        });
        if (status) return PyLong_FromLong(status);
        return pair(k, v);
    });
}

// Scratch of a call: the caller's, or `need` bytes of a new tensor.
struct Scratch {
    at::Tensor t;
    void * p = nullptr;
    size_t bytes = 0;
    Scratch(PyObject * given, size_t need, const at::Tensor & like, int device) {
        if (given) {
            t = tensor(given);
            on(t, device);
            require(t.is_contiguous() && t.numel() > 0);
        } else if (need) {
            t = at::empty({int64_t(need)}, like.options().dtype(at::kByte));
        } else {
            return;
        }
        p = const_cast<void *>(t.const_data_ptr());
        bytes = size_t(t.numel()) * t.element_size();
    }
};

Signature attend_sig{8, 8, {"self", "q", "row_seq", "row_pos", "seq_slot", "scale", "out", "scratch"}, {}};

PyObject * attend(PyObject *, PyObject * const * args, Py_ssize_t n, PyObject * kwnames) {
    return guarded([&]() -> PyObject * {
        PyObject * a[kMost];
        parse(attend_sig, args, n, kwnames, a);
        const Cache cache(a[0]);
        const at::Tensor & q = tensor(a[1]), & slot = tensor(a[4]);
        const Rows rq(q, cache.device);
        require(rq.dim == cache.c->head_dim && rq.heads % cache.c->kv_heads == 0 && slot.dim() == 1);
        const int code = dtype_of(q.scalar_type()), n_seq = count(slot.size(0));
        const auto * seq = list<int32_t>(tensor(a[2]), rq.rows, cache.device);
        const auto * pos = list<int32_t>(tensor(a[3]), rq.rows, cache.device);
        const auto * slots = list<int32_t>(slot, n_seq, cache.device);
        const float scale = number(a[5], rq.dim == 64 ? 0.125 : 0.08838834764831845);  // 1 / sqrt(head_dim)
        at::Tensor out = output(a[6], q, q.scalar_type());
        const Rows ro(out, cache.device);
        require(out.scalar_type() == q.scalar_type());
        const Scratch scratch(a[7], a[7] ? 0 : entry.attn_scratch(cache.c, rq.rows, rq.heads), q, cache.device);
        const int status = unlocked(cache.device, [&](void * stream) {
            return entry.attn(cache.c, rq.p, rq.stride, code, rq.rows, rq.heads, seq, pos, slots, n_seq, scale, ro.p, ro.stride,
                              scratch.p, scratch.bytes, stream);
        });
        return status ? PyLong_FromLong(status) : THPVariable_Wrap(std::move(out));
    });
}

Signature prompt_sig{10, 5, {"q", "k", "v", "q_offsets", "kv_offsets", "kv_begin", "kv_end", "scale", "out", "scratch"}, {}};

PyObject * prompt(PyObject *, PyObject * const * args, Py_ssize_t n, PyObject * kwnames) {
    return guarded([&]() -> PyObject * {
        PyObject * a[kMost];
        parse(prompt_sig, args, n, kwnames, a);
        const at::Tensor & q = tensor(a[0]), & k = tensor(a[1]), & v = tensor(a[2]), & offsets = tensor(a[3]);
        const int device = current_device_of(q);
        const at::ScalarType type = q.scalar_type();
        require(type == at::kHalf || type == at::kBFloat16);
        const Rows rq(q, device);
        const Keys rk(k, device, rq.dim), rv(v, device, rq.dim);
        require(k.scalar_type() == type && v.scalar_type() == type && v.sizes() == k.sizes() && offsets.dim() == 1);
        const int n_seq = count(offsets.size(0) - 1), kv_rows = count(k.size(0)), kv = count(k.size(1));
        const auto * from = list<int32_t>(offsets, int64_t(n_seq) + 1, device);
        const int32_t * begin, * end;
        if (a[4]) {
            require(!a[5] && !a[6]);
            begin = list<int32_t>(tensor(a[4]), int64_t(n_seq) + 1, device);
            end = begin + 1;
        } else {
            begin = list<int32_t>(tensor(a[5]), n_seq, device);
            end = list<int32_t>(tensor(a[6]), n_seq, device);
        }
        const float scale = number(a[7], rq.dim == 64 ? 0.125 : 0.08838834764831845);  // 1 / sqrt(head_dim)
        require(a[7] || rq.dim == 64 || rq.dim == 128);
        at::Tensor out = output(a[8], q, type);
        const Rows ro(out, device);
        const int code = dtype_of(type), out_code = dtype_of(out.scalar_type());
        require(out_code == code || out_code == EXL3CU_F32);
        const Scratch scratch(a[9], a[9] ? 0 : entry.prompt_scratch(rq.rows, n_seq, kv_rows, rq.heads, kv, rq.dim), q, device);
        const int status = unlocked(device, [&](void * stream) {
            return entry.prompt(rq.p, rq.stride, rk.p, rk.row_stride, rk.head_stride, rv.p, rv.row_stride, rv.head_stride, kv_rows, code,
                                rq.heads, kv, rq.dim, from, begin, end, n_seq, rq.rows, scale, ro.p, ro.stride, out_code, scratch.p,
                                scratch.bytes, stream);
        });
        return status ? PyLong_FromLong(status) : THPVariable_Wrap(std::move(out));
    });
}

// bind(addresses of the entries above, in order)
PyObject * bind(PyObject *, PyObject * args) {
    unsigned long long p[7];
    if (!PyArg_ParseTuple(args, "KKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6)) return nullptr;
    const auto to = [](auto & f, unsigned long long at) { f = reinterpret_cast<std::decay_t<decltype(f)>>(at); };
    to(entry.rope, p[0]);
    to(entry.append, p[1]);
    to(entry.read, p[2]);
    to(entry.attn_scratch, p[3]);
    to(entry.attn, p[4]);
    to(entry.prompt_scratch, p[5]);
    to(entry.prompt, p[6]);
    Py_RETURN_NONE;
}

template <typename F> PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"qk_norm_rope", fast(rope), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"append", fast(append), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"read", fast(read), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"attend", fast(attend), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {"prompt_attention", fast(prompt), METH_FASTCALL | METH_KEYWORDS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module{PyModuleDef_HEAD_INIT, "exl3cu_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_exl3cu_torch() {
    for (Signature * s : {&rope_sig, &append_sig, &read_sig, &attend_sig, &prompt_sig})
        for (int i = 0; i < s->count; ++i)
            if (!(s->name[i] = PyUnicode_InternFromString(s->text[i]))) return nullptr;
    PyObject * mod = PyModule_Create(&module);
    if (mod && PyModule_AddStringConstant(mod, "built_for", EXL3CU_BUILT_FOR)) Py_CLEAR(mod);  // Python's ABI, torch's version
    return mod;
}

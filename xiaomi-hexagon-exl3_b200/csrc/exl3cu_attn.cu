// Attention operators of any head geometry: the query/key norm with the rotary
// embedding, the 4-bit K/V cache's writer and reader, and attention of single
// rows over that cache.  (exl3cu_attn_prompt.cu: causal attention of packed
// prompts.)  Formats and conventions: exl3cu_attn.h.
//
// Like the hybrid decoder's kernels these are launched with programmatic
// dependent launch and touch nothing before griddepcontrol.wait.
#include "exl3cu.h"
#include "exl3cu_async.cuh"
#include "exl3cu_attn.cuh"
#include "exl3cu_attn.h"
#include "exl3cu_internal.h"

namespace exl3cu {

namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int s = 16; s; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    return v;
}

// ---- query/key norm and rotary embedding ----------------------------------------------------------

struct RopeArgs {
    const void * q;
    const void * k;
    void * q_out;
    void * k_out;
    long long q_stride, k_stride, q_out_stride, k_out_stride;
    const int32_t * row_pos;
    const float * q_w;
    const float * k_w;
    const float * inv_freq;
    float eps, factor;
    int rows, heads, kv_heads, rotary, interleaved, q_out_dtype, k_out_dtype;
};

// cos and sin of pos * f, the product and its reduction to one turn in 64 bits (pos and f have 24 bits
// each at most where it matters, so the product is exact), the functions in 32.
__device__ __forceinline__ void rope_angle(int pos, float f, float factor, float & cs, float & sn) {
    const double a = double(pos) * double(f);
    const double turns = rint(a * 0.15915494309189535);
    const float r = float(fma(-turns, 6.283185307179586, a));
    sincosf(r, &sn, &cs);
    cs *= factor;
    sn *= factor;
}

// One warp per (row, head): lane holds dimensions [lane * D/32, +D/32).
template <typename T, int D>
__global__ void __launch_bounds__(128) k_qk_norm_rope(const RopeArgs a) {
    pdl_trigger();
    pdl_wait_primary();
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const long long item = blockIdx.x * 4ll + (threadIdx.x >> 5);
    const int per_row = a.heads + a.kv_heads;
    if (item >= (long long)a.rows * per_row) return;
    const int r = int(item / per_row), h = int(item % per_row);
    const int pos = a.row_pos[r];
    if (pos < 0) return;
    const bool is_q = h < a.heads;
    const T * x = static_cast<const T *>(is_q ? a.q : a.k) +
                  (is_q ? r * a.q_stride + h * D : r * a.k_stride + (h - a.heads) * D);
    const float * w = is_q ? a.q_w : a.k_w;
    float v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f32(x[lane * E + i]);
    if (w) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) ss = fmaf(v[i], v[i], ss);
        const float inv = rsqrtf(warp_sum(ss) / float(D) + a.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = v[i] * inv * w[lane * E + i];
    }
    const int half = a.rotary / 2;
    if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const int d = lane * E + i;
            if (d < a.rotary) {
                float cs, sn;
                rope_angle(pos, a.inv_freq[d >> 1], a.factor, cs, sn);
                const float x0 = v[i], x1 = v[i + 1];
                v[i] = x0 * cs - x1 * sn;
                v[i + 1] = x1 * cs + x0 * sn;
            }
        }
    } else if (half) {
        // the partner of dimension d < half is d + half: half / E lanes further on
        const int shift = half / E;
        const bool first = lane < shift, second = lane >= shift && lane < 2 * shift;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float up = __shfl_sync(0xffffffffu, v[i], (lane + shift) & 31);
            const float down = __shfl_sync(0xffffffffu, v[i], (lane - shift) & 31);
            if (first || second) {
                const int j = (first ? lane : lane - shift) * E + i;
                float cs, sn;
                rope_angle(pos, a.inv_freq[j], a.factor, cs, sn);
                v[i] = first ? v[i] * cs - up * sn : v[i] * cs + down * sn;
            }
        }
    }
    const long long at = is_q ? r * a.q_out_stride + h * D : r * a.k_out_stride + (h - a.heads) * D;
    void * out = is_q ? a.q_out : a.k_out;
    const int dt = is_q ? a.q_out_dtype : a.k_out_dtype;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const long long p = at + lane * E + i;
        if (dt == EXL3CU_F32) static_cast<float *>(out)[p] = v[i];
        else if (dt == EXL3CU_F16) static_cast<__half *>(out)[p] = __float2half_rn(v[i]);
        else static_cast<__nv_bfloat16 *>(out)[p] = __float2bfloat16_rn(v[i]);
    }
}

// ---- the 4-bit cache -------------------------------------------------------------------------------

// One warp per (row, K or V, head): lane holds dimensions [lane * D/32, +D/32); dimension d is of group
// d mod G, G = D / 32, so a lane holds one element of every group.
template <typename T, int D>
__global__ void __launch_bounds__(128)
k_kv4_append(const Kv4 c, const T * k, long long k_stride, const T * v, long long v_stride, int rows,
             const int32_t * row_seq, const int32_t * row_pos, const int32_t * seq_slot, int n_seq) {
    pdl_trigger();
    pdl_wait_primary();
    constexpr int G = D / 32;
    const int lane = threadIdx.x & 31;
    const long long item = blockIdx.x * 4ll + (threadIdx.x >> 5);
    const int per_row = 2 * c.kv_heads;
    if (item >= (long long)rows * per_row) return;
    const int r = int(item / per_row), j = int(item % per_row);
    const bool is_v = j >= c.kv_heads;
    const int h = is_v ? j - c.kv_heads : j;
    const int seq = row_seq[r];
    if (seq < 0 || seq >= n_seq) return;
    const int slot = seq_slot[seq], pos = row_pos[r];
    if (slot < 0 || slot >= c.n_slots || pos < 0 || pos >= c.max_len) return;
    const T * x = (is_v ? v + r * v_stride : k + r * k_stride) + h * D + lane * G;
    const size_t at = (size_t(slot) * c.kv_heads + h) * c.max_len + pos;
    uint32_t code[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const float xv = to_f32(x[g]);
        const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(xv) & 0x7fffffffu);
        const __half s = kv4_scale(most);
        code[g] = kv4_code(xv, __half2float(s));
        if (lane == 0) (is_v ? c.v_scales : c.k_scales)[at * G + g] = __half_as_ushort(s);
    }
    uint8_t * out = (is_v ? c.v_codes : c.k_codes) + at * (D / 2) + lane * (G / 2);
#pragma unroll
    for (int g = 0; g < G; g += 2) out[g / 2] = uint8_t(code[g] | code[g + 1] << 4);
}

// One warp per (row, head): lane holds dimensions [lane * G, +G) of the key and of the value.
template <typename T, int D>
__global__ void __launch_bounds__(128)
k_kv4_read(const Kv4 c, const int32_t * seq_slot, const int32_t * offsets, int n_seq, int total, T * k,
           long long k_stride, T * v, long long v_stride) {
    pdl_trigger();
    pdl_wait_primary();
    constexpr int G = D / 32;
    const int lane = threadIdx.x & 31;
    const long long item = blockIdx.x * 4ll + (threadIdx.x >> 5);
    if (item >= (long long)total * c.kv_heads) return;
    const int r = int(item / c.kv_heads), h = int(item % c.kv_heads);
    const int seq = find_segment(offsets, n_seq, r);
    if (seq < 0) return;
    const int slot = seq_slot[seq], pos = r - offsets[seq];
    const bool ok = slot >= 0 && slot < c.n_slots && pos < c.max_len;
    const size_t at = ok ? (size_t(slot) * c.kv_heads + h) * c.max_len + pos : 0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const uint8_t * codes = (w ? c.v_codes : c.k_codes) + at * (D / 2) + lane * (G / 2);
        const uint16_t * scales = (w ? c.v_scales : c.k_scales) + at * G;
        T * out = (w ? v + r * v_stride : k + r * k_stride) + h * D + lane * G;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int code = (codes[g / 2] >> (4 * (g & 1))) & 15;
            out[g] = from_f32<T>(ok ? float(code - 8) * __half2float(__ushort_as_half(scales[g])) : 0.f);
        }
    }
}

// ---- attention of single rows over the cache ------------------------------------------------------

// One CTA of 4 warps per (query head, row): warp w takes positions w, w + 4, ...; one pass with the running
// maximum and sum per warp, merged in warp order.
template <typename T, int D>
__global__ void __launch_bounds__(128)
k_kv4_attn(const Kv4 c, const T * q, long long q_stride, int heads, const int32_t * row_seq, const int32_t * row_pos,
           const int32_t * seq_slot, int n_seq, float scale, T * out, long long out_stride) {
    pdl_trigger();
    pdl_wait_primary();
    constexpr int G = D / 32;
    __shared__ float sm_m[4], sm_l[4], sm_acc[4][D];
    const int h = blockIdx.x, r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int seq = row_seq[r];
    if (seq < 0 || seq >= n_seq) return;
    const int slot = seq_slot[seq];
    const int n = slot >= 0 && slot < c.n_slots ? min(row_pos[r], c.max_len - 1) + 1 : 0;
    T * dst = out + r * out_stride + h * D;
    if (n <= 0) {
        for (int d = threadIdx.x; d < D; d += 128) dst[d] = from_f32<T>(0.f);
        return;
    }
    float qv[G], acc[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        qv[g] = to_f32(q[r * q_stride + h * D + lane * G + g]);
        acc[g] = 0.f;
    }
    const size_t base = (size_t(slot) * c.kv_heads + h / (heads / c.kv_heads)) * c.max_len;
    float m = -INFINITY, l = 0.f;
    for (int p = warp; p < n; p += 4) {
        const uint8_t * kc = c.k_codes + (base + p) * (D / 2) + lane * (G / 2);
        const uint8_t * vc = c.v_codes + (base + p) * (D / 2) + lane * (G / 2);
        float s = 0.f, vv[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int sh = 4 * (g & 1);
            s = fmaf(qv[g], float(((kc[g / 2] >> sh) & 15) - 8) * __half2float(__ushort_as_half(c.k_scales[(base + p) * G + g])), s);
            vv[g] = float(((vc[g / 2] >> sh) & 15) - 8) * __half2float(__ushort_as_half(c.v_scales[(base + p) * G + g]));
        }
        s = warp_sum(s) * scale;
        const float mn = fmaxf(m, s);
        const float corr = m == -INFINITY ? 1.f : expf(m - mn), e = s == -INFINITY ? 0.f : expf(s - mn);
        l = l * corr + e;
#pragma unroll
        for (int g = 0; g < G; ++g) acc[g] = fmaf(e, vv[g], acc[g] * corr);
        m = mn;
    }
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) sm_acc[warp][lane * G + g] = acc[g];
    __syncthreads();
    if (warp) return;
    float M = -INFINITY, L = 0.f, A[G] = {};
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w]);
    for (int w = 0; w < 4; ++w) {
        if (sm_l[w] == 0.f) continue;  // a warp that saw no position
        const float f = expf(sm_m[w] - M);
        L = fmaf(sm_l[w], f, L);
#pragma unroll
        for (int g = 0; g < G; ++g) A[g] = fmaf(sm_acc[w][lane * G + g], f, A[g]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) dst[lane * G + g] = from_f32<T>(A[g] / L);
}

}  // namespace

}  // namespace exl3cu

using namespace exl3cu;

namespace {

bool dtype_ok(int dtype) { return dtype == EXL3CU_F32 || dtype == EXL3CU_F16 || dtype == EXL3CU_BF16; }

int bad(const char * what) { return api_fail(EXL3CU_INVALID_ARGUMENT, what); }

// A row-strided operand: rows of `width` elements on 16-byte boundaries.
bool rows_ok(const void * p, size_t stride, size_t width, int dtype) {
    const size_t b = dtype == EXL3CU_F32 ? 4 : 2;
    return p && stride >= width && stride <= (size_t(1) << 40) && stride * b % 16 == 0 &&
           reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

bool cache_ok(const exl3cu_kv4_cache * c) {
    return c && c->k_codes && c->k_scales && c->v_codes && c->v_scales && c->n_slots > 0 && c->kv_heads > 0 &&
           c->max_len > 0 && c->max_len % 64 == 0 && (c->head_dim == 64 || c->head_dim == 128) &&
           (reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->k_scales) |
            reinterpret_cast<uintptr_t>(c->v_codes) | reinterpret_cast<uintptr_t>(c->v_scales)) % 16 == 0;
}

Kv4 device_cache(const exl3cu_kv4_cache * c) {
    return Kv4{c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->n_slots, c->kv_heads, c->max_len};
}

constexpr const char * kBadCache =
    "kv4: bad cache (four 16-byte aligned arrays, head_dim 64 or 128, max_len a multiple of 64)";

}  // namespace

extern "C" {

int exl3cu_qk_norm_rope(const void * d_q, size_t q_stride, const void * d_k, size_t k_stride, int dtype, int rows,
                        int heads, int kv_heads, int head_dim, const int32_t * d_row_pos, const float * d_q_w,
                        const float * d_k_w, float eps, const float * d_inv_freq, int rotary_dim, int interleaved,
                        float attn_factor, void * d_q_out, size_t q_out_stride, int q_out_dtype, void * d_k_out,
                        size_t k_out_stride, int k_out_dtype, void * stream) {
    if (head_dim != 64 && head_dim != 128) return bad("qk_norm_rope: head_dim must be 64 or 128");
    if (!dtype_ok(dtype) || !dtype_ok(q_out_dtype) || (kv_heads > 0 && !dtype_ok(k_out_dtype)))
        return bad("qk_norm_rope: unknown dtype");
    if (rows < 0 || heads <= 0 || kv_heads < 0 || heads > 1024 || kv_heads > 1024)
        return bad("qk_norm_rope: bad rows or heads (heads 1..1024, kv_heads 0..1024)");
    if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16 || (rotary_dim && !d_inv_freq))
        return bad("qk_norm_rope: rotary_dim must be a multiple of 16 up to head_dim, with inv_freq");
    if (!rows) return EXL3CU_OK;
    if (!d_row_pos || !rows_ok(d_q, q_stride, size_t(heads) * head_dim, dtype) ||
        !rows_ok(d_q_out, q_out_stride, size_t(heads) * head_dim, q_out_dtype) ||
        (kv_heads && (!rows_ok(d_k, k_stride, size_t(kv_heads) * head_dim, dtype) ||
                      !rows_ok(d_k_out, k_out_stride, size_t(kv_heads) * head_dim, k_out_dtype))))
        return bad("qk_norm_rope: null or misaligned operand, or rows closer than their width");
    const RopeArgs a{d_q, d_k, d_q_out, d_k_out, (long long)q_stride, (long long)k_stride, (long long)q_out_stride,
                     (long long)k_out_stride, d_row_pos, d_q_w, d_k_w, d_inv_freq, eps, attn_factor, rows, heads,
                     kv_heads, rotary_dim, interleaved != 0, q_out_dtype, k_out_dtype};
    const long long items = (long long)rows * (heads + kv_heads);
    if (items > (1ll << 32)) return bad("qk_norm_rope: too many rows");
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        return attn_launch(head_dim == 128 ? k_qk_norm_rope<T, 128> : k_qk_norm_rope<T, 64>,
                           dim3(unsigned((items + 3) / 4)), dim3(128), 0, stream, a);
    });
}

int exl3cu_kv4_append(const exl3cu_kv4_cache * cache, const void * d_k, size_t k_stride, const void * d_v,
                      size_t v_stride, int dtype, int rows, const int32_t * d_row_seq, const int32_t * d_row_pos,
                      const int32_t * d_seq_slot, int n_seq, void * stream) {
    if (!cache_ok(cache)) return bad(kBadCache);
    if (!dtype_ok(dtype)) return bad("kv4_append: unknown dtype");
    if (rows < 0 || n_seq < 0) return bad("kv4_append: negative count");
    if (!rows || !n_seq) return EXL3CU_OK;
    const size_t width = size_t(cache->kv_heads) * cache->head_dim;
    if (!d_row_seq || !d_row_pos || !d_seq_slot || !rows_ok(d_k, k_stride, width, dtype) ||
        !rows_ok(d_v, v_stride, width, dtype))
        return bad("kv4_append: null or misaligned operand, or rows closer than their width");
    const Kv4 c = device_cache(cache);
    const long long items = 2ll * rows * cache->kv_heads;
    if (items > (1ll << 32)) return bad("kv4_append: too many rows");
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        return attn_launch(cache->head_dim == 128 ? k_kv4_append<T, 128> : k_kv4_append<T, 64>,
                           dim3(unsigned((items + 3) / 4)), dim3(128), 0, stream, c, static_cast<const T *>(d_k),
                           (long long)k_stride, static_cast<const T *>(d_v), (long long)v_stride, rows, d_row_seq,
                           d_row_pos, d_seq_slot, n_seq);
    });
}

int exl3cu_kv4_read(const exl3cu_kv4_cache * cache, const int32_t * d_seq_slot, const int32_t * d_kv_offsets, int n_seq,
                    int total_rows, void * d_k, size_t k_stride, void * d_v, size_t v_stride, int dtype,
                    void * stream) {
    if (!cache_ok(cache)) return bad(kBadCache);
    if (!dtype_ok(dtype)) return bad("kv4_read: unknown dtype");
    if (total_rows < 0 || n_seq < 0) return bad("kv4_read: negative count");
    if (!total_rows || !n_seq) return EXL3CU_OK;
    const size_t width = size_t(cache->kv_heads) * cache->head_dim;
    if (!d_seq_slot || !d_kv_offsets || !rows_ok(d_k, k_stride, width, dtype) || !rows_ok(d_v, v_stride, width, dtype))
        return bad("kv4_read: null or misaligned operand, or rows closer than their width");
    const Kv4 c = device_cache(cache);
    const long long items = (long long)total_rows * cache->kv_heads;
    if (items > (1ll << 32)) return bad("kv4_read: too many rows");
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        return attn_launch(cache->head_dim == 128 ? k_kv4_read<T, 128> : k_kv4_read<T, 64>,
                           dim3(unsigned((items + 3) / 4)), dim3(128), 0, stream, c, d_seq_slot, d_kv_offsets, n_seq,
                           total_rows, static_cast<T *>(d_k), (long long)k_stride, static_cast<T *>(d_v),
                           (long long)v_stride);
    });
}

size_t exl3cu_kv4_attn_scratch_bytes(const exl3cu_kv4_cache * cache, int rows, int heads) {
    (void)cache;
    (void)rows;
    (void)heads;
    return 0;
}

int exl3cu_kv4_attn(const exl3cu_kv4_cache * cache, const void * d_q, size_t q_stride, int dtype, int rows, int heads,
                    const int32_t * d_row_seq, const int32_t * d_row_pos, const int32_t * d_seq_slot, int n_seq,
                    float scale, void * d_out, size_t out_stride, void * d_scratch, size_t scratch_bytes,
                    void * stream) {
    if (!cache_ok(cache)) return bad(kBadCache);
    if (!dtype_ok(dtype)) return bad("kv4_attn: unknown dtype");
    if (rows < 0 || n_seq < 0 || rows > 65535) return bad("kv4_attn: rows must be 0..65535 and n_seq not negative");
    if (heads <= 0 || heads % cache->kv_heads || heads > 1024)
        return bad("kv4_attn: heads must be a multiple of kv_heads, at most 1024");
    if (!rows || !n_seq) return EXL3CU_OK;
    const size_t width = size_t(heads) * cache->head_dim;
    if (!d_row_seq || !d_row_pos || !d_seq_slot || !rows_ok(d_q, q_stride, width, dtype) ||
        !rows_ok(d_out, out_stride, width, dtype))
        return bad("kv4_attn: null or misaligned operand, or rows closer than their width");
    (void)d_scratch;
    (void)scratch_bytes;
    const Kv4 c = device_cache(cache);
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        return attn_launch(cache->head_dim == 128 ? k_kv4_attn<T, 128> : k_kv4_attn<T, 64>,
                           dim3(unsigned(heads), unsigned(rows)), dim3(128), 0, stream, c, static_cast<const T *>(d_q),
                           (long long)q_stride, heads, d_row_seq, d_row_pos, d_seq_slot, n_seq, scale,
                           static_cast<T *>(d_out), (long long)out_stride);
    });
}

}  // extern "C"

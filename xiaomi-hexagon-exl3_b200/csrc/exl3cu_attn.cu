// Attention operators for any number of heads of 64 or 128: the query/key norm with the rotary
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
#include "exl3cu_ring.h"

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <tuple>
#include <type_traits>

namespace exl3cu {

static __device__ unsigned g_attn_status;

namespace {

constexpr int kSms = 148;  // a B200's

// Constants of codes2 in registers: an instruction takes one immediate, and these need two.
struct CodeConst {
    uint32_t magic, sixteenth, minus72;
    __device__ __forceinline__ CodeConst() {
        asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
        asm volatile("mov.b32 %0, 0x2c002c00;" : "=r"(sixteenth));
        asm volatile("mov.b32 %0, 0xd480d480;" : "=r"(minus72));
    }
};

// Halves c - 8 of codes i and i + 4 of a word, i = 0 .. 3, from the word for i < 2 and from the word shifted right
// by 8 for i >= 2: the code's bits in the mantissa of 1024 make 1024 + c (or, 4 bits up, 1024 + 16 c).
template <int i> __device__ __forceinline__ uint32_t codes2(uint32_t w, const CodeConst & k) {
    uint32_t x, y;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(w), "r"(i & 1 ? 0x00f000f0u : 0x000f000fu), "r"(k.magic));
    if (i & 1) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x), "r"(k.sixteenth), "r"(k.minus72));
    else asm("add.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0xe408e408u));  // - 1032
    return y;
}

__device__ __forceinline__ float2 h2f2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }

// N elements from 16-byte aligned memory.
template <int N, typename T> __device__ __forceinline__ void load_row(const T * p, float (&x)[N]) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < N; i += V) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p + i);
        const T * e = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int j = 0; j < V; ++j) x[i + j] = to_f32(e[j]);
    }
}

// W words of 4 bytes (1, 2 or 4) from shared memory.
template <int W> __device__ __forceinline__ void lds(const unsigned char * p, uint32_t (&w)[W]) {
    if constexpr (W == 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
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

// Eight elements as they lie, and as floats side by side.
template <typename T> struct Eight {
    static constexpr int kWords = sizeof(T) / 2;
    uint4 raw[kWords];
    __device__ __forceinline__ void load(const T * p) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    __device__ __forceinline__ void get(uint64_t * x) const {
        const T * e = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = two(to_f32(e[2 * i]), to_f32(e[2 * i + 1]));
    }
};

__device__ __forceinline__ void store4(void * p, int dtype, long long at, const float * x) {
    if (dtype == EXL3CU_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p) + at) = make_float4(x[0], x[1], x[2], x[3]);
    } else if (dtype == EXL3CU_F16) {
        const __half2 lo = __floats2half2_rn(x[0], x[1]), hi = __floats2half2_rn(x[2], x[3]);
        *reinterpret_cast<uint2 *>(static_cast<__half *>(p) + at) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
    } else {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(p) + at) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
    }
}

template <typename T> __device__ __forceinline__ uint32_t pack_pair(uint64_t x) {
    const float2 v = of_two(x);
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 y = __floats2half2_rn(v.x, v.y);
        return *reinterpret_cast<const uint32_t *>(&y);
    } else {
        const __nv_bfloat162 y = __floats2bfloat162_rn(v.x, v.y);
        return *reinterpret_cast<const uint32_t *>(&y);
    }
}

// Eight elements as `dtype`.
__device__ __forceinline__ void store8(void * p, int dtype, long long at, const uint64_t * x) {
    if (dtype == EXL3CU_F32) {
        ulonglong2 * to = reinterpret_cast<ulonglong2 *>(static_cast<float *>(p) + at);
        to[0] = make_ulonglong2(x[0], x[1]);
        to[1] = make_ulonglong2(x[2], x[3]);
    } else if (dtype == EXL3CU_F16) {
        *reinterpret_cast<uint4 *>(static_cast<__half *>(p) + at) =
            make_uint4(pack_pair<__half>(x[0]), pack_pair<__half>(x[1]), pack_pair<__half>(x[2]), pack_pair<__half>(x[3]));
    } else {
        *reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p) + at) =
            make_uint4(pack_pair<__nv_bfloat16>(x[0]), pack_pair<__nv_bfloat16>(x[1]), pack_pair<__nv_bfloat16>(x[2]),
                       pack_pair<__nv_bfloat16>(x[3]));
    }
}

// D/16 threads to a head, each with two runs of eight dimensions that hold both members of its pairs ((8 j, half + 8 j)
// or 16 consecutive ones), so that the rotation needs no exchange.  A thread keeps its head (with its weights and
// addresses) and goes through the CTA's rows, the loads of the next kAhead under way; the rows' angles are computed once
// for all heads, kRopeRows rows at a time, into shared memory, behind the first rows' loads.  The CTAs of a call are
// resident together, each with an equal number of rows.  Bound by the bytes of q and k in and out (8191 rows of 20 heads of
// 16 bits, 84 MB: 17.7 us, 4.7 TB/s); a call of few rows by latency (2.7 us).  What it took there: 8 dimensions a thread,
// in accesses of 8 bytes, 26.2 us; kAhead 1 18.8; 8 rows of angles at a time 18.1.
constexpr int kRopeThreads = 320;    // at most: heads beyond kRopeThreads / (D / 16) are taken in turn
constexpr int kRopeRows = 16;
constexpr int kAhead = 2;
constexpr int kRopePerSm = 640;      // threads resident on an SM

// SAME: the outputs are of the inputs' type.
template <typename T, int D, bool SAME>
__global__ void __launch_bounds__(kRopeThreads, 2) k_qk_norm_rope(const RopeArgs a) {
    constexpr int L = D / 16;
    constexpr int kType = std::is_same_v<T, float> ? EXL3CU_F32 : std::is_same_v<T, __half> ? EXL3CU_F16 : EXL3CU_BF16;
    __shared__ __align__(16) float sm_cos[2][kRopeRows * (D / 2)], sm_sin[2][kRopeRows * (D / 2)];
    __shared__ int sm_pos[2][kRopeRows];
    pdl_trigger();
    const int half = a.rotary / 2, j = threadIdx.x % L, per_row = a.heads + a.kv_heads, step = blockDim.x / L;
    // the CTA's rows: an equal share
    const int first = int((long long)a.rows * blockIdx.x / gridDim.x), last = int((long long)a.rows * (blockIdx.x + 1) / gridDim.x);
    // the thread's two runs of dimensions, and the first of its pairs' frequencies where it rotates
    int d0 = 16 * j, d1 = 16 * j + 8, f0 = a.interleaved ? 8 * j : -1;
    if (!a.interleaved && 8 * j < half) d0 = f0 = 8 * j, d1 = half + 8 * j;
    const bool turns = a.interleaved ? d0 < a.rotary : f0 >= 0;
    f0 = max(f0, 0);
    const unsigned mask = ((1u << L) - 1u) << (threadIdx.x & 31 & ~(L - 1));
    pdl_wait_primary();
    for (int row0 = first, buf = 0; row0 < last; row0 += kRopeRows, buf ^= 1) {
        const int rows = min(kRopeRows, last - row0);
        Eight<T> ahead[kAhead][2];
        const T * x;
        long long stride;
        const auto start = [&](int h) {  // the first rows of head h
            const bool is_q = h < a.heads;
            stride = is_q ? a.q_stride : a.k_stride;
            x = (is_q ? static_cast<const T *>(a.q) + h * D : static_cast<const T *>(a.k) + (h - a.heads) * D) + row0 * stride;
#pragma unroll
            for (int u = 0; u < kAhead; ++u, x += stride)
                if (u < rows) {
                    ahead[u][0].load(x + d0);
                    ahead[u][1].load(x + d1);
                }
        };
        int h = threadIdx.x / L;
        if (h < per_row) start(h);
        if (threadIdx.x < rows) sm_pos[buf][threadIdx.x] = a.row_pos[row0 + threadIdx.x];
        for (int i = threadIdx.x; i < rows * half; i += blockDim.x) {
            const int ar = i / half, f = i - ar * half, pos = a.row_pos[row0 + ar];
            float cs, sn;
            rope_angle(max(pos, 0), a.inv_freq[f], a.factor, cs, sn);
            sm_cos[buf][ar * (D / 2) + f] = cs;
            sm_sin[buf][ar * (D / 2) + f] = sn;
        }
        __syncthreads();  // the angles; with two buffers the next chunk's are not those still in use
        while (h < per_row) {
            const bool is_q = h < a.heads;
            const long long out_stride = is_q ? a.q_out_stride : a.k_out_stride;
            const float * weights = is_q ? a.q_w : a.k_w;
            void * out = is_q ? a.q_out : a.k_out;
            const int dt = SAME ? kType : is_q ? a.q_out_dtype : a.k_out_dtype;
            long long at = row0 * out_stride + (is_q ? h : h - a.heads) * D;
            uint64_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // any alignment
                const float * at_w = weights + (i < 4 ? d0 : d1 - 8) + 2 * i;
                w[i] = weights ? two(at_w[0], at_w[1]) : 0;
            }
            const float * cos_at = sm_cos[buf] + f0, * sin_at = sm_sin[buf] + f0;
            for (int r0 = 0; r0 < rows; r0 += kAhead)
#pragma unroll
            for (int u = 0; u < kAhead; ++u, at += out_stride, cos_at += D / 2, sin_at += D / 2) {
                const int r = r0 + u;
                if (r >= rows) break;
                uint64_t v[8];
                ahead[u][0].get(v);
                ahead[u][1].get(v + 4);
                if (r + kAhead < rows) {
                    ahead[u][0].load(x + d0);
                    ahead[u][1].load(x + d1);
                    x += stride;
                }
                if (weights) {
                    uint64_t sq = mul2(v[0], v[0]);
#pragma unroll
                    for (int i = 1; i < 8; ++i) sq = fma2(v[i], v[i], sq);
                    const float2 parts = of_two(sq);
                    float ss = parts.x + parts.y;
#pragma unroll
                    for (int s = L / 2; s; s >>= 1) ss += __shfl_xor_sync(mask, ss, s);
                    const float inv = rsqrtf(ss * (1.f / D) + a.eps);
                    const uint64_t inv2 = two(inv, inv);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = mul2(mul2(v[i], inv2), w[i]);
                }
                if (turns) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {  // four pairs at a time
                        const float4 c4 = reinterpret_cast<const float4 *>(cos_at)[i], s4 = reinterpret_cast<const float4 *>(sin_at)[i];
                        if (a.interleaved) {  // (x, y) (c, c) + (y, x) (-s, s)
                            const float cs[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                uint64_t & y = v[4 * i + k];
                                const float2 of = of_two(y);
                                y = fma2(two(of.y, of.x), two(-sn[k], sn[k]), mul2(y, two(cs[k], cs[k])));
                            }
                        } else {
                            const uint64_t cs[2] = {two(c4.x, c4.y), two(c4.z, c4.w)}, sn[2] = {two(s4.x, s4.y), two(s4.z, s4.w)};
                            const uint64_t minus[2] = {two(-s4.x, -s4.y), two(-s4.z, -s4.w)};
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                uint64_t & y0 = v[2 * i + k], & y1 = v[4 + 2 * i + k];
                                const uint64_t x0 = y0, x1 = y1;
                                y0 = fma2(x1, minus[k], mul2(x0, cs[k]));
                                y1 = fma2(x0, sn[k], mul2(x1, cs[k]));
                            }
                        }
                    }
                }
                if (sm_pos[buf][r] < 0) continue;
                store8(out, dt, at + d0, v);
                store8(out, dt, at + d1, v + 4);
            }
            h += step;
            if (h < per_row) start(h);
        }
    }
}

// ---- the 4-bit cache -------------------------------------------------------------------------------

constexpr int kCacheThreads = 256;

// Codes of 8 dimensions, the first of a group 0, as a word; x two side by side, s the scales, inv = 1 / s within an ulp or
// two, 0 where s is 0.  A sum with 1.5 * 2^23 + 8 rounds to the nearest integer, ties to even, and leaves the code in its
// low bits; the constant high bits come off the assembled word at once.
//   x of 16 bits: x / s differs from a tie (n + 1/2) by at least 2^-16 unless it is one, since x has 11 bits and
//   (n + 1/2) s at most 15; rounding the approximate quotient (off by 2^-20 at most) to multiples of 2^-18 first, by a
//   sum with 48, makes ties exact and moves nothing else across one.
//   f32: the remainder x - t s is exact; where it reaches half a step (a tie, or the quotient's error) the exact
//   comparison of kv4_code decides.
template <typename T, int G>
__device__ __forceinline__ uint32_t kv4_word(const uint64_t (&x)[4], const float (&s)[G], const float (&inv)[G]) {
    constexpr float kMagic = 12582912.f + 8.f;
    constexpr uint32_t kHigh = 0x4b400000u;  // the bits of 1.5 * 2^23
    const uint64_t magic = two(kMagic, kMagic);
    uint32_t word = 0, taken = 0;
    bool close = false;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        const uint64_t inv2 = two(inv[2 * i % G], inv[(2 * i + 1) % G]);
        uint64_t w;
        if constexpr (sizeof(T) == 4) {
            w = fma2(x[i], inv2, magic);
            const float2 d = of_two(fma2(add2(magic, mul2(w, two(-1.f, -1.f))), two(s[2 * i % G], s[(2 * i + 1) % G]), x[i]));
            close = close || fabsf(d.x) >= 0.5f * s[2 * i % G] || fabsf(d.y) >= 0.5f * s[(2 * i + 1) % G];
        } else {
            w = add2(add2(fma2(x[i], inv2, two(48.f, 48.f)), two(-48.f, -48.f)), magic);
        }
        const float2 v = of_two(w);
        word = (word * 16u + __float_as_uint(v.y)) * 16u + __float_as_uint(v.x);
        taken = (taken * 16u + kHigh) * 16u + kHigh;
    }
    word -= taken;
    if (sizeof(T) == 4 && close) {
        word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = of_two(x[i]);
            word |= kv4_code(v.x, s[2 * i % G], inv[2 * i % G]) << (8 * i);
            word |= kv4_code(v.y, s[(2 * i + 1) % G], inv[(2 * i + 1) % G]) << (8 * i + 4);
        }
    }
    return word;
}

// The larger of the bits of |x|, of each half.
__device__ __forceinline__ uint32_t most2(uint32_t a, uint32_t b) { return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu); }

// The scales of a head's groups (0, 1 in the first word, 2, 3 in the second) from its D/16 lanes' dimensions, 16 each, as
// they lie; returns whether a group has a value beyond 7 times the largest scale (or one that is not finite).  |x| is
// compared as an integer, so that a NaN is the largest; those of 16 bits two at a time, even and odd groups side by side.
// Lanes halve the groups that they carry with each exchange, and come by the others' scales in the end.
template <typename T, int D>
__device__ __forceinline__ bool kv4_scales(const Eight<T> (&e)[2], unsigned mask, int j, uint32_t (&pair)[D / 64]) {
    constexpr int G = D / 32;
    constexpr uint32_t kMost = 0x48dfe400u;  // the bits of 7 * 65504
    uint32_t own;
    bool beyond;
    if constexpr (sizeof(T) == 2) {
        uint32_t m[G / 2];
#pragma unroll
        for (int g = 0; g < G / 2; ++g) {
            const auto at = [&](int i) { return reinterpret_cast<const uint32_t *>(e[i / 4].raw)[i % 4]; };
            m[g] = most2(at(g), at(g + G / 2));
#pragma unroll
            for (int i = g + G; i < 8; i += G / 2) m[g] = most2(m[g], at(i));
        }
        if constexpr (G == 4) {
            const bool up = j & 4;
            const uint32_t got = __shfl_xor_sync(mask, up ? m[0] : m[1], 4);
            m[0] = __vmaxu2(up ? m[1] : m[0], got);
        }
        m[0] = __vmaxu2(m[0], __shfl_xor_sync(mask, m[0], 2));
        m[0] = __vmaxu2(m[0], __shfl_xor_sync(mask, m[0], 1));
        const auto bits = [](uint32_t h) {  // of the f32 that it stands for
            return __float_as_uint(to_f32(*reinterpret_cast<const T *>(&h)));
        };
        const uint32_t lo = bits(m[0] & 0xffffu), hi = bits(m[0] >> 16);
        own = uint32_t(__half_as_ushort(kv4_scale(lo))) | uint32_t(__half_as_ushort(kv4_scale(hi))) << 16;
        beyond = max(lo, hi) > kMost;
    } else {
        uint32_t m[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const auto at = [&](int i) { return reinterpret_cast<const uint32_t *>(e[i / 8].raw)[i % 8] & 0x7fffffffu; };
            m[g] = at(g);
#pragma unroll
            for (int i = g + G; i < 16; i += G) m[g] = max(m[g], at(i));
        }
        if constexpr (G == 4) {
            const bool up = j & 4;
            const uint32_t a = __shfl_xor_sync(mask, up ? m[0] : m[2], 4), b = __shfl_xor_sync(mask, up ? m[1] : m[3], 4);
            m[0] = max(up ? m[2] : m[0], a);
            m[1] = max(up ? m[3] : m[1], b);
        }
        const bool up = j & 2;
        const uint32_t got = __shfl_xor_sync(mask, up ? m[0] : m[1], 2);
        m[0] = max(up ? m[1] : m[0], got);
        m[0] = max(m[0], __shfl_xor_sync(mask, m[0], 1));
        const uint32_t mine = __half_as_ushort(kv4_scale(m[0])), other = __shfl_xor_sync(mask, mine, 2);
        own = up ? other | mine << 16 : mine | other << 16;
        beyond = m[0] > kMost;
    }
    if constexpr (G == 4) {
        const uint32_t other = __shfl_xor_sync(mask, own, 4);
        pair[0] = j & 4 ? other : own;
        pair[1] = j & 4 ? own : other;
    } else {
        pair[0] = own;
    }
    return beyond;
}

// D/16 threads a (row, head), each with 16 consecutive dimensions of the key and of the value: two words of codes each,
// and 16 / G elements of every group (dimension d is of group d mod G).  24234 rows of 8 heads of 64 dimensions, 64 MB in
// and out: 17.0 us, 3.7 TB/s, at 63 % of the issue slots (8 dimensions a thread: 18.8, 79 %).  blockIdx.y is the head: the
// CTA's rows, consecutive positions of a prompt, are one piece of the cache (heads of a row side by side: 18.8).
template <typename T, int D>
__global__ void __launch_bounds__(kCacheThreads)
k_kv4_append(const Kv4 c, const T * k, long long k_stride, const T * v, long long v_stride, int rows,
             const int32_t * row_seq, const int32_t * row_pos, const int32_t * seq_slot, int n_seq) {
    constexpr int G = D / 32, L = D / 16;
    pdl_trigger();
    const int r = blockIdx.x * (kCacheThreads / L) + threadIdx.x / L, h = blockIdx.y, j = threadIdx.x % L;
    const unsigned mask = ((1u << L) - 1u) << (threadIdx.x & 31 & ~(L - 1));
    pdl_wait_primary();
    if (r >= rows) return;
    const int seq = row_seq[r], pos = row_pos[r];
    Eight<T> e[2][2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const T * src = (w ? v + r * v_stride : k + r * k_stride) + h * D + 16 * j;
        e[w][0].load(src);
        e[w][1].load(src + 8);
    }
    if (seq < 0 || seq >= n_seq) return;
    const int slot = seq_slot[seq];
    if (slot < 0 || slot >= c.n_slots || pos < 0 || pos >= c.max_len) return;
    const size_t at = (size_t(slot) * c.kv_heads + h) * c.max_len + pos;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t pair[G / 2];
        const bool beyond = kv4_scales<T, D>(e[w], mask, j, pair);
        if (!(j & 3)) reinterpret_cast<uint32_t *>((w ? c.v_scales : c.k_scales) + at * G)[j / 4] = pair[j / 4 % (G / 2)];
        float s[G], inv[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float2 f = h2f2(pair[g / 2]);
            s[g] = g & 1 ? f.y : f.x;
            inv[g] = s[g] > 0.f ? __fdividef(1.f, s[g]) : 0.f;
        }
        uint64_t x[2][4];
        e[w][0].get(x[0]);
        e[w][1].get(x[1]);
        // a group beyond the largest scale saturates; one that is not finite has codes of zero
        if (__any_sync(mask, beyond)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float2 y = of_two(x[i / 4][i % 4]);
                const float a = 7.f * s[2 * i % G], b = 7.f * s[(2 * i + 1) % G];
                y.x = inv[2 * i % G] > 0.f ? fminf(fmaxf(y.x, -a), a) : 0.f;
                y.y = inv[(2 * i + 1) % G] > 0.f ? fminf(fmaxf(y.y, -b), b) : 0.f;
                x[i / 4][i % 4] = two(y.x, y.y);
            }
        }
        reinterpret_cast<uint2 *>((w ? c.v_codes : c.k_codes) + at * (D / 2))[j] =
            make_uint2(kv4_word<T, G>(x[0], s, inv), kv4_word<T, G>(x[1], s, inv));
    }
}

// D/8 threads a (row, head), each with 8 consecutive dimensions of the key and of the value; kReadRows rows a thread,
// whose loads are under way together; the heads of a row side by side, as they lie in the output.  Bound by the bytes
// written: 50 MB 14.4 us, 3.4 TB/s, as fast as so many are filled with zeros (4 rows a thread 14.9, 1 16.7).
constexpr int kReadRows = 2;

template <typename T, int D>
__global__ void __launch_bounds__(kCacheThreads)
k_kv4_read(const Kv4 c, const int32_t * seq_slot, const int32_t * offsets, int n_seq, int total, T * k,
           long long k_stride, T * v, long long v_stride) {
    constexpr int G = D / 32, L = D / 8, kStep = kCacheThreads / L;
    pdl_trigger();
    const int blk = blockIdx.x / c.kv_heads, h = blockIdx.x - blk * c.kv_heads, j = threadIdx.x % L;
    const int first = blk * (kReadRows * kStep) + threadIdx.x / L;  // rows first, first + kStep, ...
    const CodeConst kc2;
    pdl_wait_primary();
    if (first >= total) return;
    int seq = find_segment(offsets, n_seq, first);
    const int end = min(offsets[n_seq], total);
    uint32_t codes[kReadRows][2], scales[kReadRows][2][G / 2];
    bool live[kReadRows];
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
        const int r = first + u * kStep;
        live[u] = false;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            codes[u][w] = 0x88888888u;
#pragma unroll
            for (int g = 0; g < G / 2; ++g) scales[u][w][g] = 0;
        }
        if (r >= end) continue;
        if (seq < 0) seq = find_segment(offsets, n_seq, r);
        if (seq < 0) continue;
        while (r >= offsets[seq + 1]) ++seq;  // ends: r < offsets[n_seq]
        live[u] = true;
        const int slot = seq_slot[seq], pos = r - offsets[seq];
        if (slot < 0 || slot >= c.n_slots || pos >= c.max_len) continue;  // zeros
        const size_t at = (size_t(slot) * c.kv_heads + h) * c.max_len + pos;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            codes[u][w] = reinterpret_cast<const uint32_t *>((w ? c.v_codes : c.k_codes) + at * (D / 2))[j];
            lds(reinterpret_cast<const unsigned char *>((w ? c.v_scales : c.k_scales) + at * G), scales[u][w]);
        }
    }
#pragma unroll
    for (int u = 0; u < kReadRows; ++u) {
        if (!live[u]) continue;
        const long long r = first + u * kStep;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float s[G], x[8];
#pragma unroll
            for (int g = 0; g < G; g += 2) {
                const float2 f = h2f2(scales[u][w][g / 2]);
                s[g] = f.x;
                s[g + 1] = f.y;
            }
            const uint32_t lo = codes[u][w], hi = lo >> 8;
            const uint32_t pairs[4] = {codes2<0>(lo, kc2), codes2<1>(lo, kc2), codes2<2>(hi, kc2), codes2<3>(hi, kc2)};
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // codes i and i + 4, less 8
                const float2 f = h2f2(pairs[i]);
                x[i] = f.x * s[i % G];
                x[i + 4] = f.y * s[i % G];
            }
            T * out = (w ? v + r * v_stride : k + r * k_stride) + h * D + 8 * j;
            if constexpr (sizeof(T) == 4) {
                store4(out, EXL3CU_F32, 0, x);
                store4(out, EXL3CU_F32, 4, x + 4);
            } else {
                uint4 q;
                T * e = reinterpret_cast<T *>(&q);
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
                *reinterpret_cast<uint4 *>(out) = q;
            }
        }
    }
}

// ---- attention of single rows over the cache ------------------------------------------------------
//
// One pass over the keys of a row in tiles of 64, on the matrix instructions, with the running maximum and sum
// of a softmax.  The bytes of the cache (2 (D/2 + D/16) a key and K/V head) are its floor, if a code costs few
// instructions; so codes are never multiplied by their scales.  8 rows of 131072 positions (604 MB): 117 us, 5.2 TB/s;
// the loads alone 94.  The difference is a tile's chain of products, softmax and products with the three warps that a
// scheduler has: a tenth fewer instructions (uncentred codes on the key side) gave 118 for 119, copies of keys and values
// that start separately 124.
//
//   Codes become halves by one logic operation on two at a time (into the mantissa of 1024) and one multiply-add
//   (to c - 8, exact), after a shift for every other four.
//   Scales stay out of the operands.  A score is sum over groups of s_g (q_g . codes_g): a group (d mod D/32) is
//   two steps of 16 of the product, so s_g multiplies the group's sum.  On the value side the weight times s_g is the
//   other operand, one fragment per group; the 16 dimensions of a product's rows are of one group.
//
//   S^T [16 keys x 8] = K codes (A, as they lie: lane t of a row's four holds 16 bytes) times q (B).
//   O^T [16 dimensions x 8] += V codes (A: pairs of keys brought together by a byte permutation) times weights
//   (B: the score fragment, transposed by movmatrix).
//
// Columns: 8 heads of 16-bit rows, or, where no more than 4 share a K/V head, one head to a pair of columns, which
// halves what a lane computes around the products; of f32 rows the pair's second column holds what the first one's
// rounding left, 2^11 times as large so that it keeps its digits where x is small: x = hi + 2^-11 lo to 2^-22 of x down to
// 2^-23 of the largest, and to 2^-45 of the largest below.  (16-bit rows: weights rounded to 2^-11 of their value, the
// result's own precision.)
// Both operands are scaled by powers of two into the half's range: q by its largest element, the weights by the largest
// value scale seen of their group, so that nothing overflows and a group of small values beside one of large ones keeps
// its digits.  The maximum that the weights refer to follows the true one when it has grown by more than 2^kLazy.  Masked
// keys get a score of -inf and scales of zero; codes are finite whatever they are.
//
// The tiles of all rows form one list that is cut into equal shares, one per CTA, so that a batch of a long and
// many short contexts fills the GPU evenly (a row counts kRowCost tiles more than it has: what taking up a row costs
// a CTA).  A CTA's part of a row that it does not hold whole goes to scratch as (maximum, sum, accumulator), and
// k_kv4_merge joins the parts in order.  (Few rows of few positions: a cluster of CTAs to a row instead.)

constexpr int kKeys = 64;        // keys per tile
constexpr int kAttnWarps = 4;    // warps of a CTA, each with tiles of its own
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr int kAttnCtas = 3;     // per SM
constexpr int kScanThreads = 128;
static_assert(kAttnThreads >= kScanThreads, "the rows are scanned by the first 128 threads");
constexpr int kStages = 2;       // tiles in flight per warp
constexpr int kSplitRows = 256;  // rows up to which the tiles of all rows are cut into equal shares
constexpr int kRowCost = 8;      // 8 rows between 1 and 32768 positions: 19.0 us with 2, 15.0 with 8, 15.1 with 12
constexpr int kPlanFloats = 2 * kSplitRows;  // scratch begins with (first share, shares) of every row
constexpr int kMinShare = 4;     // tiles of a share: one per warp at least
// Few rows in a cache of few positions: a cluster of CTAs takes a row and joins its parts from their shared memory, which
// spares the second kernel: 1 row behind 767 positions 6.8 us (f32; with shares 8.6), behind 2047 6.5 (bf16; 9.3), 8 rows
// behind 4095 11.7 (14.7).  Above 4096 positions, or with more clusters than are resident together, shares are faster:
// 8191 positions 10.6 against 9.6, 32 rows of 767 20.8 against 13.8.
constexpr int kCluster = 8;
constexpr int kClusterTiles = 64;
constexpr int kLazy = 6, kTop = 15 - kLazy;  // weights times value scales are up to 2^kTop, 2^15 before m moves
constexpr float kLow = 2048.f;   // of the low parts of f32 operands

template <int D> struct Kv4Tile {
    static constexpr int kCodes = kKeys * D / 2, kScales = kKeys * D / 16;  // bytes of one of K and V
    static constexpr int kBytes = 2 * (kCodes + kScales);
};

// How the tiles are divided: a CTA a row; equal shares of all rows' tiles; a cluster of CTAs a row.
enum Split { kWhole, kShares, kClusters };

struct Kv4Attn {
    Kv4 c;
    const void * q;
    void * out;
    long long q_stride, out_stride;
    const int32_t * row_seq;
    const int32_t * row_pos;
    const int32_t * seq_slot;
    float * part;  // kPlanFloats; [y][x][2][HC][D + 4]: a CTA's row that it begins and does not end, and the one
                   // that it goes on with
    int rows, n_seq, heads, chunks;
    int split;          // see Split
    float scale_log2;   // scale * log2(e)
};

// Visible keys of row r and its slot: -1 keys for a row of no sequence.
__device__ __forceinline__ int visible(const Kv4Attn & a, int r, int & slot) {
    const int seq = a.row_seq[r], pos = a.row_pos[r];
    slot = 0;
    if (seq < 0 || seq >= a.n_seq) return -1;
    slot = a.seq_slot[seq];
    return slot >= 0 && slot < a.c.n_slots ? max(0, min(pos, a.c.max_len - 1) + 1) : 0;
}

__device__ __forceinline__ int tiles_of(int n) { return (max(n, 0) + kKeys - 1) / kKeys; }
__device__ __forceinline__ int list_of(int n) { return n > 0 ? tiles_of(n) + kRowCost : 0; }

// Visible keys and slots of rows 2 i and 2 i + 1 for thread i of the first 128, the list before them, and the whole
// list's length for every thread.  sm: 4 ints.
__device__ __forceinline__ void scan_rows(const Kv4Attn & a, int (&n)[2], int (&slot)[2], int & before, int & total,
                                          int * sm) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = threadIdx.x * 2 + i;
        n[i] = -1;
        if (r < a.rows && threadIdx.x < kScanThreads) n[i] = visible(a, r, slot[i]);
    }
    const int mine = list_of(n[0]) + list_of(n[1]);
    int upto = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += o;
    }
    if (lane == 31 && warp < kScanThreads / 32) sm[warp] = upto;
    __syncthreads();
    before = upto - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < warp) before += sm[w];
        total += sm[w];
    }
}

__device__ __forceinline__ int share_of(int total, int shares) {
    const int each = (total + shares - 1) / shares;
    return max(kMinShare, (each + kAttnWarps - 1) / kAttnWarps * kAttnWarps);
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// d = a b.
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    uint32_t y;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 .. 127

// The key of a 16-key step that row g (and, 8 further, row g + 8) of the score fragment stands for.  Chosen so
// that both the rows read for the scores (g = 2 i, 2 i + 1 together) and those read for the values (g = 2 t) fall
// on different banks as far as a row of 64 or 32 bytes allows.
template <int D> __device__ __forceinline__ int key_of(int g) {
    return g & 1 ? 4 + ((g >> 1) ^ (D == 128 ? 1 : 2)) : g >> 1;
}

template <typename T, int D, int HC>
__global__ void __launch_bounds__(kAttnThreads, kAttnCtas) k_kv4_attn(const Kv4Attn a) {
    using Tile = Kv4Tile<D>;
    constexpr int G = D / 32, H = HC / 4;  // groups, heads of a lane's scores
    constexpr bool PAIR = HC == 4, LO = sizeof(T) == 4;  // a head to two columns; the second one its low halves
    static_assert(!LO || PAIR, "f32 rows take two columns a head");
    extern __shared__ __align__(128) unsigned char ring_all[];
    __shared__ uint64_t full[kAttnWarps][kStages];
    __shared__ int sm_n[kSplitRows], sm_slot[kSplitRows], sm_scan[4], sm_row, sm_off;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char * ring = ring_all + warp * kStages * Tile::kBytes;
    const int share_heads = a.heads / a.c.kv_heads;
    const int kvh = blockIdx.y / a.chunks, chunk = blockIdx.y % a.chunks;
    const int head0 = kvh * share_heads + chunk * HC, nh = min(HC, share_heads - chunk * HC);
    T * const out = static_cast<T *>(a.out) + head0 * D;
    pdl_trigger();
    if (threadIdx.x < kAttnWarps * kStages) mbar_init(&full[0][0] + threadIdx.x, 1);
    mbar_init_fence();
    pdl_wait_primary();

    const auto zero_row = [&](int r) {
        for (int i = 0; i < nh * D; ++i) out[r * a.out_stride + i] = from_f32<T>(0.f);
    };
    // the next row (of the list; row0 + row of the call), where in it to begin, what is left of the share
    int row = 0, off = 0, left;
    const int row0 = a.split == kShares ? 0 : a.split == kClusters ? blockIdx.x / kCluster : blockIdx.x;
    if (a.split == kShares) {
        int n[2], slot[2], before, total;
        scan_rows(a, n, slot, before, total, sm_scan);
        const int share = share_of(total, gridDim.x), begin = blockIdx.x * share;
        left = min(share, total - begin);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = threadIdx.x * 2 + i, list = list_of(n[i]);
            if (r < a.rows && r < kSplitRows) {
                sm_n[r] = n[i];
                sm_slot[r] = slot[i];
            }
            if (n[i] == 0 && r % gridDim.x == blockIdx.x) zero_row(r);
            if (before <= begin && begin < before + list) {
                sm_row = r;
                sm_off = begin - before;
            }
            if (blockIdx.x == 0 && blockIdx.y == 0 && r < a.rows && r < kSplitRows) {
                const int x0 = before / share;
                reinterpret_cast<int2 *>(a.part)[r] = make_int2(x0, n[i] > 0 ? (before + tiles_of(n[i]) - 1) / share - x0 + 1 : 0);
            }
            before += list;
        }
        __syncthreads();
        if (left <= 0) return;
        row = sm_row;
        off = sm_off;
    } else {
        int slot;
        const int n = visible(a, row0, slot);
        if (threadIdx.x == 0) {
            sm_n[0] = n;
            sm_slot[0] = slot;
            if (n == 0 && (a.split == kWhole || blockIdx.x % kCluster == 0)) zero_row(row0);
        }
        __syncthreads();
        if (n <= 0) return;  // the whole cluster
        left = list_of(n);
        if (a.split == kClusters) {
            const int share = (tiles_of(n) + kCluster - 1) / kCluster;
            off = blockIdx.x % kCluster * share;
            left = share;
        }
    }

    const CodeConst kc2;
    CopyRing<kStages> copies;  // tiles of this warp
    const auto arrived = [&](unsigned slot, unsigned parity) { return bool(__all_sync(0xffffffffu, mbar_wait(&full[warp][slot], parity))); };
    while (left > 0) {
        const int n = sm_n[row], tiles = tiles_of(n), t0 = min(off, tiles), t1 = min(tiles, off + left);
        left = a.split == kClusters ? 0 : left - min(left, list_of(n) - off);
        off = 0;
        const int call_row = row0 + row, slot = sm_slot[row];
        ++row;
        if (t0 >= t1) continue;
        const size_t base = (size_t(slot) * a.c.kv_heads + kvh) * a.c.max_len;
        const auto start = [&](int tile, unsigned to) {
            unsigned char * dst = ring + to * Tile::kBytes;
            uint64_t * bar = &full[warp][to];
            if (lane == 0) {
                const size_t key = base + size_t(tile) * kKeys;
                mbar_arrive_expect_tx(bar, Tile::kBytes);
                bulk_g2s(dst, a.c.k_codes + key * (D / 2), Tile::kCodes, bar);
                bulk_g2s(dst + Tile::kCodes, a.c.k_scales + key * G, Tile::kScales, bar);
                bulk_g2s(dst + Tile::kCodes + Tile::kScales, a.c.v_codes + key * (D / 2), Tile::kCodes, bar);
                bulk_g2s(dst + 2 * Tile::kCodes + Tile::kScales, a.c.v_scales + key * G, Tile::kScales, bar);
            }
        };
#pragma unroll
        for (int i = 0; i < kStages; ++i)
            if (t0 + warp + i * kAttnWarps < t1) start(t0 + warp + i * kAttnWarps, copies.slot(i));

        // q as the B operand: column g is a head (PAIR: half of one); this lane's dimensions are
        // [t D/4, +D/4), words of 8, codes i and i + 4 of a word a pair.  Scaled by 2^e to a largest element in [2^8, 2^9).
        uint32_t qb[D / 16][2];
        float cs[H];
        {
            const int col_head = PAIR ? g >> 1 : g;
            float x[D / 4], top = 0.f;
            const T * src = static_cast<const T *>(a.q) + call_row * a.q_stride + (head0 + min(col_head, nh - 1)) * D + t * (D / 4);
            load_row<D / 4>(src, x);
#pragma unroll
            for (int i = 0; i < D / 4; ++i) {
                if (col_head >= nh) x[i] = 0.f;
                top = fmaxf(top, fabsf(x[i]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int ex = int(__float_as_uint(top) >> 23);  // 255: an infinity
            const int e = ex == 255 ? 0 : min(135 - ex, 126);  // f32 has no smaller normal than 2^-126, which becomes 1
            const float up = pow2(e);
#pragma unroll
            for (int i = 0; i < D / 4; ++i) {
                x[i] *= up;
                if (LO) {
                    const float hi = __half2float(__float2half_rn(x[i]));
                    x[i] = g & 1 ? (x[i] - hi) * kLow : hi;
                } else if (PAIR && (g & 1)) {
                    x[i] = 0.f;
                }
            }
#pragma unroll
            for (int st = 0; st < D / 16; ++st) {
                const int i = st & 3, w = 2 * (st >> 2);  // code of a word, first of the step's two words
                qb[st][0] = pack_h2(x[8 * w + i], x[8 * w + i + 4]);
                qb[st][1] = pack_h2(x[8 * w + 8 + i], x[8 * w + 12 + i]);
            }
#pragma unroll
            for (int j = 0; j < H; ++j) {  // the score's columns are 2 t and 2 t + 1
                const int eh = __shfl_sync(0xffffffffu, e, 8 * t + 4 * j);
                cs[j] = fminf(fmaxf(a.scale_log2 * pow2(-eh), 1.2e-38f), 3e38f);  // 0 or inf would meet inf or 0
            }
        }

        // accumulators; the score that weights refer to (before cs); sum of the weights.  Weights are
        // exp2((s - m) cs + 14 + kTop - ev), ev the exponent of the largest value scale seen, which is below 2^(ev - 14).
        // The value scales of a group whose own largest is smaller are raised by what it is smaller, a power of two up to
        // 2^15, before they meet the weights: exact in a half, and a group 2^15 further down still has its weights at
        // 2^(kTop - 15).  evs: the groups' own exponents as they stand in a half, two to a word.  (Accumulators o[i] are
        // of group i mod G.)
        float o[D / 16][4] = {}, m[H], l[H] = {};
#pragma unroll
        for (int j = 0; j < H; ++j) m[j] = -INFINITY;
        int ev = 0;
        uint32_t evs[G / 2] = {};
        // exponents of the groups' largest scales as raised, in a half's place: no more than 15 below ev
        const auto raised = [&](int i) { return __vmaxu2(evs[i], uint32_t(max(ev - 15, 0)) * 0x04000400u); };
        const auto exponent = [&](int j) { return int(raised(j / 2) >> (16 * (j & 1) + 10) & 31u); };  // of group j
        int tile = t0 + warp;
        for (; tile < t1; tile += kAttnWarps) {
            const unsigned char * kc = ring + copies.slot() * Tile::kBytes;
            const unsigned char * ks = kc + Tile::kCodes, * vc = ks + Tile::kScales, * vs = vc + Tile::kCodes;
            if (!copies.next(arrived)) break;
            const int keys = n - tile * kKeys;  // visible keys of the tile, >= 1
            if (keys < kKeys) {  // what lies behind them may not be finite: scales of zero
                uint32_t * z = reinterpret_cast<uint32_t *>(const_cast<unsigned char *>(ks));
                for (int i = keys * (G / 2) + lane; i < kKeys * (G / 2); i += 32) {
                    z[i] = 0;
                    z[i + (Tile::kScales + Tile::kCodes) / 4] = 0;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next copy into the slot
                __syncwarp();
            }
            // scores of keys 16 x + key_of(g) (+ 8), heads t (PAIR) or 2 t, 2 t + 1
            float sc[4][2][H];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int k0 = 16 * x + key_of<D>(g);
                uint32_t w0[D / 32], w1[D / 32], u0[D / 32], u1[D / 32], s0[G / 2], s1[G / 2];
                lds(kc + k0 * (D / 2) + t * (D / 8), w0);
                lds(kc + (k0 + 8) * (D / 2) + t * (D / 8), w1);
                lds(ks + k0 * (2 * G), s0);
                lds(ks + (k0 + 8) * (2 * G), s1);
#pragma unroll
                for (int w = 0; w < D / 32; ++w) {
                    u0[w] = w0[w] >> 8;
                    u1[w] = w1[w] >> 8;
                }
                float acc[G][4];
                const auto take = [&](auto ic) {  // codes I and I + 4 of the words: group I mod G
                    constexpr int I = decltype(ic)::value;
#pragma unroll
                    for (int w = 0; w < D / 32; w += 2) {
                        const uint32_t f[4] = {codes2<I>(I < 2 ? w0[w] : u0[w], kc2), codes2<I>(I < 2 ? w1[w] : u1[w], kc2),
                                               codes2<I>(I < 2 ? w0[w + 1] : u0[w + 1], kc2), codes2<I>(I < 2 ? w1[w + 1] : u1[w + 1], kc2)};
                        if (w == 0 && I < G) mma16816_first(acc[I % G], f, qb[2 * w + I][0], qb[2 * w + I][1]);
                        else mma16816(acc[I % G], f, qb[2 * w + I][0], qb[2 * w + I][1]);
                    }
                };
                take(std::integral_constant<int, 0>{});
                take(std::integral_constant<int, 1>{});
                take(std::integral_constant<int, 2>{});
                take(std::integral_constant<int, 3>{});
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    const float2 f0 = h2f2(s0[j / 2]), f1 = h2f2(s1[j / 2]);
                    const float a0 = j & 1 ? f0.y : f0.x, a1 = j & 1 ? f1.y : f1.x;
#pragma unroll
                    for (int jj = 0; jj < H; ++jj) {
                        const float v0 = LO ? fmaf(acc[j][1], 1.f / kLow, acc[j][0]) : acc[j][jj];
                        const float v1 = LO ? fmaf(acc[j][3], 1.f / kLow, acc[j][2]) : acc[j][2 + jj];
                        sc[x][0][jj] = j ? fmaf(a0, v0, sc[x][0][jj]) : a0 * v0;
                        sc[x][1][jj] = j ? fmaf(a1, v1, sc[x][1][jj]) : a1 * v1;
                    }
                }
            }
            if (keys < kKeys) {
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y)
                        if (16 * x + key_of<D>(g) + 8 * y >= keys)
#pragma unroll
                            for (int j = 0; j < H; ++j) sc[x][y][j] = -INFINITY;
            }
            // exponents of the groups' largest value scales of the lane's two keys; the lane's largest scores.  The others'
            // are asked for only where something has moved: exchanges would stand in every tile's way.
            bool moved = false;
            {
                uint32_t w[G];
                lds(vs + lane * (4 * G), w);
#pragma unroll
                for (int i = 0; i < G / 2; ++i)
                    moved = moved || __vmaxu2(__vmaxu2(w[i] & 0x7c007c00u, w[i + G / 2] & 0x7c007c00u), evs[i]) != evs[i];
            }
            float mx[H];
#pragma unroll
            for (int j = 0; j < H; ++j) {
                mx[j] = max3(m[j], sc[0][0][j], sc[0][1][j]);
#pragma unroll
                for (int x = 1; x < 4; ++x) mx[j] = max3(mx[j], sc[x][0][j], sc[x][1][j]);
                moved = moved || (mx[j] - m[j]) * cs[j] > float(kLazy);  // no: both -inf
            }
            if (__any_sync(0xffffffffu, moved)) {
                int before[G];
#pragma unroll
                for (int i = 0; i < G; ++i) before[i] = exponent(i);
                const int ev_before = ev;
                {
                    uint32_t w[G];
                    lds(vs + lane * (4 * G), w);
#pragma unroll
                    for (int i = 0; i < G / 2; ++i) {
                        uint32_t e = 0;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {  // a scale that is not finite does not count: its group's result is not either
                            const uint32_t x = w[i + k * (G / 2)] & 0x7c007c00u;
                            e = __vmaxu2(e, x & ~__vcmpeq2(x, 0x7c007c00u));
                        }
                        const uint32_t lo = __reduce_max_sync(0xffffffffu, e & 0xffffu), hi = __reduce_max_sync(0xffffffffu, e >> 16);
                        evs[i] = __vmaxu2(evs[i], lo | hi << 16);
                        ev = max(ev, int(max(evs[i] & 0xffffu, evs[i] >> 16) >> 10));
                    }
                }
                float f[H];
#pragma unroll
                for (int j = 0; j < H; ++j) {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], x));
                    f[j] = mx[j] == m[j] ? 1.f : exp2_approx((m[j] - mx[j]) * cs[j]);
                    m[j] = mx[j];
                }
                if (tile != t0 + warp) {  // sums so far
                    float down[G];
#pragma unroll
                    for (int i = 0; i < G; ++i) down[i] = pow2(before[i] - exponent(i));
#pragma unroll
                    for (int j = 0; j < H; ++j) {
                        l[j] *= f[j] * pow2(ev_before - ev);
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) {
                            const float fg = f[j] * down[i % G];
                            o[i][j] *= fg;
                            o[i][2 + j] *= fg;
                            if (LO) {
                                o[i][1] *= fg;
                                o[i][3] *= fg;
                            }
                        }
                    }
                }
            }
            uint32_t raise[G / 2];  // 2^(ev - the exponent as raised), two halves
#pragma unroll
            for (int i = 0; i < G / 2; ++i) raise[i] = uint32_t(15 + ev) * 0x04000400u - raised(i);
            // the difference to m before the factor: with a rounded m cs in its place, scores above 2^24 would be off by
            // whole powers of two
            const float top = float(14 + kTop - ev);
            float less[H];
#pragma unroll
            for (int j = 0; j < H; ++j) less[j] = m[j] == -INFINITY ? 0.f : -m[j];
            const uint64_t less2 = two(less[0], less[H - 1]), cs2 = two(cs[0], cs[H - 1]), top2 = two(top, top);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int k0 = 16 * x + key_of<D>(g);
                uint32_t s0[G / 2], s1[G / 2];
                lds(vs + k0 * (2 * G), s0);
                lds(vs + (k0 + 8) * (2 * G), s1);
#pragma unroll
                for (int j = 0; j < G / 2; ++j) {
                    asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(s0[j]) : "r"(raise[j]));
                    asm("mul.rn.f16x2 %0, %0, %1;" : "+r"(s1[j]) : "r"(raise[j]));
                }
                float p[2][H];
#pragma unroll
                for (int i = 0; i < H; ++i) {  // two at a time: the keys of a head (PAIR), or the heads of a key
                    const float2 e = of_two(fma2(add2(two(sc[x][PAIR ? 0 : i][0], PAIR ? sc[x][1][0] : sc[x][i][H - 1]), less2), cs2, top2));
                    p[PAIR ? 0 : i][0] = exp2_approx(e.x);
                    p[PAIR ? 1 : i][H - 1] = exp2_approx(e.y);
                    l[0] += p[PAIR ? 0 : i][0];
                    l[H - 1] += p[PAIR ? 1 : i][H - 1];
                }
                uint32_t pb[G][2];
#pragma unroll
                for (int j = 0; j < G; ++j)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float2 f = h2f2(y ? s1[j / 2] : s0[j / 2]);
                        const float sv = j & 1 ? f.y : f.x, v0 = p[y][0] * sv;
                        pb[j][y] = transpose8x8(LO ? pack_h2(v0, (v0 - __half2float(__float2half_rn(v0))) * kLow)
                                                   : pack_h2(v0, PAIR ? 0.f : p[y][H - 1] * sv));
                    }
                // values of keys 2 t, 2 t + 1 and 8 further (as the score rows count them): dimensions of word(s) g
                uint32_t va[D / 64], vb[D / 64], vc2[D / 64], vd[D / 64];
                const int ka = 16 * x + t, kb = 16 * x + 4 + (t ^ (D == 128 ? 1 : 2));
                lds(vc + ka * (D / 2) + g * (D / 16), va);
                lds(vc + kb * (D / 2) + g * (D / 16), vb);
                lds(vc + (ka + 8) * (D / 2) + g * (D / 16), vc2);
                lds(vc + (kb + 8) * (D / 2) + g * (D / 16), vd);
                // codes 0-3 and 4-7 of two keys in a word, and the same shifted for codes 2, 3 and 6, 7
                uint32_t lo01[2][D / 64], hi01[2][D / 64], lo23[2][D / 64], hi23[2][D / 64];
#pragma unroll
                for (int w = 0; w < D / 64; ++w) {
                    lo01[0][w] = __byte_perm(va[w], vb[w], 0x5410);
                    hi01[0][w] = __byte_perm(va[w], vb[w], 0x7632);
                    lo23[0][w] = __byte_perm(vc2[w], vd[w], 0x5410);
                    hi23[0][w] = __byte_perm(vc2[w], vd[w], 0x7632);
                    lo01[1][w] = lo01[0][w] >> 8;
                    hi01[1][w] = hi01[0][w] >> 8;
                    lo23[1][w] = lo23[0][w] >> 8;
                    hi23[1][w] = hi23[0][w] >> 8;
                }
                const auto take = [&](auto ic) {
                    constexpr int I = decltype(ic)::value, S = I / 2;
                    if constexpr (D == 128) {  // dimensions 16 g + I, 16 g + 8 + I; then the same 4 further
                        const uint32_t f[4] = {codes2<I>(lo01[S][0], kc2), codes2<I>(lo01[S][1], kc2), codes2<I>(lo23[S][0], kc2), codes2<I>(lo23[S][1], kc2)};
                        mma16816(o[I], f, pb[I % G][0], pb[I % G][1]);
                        const uint32_t h[4] = {codes2<I>(hi01[S][0], kc2), codes2<I>(hi01[S][1], kc2), codes2<I>(hi23[S][0], kc2), codes2<I>(hi23[S][1], kc2)};
                        mma16816(o[I + 4], h, pb[I % G][0], pb[I % G][1]);
                    } else {  // dimensions 8 g + I, 8 g + 4 + I
                        const uint32_t f[4] = {codes2<I>(lo01[S][0], kc2), codes2<I>(hi01[S][0], kc2), codes2<I>(lo23[S][0], kc2), codes2<I>(hi23[S][0], kc2)};
                        mma16816(o[I], f, pb[I % G][0], pb[I % G][1]);
                    }
                };
                take(std::integral_constant<int, 0>{});
                take(std::integral_constant<int, 1>{});
                take(std::integral_constant<int, 2>{});
                take(std::integral_constant<int, 3>{});
            }
            __syncwarp();  // every lane has read the tile
            if (tile + kStages * kAttnWarps < t1) start(tile + kStages * kAttnWarps, copies.slot(kStages - 1));
        }

        // short of the end after a wait that ran out: copies in flight end before the CTA does
        copies.drain(min(kStages, (t1 - tile + kAttnWarps - 1) / kAttnWarps), arrived);
        constexpr int kRec = D + 4;
        if (!__syncthreads_and(tile >= t1)) {
            // no result: a row that the CTA has to itself stays as it was, and in the parts that a join will look for here
            // a maximum that is NaN makes it the result
            if (threadIdx.x == 0) atomicOr(&g_attn_status, kStatusWaitTimeout);
            if (a.split == kShares && threadIdx.x < (t0 ? 2 * HC : HC))  // record 1, if any, comes before record 0
                a.part[kPlanFloats + ((size_t(blockIdx.y) * gridDim.x + blockIdx.x) * (2 * HC) + threadIdx.x) * kRec + D] = NAN;
            if (a.split == kClusters && threadIdx.x < HC)
                reinterpret_cast<float *>(ring_all)[(HC + threadIdx.x) * kRec + D] = NAN;
            break;
        }
        // the warp's part: sums over the lanes of a head, then into the warp's own ring (its copies have landed):
        // [HC][D + 4], accumulator, maximum (times cs), sum
        float * const mine = reinterpret_cast<float *>(ring);
        float back[G];
#pragma unroll
        for (int i = 0; i < G; ++i) back[i] = pow2(exponent(i) - 14 - kTop);
#pragma unroll
        for (int j = 0; j < H; ++j) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[j] += __shfl_xor_sync(0xffffffffu, l[j], x);
            float * rec = mine + (PAIR ? t : 2 * t + j) * kRec;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const int d = D == 128 ? 16 * g + i : 8 * g + i;
                rec[d] = (LO ? fmaf(o[i][1], 1.f / kLow, o[i][0]) : o[i][j]) * back[i % G];
                rec[d + (D == 128 ? 8 : 4)] = (LO ? fmaf(o[i][3], 1.f / kLow, o[i][2]) : o[i][2 + j]) * back[i % G];
            }
            if (g == 0) {
                rec[D] = m[j] * cs[j];
                rec[D + 1] = l[j] * pow2(ev - 14 - kTop);
            }
        }
        const bool whole = t0 == 0 && t1 == tiles;
        __syncthreads();
        float * part = whole ? nullptr
                       : a.split == kClusters
                           ? reinterpret_cast<float *>(ring_all) + HC * kRec  // behind the first warp's record
                           : a.part + kPlanFloats + ((size_t(blockIdx.y) * gridDim.x + blockIdx.x) * 2 + (t0 ? 1 : 0)) * (HC * kRec);
        for (int i = threadIdx.x; i < nh * D; i += kAttnThreads) {
            const int h = i / D, d = i % D;
            const float * rec = reinterpret_cast<const float *>(ring_all) + h * kRec;
            constexpr int kNext = kStages * Tile::kBytes / 4;
            float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) M = fmaxf(M, rec[w * kNext + D]);
            const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) {
                const float f = exp2_approx(rec[w * kNext + D] - ref);
                L = fmaf(rec[w * kNext + D + 1], f, L);
                A = fmaf(rec[w * kNext + d], f, A);
            }
            if (whole) {
                out[call_row * a.out_stride + i] = from_f32<T>(A / L);
            } else {
                part[h * kRec + d] = A;
                if (d == 0) {
                    part[h * kRec + D] = M;
                    part[h * kRec + D + 1] = L;
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next copies overwrite these records
        __syncthreads();
    }
    if (a.split == kClusters) {  // join the parts, in order; the outputs are dealt out among the cluster's threads
        namespace cg = cooperative_groups;
        constexpr int kRec = D + 4;
        const int tiles = tiles_of(sm_n[0]), share = (tiles + kCluster - 1) / kCluster, used = (tiles + share - 1) / share;
        if (used == 1) return;  // the whole cluster
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        for (int i = blockIdx.x % kCluster * kAttnThreads + threadIdx.x; i < nh * D; i += kCluster * kAttnThreads) {
            float M[kCluster], L = 0.f, A = 0.f, top = -INFINITY;
            const float * rec = reinterpret_cast<const float *>(ring_all) + HC * kRec + i / D * kRec;
#pragma unroll
            for (int u = 0; u < kCluster; ++u) {
                M[u] = u < used ? cluster.map_shared_rank(rec, u)[D] : -INFINITY;
                top = fmaxf(top, M[u]);
            }
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int u = 0; u < kCluster; ++u)
                if (u < used) {
                    const float * r = cluster.map_shared_rank(rec, u);
                    const float f = exp2_approx(M[u] - ref);
                    L = fmaf(r[D + 1], f, L);
                    A = fmaf(r[i % D], f, A);
                }
            out[row0 * a.out_stride + i] = from_f32<T>(A / L);
        }
        cluster.sync();  // the others' reads
    }
}

// Joins the parts of the rows that were cut, in a fixed order.  WIDE (few rows, so many parts to each): a CTA per
// (row, K/V head chunk, head), a thread per dimension and kGroups-th part.  Otherwise a CTA per (row, K/V head chunk),
// a thread per output.  Bound by latency: the parts' loads go out together, kBatch to a thread.
constexpr int kMergeThreads = 1024;

template <typename T, int D, int HC, bool WIDE>
__global__ void __launch_bounds__(WIDE ? kMergeThreads : HC * D) k_kv4_merge(const Kv4Attn a, int shares) {
    constexpr int kRec = D + 4, kGroups = WIDE ? kMergeThreads / D : 1, kBatch = WIDE ? 14 : 4;
    __shared__ float sm_a[kGroups][D], sm_m[kGroups], sm_l[kGroups];
    const int row = blockIdx.x, y = blockIdx.y;
    pdl_trigger();
    pdl_wait_primary();
    const int2 plan = reinterpret_cast<const int2 *>(a.part)[row];  // first share, shares
    if (plan.y <= 1) return;
    const int share_heads = a.heads / a.c.kv_heads, chunk = y % a.chunks;
    const int h = WIDE ? blockIdx.z : threadIdx.x / D, d = threadIdx.x % D, group = WIDE ? threadIdx.x / D : 0;
    if (h >= min(HC, share_heads - chunk * HC)) return;
    const float * const base = a.part + kPlanFloats + ((size_t(y) * shares + plan.x) * 2 * HC + h) * kRec;
    float M = -INFINITY, L = 0.f, A = 0.f;
    for (int i0 = group; i0 < plan.y; i0 += kBatch * kGroups) {
        float vm[kBatch], vl[kBatch], va[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = min(i0 + kGroups * u, plan.y - 1);
            // a CTA's record 0 is the row that it begins and does not end, record 1 the row that it goes on with
            const float * r = base + (size_t(i) * 2 + (i > 0)) * HC * kRec;
            vm[u] = r[D];
            vl[u] = r[D + 1];
            va[u] = r[d];
        }
        float mn = M;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) mn = fmaxf(mn, vm[u]);
        const float ref = mn == -INFINITY ? 0.f : mn, f0 = exp2_approx(M - ref);
        L *= f0;
        A *= f0;
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (i0 + kGroups * u < plan.y) {
                const float f = exp2_approx(vm[u] - ref);
                L = fmaf(vl[u], f, L);
                A = fmaf(va[u], f, A);
            }
        M = mn;
    }
    if constexpr (WIDE) {
        sm_a[group][d] = A;
        if (d == 0) {
            sm_m[group] = M;
            sm_l[group] = L;
        }
        __syncthreads();
        if (group) return;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) M = fmaxf(M, sm_m[i]);
        const float ref = M == -INFINITY ? 0.f : M;
        L = A = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            const float f = exp2_approx(sm_m[i] - ref);
            L = fmaf(sm_l[i], f, L);
            A = fmaf(sm_a[i][d], f, A);
        }
    }
    static_cast<T *>(a.out)[row * a.out_stride + (y / a.chunks * share_heads + chunk * HC + h) * D + d] = from_f32<T>(A / L);
}

// How a call is cut up: shares (CTAs) per K/V head chunk, 0 for one CTA per row.
struct AttnPlan {
    int heads_per_cta, chunks, ys, shares;
    Split split;
    size_t scratch;
};

AttnPlan plan_attn(const exl3cu_kv4_cache * c, int rows, int heads, int dtype) {
    AttnPlan p;
    const int share_heads = heads / c->kv_heads;
    p.heads_per_cta = dtype == EXL3CU_F32 || share_heads <= 4 ? 4 : 8;
    p.chunks = (share_heads + p.heads_per_cta - 1) / p.heads_per_cta;
    p.ys = c->kv_heads * p.chunks;
    p.shares = 0;
    p.scratch = 0;
    p.split = kWhole;
    if (rows > kSplitRows) return p;
    p.split = c->max_len / kKeys <= kClusterTiles && (long long)rows * p.ys * kCluster <= kAttnCtas * kSms ? kClusters : kShares;
    // as many CTAs as are resident together (three per SM), no more than there can be shares
    const long long most = ((long long)rows * (c->max_len / kKeys + kRowCost) + kMinShare - 1) / kMinShare;
    p.shares = int(std::max(1ll, std::min((long long)(kAttnCtas * kSms / p.ys), most)));
    p.scratch = kPlanFloats * sizeof(float) + size_t(p.ys) * p.shares * 2 * p.heads_per_cta * (c->head_dim + 4) * sizeof(float);
    return p;
}

}  // namespace

cudaError_t attn_read_status(unsigned * out, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(out, g_attn_status, sizeof(unsigned));
    if (e == cudaSuccess && clear && *out) {
        const unsigned zero = 0;
        e = cudaMemcpyToSymbol(g_attn_status, &zero, sizeof(unsigned));
    }
    return e;
}

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
           c->kv_heads <= 1024 && c->max_len > 0 && c->max_len % 64 == 0 && c->max_len <= 1 << 27 && (c->head_dim == 64 || c->head_dim == 128) &&
           (reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->k_scales) |
            reinterpret_cast<uintptr_t>(c->v_codes) | reinterpret_cast<uintptr_t>(c->v_scales)) % 16 == 0;
}

Kv4 device_cache(const exl3cu_kv4_cache * c) {
    return Kv4{c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->n_slots, c->kv_heads, c->max_len};
}

// Words of 8 bytes, each read as the kind of the parameter that it becomes.
struct Words {
    const char * at;
    template <typename P> P next() {
        P v;
        memcpy(&v, at, 8);
        at += 8;
        return v;
    }
    operator int() { return int(next<long long>()); }
    operator size_t() { return next<size_t>(); }
    operator float() { return float(next<double>()); }
    template <typename P> operator P *() { return next<P *>(); }
};

template <typename... A> int call_with_words(int (*f)(A...), const void * words) {
    Words w{static_cast<const char *>(words)};
    const std::tuple<A...> args{static_cast<A>(w)...};  // braces: evaluated in order
    return std::apply(f, args);
}

constexpr const char * kBadCache =
    "kv4: bad cache (four 16-byte aligned arrays, head_dim 64 or 128, max_len a multiple of 64 up to 2^27)";

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
    const bool same = q_out_dtype == dtype && (!kv_heads || k_out_dtype == dtype);
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        const int lanes = head_dim / 16;
        const int threads = (std::min((heads + kv_heads) * lanes, kRopeThreads) + 31) / 32 * 32;
        const dim3 grid(unsigned(std::min(rows, kRopePerSm / threads * kSms))), block{unsigned(threads)};
        if (head_dim == 128)
            return attn_launch(same ? k_qk_norm_rope<T, 128, true> : k_qk_norm_rope<T, 128, false>, grid, block, 0, stream, 1, a);
        return attn_launch(same ? k_qk_norm_rope<T, 64, true> : k_qk_norm_rope<T, 64, false>, grid, block, 0, stream, 1, a);
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
    const int per_cta = kCacheThreads / (cache->head_dim / 16);
    const dim3 grid(unsigned((rows - 1) / per_cta + 1), unsigned(cache->kv_heads));
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        return attn_launch(cache->head_dim == 128 ? k_kv4_append<T, 128> : k_kv4_append<T, 64>,
                           grid, dim3(kCacheThreads), 0, stream, 1, c, static_cast<const T *>(d_k),
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
    const int per_cta = kReadRows * (kCacheThreads / (cache->head_dim / 8));
    const dim3 grid(unsigned((total_rows - 1) / per_cta + 1) * unsigned(cache->kv_heads));
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        return attn_launch(cache->head_dim == 128 ? k_kv4_read<T, 128> : k_kv4_read<T, 64>,
                           grid, dim3(kCacheThreads), 0, stream, 1, c, d_seq_slot, d_kv_offsets, n_seq,
                           total_rows, static_cast<T *>(d_k), (long long)k_stride, static_cast<T *>(d_v),
                           (long long)v_stride);
    });
}

size_t exl3cu_kv4_attn_scratch_bytes(const exl3cu_kv4_cache * cache, int rows, int heads) {
    if (!cache_ok(cache) || rows <= 0 || heads <= 0 || heads % cache->kv_heads) return 0;
    // the larger of the two forms: f32 rows, and 16-bit rows
    return std::max(plan_attn(cache, rows, heads, EXL3CU_F32).scratch, plan_attn(cache, rows, heads, EXL3CU_F16).scratch);
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
    if (!(scale > 0.f) || scale > 1e30f) return bad("kv4_attn: scale must be positive and finite");
    if (!rows || !n_seq) return EXL3CU_OK;
    const size_t width = size_t(heads) * cache->head_dim;
    if (!d_row_seq || !d_row_pos || !d_seq_slot || !rows_ok(d_q, q_stride, width, dtype) ||
        !rows_ok(d_out, out_stride, width, dtype))
        return bad("kv4_attn: null or misaligned operand, or rows closer than their width");
    const AttnPlan p = plan_attn(cache, rows, heads, dtype);
    if (p.scratch && (!d_scratch || scratch_bytes < p.scratch || reinterpret_cast<uintptr_t>(d_scratch) % 16))
        return bad("kv4_attn: scratch missing, misaligned or too small (exl3cu_kv4_attn_scratch_bytes)");
    const Kv4Attn a{device_cache(cache), d_q, d_out, (long long)q_stride, (long long)out_stride, d_row_seq, d_row_pos,
                    d_seq_slot, static_cast<float *>(d_scratch), rows, n_seq, heads, p.chunks, p.split,
                    scale * 1.4426950408889634f};
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        const auto run = [&](auto dim, auto heads_per_cta) {
            constexpr int D = decltype(dim)::value, HC = decltype(heads_per_cta)::value;
            constexpr int smem = kAttnWarps * kStages * Kv4Tile<D>::kBytes;
            static_assert(size_t(HC) * (D + 4) * 4 <= kStages * Kv4Tile<D>::kBytes, "a warp's record fits its ring");
            int dev = 0;
            if (cudaGetDevice(&dev) != cudaSuccess) return api_cuda_fail(cudaGetLastError(), "kv4_attn");
            static std::atomic<unsigned long long> done{0};  // devices whose kernel may use that much shared memory
            const unsigned long long bit = 1ull << (dev & 63);
            if (!(done.load() & bit)) {
                const cudaError_t e =
                    cudaFuncSetAttribute(k_kv4_attn<T, D, HC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
                if (e != cudaSuccess) return api_cuda_fail(e, "kv4_attn: shared memory");
                done.fetch_or(bit);
            }
            const int ctas = p.split == kShares ? p.shares : p.split == kClusters ? rows * kCluster : rows;
            const int rc = attn_launch(k_kv4_attn<T, D, HC>, dim3(unsigned(ctas), unsigned(p.ys)), dim3(kAttnThreads), size_t(smem),
                                       stream, p.split == kClusters ? kCluster : 1, a);
            if (rc || p.split != kShares) return rc;
            // a row has about shares / rows parts: above 8, a CTA per head, below, one for all heads of a K/V head
            if (p.shares > 8 * rows)
                return attn_launch(k_kv4_merge<T, D, HC, true>, dim3(unsigned(rows), unsigned(p.ys), HC),
                                   dim3(kMergeThreads), 0, stream, 1, a, p.shares);
            return attn_launch(k_kv4_merge<T, D, HC, false>, dim3(unsigned(rows), unsigned(p.ys)), dim3(HC * D), 0,
                               stream, 1, a, p.shares);
        };
        constexpr std::integral_constant<int, 64> d64;
        constexpr std::integral_constant<int, 128> d128;
        constexpr std::integral_constant<int, 4> h4;
        if constexpr (sizeof(T) == 2) {
            constexpr std::integral_constant<int, 8> h8;
            if (p.heads_per_cta == 8) return cache->head_dim == 128 ? run(d128, h8) : run(d64, h8);
        }
        return cache->head_dim == 128 ? run(d128, h4) : run(d64, h4);
    });
}

int exl3cu_attn_words(int call, const void * words) {
    if (!words) return bad("attn_words: words is NULL");
    switch (call) {
        case EXL3CU_CALL_QK_NORM_ROPE: return call_with_words(exl3cu_qk_norm_rope, words);
        case EXL3CU_CALL_KV4_APPEND: return call_with_words(exl3cu_kv4_append, words);
        case EXL3CU_CALL_KV4_READ: return call_with_words(exl3cu_kv4_read, words);
        case EXL3CU_CALL_KV4_ATTN: return call_with_words(exl3cu_kv4_attn, words);
        case EXL3CU_CALL_PROMPT_ATTN: return call_with_words(exl3cu_prompt_attn, words);
        default: return bad("attn_words: unknown call");
    }
}

}  // extern "C"

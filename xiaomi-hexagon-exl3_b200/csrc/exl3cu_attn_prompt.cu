// Causal attention of packed sequences with grouped heads (exl3cu_prompt_attn; contract in exl3cu_attn.h).
#include "exl3cu.h"
#include "exl3cu_async.cuh"
#include "exl3cu_attn.cuh"
#include "exl3cu_attn.h"
#include "exl3cu_internal.h"

namespace exl3cu {

namespace {

struct PromptArgs {
    const void * q;
    const void * k;
    const void * v;
    void * out;
    long long q_stride, k_row, k_head, v_row, v_head, out_stride;
    const int32_t * q_offsets;
    const int32_t * kv_begin;
    const int32_t * kv_end;
    int n_seq, q_rows, kv_rows, heads, kv_heads, out_dtype;
    float scale;
};

// One warp per (query row, head), one pass over the visible keys: lane holds dimensions [lane * D/32, +D/32).
template <typename T, int D>
__global__ void __launch_bounds__(128) k_prompt_attn(const PromptArgs a) {
    pdl_trigger();
    pdl_wait_primary();
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const long long item = blockIdx.x * 4ll + (threadIdx.x >> 5);
    if (item >= (long long)a.q_rows * a.heads) return;
    const int r = int(item / a.heads), h = int(item % a.heads);
    const int s = find_segment(a.q_offsets, a.n_seq, r);
    if (s < 0) return;
    const int k0 = max(a.kv_begin[s], 0), k1 = min(a.kv_end[s], a.kv_rows);
    const int n = k1 - k0 - (a.q_offsets[s + 1] - 1 - r);  // visible keys
    const int kvh = h / (a.heads / a.kv_heads);
    const T * q = static_cast<const T *>(a.q) + r * a.q_stride + h * D + lane * E;
    const T * k = static_cast<const T *>(a.k) + k0 * a.k_row + kvh * a.k_head + lane * E;
    const T * v = static_cast<const T *>(a.v) + k0 * a.v_row + kvh * a.v_head + lane * E;
    float qv[E], acc[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        qv[i] = to_f32(q[i]);
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int p = 0; p < n; ++p) {
        float sc = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) sc = fmaf(qv[i], to_f32(k[p * a.k_row + i]), sc);
#pragma unroll
        for (int x = 16; x; x >>= 1) sc += __shfl_xor_sync(0xffffffffu, sc, x);
        sc *= a.scale;
        const float mn = fmaxf(m, sc);
        const float corr = m == -INFINITY ? 1.f : expf(m - mn), e = sc == -INFINITY ? 0.f : expf(sc - mn);
        l = l * corr + e;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] = fmaf(e, to_f32(v[p * a.v_row + i]), acc[i] * corr);
        m = mn;
    }
    const long long at = r * a.out_stride + h * D + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float o = n > 0 ? acc[i] / l : 0.f;
        if (a.out_dtype == EXL3CU_F32) static_cast<float *>(a.out)[at + i] = o;
        else static_cast<T *>(a.out)[at + i] = from_f32<T>(o);
    }
}

}  // namespace

}  // namespace exl3cu

using namespace exl3cu;

extern "C" int exl3cu_prompt_attn(const void * d_q, size_t q_stride, const void * d_k, size_t k_row_stride,
                                  size_t k_head_stride, const void * d_v, size_t v_row_stride, size_t v_head_stride,
                                  int kv_rows, int dtype, int heads, int kv_heads, int head_dim,
                                  const int32_t * d_q_offsets, const int32_t * d_kv_begin, const int32_t * d_kv_end,
                                  int n_seq, int q_rows, float scale, void * d_out, size_t out_stride, int out_dtype,
                                  void * stream) {
    const auto bad = [](const char * what) { return api_fail(EXL3CU_INVALID_ARGUMENT, what); };
    if (head_dim != 64 && head_dim != 128) return bad("prompt_attn: head_dim must be 64 or 128");
    if (dtype != EXL3CU_F16 && dtype != EXL3CU_BF16) return bad("prompt_attn: q, k and v must be f16 or bf16");
    if (out_dtype != dtype && out_dtype != EXL3CU_F32) return bad("prompt_attn: out must be f32 or of q's type");
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 1024)
        return bad("prompt_attn: heads must be a multiple of kv_heads, at most 1024");
    if (n_seq < 0 || q_rows < 0 || kv_rows < 0) return bad("prompt_attn: negative count");
    if (!n_seq || !q_rows) return EXL3CU_OK;
    constexpr size_t kMaxStride = size_t(1) << 36;  // 2^37 bytes: below the tensor map's limit
    const auto aligned = [](const void * p) { return p && reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const auto stride_ok = [&](size_t s, size_t least, size_t unit) { return s >= least && s <= kMaxStride && s % unit == 0; };
    const size_t width = size_t(heads) * head_dim;
    if (!aligned(d_q) || !aligned(d_out) || !stride_ok(q_stride, width, 8) ||
        !stride_ok(out_stride, width, out_dtype == EXL3CU_F32 ? 4 : 8))
        return bad("prompt_attn: q or out null or misaligned, or rows closer than their width");
    if (kv_rows && (!aligned(d_k) || !aligned(d_v) || !stride_ok(k_row_stride, head_dim, 8) ||
                    !stride_ok(v_row_stride, head_dim, 8) || !stride_ok(k_head_stride, head_dim, 8) ||
                    !stride_ok(v_head_stride, head_dim, 8)))
        return bad("prompt_attn: k or v null or misaligned, or a stride below head_dim or no multiple of 8");
    if (!d_q_offsets || !d_kv_begin || !d_kv_end) return bad("prompt_attn: offsets are NULL");
    const PromptArgs a{d_q, d_k, d_v, d_out, (long long)q_stride, (long long)k_row_stride, (long long)k_head_stride,
                       (long long)v_row_stride, (long long)v_head_stride, (long long)out_stride, d_q_offsets, d_kv_begin,
                       d_kv_end, n_seq, q_rows, kv_rows, heads, kv_heads, out_dtype, scale};
    const long long items = (long long)q_rows * heads;
    if (items > (1ll << 32)) return bad("prompt_attn: too many query rows");
    const dim3 grid(unsigned((items + 3) / 4)), block(128);
    if (dtype == EXL3CU_F16)
        return attn_launch(head_dim == 128 ? k_prompt_attn<__half, 128> : k_prompt_attn<__half, 64>, grid, block, 0,
                           stream, a);
    return attn_launch(head_dim == 128 ? k_prompt_attn<__nv_bfloat16, 128> : k_prompt_attn<__nv_bfloat16, 64>, grid,
                       block, 0, stream, a);
}

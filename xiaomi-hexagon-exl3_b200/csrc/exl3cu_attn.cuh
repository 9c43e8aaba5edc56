// Shared by the attention operators (exl3cu_attn.cu, exl3cu_attn_prompt.cu): element types, the 4-bit
// code and scale of a cached value, and the launch helper.
#pragma once
#include "exl3cu.h"
#include "exl3cu_attn.h"
#include "exl3cu_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace exl3cu {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two floats side by side, the operands of the two-wide instructions.
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t y;
    asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(lo), "f"(hi));
    return y;
}
__device__ __forceinline__ float2 of_two(uint64_t x) {
    float2 y;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
    return y;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t y;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
    return y;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t y;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t y;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
    return y;
}

// exl3cu_kv4_cache without head_dim (a template argument of the kernels).
struct Kv4 {
    uint8_t * k_codes;
    uint16_t * k_scales;
    uint8_t * v_codes;
    uint16_t * v_scales;
    int n_slots, kv_heads, max_len;
};

// The scale of a group from the bits of its largest |x| (compared as integers, so that a NaN is the
// largest): the smallest half with 7 * scale >= |x|, at most 65504.  The half nearest to the quotient is that one
// or the one below it, and 7 times a half is exact.
__device__ __forceinline__ __half kv4_scale(uint32_t most_bits) {
    const float most = __uint_as_float(most_bits);
    const __half near = __float2half_rn(fminf(most * (1.f / 7.f), 65504.f));
    uint32_t bits = __half_as_ushort(near);
    if (7.f * __half2float(near) < most && bits < 0x7bffu) ++bits;
    return __ushort_as_half(most_bits >= 0x7f800000u ? 0x7fff : bits);  // an infinity or a NaN in the group
}

// 8 + x / s rounded to the nearest integer, ties to even, from -7 to 7; inv about 1 / s.  The approximate quotient is at
// most one step off; x - t s is exact (t s has 15 bits at most, and t s and x are within a factor of
// two of one another where t is not zero), and so is its comparison with s / 2.
__device__ __forceinline__ uint32_t kv4_code(float x, float s, float inv) {
    if (!(s > 0.f)) return 8u;  // a group of zeros, or a NaN scale
    float t = rintf(x * inv);
    t = fminf(fmaxf(t, -8.f), 8.f);  // saturated groups
    const float d = fmaf(-t, s, x), h = 0.5f * s;
    const bool odd = (int(t) & 1) != 0;
    if (d > h || (d == h && odd)) t += 1.f;
    else if (d < -h || (d == -h && odd)) t -= 1.f;
    return uint32_t(int(fminf(fmaxf(t, -7.f), 7.f)) + 8);
}

// The segment s of [offsets[s], offsets[s + 1]) that holds row r, or -1.  Offsets ascend; empty segments hold
// nothing.
__device__ __forceinline__ int find_segment(const int32_t * offsets, int n, int r) {
    if (r < offsets[0] || r >= offsets[n]) return -1;
    int lo = 0, hi = n;  // offsets[lo] <= r < offsets[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= r) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Calls f with a value of the element type that `dtype` names.
template <typename F>
int with_type(int dtype, F && f) {
    if (dtype == EXL3CU_F32) return f(float{});
    if (dtype == EXL3CU_F16) return f(__half{});
    return f(__nv_bfloat16{});
}

// Launch with programmatic stream serialization (the kernels wait for their predecessor with
// griddepcontrol.wait before touching memory); clusters of
// `cluster` CTAs along x.
template <typename... KArgs, typename... Args>
int attn_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, void * stream, int cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
    if (e == cudaSuccess) return EXL3CU_OK;
    (void)cudaGetLastError();
    return api_cuda_fail(e, "attention operator");
}

}  // namespace exl3cu

// Causal attention of packed sequences with grouped heads on the 5th-generation tensor cores
// (exl3cu_prompt_attn; contract in exl3cu_attn.h).
//
// out = softmax(scale Q K^T) V per query head, one pass over the keys in tiles of 128 with a running
// maximum and sum per query row.  4 D flops a visible (query, key) pair and head: bound by the tensor cores
// and, at the same rate at D = 128, by the exponentials (16 a clock and SM).  16384 tokens, 16 heads of 128:
// 836 us, 1315 TFLOP/s, in short runs; 975 us, 1128 TFLOP/s, in long ones, which the power limit holds back; 37 tokens
// 7.2 us.
//
// One CTA serves one sequence's block of query rows for a group of P heads that share a K/V head (P: the largest
// power of two, at most 16, that divides heads / kv_heads): two tiles of 128 rows, row = position * P + head, so
// that the heads of a group share the K/V tiles and a causal block wastes at most one tile of keys.  The
// blocks of a sequence are launched longest first.
//
// Per tile of keys:  S = Q K^T (tcgen05, operands in shared memory by TMA, 128-byte swizzle), S in TMEM;
// a thread owns a row of S: maximum, P = exp2(scale log2e (S - m)), a quarter of them on the multiply-add pipe,
// row sum in f32, P rounded to the 16-bit type (half a step each: the product takes 16-bit operands) and stored over S
// in TMEM;  O += P V, begun when three quarters of P are there, with P from TMEM, V from shared memory as it lies (MN-major), O in
// TMEM.  The maximum that the weights refer to follows the true one only when it has grown by more than 2^8, so O is
// rescaled rarely.
//
// (Two threads a row instead of one: the exponentials of a tile take no less time, 1235 against 877 us at 16384
// tokens.)
//
// Warps: 0-3 and 4-7 the rows of the two tiles; 8 loads; 9 issues the products and owns TMEM.  While one
// tile's rows work on their exponentials, the other tile's products run.
//
// Values that a row does not see must not reach it even if they are not finite (0 * NaN is NaN in a product).
// Scores are replaced where masked.  For values the load warp reads the tiles of V in which some row's view
// ends, sets elements that are not finite to zero and notes per dimension the first key that held a NaN, +inf
// or -inf; the rows that see that key get it back at the end.
//
// Every wait is bounded; a wait that runs out sets a status bit, and the CTA ends without its result.
#include "exl3cu.h"
#include "exl3cu_async.cuh"
#include "exl3cu_attn.cuh"
#include "exl3cu_attn.h"
#include "exl3cu_internal.h"

#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace exl3cu {

static __device__ unsigned g_prompt_status;

namespace {

constexpr int kTile = 128;      // keys per tile, rows per query tile
constexpr int kThreads = 384;   // 8 warps of rows, load warp, product warp, two idle
// Registers a thread: a row's 128 scores need more than the 168 that 384 threads can have alike.  The last four
// warps give theirs up to the rows' eight: 8 * 216 + 4 * 72 = 12 * 168.
constexpr int kRegs = 168, kRegsRows = 216, kRegsRest = 72;
static_assert(8 * kRegsRows + 4 * kRegsRest <= 12 * kRegs, "more registers than the launch has would wait forever");
constexpr int kBlockBytes = kTile * 128;  // 64 dimensions of 128 rows
constexpr int kEarly = 96;      // keys of a tile whose weights are handed to the products before the others are computed
// Weights are scaled by 2^kShift, up to 2^14 when the maximum lags by its 2^8: so that a half holds those of a
// long, flat tail too (2^-30 of the largest), and none overflows.
constexpr int kShift = 6;
constexpr float kFar = 134217728.f;  // 2^27: scores (times log2 e) that a weight's exponent can still tell apart
// Tiles of keys of a share at least, where a block's keys are shared among CTAs: 512 rows behind 1000 keys 21.5 us with 4,
// 25.3 with 6, 25.7 without sharing; behind 4000 keys 29.7, 29.6 with 6, 33.7 with 10, 62.5 without.
constexpr int kMinSplit = 4;
constexpr int kMaxSplits = 16;
constexpr uint32_t kNever = 0x7fffffffu;
// Tiles of keys in which some row's view ends: a CTA's rows see at most 255 keys more than its first, which is
// at most three tiles.
constexpr int kMasked = 3;

template <int D> struct Shape {
    static constexpr int kBlocks = D / 64;                     // 64-dimension blocks of a row
    static constexpr int kTileBytes = kBlocks * kBlockBytes;
    static constexpr int kSlots = D == 128 ? 5 : 8;            // ring of K and V tiles
    static constexpr int kSmem = 2 * kTileBytes + kSlots * kTileBytes + 2048 + 1024;
};
static_assert(Shape<128>::kSmem <= 232448 && 2 * Shape<64>::kSmem > 232448, "one CTA per SM: it holds all of TMEM");

struct PromptArgs {
    void * out;
    long long out_stride;
    const int32_t * q_offsets;
    const int32_t * kv_begin;
    const int32_t * kv_end;
    int n_seq, q_rows, kv_rows, heads, kv_heads, out_f32;
    int log_p;        // heads per group P = 1 << log_p
    int splits;       // CTAs that share a block's keys, blockIdx.y; more than 1 only with scratch
    float * part;     // [blocks][splits][2 kTile][D] accumulators, then as many (reference, sum)
    float scale_log2; // scale * log2(e)
};

// A shared-memory operand's descriptor: the low word (address and leading offset) moves with the operand, the high
// word (stride of 8 rows 1024 bytes, descriptor version for sm_100, 128-byte swizzle) is the same for all here.
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo) {
    return ((saddr >> 4) & 0x3fffu) | ((lbo >> 4) & 0x3fffu) << 16;
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ void commit(uint64_t * bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D = A B (+ D): both operands in shared memory / A in TMEM.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 x, {%1, %4};\n\tmov.b64 y, {%2, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(kDescHigh), "r"(uint32_t(acc))
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 y, {%2, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(kDescHigh), "r"(uint32_t(acc))
        : "memory");
}

// 32 consecutive TMEM columns of this thread's lane (landed() before use).
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t * r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// wait_ld() for N columns: what uses them stays behind it.
template <int N> __device__ __forceinline__ void landed(uint32_t * r) {
    wait_ld();
#pragma unroll
    for (int i = 0; i < N; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t * r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t * r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// A box of the map at (x, y, z) into shared memory; x is a multiple of 64 elements.
__device__ __forceinline__ void tma_load(void * dst, const CUtensorMap * map, int x, int y, int z, uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_addr(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The largest of three, a NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// 2^x of two x from -126 to 127 on the multiply-add pipe (the exponential unit does 16 a clock and SM, which is as
// long as the products take): x = n + f, |f| <= 1/2, by a sum with 1.5 * 2^23; 2^f by a polynomial of degree 4 fitted
// for the least relative error on [-1/2, 1/2], 2.6e-6 at most; n goes into the exponent.
__device__ __forceinline__ float2 exp2_two(uint64_t x) {
    const float2 v = of_two(x);
    x = two(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
    const uint64_t magic = two(12582912.f, 12582912.f);
    const uint64_t t = add2(x, magic);
    const uint64_t f = add2(x, fma2(t, two(-1.f, -1.f), magic));  // x - n
    uint64_t y = fma2(f, two(9.570096619e-3f, 9.570096619e-3f), two(5.591785908e-2f, 5.591785908e-2f));
    y = fma2(y, f, two(0.2402474433f, 0.2402474433f));
    y = fma2(y, f, two(0.6931217909f, 0.6931217909f));
    y = fma2(y, f, two(0.9999992847f, 0.9999992847f));
    const float2 n = of_two(t), r = of_two(y);
    return make_float2(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(n.x) << 23)),
                       __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(n.y) << 23)));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t y;
    if constexpr (std::is_same_v<T, __half>) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
    return y;
}

// A block of query rows: positions p0 .. of a sequence with query rows [q0, q1) and keys [k0, k1).
struct Work {
    int seq;  // -1: none
    int q0, q1, k0, k1, p0;
};

// Block `blk` of the call, by one warp: blocks of all sequences in order, counted from the end so that a
// sequence's longest block starts first.  A lane holds a sequence; up to 32 are read once.
__device__ __forceinline__ void find_block(const PromptArgs & a, int blk, Work & out) {
    constexpr int kLogRows = 8;
    static_assert(1 << kLogRows == 2 * kTile, "rows of a block");
    const int lane = threadIdx.x & 31, log_positions = kLogRows - a.log_p, positions = 1 << log_positions;
    int q0 = 0, q1 = 0, k0 = 0, k1 = 0;
    const auto read = [&](int s) {
        q0 = q1 = k0 = k1 = 0;
        if (s < a.n_seq) {
            q0 = max(a.q_offsets[s], 0);
            q1 = min(a.q_offsets[s + 1], a.q_rows);
            k0 = min(max(a.kv_begin[s], 0), a.kv_rows);
            k1 = max(min(a.kv_end[s], a.kv_rows), k0);
        }
        return q1 > q0 ? (q1 - q0 + positions - 1) >> log_positions : 0;
    };
    int total = 0, mine = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
        mine = read(s0 + lane);
        total += int(__reduce_add_sync(0xffffffffu, unsigned(mine)));
    }
    int want = total - 1 - blk;
    if (lane == 0) out.seq = -1;
    __syncwarp();
    for (int s0 = 0; want >= 0 && s0 < a.n_seq; s0 += 32) {
        if (a.n_seq > 32) mine = read(s0 + lane);
        int upto = mine;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, x);
            if (lane >= x) upto += o;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, want < upto);
        if (hit) {
            if (lane == __ffs(hit) - 1) out = Work{s0 + lane, q0, q1, k0, k1, (want - (upto - mine)) * positions};
            break;
        }
        want -= __shfl_sync(0xffffffffu, upto, 31);
    }
    __syncwarp();
}

// How a block's keys are shared: tiles of a share, shares that have any.
struct Split {
    int tiles, used;
};
__device__ __forceinline__ Split split_of(const PromptArgs & a, const Work & w) {
    const int nq = w.q1 - w.q0, last = min(w.p0 + (2 * kTile >> a.log_p), nq) - 1;  // the block's last position sees most
    const int all = (max(0, last + 1 + (w.k1 - w.k0) - nq) + kTile - 1) / kTile;
    if (a.splits == 1) return Split{max(all, 1), 1};  // no divisions: a short prompt waits for them
    const int tiles = max(kMinSplit, (all + a.splits - 1) / a.splits);
    return Split{tiles, max(1, (all + tiles - 1) / tiles)};
}

// A CTA's share of its block, as if there were no other keys: every position's view is cut to it.
struct View {
    bool work, part;  // part: other CTAs have shares of the block too
    int q0, k0, nq, p0, keys, ahead;
    __device__ __forceinline__ View(const PromptArgs & a, const Work & w) {
        const Split split = split_of(a, w);
        work = w.seq >= 0 && int(blockIdx.y) < split.used;
        part = split.used > 1;
        const int key0 = part ? int(blockIdx.y) * split.tiles * kTile : 0, all = w.k1 - w.k0;
        q0 = w.q0;
        k0 = w.k0 + key0;
        nq = w.q1 - w.q0;
        p0 = w.p0;
        keys = part ? min(all - key0, split.tiles * kTile) : all;
        ahead = all - nq - key0;
    }
    // keys of the share that position p of the sequence sees
    __device__ __forceinline__ int sees(int p) const { return work && p < nq ? max(0, min(keys, p + 1 + ahead)) : 0; }
};

struct Bars {
    uint64_t full[8], empty[8], q_full, clean[kMasked], s_full[2], p_full[2][2], o_done[2];
    uint32_t tmem, dirty;
    Work work;
};

// Elements of a 16-bit pair whose exponent is all ones, as a mask of the pair.
template <typename T> __device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    constexpr uint32_t e = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
    return ((w & e) == e ? 0xffffu : 0u) | ((w >> 16 & e) == e ? 0xffff0000u : 0u);
}

// Clears what is not finite in keys [first, 128) of the V tile at `tile` (whose keys start at `base`); first
// keys that held a NaN, +inf or -inf go to seen[0 .. 2][dimension], keys from `keys` on are only cleared.
template <typename T, int D>
__device__ __noinline__ void clean_found(unsigned char * tile, int first, int base, int keys, uint32_t * seen,
                                         uint32_t * dirty) {
    const int lane = threadIdx.x & 31;
    constexpr uint32_t e = std::is_same_v<T, __half> ? 0x7c00u : 0x7f80u;
    for (int b = 0; b < D / 64; ++b)
        for (int r = (first & ~3) + (lane >> 3); r < kTile; r += 4) {
            uint32_t * at = reinterpret_cast<uint32_t *>(tile + b * kBlockBytes + r * 128 + (lane & 7) * 16);
            const int d0 = b * 64 + (((lane & 7) ^ (r & 7)) << 3);  // the swizzle: 16-byte chunk ^ (row mod 8)
            for (int i = 0; i < 4 && r >= first; ++i) {
                const uint32_t v = at[i], mask = not_finite<T>(v);
                if (!mask) continue;
                at[i] = v & ~mask;
                for (int h = 0; h < 2; ++h)
                    if ((mask >> 16 * h & 1u) && base + r < keys) {
                        const uint32_t x = v >> 16 * h & 0xffffu;
                        const int kind = (x & 0x7fffu) != e ? 0 : x & 0x8000u ? 2 : 1;
                        atomicMin(seen + kind * D + d0 + 2 * i + h, uint32_t(base + r));
                        *dirty = 1u;
                    }
            }
        }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the products read them
}

// The same; reads only where all is finite, which is what a short prompt waits for: the loads of a pass go out
// together (64 16-byte loads a lane took 8700 cycles with the clearing between them).
template <typename T, int D>
__device__ __forceinline__ void clean_values(unsigned char * tile, int first, int base, int keys, uint32_t * seen,
                                             uint32_t * dirty) {
    const int lane = threadIdx.x & 31;
    constexpr uint32_t e2 = std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t one = std::is_same_v<T, __half> ? 0x04000400u : 0x00800080u;
    uint32_t any = 0;
    // 8 lanes to a 128-byte row of a block, 4 rows at a time; rows before `first` may be read, and decide nothing wrong
    for (int r0 = first & ~31; r0 < kTile; r0 += 32)
#pragma unroll
        for (int b = 0; b < D / 64; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint4 w = *reinterpret_cast<const uint4 *>(tile + b * kBlockBytes + (r0 + 4 * i) * 128 + lane * 16);
                // an exponent of all ones carries into the sign's place
                any |= ((w.x & e2) + one) | ((w.y & e2) + one) | ((w.z & e2) + one) | ((w.w & e2) + one);
            }
    if (__any_sync(0xffffffffu, (any & 0x80008000u) != 0u)) clean_found<T, D>(tile, first, base, keys, seen, dirty);
    __syncwarp();
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
k_prompt_attn(const PromptArgs a, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v) {
    using Sh = Shape<D>;
    extern __shared__ unsigned char raw[];
    unsigned char * smem = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
    unsigned char * sq = smem;                          // two query tiles
    unsigned char * ring = smem + 2 * Sh::kTileBytes;
    uint32_t * seen = reinterpret_cast<uint32_t *>(ring + Sh::kSlots * Sh::kTileBytes);  // [3][D]
    Bars & bars = *reinterpret_cast<Bars *>(seen + 3 * 128);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();

    const int groups = a.heads >> a.log_p;
    const int hg = int(blockIdx.x) % groups, blk = int(blockIdx.x) / groups;
    const int head0 = hg << a.log_p, kvh = head0 / (a.heads / a.kv_heads);
    const int ppt = kTile >> a.log_p;  // positions per tile

    if (warp == 8) {
        if (lane == 0) {
            for (int i = 0; i < Sh::kSlots; ++i) {
                mbar_init(&bars.full[i], 1);
                mbar_init(&bars.empty[i], 1);
            }
            mbar_init(&bars.q_full, 1);
            for (int i = 0; i < kMasked; ++i) mbar_init(&bars.clean[i], 1);
            for (int t = 0; t < 2; ++t) {
                mbar_init(&bars.s_full[t], 1);
                for (int i = 0; i < 2; ++i) mbar_init(&bars.p_full[t][i], 4);  // the tile's warps
                mbar_init(&bars.o_done[t], 1);
            }
            bars.dirty = 0;
            mbar_init_fence();
            for (const CUtensorMap * map : {&map_q, &map_k, &map_v})
                asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
        }
    } else if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&bars.tmem)),
                     "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (warp == 0) {
        pdl_wait_primary();
        find_block(a, blk, bars.work);
    }
    for (int i = threadIdx.x; i < 3 * D; i += kThreads) seen[i] = kNever;
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = bars.tmem;
    const View view(a, bars.work);
    const auto tiles_of = [&](int t) {
        const int first = view.p0 + t * ppt;
        return first >= view.nq ? 0 : (view.sees(min(first + ppt, view.nq) - 1) + kTile - 1) / kTile;
    };
    const int nt[2] = {tiles_of(0), tiles_of(1)};
    const int n = max(nt[0], nt[1]);
    const int all_see = view.sees(view.p0);  // keys that every row of the CTA sees
    const int masked0 = all_see / kTile;     // first tile of keys in which some row's view ends

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
    if (warp == 8) {
        // ---- loads, and the cleaning of V where views end ----
        pdl_wait_primary();
        if (n > 0) {
            if (lane == 0) {
                mbar_arrive_expect_tx(&bars.q_full, uint32_t(2 * Sh::kTileBytes));
                for (int t = 0; t < 2; ++t)
                    for (int b = 0; b < Sh::kBlocks; ++b)
                        tma_load(sq + t * Sh::kTileBytes + b * kBlockBytes, &map_q, b * 64, head0, view.q0 + view.p0 + t * ppt,
                                 &bars.q_full);
            }
            bool ok = true;
            int it = 0;
            for (int j = 0; j <= n && ok; ++j) {
                if (j < n) {
                    for (int w = 0; w < 2 && ok; ++w, ++it) {
                        const int slot = it % Sh::kSlots;
                        if (it >= Sh::kSlots) ok = mbar_wait_sleep(&bars.empty[slot], unsigned(it / Sh::kSlots - 1) & 1u);
                        if (ok && lane == 0) {
                            mbar_arrive_expect_tx(&bars.full[slot], uint32_t(Sh::kTileBytes));
                            for (int b = 0; b < Sh::kBlocks; ++b)
                                tma_load(ring + slot * Sh::kTileBytes + b * kBlockBytes, w ? &map_v : &map_k, b * 64,
                                         kvh, view.k0 + j * kTile, &bars.full[slot]);
                        }
                        ok = __all_sync(0xffffffffu, ok);
                    }
                }
                // one tile behind the loads, so that the next tile's are under way
                if (ok && j > 0 && j - 1 >= masked0) {
                    const int vi = 2 * (j - 1) + 1, slot = vi % Sh::kSlots;
                    ok = __all_sync(0xffffffffu, mbar_wait_sleep(&bars.full[slot], unsigned(vi / Sh::kSlots) & 1u));
                    if (ok) {
                        clean_values<T, D>(ring + slot * Sh::kTileBytes, max(0, all_see - (j - 1) * kTile), (j - 1) * kTile,
                                           view.keys, seen, &bars.dirty);
                        if (lane == 0) mbar_arrive(&bars.clean[j - 1 - masked0]);
                    }
                }
            }
            if (!ok) {
                if (lane == 0) atomicOr(&g_prompt_status, kStatusWaitTimeout);
                for (int i = max(0, it - Sh::kSlots); i < it; ++i)  // copies in flight end before the CTA does
                    (void)mbar_wait_sleep(&bars.full[i % Sh::kSlots], unsigned(i / Sh::kSlots) & 1u);
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        // ---- products ----
        // The warp stays together and one lane issues, so that addresses and descriptors live in uniform registers:
        // a lone thread spends more time on preparing the instructions than the tensor cores on carrying them out.
        constexpr uint32_t type = std::is_same_v<T, __half> ? 0u : 1u;
        constexpr uint32_t common = 1u << 4 | type << 7 | type << 10 | 8u << 24;  // f32 sums, M = 128
        constexpr uint32_t idesc_s = common | uint32_t(kTile >> 3) << 17;
        constexpr uint32_t idesc_o = common | uint32_t(D >> 3) << 17 | 1u << 16;  // V: MN-major
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const int n0 = __shfl_sync(0xffffffffu, nt[0], 0), n1 = __shfl_sync(0xffffffffu, nt[1], 0), nn = max(n0, n1);
        const int first_masked = __shfl_sync(0xffffffffu, masked0, 0);
        const uint32_t desc_q = desc_low(smem_addr(sq), 16), desc_k = desc_low(smem_addr(ring), 16);
        const uint32_t desc_v = desc_low(smem_addr(ring), kBlockBytes);
        constexpr uint32_t tile16 = Sh::kTileBytes >> 4;
        const auto product_s = [&](int t, int slot) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t at = uint32_t((kk / 4) * kBlockBytes + (kk % 4) * 32) >> 4;
                mma_ss(tm + t * 128, desc_q + t * tile16 + at, desc_k + slot * tile16 + at, idesc_s, kk > 0);
            }
        };
        const auto product_o = [&](int t, int slot, int part, bool add) {
#pragma unroll
            for (int kk = 0; kk < kTile / 16; ++kk)
                if ((kk >= kEarly / 16) == (part != 0))
                    mma_ts(tm + 256 + t * 128, tm + t * 128 + kk * 8, desc_v + slot * tile16 + kk * (2048 >> 4), idesc_o, add || kk > 0);
        };
        bool ok = true;
        // every lane has seen the phase, or none goes on
        const auto wait = [&](uint64_t & bar, unsigned parity) {
            ok = ok && __all_sync(0xffffffffu, mbar_wait(&bar, parity));
        };
        // a slot is handed back only where a later load waits for it: no arrival outlives the CTA
        const auto returns = [&](int item) { return item + Sh::kSlots < 2 * nn; };
        if (nn > 0) {
            wait(bars.q_full, 0);
            wait(bars.full[0], 0);
            if (ok && elect()) {
                for (int t = 0; t < 2; ++t)
                    if ((t ? n1 : n0) > 0) {
                        product_s(t, 0);
                        commit(&bars.s_full[t]);
                    }
                if (returns(0)) commit(&bars.empty[0]);
            }
            __syncwarp();
        }
        int vs = 1, ks = 2;               // slots of this tile's values and the next one's keys
        unsigned vphase = 0, kphase = 0;  // and their barriers' phases
        for (int j = 0; j < nn && ok; ++j) {
            wait(bars.full[vs], vphase);
            if (j >= first_masked) wait(bars.clean[j - first_masked], 0);
            if (j + 1 < nn) wait(bars.full[ks], kphase);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int mine = t ? n1 : n0, other = t ? n0 : n1;
                if (j < mine) {
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        wait(bars.p_full[t][part], unsigned(j) & 1u);
                        fence_after();
                        if (ok && elect()) {
                            product_o(t, vs, part, part || j > 0);
                            if (part) {
                                if (j + 1 == mine) commit(&bars.o_done[t]);
                                // the tile's last user of the values, and of the next keys
                                if ((t || j >= other) && returns(2 * j + 1)) commit(&bars.empty[vs]);
                                if (j + 1 < mine) {
                                    product_s(t, ks);
                                    commit(&bars.s_full[t]);
                                    if ((t || j + 1 >= other) && returns(2 * j + 2)) commit(&bars.empty[ks]);
                                }
                            }
                        }
                        __syncwarp();
                    }
                }
            }
            vs += 2;
            if (vs >= Sh::kSlots) vs -= Sh::kSlots, vphase ^= 1u;
            ks += 2;
            if (ks >= Sh::kSlots) ks -= Sh::kSlots, kphase ^= 1u;
        }
        if (!ok && lane == 0) atomicOr(&g_prompt_status, kStatusWaitTimeout);
        __syncwarp();
    }
    } else {
        // ---- rows: thread = row of tile t ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsRows));
        const int t = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + 256 + t * 128;
        const int lim = view.sees(view.p0 + t * ppt + (row >> a.log_p));
        const int tile_sees = view.sees(view.p0 + t * ppt);
        const float c = a.scale_log2, far = fminf(kFar / c, 3e38f);
        float m = -INFINITY, sum = 0.f;
        const int tiles = nt[t];
        bool ok = true;
        for (int j = 0; j < tiles; ++j) {
            ok = __all_sync(0xffffffffu, mbar_wait(&bars.s_full[t], unsigned(j) & 1u));
            if (!ok) break;
            fence_after();
            uint32_t s[kTile];
            const bool edge = (j + 1) * kTile > tile_sees;  // some row does not see all of the tile
            const int left = lim - j * kTile;
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_ld(ts + 32 * i, s + 32 * i);
            landed<kTile>(s);
            if (edge) {
#pragma unroll
                for (int x = 0; x < kTile; ++x) s[x] = x < left ? s[x] : 0xff800000u;
            }
            float mx[4] = {m, m, m, m};
#pragma unroll
            for (int x = 0; x < kTile; x += 2)
                mx[x / 2 % 4] = max3(mx[x / 2 % 4], __uint_as_float(s[x]), __uint_as_float(s[x + 1]));
            const float top = max3(mx[0], mx[1], max3(mx[2], mx[3], mx[3]));
            // m: what the weights refer to (or -kFar, where it is below that).  It moves with the first tile, and when the
            // true maximum is more than 2^8 above (or a NaN, which then stays); then the sums so far are scaled down.
            if (__any_sync(0xffffffffu, !((top - m) * c <= 8.f))) {
                const float f = exp2_fast((fmaxf(m, -far) - fmaxf(top, -far)) * c);
                m = top;
                sum *= f;
                if (j > 0) {  // every product up to the tile before is complete: S of this tile came after them
                    for (int i = 0; i < D; i += 32) {
                        uint32_t o[32];
                        tmem_ld(to + i, o);
                        landed<32>(o);
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                        tmem_st(to + i, o);
                    }
                }
            }
            // m c is rounded up, so that no weight overflows; the rounding takes up to 2^-16 off all of them where |m c|
            // comes to kFar, and a half has room for that.  (+inf among the scores: all NaN, as inf - inf is.)
            const float mc = __fmaf_ru(fmaxf(m, -far), c, -float(kShift));
            const uint64_t c2 = two(c, c), mc2 = two(-mc, -mc);
            uint64_t add[2] = {0, 0};
            // masked scores have to become 0: at a view's end the polynomial is not used
            const auto weights = [&](auto polynomial, int need) {
                const auto some = [&](auto from, auto to_key) {
#pragma unroll
                    for (int i = decltype(from)::value; i < decltype(to_key)::value; i += 2) {
                        const uint64_t x = fma2(two(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), c2, mc2);
                        float2 e;
                        if (decltype(polynomial)::value && i / 2 % 4 == 3) {
                            e = exp2_two(x);
                        } else {
                            e = of_two(x);
                            e.x = exp2_fast(e.x);
                            e.y = exp2_fast(e.y);
                        }
                        add[i / 2 % 2] = add2(add[i / 2 % 2], two(e.x, e.y));
                        s[i / 2] = pack2<T>(e.x, e.y);
                    }
                };
                const auto hand_over = [&](int part) {
                    wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.p_full[t][part]);
                };
                if constexpr (decltype(polynomial)::value) {
                    some(std::integral_constant<int, 0>{}, std::integral_constant<int, kEarly>{});
                } else {  // no row of the warp sees keys from `need` on
                    const auto third = [&](auto from) {
                        constexpr int at = decltype(from)::value;
                        if (at < need) some(from, std::integral_constant<int, at + 32>{});
                        else
#pragma unroll
                            for (int i = at / 2; i < at / 2 + 16; ++i) s[i] = 0;
                    };
                    third(std::integral_constant<int, 0>{});
                    third(std::integral_constant<int, 32>{});
                    third(std::integral_constant<int, 64>{});
                }
                tmem_st(ts, s);
                tmem_st16(ts + 32, s + 32);
                hand_over(0);
                if (decltype(polynomial)::value || kEarly < need) {
                    some(std::integral_constant<int, kEarly>{}, std::integral_constant<int, kTile>{});
                } else {
#pragma unroll
                    for (int i = kEarly / 2; i < kTile / 2; ++i) s[i] = 0;
                }
                tmem_st16(ts + 48, s + 48);
                hand_over(1);
            };
            if (edge) weights(std::false_type{}, __reduce_max_sync(0xffffffffu, left));
            else weights(std::true_type{}, kTile);
            const float2 added = of_two(add2(add[0], add[1]));
            sum += added.x + added.y;
        }
        if (ok && tiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars.o_done[t], 0));
        if (ok && tiles == 0 && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(&bars.q_full, 0));  // a copy to the stage
        if (!ok && lane == 0) atomicOr(&g_prompt_status, kStatusWaitTimeout);
        fence_after();
        // read again: the loop needs the registers
        const View end(a, bars.work);
        const int p = end.p0 + t * ppt + (row >> a.log_p);
        const bool live = end.work && ok && p < end.nq, part = end.part;
        // nothing from -kFar on (scores of -inf alone), or something above kFar: NaN
        const float inv = part ? 1.f : lim <= 0 ? 0.f : m >= -far && m <= far ? 1.f / sum : NAN;
        const bool dirty = *reinterpret_cast<volatile uint32_t *>(&bars.dirty) != 0u;
        // a share's part goes to scratch as it is, in f32, with what its weights refer to
        const bool f32 = part || a.out_f32;
        const size_t rec0 = (size_t(blockIdx.x) * a.splits + blockIdx.y) * (2 * kTile) + t * kTile, rec = rec0 + row;
        char * const out = static_cast<char *>(part ? a.part : a.out);
        if (part && end.work && p < end.nq) {  // NaN after a wait that ran out: the join makes it the row's result
            const float mr = !ok || !(m <= far) ? NAN : m < -far ? -INFINITY : __fmaf_ru(m, c, -float(kShift));
            reinterpret_cast<float2 *>(a.part + size_t(gridDim.x) * a.splits * (2 * kTile) * D)[rec] = make_float2(mr, sum);
        }
        // Rows go out by way of the query tile's memory (its products are complete), 2 D bytes of a row at a time, so that
        // its lanes write them together: a row to a lane and 16 bytes at a time take a wavefront per row.
        if (__any_sync(0xffffffffu, live)) {
            constexpr int kRowBytes = 2 * D, kChunks = kRowBytes / 16, kAtOnce = 32 / kChunks;  // rows written together
            unsigned char * const stage = sq + t * Sh::kTileBytes + (warp & 3) * 32 * kRowBytes;
            const auto place = [&](int r, int chunk) {
                return reinterpret_cast<uint4 *>(stage + r * kRowBytes + ((chunk & ~7) | ((chunk ^ r) & 7)) * 16);
            };
            const auto values = [&](int from, uint32_t * o) {  // 32 dimensions, scaled
#pragma unroll
                for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * inv);
                if (dirty) {
#pragma unroll
                    for (int x = 0; x < 32; ++x) {
                        float v = __uint_as_float(o[x]);
                        if (seen[D + from + x] < uint32_t(lim)) v += INFINITY;
                        if (seen[2 * D + from + x] < uint32_t(lim)) v -= INFINITY;
                        if (seen[from + x] < uint32_t(lim)) v = NAN;
                        o[x] = __float_as_uint(v);
                    }
                }
            };
            // the rows' places: row r of the warp is head (r mod P) of position r / P
            const int first = (warp & 3) * 32, chunk = lane % kChunks, heads_mask = (1 << a.log_p) - 1;
            const auto write = [&](int column) {  // bytes
                __syncwarp();
#pragma unroll 8
                for (int r = lane / kChunks; r < 32; r += kAtOnce) {
                    const uint4 w = *place(r, chunk);
                    const int position = end.p0 + t * ppt + ((first + r) >> a.log_p), head = head0 + ((first + r) & heads_mask);
                    const long long at = part ? (long long)(rec0 + first + r) * D : (long long)(end.q0 + position) * a.out_stride + head * D;
                    if (position < end.nq && end.work && ok)
                        *reinterpret_cast<uint4 *>(out + at * (f32 ? 4 : 2) + column + chunk * 16) = w;
                }
                __syncwarp();
            };
            uint32_t o[D];
            if (tiles > 0 && ok) {
#pragma unroll
                for (int i = 0; i < D; i += 32) tmem_ld(to + i, o + i);
                landed<D>(o);  // a row that sees nothing has sums of zero: its weights were, and the values are clean
            } else {
#pragma unroll
                for (int i = 0; i < D; ++i) o[i] = 0;
            }
#pragma unroll
            for (int i = 0; i < D; i += 32) values(i, o + i);
            if (f32) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int x = 0; x < kChunks; ++x) {
                        const uint32_t * e = o + half * (D / 2) + 4 * x;
                        *place(lane, x) = make_uint4(e[0], e[1], e[2], e[3]);
                    }
                    write(half * kRowBytes);
                }
            } else {
#pragma unroll
                for (int x = 0; x < kChunks; ++x) {
                    const auto pair = [&](int i) { return pack2<T>(__uint_as_float(o[8 * x + 2 * i]), __uint_as_float(o[8 * x + 2 * i + 1])); };
                    *place(lane, x) = make_uint4(pair(0), pair(1), pair(2), pair(3));
                }
                write(0);
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 9)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// Joins a block's shares, in order: a warp to a row of the block, 32 rows to a CTA.  Bound by the bytes of the parts.
template <typename T, int D>
__global__ void __launch_bounds__(256) k_prompt_merge(const PromptArgs a) {
    __shared__ Work sm_work;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_trigger();
    pdl_wait_primary();
    const int groups = a.heads >> a.log_p;
    if (warp == 0) find_block(a, int(blockIdx.x) / groups, sm_work);
    __syncthreads();
    const Work w = sm_work;
    if (w.seq < 0) return;
    const int used = split_of(a, w).used, nq = w.q1 - w.q0;
    if (used <= 1) return;
    constexpr int E = D / 32;
    for (int i = 0; i < 4; ++i) {
        const int row = blockIdx.y * 32 + warp * 4 + i;  // of the block's two tiles
        const int p = w.p0 + (row >> a.log_p), head = ((int(blockIdx.x) % groups) << a.log_p) + (row & ((1 << a.log_p) - 1));
        if (p >= nq) continue;
        const size_t rec = size_t(blockIdx.x) * a.splits * (2 * kTile) + row;
        const float2 * refs = reinterpret_cast<const float2 *>(a.part + size_t(gridDim.x) * a.splits * (2 * kTile) * D) + rec;
        float2 mine = lane < used ? refs[lane * (2 * kTile)] : make_float2(-INFINITY, 0.f);
        float o[kMaxSplits][E];
#pragma unroll
        for (int z = 0; z < kMaxSplits; ++z) {
            if (z >= used) break;
            const float * x = a.part + (rec + size_t(z) * (2 * kTile)) * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) o[z][e] = x[e];
        }
        float top = mine.x;
#pragma unroll
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float f = exp2_fast(mine.x - (top == -INFINITY ? 0.f : top));
        float sum = mine.y * f;
#pragma unroll
        for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        float v[E] = {};
#pragma unroll
        for (int z = 0; z < kMaxSplits; ++z) {
            if (z >= used) break;
            const float fz = __shfl_sync(0xffffffffu, f, z);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = fmaf(o[z][e], fz, v[e]);
        }
        const bool any = p + 1 + w.k1 - w.k0 - nq > 0;
        const long long at = (long long)(w.q0 + p) * a.out_stride + head * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float y = any ? v[e] / sum : 0.f;
            if (a.out_f32) static_cast<float *>(a.out)[at + e] = y;
            else static_cast<T *>(a.out)[at + e] = from_f32<T>(y);
        }
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void * p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// Rows of `heads` heads of D 16-bit values; boxes of 64 values x box_heads x box_rows.
bool encode(CUtensorMap * map, const void * p, bool bf16, int D, size_t heads, size_t rows, size_t head_stride,
            size_t row_stride, unsigned box_heads, unsigned box_rows) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[3] = {cuuint64_t(D), heads, rows};
    const cuuint64_t strides[2] = {head_stride * 2, row_stride * 2};
    const cuuint32_t box[3] = {64, box_heads, box_rows}, steps[3] = {1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(p), dims,
              strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

std::atomic<unsigned long long> g_attr[4];

template <typename T, int D>
int launch(const PromptArgs & a, const CUtensorMap (&maps)[3], unsigned blocks, void * stream) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return api_cuda_fail(cudaGetLastError(), "prompt_attn");
    auto & done = g_attr[(std::is_same_v<T, __half> ? 0 : 2) + (D == 128)];
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(done.load() & bit)) {
        const cudaError_t e =
            cudaFuncSetAttribute(k_prompt_attn<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
        if (e != cudaSuccess) return api_cuda_fail(e, "prompt_attn: shared memory");
        cudaFuncAttributes f;
        if (cudaFuncGetAttributes(&f, k_prompt_attn<T, D>) != cudaSuccess || f.numRegs != kRegs)
            return api_fail(EXL3CU_NO_SUPPORT, "prompt_attn: built with another number of registers than it divides up");
        done.fetch_or(bit);
    }
    const int rc = attn_launch(k_prompt_attn<T, D>, dim3(blocks, unsigned(a.splits)), dim3(kThreads), size_t(Shape<D>::kSmem),
                               stream, 1, a, maps[0], maps[1], maps[2]);
    if (rc || a.splits == 1) return rc;
    return attn_launch(k_prompt_merge<T, D>, dim3(blocks, 2 * kTile / 32), dim3(256), 0, stream, 1, a);
}

constexpr int kSms = 148;  // a B200's

struct Plan {
    int log_p;         // heads per CTA: the power of two in heads / kv_heads, at most 16
    long long blocks;  // of all sequences: at most one part block per sequence more than the rows fill
    int splits;
    size_t scratch;
};

// A block's keys are shared among CTAs where the blocks alone leave most SMs idle (a prompt's chunk of 512 rows
// behind a long start is 32 blocks for 148 SMs) and there are keys for it.
Plan plan_prompt(int q_rows, int n_seq, int kv_rows, int heads, int kv_heads, int head_dim) {
    Plan p{0, 0, 1, 0};
    while (p.log_p < 4 && (heads / kv_heads) % (2 << p.log_p) == 0) ++p.log_p;
    p.blocks = ((long long)q_rows / (2 * kTile >> p.log_p) + n_seq) * (heads >> p.log_p);
    const long long tiles = ((long long)kv_rows + kTile - 1) / kTile;
    if (tiles >= 3 * kMinSplit)  // two short shares and joining them take as long as one
        p.splits = int(std::max(1ll, std::min({kSms / std::max(p.blocks, 1ll), tiles / kMinSplit, (long long)kMaxSplits})));
    p.scratch = p.splits > 1 ? size_t(p.blocks) * p.splits * (2 * kTile) * (head_dim + 2) * sizeof(float) : 0;
    return p;
}

}  // namespace

cudaError_t prompt_read_status(unsigned * out, bool clear) {
    cudaError_t e = cudaMemcpyFromSymbol(out, g_prompt_status, sizeof(unsigned));
    if (e == cudaSuccess && clear && *out) {
        const unsigned zero = 0;
        e = cudaMemcpyToSymbol(g_prompt_status, &zero, sizeof(unsigned));
    }
    return e;
}

}  // namespace exl3cu

using namespace exl3cu;

extern "C" int exl3cu_prompt_attn(const void * d_q, size_t q_stride, const void * d_k, size_t k_row_stride,
                                  size_t k_head_stride, const void * d_v, size_t v_row_stride, size_t v_head_stride,
                                  int kv_rows, int dtype, int heads, int kv_heads, int head_dim,
                                  const int32_t * d_q_offsets, const int32_t * d_kv_begin, const int32_t * d_kv_end,
                                  int n_seq, int q_rows, float scale, void * d_out, size_t out_stride, int out_dtype,
                                  void * d_scratch, size_t scratch_bytes, void * stream) {
    const auto bad = [](const char * what) { return api_fail(EXL3CU_INVALID_ARGUMENT, what); };
    if (head_dim != 64 && head_dim != 128) return bad("prompt_attn: head_dim must be 64 or 128");
    if (dtype != EXL3CU_F16 && dtype != EXL3CU_BF16) return bad("prompt_attn: q, k and v must be f16 or bf16");
    if (out_dtype != dtype && out_dtype != EXL3CU_F32) return bad("prompt_attn: out must be f32 or of q's type");
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads > 1024)
        return bad("prompt_attn: heads must be a multiple of kv_heads, at most 1024");
    if (n_seq < 0 || q_rows < 0 || kv_rows < 0) return bad("prompt_attn: negative count");
    if (!(scale > 0.f) || scale > 1e30f) return bad("prompt_attn: scale must be positive and finite");
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

    Plan plan = plan_prompt(q_rows, n_seq, kv_rows, heads, kv_heads, head_dim);
    if (!d_scratch) plan.splits = 1;  // without scratch a block has its keys to itself
    else if (plan.splits > 1 && (scratch_bytes < plan.scratch || !aligned(d_scratch)))
        return bad("prompt_attn: scratch misaligned or too small (exl3cu_prompt_attn_scratch_bytes)");
    const int log_p = plan.log_p;
    const long long blocks = plan.blocks;
    if (blocks > 0x7fffffffll) return bad("prompt_attn: too many query rows");
    const bool bf16 = dtype == EXL3CU_BF16;
    CUtensorMap maps[3];
    const bool any = kv_rows > 0;  // without keys the maps of k and v are never used
    if (!encode(&maps[0], d_q, bf16, head_dim, size_t(heads), size_t(q_rows), size_t(head_dim), q_stride, 1u << log_p,
                unsigned(kTile >> log_p)) ||
        !encode(&maps[1], any ? d_k : d_q, bf16, head_dim, any ? size_t(kv_heads) : 1, any ? size_t(kv_rows) : 1,
                any ? k_head_stride : head_dim, any ? k_row_stride : head_dim, 1, kTile) ||
        !encode(&maps[2], any ? d_v : d_q, bf16, head_dim, any ? size_t(kv_heads) : 1, any ? size_t(kv_rows) : 1,
                any ? v_head_stride : head_dim, any ? v_row_stride : head_dim, 1, kTile))
        return api_fail(EXL3CU_CUDA_ERROR, "prompt_attn: cuTensorMapEncodeTiled failed");
    const PromptArgs a{d_out, (long long)out_stride, d_q_offsets, d_kv_begin, d_kv_end, n_seq, q_rows, kv_rows, heads,
                       kv_heads, out_dtype == EXL3CU_F32, log_p, plan.splits, static_cast<float *>(d_scratch),
                       scale * 1.4426950408889634f};
    if (!bf16)
        return head_dim == 128 ? launch<__half, 128>(a, maps, unsigned(blocks), stream)
                               : launch<__half, 64>(a, maps, unsigned(blocks), stream);
    return head_dim == 128 ? launch<__nv_bfloat16, 128>(a, maps, unsigned(blocks), stream)
                           : launch<__nv_bfloat16, 64>(a, maps, unsigned(blocks), stream);
}

extern "C" size_t exl3cu_prompt_attn_scratch_bytes(int q_rows, int n_seq, int kv_rows, int heads, int kv_heads,
                                                   int head_dim) {
    if (q_rows <= 0 || n_seq <= 0 || kv_rows <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
    return plan_prompt(q_rows, n_seq, kv_rows, heads, kv_heads, head_dim).scratch;
}

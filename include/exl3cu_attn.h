/* Attention operators for any number of heads (libexl3cu): query/key norms with
 * the rotary embedding, a K/V cache held in 4 bits, attention of single tokens
 * over that cache, and causal attention of packed prompts on the tensor cores.
 *
 * They stand beside the fixed-geometry kernels of exl3cu_hybrid.h, whose row
 * conventions they share: row r of a step belongs to step sequence row_seq[r]
 * at position row_pos[r]; step sequence s uses cache slot seq_slot[s].  All
 * pointers are device pointers on the current device; calls are stream-ordered
 * and neither allocate nor synchronise, so they can be captured in a CUDA graph.
 * No counterpart in the reference tree, whose attention is upstream llama.cpp's
 * (patches/llama-exl3.patch:175-183 routes FLASH_ATTN_EXT).
 *
 * Types: EXL3CU_F32, EXL3CU_F16 and EXL3CU_BF16.  Sums, softmax statistics and
 * norms are held in 32 bits whatever the type; the weights of a softmax are
 * rounded to 16 bits where they enter a product, as said below.  head_dim is 64
 * or 128.  A row's
 * heads are contiguous (head h of row r starts at r * stride + h * head_dim);
 * strides count elements.  Rows start on 16-byte boundaries.
 */
#ifndef EXL3CU_ATTN_H
#define EXL3CU_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define EXL3CU_BF16 4 /* beside enum exl3cu_dtype's F32 and F16; 2 and 3 are the operator's input forms */

/* Per row r and head: y = x * rsqrt(mean(x^2) + eps) * w (q_w / k_w, f32
 * [head_dim]; NULL: no norm, y = x), then the first rotary_dim dimensions are
 * rotated by the angles row_pos[r] * inv_freq[i] (f32 [rotary_dim / 2]), cosine
 * and sine multiplied by attn_factor; the pairs are (i, i + rotary_dim / 2), or
 * (2i, 2i + 1) when interleaved.  The remaining dimensions keep y.  Angles are
 * reduced in 64 bits, so positions of millions lose nothing.  rotary_dim is
 * even, from 0 to head_dim, a multiple of 16 when not 0.  Rows of a negative
 * position are not written (packed rows past the last sequence).  q_out may be q,
 * and k_out may be k (same type and stride).  kv_heads may be 0 (no keys). */
int exl3cu_qk_norm_rope(const void * d_q, size_t q_stride, const void * d_k, size_t k_stride, int dtype, int rows,
                        int heads, int kv_heads, int head_dim, const int32_t * d_row_pos, const float * d_q_w,
                        const float * d_k_w, float eps, const float * d_inv_freq, int rotary_dim, int interleaved,
                        float attn_factor, void * d_q_out, size_t q_out_stride, int q_out_dtype, void * d_k_out,
                        size_t k_out_stride, int k_out_dtype, void * stream);

/* A K/V cache in 4 bits.  One position of one K/V head is head_dim / 2 bytes of
 * codes (dimension 2i in the low half of byte i, 2i + 1 in the high half) and
 * G = head_dim / 32 half-precision scales; dimension d belongs to group d mod G
 * and stands for (code - 8) * scale.
 *   codes   [n_slots][kv_heads][max_len][head_dim / 2]
 *   scales  [n_slots][kv_heads][max_len][G]
 * max_len is a multiple of 64, at most 2^27, kv_heads at most 1024, and the arrays start
 * on 16-byte boundaries. */
typedef struct exl3cu_kv4_cache {
    uint8_t * k_codes;
    uint16_t * k_scales;
    uint8_t * v_codes;
    uint16_t * v_scales;
    int n_slots;
    int kv_heads;
    int max_len;
    int head_dim;
} exl3cu_kv4_cache;

/* Quantises each row's keys and values into the cache at (slot, position).  The
 * scale of a group is the smallest half with 7 * scale >= max |x| (at most 65504,
 * where larger values saturate), the code 8 + x / scale rounded to nearest, ties
 * to even.  A group that holds an infinity or a NaN gets a NaN scale: it reads
 * back as NaN.  Rows whose sequence is outside [0, n_seq), whose slot is outside
 * the cache or whose position is outside [0, max_len) are skipped.  Two rows of
 * one call at the same slot and position leave that position undefined. */
int exl3cu_kv4_append(const exl3cu_kv4_cache * cache, const void * d_k, size_t k_stride, const void * d_v,
                      size_t v_stride, int dtype, int rows, const int32_t * d_row_seq, const int32_t * d_row_pos,
                      const int32_t * d_seq_slot, int n_seq, void * stream);

/* Reads positions back as packed rows: row r of [kv_offsets[s], kv_offsets[s+1])
 * (kv_offsets: n_seq + 1 ascending entries) gets position r - kv_offsets[s] of
 * sequence s's slot.  A row whose slot or position is outside the cache becomes
 * zero; rows from kv_offsets[n_seq] on are left as they were.  total_rows is the
 * rows that d_k and d_v hold. */
int exl3cu_kv4_read(const exl3cu_kv4_cache * cache, const int32_t * d_seq_slot, const int32_t * d_kv_offsets, int n_seq,
                    int total_rows, void * d_k, size_t k_stride, void * d_v, size_t v_stride, int dtype, void * stream);

/* Attention of single rows over the cache: query head h of row r attends to
 * positions 0 .. min(row_pos[r], max_len - 1) of its slot, K/V head
 * h / (heads / kv_heads); out = softmax(scale * q . k) v, scale > 0, at most
 * 65535 rows.  A row of a negative
 * position, or of a slot outside the cache, becomes zero (nothing is visible); a
 * row whose sequence is outside [0, n_seq) is left as it was.  What the cache
 * holds past the last visible position never reaches a result.  A weight times a
 * value's scale is rounded to a half for rows of 16 bits (by 2^-11 of it at most),
 * to two for f32 (2^-22).  d_scratch:
 * exl3cu_kv4_attn_scratch_bytes() bytes, 16-byte aligned, contents arbitrary; two
 * calls that may run at the same time need scratch of their own. */
size_t exl3cu_kv4_attn_scratch_bytes(const exl3cu_kv4_cache * cache, int rows, int heads);
int exl3cu_kv4_attn(const exl3cu_kv4_cache * cache, const void * d_q, size_t q_stride, int dtype, int rows, int heads,
                    const int32_t * d_row_seq, const int32_t * d_row_pos, const int32_t * d_seq_slot, int n_seq,
                    float scale, void * d_out, size_t out_stride, void * d_scratch, size_t scratch_bytes,
                    void * stream);

/* Causal attention of packed sequences.  Sequence s has query rows
 * [q_offsets[s], q_offsets[s+1]) and key/value rows [kv_begin[s], kv_end[s]); its
 * last query sees all of its keys, the one before it all but the last, and so on:
 * query i sees keys 0 .. i + (keys - queries).  A query that sees nothing (more
 * queries than keys) becomes zero.  Query head h uses K/V head h / (heads /
 * kv_heads).  Row r, head h of k starts at r * k_row_stride + h * k_head_stride,
 * so rows may be packed or lie in a slot cache [slots][kv_heads][max_len][head_dim]
 * (kv_begin = slot * kv_heads * max_len); kv_rows is the number of rows that every
 * head can address.  A key or value that a query does not see never reaches its
 * result, whatever it holds.  Packed K/V: kv_begin = offsets, kv_end = offsets + 1.
 * dtype (q, k, v): EXL3CU_F16 or EXL3CU_BF16; scale > 0; out_dtype: the same or EXL3CU_F32.
 * Weights are rounded to q's type (by 2^-11 of each at most for f16, 2^-8 for bf16).
 * A row whose largest score (scale * q . k) is beyond 2^26 in size may become NaN.
 * Query rows outside every sequence are left as they were; q_rows is the rows
 * that d_q and d_out hold.  With d_scratch (exl3cu_prompt_attn_scratch_bytes()
 * bytes, 16-byte aligned, contents arbitrary; calls that may run at the same time
 * need scratch of their own) a call of few query rows and many keys divides the
 * keys over the GPU; NULL: it does not. */
size_t exl3cu_prompt_attn_scratch_bytes(int q_rows, int n_seq, int kv_rows, int heads, int kv_heads, int head_dim);
int exl3cu_prompt_attn(const void * d_q, size_t q_stride, const void * d_k, size_t k_row_stride, size_t k_head_stride,
                       const void * d_v, size_t v_row_stride, size_t v_head_stride, int kv_rows, int dtype, int heads,
                       int kv_heads, int head_dim, const int32_t * d_q_offsets, const int32_t * d_kv_begin,
                       const int32_t * d_kv_end, int n_seq, int q_rows, float scale, void * d_out, size_t out_stride,
                       int out_dtype, void * d_scratch, size_t scratch_bytes, void * stream);

/* The calls above for bindings whose conversion of arguments costs more than a launch (ctypes: 24 arguments
 * about 6 us): `words` are the arguments of the call in order, 8 bytes each; integers and pointers as 64-bit
 * integers, the floats as doubles. */
enum exl3cu_attn_call {
    EXL3CU_CALL_QK_NORM_ROPE = 0,
    EXL3CU_CALL_KV4_APPEND = 1,
    EXL3CU_CALL_KV4_READ = 2,
    EXL3CU_CALL_KV4_ATTN = 3,
    EXL3CU_CALL_PROMPT_ATTN = 4
};
int exl3cu_attn_words(int call, const void * words);

#ifdef __cplusplus
}
#endif

#endif /* EXL3CU_ATTN_H */

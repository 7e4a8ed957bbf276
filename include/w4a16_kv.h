/*
 * w4a16_kv.h -- C ABI of the 8-bit key/value cache: rotary positions, writing
 * keys and values into the cache, reading it back, and attention over it.
 * The conventions of w4a16_hip.h hold (device pointers, return codes,
 * w4a16_last_error(), work enqueued on `stream`, nothing allocated or
 * synchronised, so every call may be captured in a HIP graph).
 *
 * The cache. Codes [batch, kv_heads, slots, head_dim], one byte each, int8 or
 * OCP e4m3; a row of head_dim codes is contiguous and rows follow each other
 * (slot stride head_dim), batch and head strides are free multiples of 16.
 * Scales fp32 [batch, kv_heads, ceil(slots / block)], one for each `block`
 * consecutive slots of a head; a value is code * scale. Scales are powers of
 * two from 2^-40 to 2^40, so that scaling rounds nothing.
 *
 * Tokens. Rows [batch, tokens, heads, head_dim] of fp16 or bf16 with any
 * batch, token and head strides (a view of a q|k|v projection's rows). Token t
 * of sequence b has position (and slot) start[b] + t. counts[b] of a
 * sequence's `tokens` rows are tokens and the rest is padding; NULL: all are.
 * start and counts are device int64 [batch]; counts below 0 read as 0, above
 * `tokens` as `tokens`.
 */
#ifndef W4A16_KV_H
#define W4A16_KV_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Types of token rows, and (with FP32) of what w4a16_kv_read writes. */
#define W4A16_FP16 0
#define W4A16_BF16 1
#define W4A16_FP32 2

/* Types of codes. */
#define W4A16_KV_INT8 0
#define W4A16_KV_FP8 1               /* e4m3, OCP: largest value 448, no infinities */

/* Token rows: element (b, t, h, i) at data[b batch_stride + t token_stride + h head_stride + i]. */
typedef struct w4a16_kv_rows {
    const void* data;
    int64_t batch_stride, token_stride, head_stride;   /* in elements */
} w4a16_kv_rows;

/* Keys or values of a cache. Strides in codes and in scales; the rest is dense. */
typedef struct w4a16_kv_codes {
    void* codes;
    float* scales;
    int64_t batch_stride, head_stride;
    int64_t scale_batch_stride, scale_head_stride;
} w4a16_kv_codes;

typedef struct w4a16_kv_cache {
    w4a16_kv_codes k, v;
    int64_t batch, kv_heads, slots, head_dim;   /* head_dim 64, 128 or 256 */
    int64_t block;                              /* slots of a scale: 16, 32, 64 or 128 */
    int code_type;                              /* W4A16_KV_INT8 or W4A16_KV_FP8 */
} w4a16_kv_cache;

/*
 * Rotary positions: out [batch, tokens, heads, head_dim] (contiguous) = x
 * rotated in its first `rot` dims by row positions[b pos_batch_stride + t
 * pos_token_stride] of the tables cos / sin fp32 [table_rows, rot / 2]; the
 * dims past rot are copied. Pair i is dims (i, i + rot / 2), or (2 i, 2 i + 1)
 * with interleaved != 0: y1 = x1 c - x2 s, y2 = x2 c + x1 s, each product and
 * sum rounded to fp32, the result once to the rows' type. A position outside
 * the tables writes NaN to the rotated dims. rot even, 2 <= rot <= head_dim.
 * out may be x's own memory where x is contiguous.
 */
int w4a16_rotary(const w4a16_kv_rows* x, void* out, int64_t batch, int64_t tokens, int64_t heads, int64_t head_dim,
                 const float* cos_table, const float* sin_table, int64_t table_rows, int64_t rot,
                 const int64_t* positions, int64_t pos_batch_stride, int64_t pos_token_stride, int interleaved,
                 int type, void* stream);

/*
 * Writes the tokens' keys and values into their slots. For each block that
 * gets tokens, with A the largest magnitude among them (NaN left out, an
 * infinity as the type's largest finite value) and M the largest code (127 or
 * 448): the scale is 2^e, e the smallest integer in [-40, 40] with A <= M 2^e,
 * or the block's present scale if that is larger and the block holds earlier
 * tokens (slots below start). Earlier tokens' codes are rescaled where the
 * scale grows (code * old / new, rounded half to even). New codes are value /
 * scale rounded half to even and saturated; NaN becomes 0. Slots behind the
 * new tokens are taken to be free: they keep their codes, whose values change
 * with the scale (a sequence grows, or is taken back to an earlier length and
 * written on from there). Tokens whose slot lies outside the cache are not
 * written. Rows of codes and of scales share no memory with each other, keys
 * with values among them (strides that interleave them are fine).
 */
int w4a16_kv_write(const w4a16_kv_rows* k, const w4a16_kv_rows* v, int64_t tokens, const w4a16_kv_cache* cache,
                   const int64_t* start, const int64_t* counts, int type, void* stream);

/*
 * Rotary positions of q and k, and w4a16_kv_write of the rotated k (rounded
 * to its type first) and of v, in one launch: the results of the two calls
 * above. q_out [batch, tokens, heads, head_dim] contiguous, padding rows zero,
 * positions outside the cache NaN in the rotated dims. rot a multiple of 16,
 * table_rows >= slots.
 */
int w4a16_rotary_kv_write(const w4a16_kv_rows* q, void* q_out, int64_t heads, const w4a16_kv_rows* k,
                          const w4a16_kv_rows* v, int64_t tokens, const float* cos_table, const float* sin_table,
                          int64_t table_rows, int64_t rot, int interleaved, const w4a16_kv_cache* cache,
                          const int64_t* start, const int64_t* counts, int type, void* stream);

/*
 * Reads keys or values back: out [batch, kv_heads, slots, head_dim]
 * (contiguous, out_type fp16, bf16 or fp32) = code * scale, rounded once and
 * saturated at the type's largest finite value (NaN codes stay NaN). head_dim
 * a multiple of 16.
 */
int w4a16_kv_read(const w4a16_kv_codes* side, void* out, int64_t batch, int64_t kv_heads, int64_t slots,
                  int64_t head_dim, int64_t block, int code_type, int out_type, void* stream);

/*
 * Attention of the tokens' queries over the cache: out [batch, tokens, heads,
 * head_dim] (contiguous, the type of q) = sum_j w_j v_j over the slots j = 0
 * .. start[b] + t, w = softmax(scale q.k_j). heads a multiple of kv_heads;
 * query head h reads KV head h / (heads / kv_heads). The tokens' own keys and
 * values must be in the cache (w4a16_kv_write first). Padding rows come out
 * zero, rows at positions outside the cache NaN. Slots behind a sequence's
 * last token may hold anything; the codes of those that a row of the call sees
 * are numbers (w4a16_kv_write writes no others: an e4m3 NaN among the values
 * may turn other rows of the call into NaN, too).
 * Scores and sums are fp32. In the second product a weight times its value's
 * scale is an fp16 number: off by 2^-11 of itself down to 2^-21 of the row's
 * largest, by 2^-32 of the largest below. bf16 queries enter the first one as
 * fp16 times a power of two per row: exact down to 2^-31 of the row's largest
 * value, off by 2^-39 of it below. The same call gives the same bits.
 * workspace: w4a16_kv_attention_workspace_bytes(...) bytes (0: none needed),
 * 16-byte aligned, contents ignored, not shared by calls that overlap.
 */
int64_t w4a16_kv_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                           int64_t slots, int64_t head_dim);
int w4a16_kv_attention(const w4a16_kv_rows* q, void* out, int64_t tokens, int64_t heads, const w4a16_kv_cache* cache,
                       const int64_t* start, const int64_t* counts, float scale, int type, void* workspace,
                       int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* W4A16_KV_H */

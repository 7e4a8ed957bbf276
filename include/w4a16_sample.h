/*
 * w4a16_sample.h -- C ABI of sampling: a token from each row of logits. The
 * conventions of w4a16_hip.h hold (device pointers, return codes,
 * w4a16_last_error(), work enqueued on `stream`, nothing allocated or
 * synchronised, so every call may be captured in a HIP graph).
 */
#ifndef W4A16_SAMPLE_H
#define W4A16_SAMPLE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * How a row's token is drawn. A pointer (device memory, one value a row) takes
 * the place of the number above it where it is not NULL.
 *   temperature  0 (or, in a row's value, anything that is not above 0): the
 *                first of the largest logits
 *   top_k        tokens that are kept; 0 (a row's value: 0 or less): all
 *   top_p        share of the kept tokens' probability; 1 (a row's value: 1 or
 *                more, NaN): all
 *   min_p        least probability relative to the largest; 0 (a row's value: 0
 *                or less, NaN): none; above 1 as 1
 */
typedef struct w4a16_sample_settings {
    double temperature;
    int64_t top_k;
    double top_p, min_p;
    const float* temperatures;
    const int64_t* top_ks;
    const float *top_ps, *min_ps;
} w4a16_sample_settings;

/*
 * tokens[r] of the row logits[r row_stride ..], n logits x of `type`
 * (W4A16_FP16, W4A16_BF16 or W4A16_FP32), 1 <= n <= 524288, drawn by the number
 * random[r] in [0, 1):
 *   weights w_i = exp((x_i - max x) / temperature), 0 for x_i = -inf;
 *   tokens in falling order of x, equal ones by index: the first top_k are kept,
 *   of those each one before which less than top_p of their weight lies, and of
 *   those each with w_i >= min_p;
 *   the token is the first, by index, at which the running sum of the kept
 *   weights exceeds random[r] times their sum.
 * A number below 0 or NaN reads as 0, one of 1 or more gives the last token of a
 * weight. Weights are held to 2^-38 of themselves and rounded to whole multiples
 * of 2^-44 of the largest one (smaller ones count as 0), their sums are exact: the
 * same call gives the same tokens. A row with NaN gives the first NaN's index and a
 * row of -inf token 0, as argmax does; where logits are +inf, those alone have weight.
 * tokens share no memory with the other arguments.
 */
int w4a16_sample(const void* logits, int64_t rows, int64_t n, int64_t row_stride, int type, const float* random,
                 const w4a16_sample_settings* settings, int64_t* tokens, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* W4A16_SAMPLE_H */

/*
 * gguf_hip_sample.h — sampling a token per row of logits: C ABI of libgguf_hip, next to
 * gguf_hip_argmax of gguf_hip.h (same conventions).
 */
#ifndef GGUF_HIP_SAMPLE_H
#define GGUF_HIP_SAMPLE_H

#include "gguf_hip.h"

#ifdef __cplusplus
extern "C" {
#endif
#pragma GCC visibility push(default)

#define GGUF_HIP_SAMPLE_MAX_VOCAB 1048576
#define GGUF_HIP_SAMPLE_MAX_ROWS 65535

/* One token per row of f32 logits [rows][ld], from the given random numbers.
 *
 * A row's tokens are taken in descending order of their logits, equal ones in ascending order
 * of their index; w = exp((logit - largest) / temperature).  Kept is a run of them from the
 * first on, the shortest that one of these asks for, but at least one token:
 *   top_k  the first top_k                                          (off where top_k <= 0)
 *   top_p  the fewest whose w sum to top_p times the sum of the first top_k, or more
 *                                                                   (off where top_p >= 1)
 *   min_p  those with w >= min_p                                    (off where min_p <= 0)
 * Drawn is the first kept token at which the running sum of w exceeds u times the kept sum.
 * temperature <= 0 (or NaN): the first token.  u is taken into 0 <= u < 1 (NaN as 0); NaN in
 * top_p and min_p: off.  A NaN or -infinite logit is never drawn; where the largest is
 * infinite, only the infinite ones are.  A row with nothing to draw gives token 0, as
 * gguf_hip_argmax does, with probability 0.
 * probs (may be NULL): w of the drawn token over the kept sum; 1 where temperature <= 0.
 *
 * u [rows]; temperature, top_k, top_p and min_p are device arrays [rows] or NULL, for which
 * the value beside counts for every row.  w is computed in f64 and summed in 64-bit integers
 * as multiples of 2^-43, so that the result depends neither on timing nor on how a row is
 * split.  work: gguf_hip_sample_workspace bytes, 16-byte aligned, no initial value; calls that
 * share it must not overlap. */
int gguf_hip_sample(const float *logits, int64_t ld, int64_t rows, int64_t vocab, const float *u,
                    const float *temperature, float temperature_all, const int32_t *top_k,
                    int32_t top_k_all, const float *top_p, float top_p_all, const float *min_p,
                    float min_p_all, int64_t *out, float *probs, void *work, int64_t work_bytes,
                    void *stream);

/* Bytes of its workspace; negative on bad shapes. */
int64_t gguf_hip_sample_workspace(int64_t rows, int64_t vocab);

#pragma GCC visibility pop
#ifdef __cplusplus
}
#endif

#endif /* GGUF_HIP_SAMPLE_H */

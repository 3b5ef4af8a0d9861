/*
 * gguf_hip_kv4.h — KV cache held in 4 bits: C ABI of libgguf_hip, next to the
 * f32 caches of gguf_hip.h (same conventions: plain device pointers, validation
 * before any HIP call, GGUF_HIP_ERR_* codes, gguf_hip_last_error, no host sync,
 * no device allocation; every call can be captured in a graph).
 *
 * A cached value is d * (c - 8): blocks of 32 channels share an f16 scale d, c is a
 * 4-bit code.  The codes are those of Q4_0 rows quantized as this package's
 * quantizer does: d = f16(max / -8) with max the block's element of largest
 * magnitude (the first of several), c = clamp(rint(x / d) + 8, 0, 15) (8 where d is
 * zero), in f32 arithmetic.  |x| has to stay below 524160 (d is finite).
 *
 * One layer's cache is n_seq * n_kv_heads lists of `slots` slots (a multiple of 32),
 * list (s, h) at byte (s * n_kv_heads + h) * (slots / 32) * 36 * head_dim.  A list is
 * tiles of 32 slots, 36 * head_dim bytes each, NB = head_dim / 32:
 *   K codes  [slot 32][g 4][block NB][4]: byte i holds channels 32 block + 8 g + i
 *            (low nibble) and 32 block + 8 g + 4 + i (high nibble);
 *   V codes  [group 8][n 16][block NB][slot of the group 4]: channels 32 block + n
 *            (low nibble) and 32 block + 16 + n (high nibble) of slot 4 group + s;
 *   K scales [group 8][block NB][slot of the group 4] f16, then V scales alike.
 *
 * Per sequence s (device int64 arrays): lengths[s] slots of every KV head are in use,
 * and pos[s] is the RoPE position of its next token.  The two differ once slots have
 * been evicted; attention itself does not depend on the order of the slots.
 * Two optional arrays [n_seq][n_kv_heads][slots] go with the slots: `positions` (int32,
 * the RoPE position of the token in the slot) and `weights` (f32, attention weight).
 *
 * Supported: head_dim 64, 128 or 256; n_heads 1..8 times n_kv_heads; f32 rows
 * qkv = [q (n_heads * head_dim) | k | v (n_kv_heads * head_dim each)] with a row stride
 * ldqkv (floats, a multiple of 4); cos / sin tables [rope_rows][head_dim / 2].
 */
#ifndef GGUF_HIP_KV4_H
#define GGUF_HIP_KV4_H

#include "gguf_hip.h"

#ifdef __cplusplus
extern "C" {
#endif
#pragma GCC visibility push(default)

#define GGUF_HIP_KV4_TILE 32
#define GGUF_HIP_KV4_MAX_SLOTS 1048576
#define GGUF_HIP_KV4_MAX_ROWS 64 /* new rows per sequence of one attention call */

/* What gguf_hip_kv4_attention does with `weights`. */
#define GGUF_HIP_KV4_WEIGHTS_NONE 0
#define GGUF_HIP_KV4_WEIGHTS_STORE 1
#define GGUF_HIP_KV4_WEIGHTS_ADD 2

/* Bytes of one layer's cache; negative on bad shapes. */
int64_t gguf_hip_kv4_bytes(int n_seq, int n_kv_heads, int head_dim, int64_t slots);

/* Rows of one or more sequences into their caches: k after rotate_half RoPE
 * (rope.wgsl:1-10; every product and sum rounded to f32) and v, quantized.
 * Sequence s owns rows starts[s] .. starts[s + 1] - 1 of qkv (device int64
 * [n_seq + 1], ascending; NULL: n_rows / n_seq rows each, in order).  Its row i goes
 * to slot lengths[s] + i with position pos[s] + i.  Rows past starts[n_seq], rows whose
 * slot or position lies past the cache or the tables, and rows of a sequence with
 * lengths[s] < 0 or pos[s] < 0, are not stored.  Neither lengths nor pos is changed.
 * positions / weights (may be NULL): the stored slots get their position and weight 0.
 * One launch; n_rows == 0 is a no-op, more than 2^25 are refused. */
int gguf_hip_kv4_append(const float *qkv, int64_t ldqkv, int64_t n_rows, const int64_t *starts,
                        const int64_t *lengths, const int64_t *pos, const float *cos_table,
                        const float *sin_table, int64_t rope_rows, void *kv, int32_t *positions,
                        float *weights, int n_seq, int n_heads, int n_kv_heads, int head_dim,
                        int64_t slots, void *stream);

/* Attention of `rows` (1 .. GGUF_HIP_KV4_MAX_ROWS) new rows of each sequence over its
 * cache.  Row i of sequence s is row s * rows + i of qkv and out, stands at position
 * pos[s] + i and sees slots 0 .. lengths[s] + i; query head h reads KV head
 * h / (n_heads / n_kv_heads), softmax scaled by 1 / sqrt(head_dim).
 * store != 0: the rows' k and v are first stored in slots lengths[s] .. + rows - 1
 * (as gguf_hip_kv4_append).  store == 0: those slots hold them already.
 * weights (WEIGHTS_STORE / WEIGHTS_ADD): for each slot a row of this call sees, the
 * softmax weights summed over the rows and over the query heads of its KV head are
 * written or added; other slots are left as they are.
 * A sequence with lengths[s] < 0, lengths[s] + rows > slots, pos[s] < 0 or
 * pos[s] + rows > rope_rows takes no part: nothing of it is written.  lengths and pos are
 * not changed.  out must not overlap qkv.  work: gguf_hip_kv4_attention_workspace bytes,
 * 16-byte aligned, no initial value; calls that share it must not overlap.  Results do
 * not depend on timing.  f32-grade: codes enter the f16 matrix cores exactly, queries and
 * probabilities times V's scales as two f16 parts each, 22 bits of each product down to
 * 2^-13 of a row's largest, below that 2^-35 of it. */
int gguf_hip_kv4_attention(const float *qkv, int64_t ldqkv, int rows, const int64_t *lengths,
                           const int64_t *pos, const float *cos_table, const float *sin_table,
                           int64_t rope_rows, void *kv, int store, int32_t *positions,
                           float *weights, int weights_mode, float *out, int64_t ldo, int n_seq,
                           int n_heads, int n_kv_heads, int head_dim, int64_t slots, void *work,
                           int64_t work_bytes, void *stream);

/* Bytes of its workspace; negative on bad shapes. */
int64_t gguf_hip_kv4_attention_workspace(int rows, int weights_mode, int n_seq, int n_heads,
                                         int n_kv_heads, int head_dim, int64_t slots);

/* Slots 0 .. lengths[s] - 1 as f32 rows: k_out / v_out [n_layers][n_seq][n_kv_heads]
 * [out_slots][head_dim] of caches [n_layers] (each gguf_hip_kv4_bytes long).  Slots from
 * out_slots on are not read, rows from lengths[s] on not written, and nothing of a
 * sequence with lengths[s] > slots.  The layout is that of
 * the f32 caches of gguf_hip_attention_prefill. */
int gguf_hip_kv4_load(const void *kv, const int64_t *lengths, float *k_out, float *v_out,
                      int64_t out_slots, int n_layers, int n_seq, int n_kv_heads, int head_dim,
                      int64_t slots, void *stream);

/* Eviction.  Every list (layer, sequence, KV head) of a sequence with
 * lengths[s] > keep and lengths[s] >= trigger is cut back to `keep` slots: those of
 * largest weight (of equal ones the lower slot; NaN counts least), where slots with
 * positions >= pos[s] - recent or < sinks come before all others, whatever their weights
 * (recent + sinks <= keep).  A kept slot below `keep` stays where it is; the kept slots
 * from `keep` on move, in order, into the slots below it that were given up.  Slots from
 * `keep` on keep their bytes.  weights / positions [n_layers][n_seq][n_kv_heads][slots] of
 * the remaining slots go to weights_out / positions_out (the same arrays: in place), the
 * new lengths to lengths_out (may be lengths).  Sequences that are not cut keep their
 * caches, weights, positions and lengths.  weights and positions are 16-byte aligned.
 * Two launches.  work: gguf_hip_kv4_evict_workspace bytes, 16-byte aligned, no initial
 * value; calls that share it must not overlap. */
int gguf_hip_kv4_evict(void *kv, const float *weights, const int32_t *positions,
                       const int64_t *lengths, const int64_t *pos, int64_t keep, int64_t trigger,
                       int64_t recent, int64_t sinks, float *weights_out, int32_t *positions_out,
                       int64_t *lengths_out, int n_layers, int n_seq, int n_kv_heads, int head_dim,
                       int64_t slots, void *work, int64_t work_bytes, void *stream);

/* Bytes of its workspace; negative on bad shapes. */
int64_t gguf_hip_kv4_evict_workspace(int n_layers, int n_seq, int n_kv_heads, int head_dim,
                                     int64_t slots);

#pragma GCC visibility pop
#ifdef __cplusplus
}
#endif

#endif /* GGUF_HIP_KV4_H */

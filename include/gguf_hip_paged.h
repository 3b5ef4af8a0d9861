/*
 * gguf_hip_paged.h — KV cache in pages that sequences can share: C ABI of libgguf_hip,
 * next to the f32 caches of gguf_hip.h and the 4-bit ones of gguf_hip_kv4.h (same
 * conventions: plain device pointers, validation before any HIP call, GGUF_HIP_ERR_*
 * codes, gguf_hip_last_error, no host sync, no device allocation; every call can be
 * captured in a graph).
 *
 * A page holds `page` slots (16, 32, 64, 128 or 256) of every KV head of one layer, in
 * f16 or bf16, 4 * n_kv_heads * page * head_dim bytes:
 *   K  [KV head][slot][head_dim]
 *   V  [KV head][slot / 16][head_dim][slot % 16]
 * One layer's pool is n_pages pages; several layers' pools follow each other, and a page
 * number means that page of every layer.
 *
 * Per sequence s: tables[s][columns] (device int32): the pages of its slots in order, slot
 * t in page tables[s][t / page], an entry outside 0 .. n_pages - 1 (-1) for none; lengths[s]
 * (device int64): the slots in use.  Slot t holds the token at RoPE position t.  refs[p]
 * (device int32): how many table entries hold page p; 0 is a free page.
 * Optional, device int64: room[s]: slots from room[s] on are not written (the end of what
 * gguf_hip_paged_grow gave the sequence, so that a page which others hold is never written;
 * without it the caller sees to that).
 *
 * Supported: head_dim 64, 128 or 256; n_heads 1..8 times n_kv_heads; f32 rows
 * qkv = [q (n_heads * head_dim) | k | v (n_kv_heads * head_dim each)] with a row stride
 * ldqkv (floats, a multiple of 4); cos / sin tables [rope_rows][head_dim / 2]; up to
 * GGUF_HIP_PAGED_MAX_SEQS sequences of up to GGUF_HIP_PAGED_MAX_SLOTS slots and up to
 * GGUF_HIP_PAGED_MAX_PAGES pages.
 */
#ifndef GGUF_HIP_PAGED_H
#define GGUF_HIP_PAGED_H

#include "gguf_hip.h"

#ifdef __cplusplus
extern "C" {
#endif
#pragma GCC visibility push(default)

#define GGUF_HIP_PAGED_F16 1
#define GGUF_HIP_PAGED_BF16 2
#define GGUF_HIP_PAGED_MAX_SEQS 4096
#define GGUF_HIP_PAGED_MAX_SLOTS 4194304
#define GGUF_HIP_PAGED_MAX_PAGES 16777216

/* Bytes of one layer's pool; negative on bad shapes. */
int64_t gguf_hip_paged_bytes(int64_t n_pages, int page, int n_kv_heads, int head_dim);

/* Rows of one or more sequences into their pages: k after rotate_half RoPE (rope.wgsl:1-10;
 * every product and sum rounded to f32) and v, each rounded to the pages' type (to nearest,
 * ties to even: f16 overflows to infinity from 65520 on).
 * Sequence s owns rows starts[s] .. starts[s + 1] - 1 of qkv (device int64 [n_seq + 1],
 * ascending; NULL: n_rows / n_seq rows each, in order).  Its row i goes to slot
 * lengths[s] + i.  Rows past starts[n_seq], rows of a sequence with lengths[s] < 0, and rows
 * whose slot has no page or lies past the table, the RoPE tables or room[s], are not stored.
 * lengths is not changed.  One launch; n_rows == 0 is a no-op, more than 2^25 are refused. */
int gguf_hip_paged_append(const float *qkv, int64_t ldqkv, int64_t n_rows, const int64_t *starts,
                          const int64_t *lengths, const int64_t *room, const int32_t *tables,
                          const float *cos_table, const float *sin_table, int64_t rope_rows,
                          void *kv, int dtype, int64_t n_pages, int page, int64_t columns,
                          int n_seq, int n_heads, int n_kv_heads, int head_dim, void *stream);

/* Attention of one new row of each sequence: row s of qkv is stored in slot lengths[s] (as
 * gguf_hip_paged_append) and attends to slots 0 .. lengths[s]; query head h reads KV head
 * h / (n_heads / n_kv_heads), softmax scaled by 1 / sqrt(head_dim).  A slot whose table entry
 * names no page is not seen.  A sequence whose row cannot be stored (lengths[s] < 0, no page,
 * past the tables or room[s]) takes no part: neither its pages nor its row of out is written.
 * lengths is not changed.  out must not overlap qkv.  work: gguf_hip_paged_attention_workspace
 * bytes, 16-byte aligned, no initial value; calls that share it must not overlap.  Results do
 * not depend on timing.  f32-grade: K and V enter the matrix cores as they are, queries and
 * probabilities as two f16 parts each (22 bits of each product down to 2^-13 of a row's
 * largest, below that 2^-35 of it) or three bf16 parts (24 bits).  Since a part may be zero, a
 * head that sees an infinite K or V may be NaN where exact sums would not be. */
int gguf_hip_paged_attention(const float *qkv, int64_t ldqkv, const int64_t *lengths,
                             const int64_t *room, const int32_t *tables, const float *cos_table,
                             const float *sin_table, int64_t rope_rows, void *kv, int dtype,
                             float *out, int64_t ldo, int64_t n_pages, int page, int64_t columns,
                             int n_seq, int n_heads, int n_kv_heads, int head_dim, void *work,
                             int64_t work_bytes, void *stream);

/* Bytes of its workspace; negative on bad shapes. */
int64_t gguf_hip_paged_attention_workspace(int page, int64_t columns, int n_seq, int n_heads,
                                           int n_kv_heads, int head_dim);

/* Slots 0 .. lengths[s] - 1 as f32 rows: k_out / v_out [n_seq][n_kv_heads][out_slots][head_dim]
 * of one layer's pool.  Slots from out_slots on are not read; rows from lengths[s] on, and rows
 * of slots without a page, are not written.  For one sequence the layout is that of the f32
 * caches of gguf_hip_attention_prefill. */
int gguf_hip_paged_load(const void *kv, int dtype, const int32_t *tables, const int64_t *lengths,
                        float *k_out, float *v_out, int64_t out_slots, int64_t n_pages, int page,
                        int64_t columns, int n_seq, int n_kv_heads, int head_dim, void *stream);

/* Sequence s becomes a fork of sequence parents[s] (device int64) as that was before the call:
 * its table and length are the parent's, whose pages it shares.  parents[s] == s leaves it as
 * it is; a parent outside 0 .. n_seq - 1 (-1) frees it: no pages, length 0.  refs of the pages
 * given up and taken are counted down and up.  The results go to tables_out / lengths_out /
 * refs_out, each the same array as its input (in place) or one that overlaps no other; nothing
 * else is changed.  One launch, or two where refs_out is another array and large. */
int gguf_hip_paged_fork(const int32_t *tables, const int64_t *lengths, const int32_t *refs,
                        const int64_t *parents, int32_t *tables_out, int64_t *lengths_out,
                        int32_t *refs_out, int64_t n_pages, int64_t columns, int n_seq,
                        void *stream);

/* Room for rows[s] (device int64) more rows of each sequence, in place.  In the order of the
 * sequences, and for each in the order of the columns lengths[s] / page ..
 * (lengths[s] + rows[s] - 1) / page (as far as the table goes): an entry without a page gets the
 * lowest free page; an entry whose page other entries hold too (refs > 1) gets the lowest free
 * page in its place, and if the page has slots in use by the sequence, their blocks of 16 slots
 * are copied in all n_layers layers.  A sequence for which no free page is left gets no further
 * ones.  room[s]: the end of the slots that the sequence may now write, lengths[s] at least (0
 * where lengths[s] < 0); it is lengths[s] where rows[s] <= 0.  lengths is not changed, and room
 * must not overlap it or rows.  refs is 16-byte aligned.
 * Two launches.  work: gguf_hip_paged_grow_workspace bytes, 16-byte aligned, no initial value;
 * calls that share it must not overlap. */
int gguf_hip_paged_grow(void *kv, int32_t *tables, const int64_t *lengths, int32_t *refs,
                        const int64_t *rows, int64_t *room, int n_layers, int64_t n_pages,
                        int page, int64_t columns, int n_seq, int n_kv_heads, int head_dim,
                        void *work, int64_t work_bytes, void *stream);

/* Bytes of its workspace; negative on bad shapes. */
int64_t gguf_hip_paged_grow_workspace(int64_t n_pages, int page, int64_t columns, int n_seq);

/* Moves the pages in use (refs > 0) into the pages 0 .. n - 1, n their number: those from n on
 * move, in order, into the free ones below n, in order; the others stay.  All n_layers layers
 * move alike; the bytes of the pages that were left stay.  Table entries and refs follow, to
 * tables_out and refs_out (each the same array as its input or one that overlaps no other);
 * live[0] (device int64) is n.  refs is 16-byte aligned.  Two launches.  work: gguf_hip_paged_compact_workspace bytes,
 * 16-byte aligned, no initial value; calls that share it must not overlap. */
int gguf_hip_paged_compact(void *kv, const int32_t *tables, const int32_t *refs,
                           int32_t *tables_out, int32_t *refs_out, int64_t *live, int n_layers,
                           int64_t n_pages, int page, int64_t columns, int n_seq, int n_kv_heads,
                           int head_dim, void *work, int64_t work_bytes, void *stream);

/* Bytes of its workspace; negative on bad shapes. */
int64_t gguf_hip_paged_compact_workspace(int64_t n_pages, int64_t columns, int n_seq);

#pragma GCC visibility pop
#ifdef __cplusplus
}
#endif

#endif /* GGUF_HIP_PAGED_H */

// The KV cache in pages (layout: gguf_hip_paged.h): what its kernels share.
#pragma once

#include "kv4.hpp"

namespace gguf {

typedef __bf16 bhalf_t;
typedef __bf16 bhalf2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bhalf8_t __attribute__((ext_vector_type(8)));

constexpr int kPageBlock = 16;  // slots of a block

// The arguments that calls over rows have: one layer's pool and its sequences.
struct PagedCache {
  uint16_t *kv;
  const int32_t *tables;   // [n_seq][columns]
  const int64_t *lengths, *room;  // room may be null
  const float *cs, *sn;    // RoPE tables [rope_rows][hd / 2]
  int64_t rope_rows;
  int n_pages, page, shift;  // page = 1 << shift
  int columns, n_seq, nh, nkv, hd;
  bool bf16;
};

// A load of what no call changes while it runs, by a scalar instruction where the address is uniform.
template <typename T>
__device__ __forceinline__ T steady(const T *p) {
  return *(const __attribute__((address_space(4))) T *)(uintptr_t)p;
}

// The slots that a call may store in sequence s: below the table's, the RoPE tables' and room's end.
__device__ __forceinline__ int64_t paged_end(const PagedCache &c, int64_t s) {
  int64_t end = (int64_t)c.columns << c.shift;
  end = end < c.rope_rows ? end : c.rope_rows;
  if (c.room) end = end < steady(c.room + s) ? end : steady(c.room + s);
  return end < 0 ? 0 : end;
}
// 16-bit values from the start of page p to those of KV head h, slot j: its K row, and its V (channel
// e at + e * 16).
__device__ __forceinline__ int64_t paged_k_at(const PagedCache &c, int64_t p, int h, int j) {
  return (((p * 2 * c.nkv + h) << c.shift) + j) * c.hd;
}
__device__ __forceinline__ int64_t paged_v_at(const PagedCache &c, int64_t p, int h, int j) {
  return (((p * 2 + 1) * c.nkv + h) << c.shift) * c.hd + (int64_t)(j >> 4) * (16 * c.hd) + (j & 15);
}

// Four channels rounded to a page's type, to nearest.
template <bool BF>
__device__ __forceinline__ uint2 paged_round(const float (&y)[4]) {
  uint16_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = BF ? __builtin_bit_cast(uint16_t, (bhalf_t)y[i]) : __builtin_bit_cast(uint16_t, (half_t)y[i]);
  return make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
}

// A row's channels after RoPE if it is of K, every product and sum rounded (no contraction).
template <int HD>
__device__ __forceinline__ void paged_turn(const Kv4Row<HD> &x, int q, bool is_k, float (&y)[4]) {
#pragma clang fp contract(off)
  const float v[4] = {x.y.x, x.y.y, x.y.z, x.y.w};
  const float c[4] = {x.c.x, x.c.y, x.c.z, x.c.w}, s[4] = {x.s.x, x.s.y, x.s.z, x.s.w};
  const bool low = q < Kv4Row<HD>::LANES / 2;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float o = Kv4Row<HD>::other(v[j]), a = v[j] * c[j], b = o * s[j];
    const float turned = low ? a - b : a + b;
    y[j] = is_k ? turned : v[j];
  }
}

// v + those of the lanes below it in the wave.
__device__ __forceinline__ int lanes_before(int v) {
  int run = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(run, o);
    if ((int)(threadIdx.x & 63) >= o) run += x;
  }
  return run;
}

hipError_t launch_paged_append(const PagedCache &c, const float *qkv, int64_t ldq, int64_t n_rows,
                               const int64_t *starts, hipStream_t s);
hipError_t launch_paged_load(const PagedCache &c, float *k, float *v, int64_t out_slots,
                             hipStream_t s);

struct PagedAttn {
  const float *qkv;
  int64_t ldq;
  float *out;
  int64_t ldo;
  void *work;
};
int64_t paged_attention_work_bytes(int page, int64_t columns, int n_seq, int nh, int nkv, int hd);
hipError_t launch_paged_attention(const PagedCache &c, const PagedAttn &a, hipStream_t s);

hipError_t launch_paged_fork(const int32_t *tables, const int64_t *lengths, const int32_t *refs,
                             const int64_t *parents, int32_t *tables_out, int64_t *lengths_out,
                             int32_t *refs_out, int n_pages, int columns, int n_seq, hipStream_t s);

// Pages of all layers and the tables over them.
struct PagedPool {
  uint16_t *kv;
  int n_layers, n_pages, page, shift, columns, n_seq;
  int64_t page_values, head_values;  // 16-bit values of a page of one layer, and of K or V of a head
};
int64_t paged_grow_work_bytes(int n_seq);
hipError_t launch_paged_grow(const PagedPool &c, int32_t *tables, const int64_t *lengths,
                             int32_t *refs, const int64_t *rows, int64_t *room, void *work,
                             hipStream_t s);
int64_t paged_compact_work_bytes(int64_t n_pages);
hipError_t launch_paged_compact(const PagedPool &c, const int32_t *tables, const int32_t *refs,
                                int32_t *tables_out, int32_t *refs_out, int64_t *live, void *work,
                                hipStream_t s);

struct SampleArgs {
  const float *logits;
  int64_t ld;
  int rows, vocab;
  const float *u, *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  float temperature_all;
  int32_t top_k_all;
  float top_p_all, min_p_all;
  int64_t *out;
  float *probs;
  void *work;
};
int64_t sample_work_bytes(int64_t rows, int64_t vocab);
hipError_t launch_sample(const SampleArgs &a, hipStream_t s);

}  // namespace gguf

// The 4-bit KV cache (layout: gguf_hip_kv4.h): what its kernels share.
#pragma once

#include "common.hpp"

namespace gguf {

constexpr int kKv4Tile = 32;

template <int HD>
struct Kv4 {
  static constexpr int NB = HD / 32;           // blocks (scales) per slot
  static constexpr int TB = 36 * HD;           // bytes per tile of 32 slots
  static constexpr int VO = 16 * HD;           // V codes, K scales, V scales within a tile
  static constexpr int KS = 32 * HD, VS = 34 * HD;
};

// The arguments that every call has: one layer's cache and its sequences.
struct Kv4Cache {
  uint8_t *kv;
  const int64_t *lengths, *pos;
  const float *cs, *sn;  // RoPE tables [rope_rows][hd / 2]
  int32_t *positions;    // may be null
  float *weights;        // may be null
  int64_t rope_rows;
  int n_seq, nh, nkv, hd, slots;
};

__device__ __forceinline__ uint8_t *kv4_list(uint8_t *kv, int64_t list, int slots, int tile_bytes) {
  return kv + list * (int64_t)(slots / kKv4Tile) * tile_bytes;
}

// One row of K (roped with the table rows c, s) or V into slot `slot` of a list, by one
// wave: lane l holds channels l, l + 64, ...  The rounding of every step is fixed (no
// contraction), so that the codes can be restated bit for bit.
template <int HD, bool IS_K>
__device__ __forceinline__ void kv4_store_row(uint8_t *list, int slot, const float *__restrict__ x,
                                              const float *__restrict__ c,
                                              const float *__restrict__ s, int lane) {
#pragma clang fp contract(off)
  using L = Kv4<HD>;
  constexpr int R = HD / 64, half = HD / 2;
  float y[R];
#pragma unroll
  for (int r = 0; r < R; ++r) y[r] = x[lane + 64 * r];
  if constexpr (IS_K) {
    if constexpr (HD == 64) {
      const float o = __shfl_xor(y[0], 32), cv = c[lane & 31], sv = s[lane & 31];
      const float a = y[0] * cv, b = o * sv;
      y[0] = lane < 32 ? a - b : a + b;
    } else {
#pragma unroll
      for (int r = 0; r < R / 2; ++r) {
        const float cv = c[lane + 64 * r], sv = s[lane + 64 * r];
        const float a = y[r], b = y[r + R / 2];
        const float ac = a * cv, bs = b * sv, bc = b * cv, as = a * sv;
        y[r] = ac - bs;
        y[r + R / 2] = bc + as;
      }
    }
  }
  uint8_t *tile = list + (int64_t)(slot / kKv4Tile) * L::TB;
  const int j = slot % kKv4Tile;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float a = fabsf(y[r]);
    float m = a;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const uint32_t eq = (uint32_t)(__ballot(a == m) >> (lane & 32));
    const int first = eq ? __builtin_ctz(eq) : 0;  // none: every element is NaN
    float d32 = __shfl(y[r], (lane & 32) + first) * -0.125f;
    // the product by itself: fused into the conversion it is added to +0, and -0 is lost
    asm volatile("" : "+v"(d32));
    const half_t d = (half_t)d32;
    const float df = (float)d;
    const float q = df != 0.f ? rintf(y[r] / df) + 8.f : 8.f;
    const int code = (int)fminf(fmaxf(q, 0.f), 15.f);
    const int b = 2 * r + (lane >> 5);
    if constexpr (IS_K) {
      const int hi = __shfl(code, lane + 4);
      if ((lane & 7) < 4)
        tile[j * half + (((lane >> 3) & 3) * L::NB + b) * 4 + (lane & 3)] =
            (uint8_t)(code | (hi << 4));
    } else {
      const int hi = __shfl(code, lane + 16);
      if ((lane & 31) < 16)
        tile[L::VO + (j >> 2) * (2 * HD) + ((lane & 15) * L::NB + b) * 4 + (j & 3)] =
            (uint8_t)(code | (hi << 4));
    }
    if ((lane & 31) == 0)
      *(half_t *)(tile + (IS_K ? L::KS : L::VS) + ((j >> 2) * L::NB + b) * 8 + (j & 3) * 2) = d;
  }
}

hipError_t launch_kv4_append(const Kv4Cache &c, const float *qkv, int64_t ldq, int64_t n_rows,
                             const int64_t *starts, hipStream_t s);
hipError_t launch_kv4_load(const uint8_t *kv, const int64_t *lengths, float *k, float *v,
                           int64_t out_slots, int n_layers, int n_seq, int nkv, int hd, int slots,
                           hipStream_t s);

struct Kv4Attn {
  const float *qkv;
  int64_t ldq;
  int rows;
  bool store;
  int weights_mode;
  float *out;
  int64_t ldo;
  void *work;
};
int64_t kv4_attention_work_bytes(int rows, bool weights, int n_seq, int nh, int nkv, int hd,
                                 int slots);
hipError_t launch_kv4_attention(const Kv4Cache &c, const Kv4Attn &a, hipStream_t s);

struct Kv4Evict {
  int64_t keep, trigger, recent, sinks;
  const float *weights;
  const int32_t *positions;
  float *weights_out;
  int32_t *positions_out;
  int64_t *lengths_out;
  void *work;
  int n_layers;
};
int64_t kv4_evict_work_bytes(int64_t lists, int slots);
hipError_t launch_kv4_evict(const Kv4Cache &c, const Kv4Evict &e, hipStream_t s);

}  // namespace gguf

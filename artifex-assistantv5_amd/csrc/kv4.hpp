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

// Lane l's channels l, l + 64, ... of a row, and for a K row its cos / sin.
template <int HD>
struct Kv4Row {
  static constexpr int R = HD / 64, T = HD == 64 ? 1 : R / 2;
  float y[R], c[T], s[T];
  __device__ __forceinline__ void load(const float *__restrict__ x, int lane) {
#pragma unroll
    for (int r = 0; r < R; ++r) y[r] = x[lane + 64 * r];
  }
  __device__ __forceinline__ void load_turn(const float *__restrict__ cr,
                                            const float *__restrict__ sr, int lane) {
#pragma unroll
    for (int r = 0; r < T; ++r) {
      const int i = HD == 64 ? lane & 31 : lane + 64 * r;
      c[r] = cr[i];
      s[r] = sr[i];
    }
  }
};

// The value of lane l ^ 16 / l ^ 32 (the two results of a swap are both lanes' values).
__device__ __forceinline__ uint32_t from_xor16(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return r[0] ^ r[1] ^ v;
}
__device__ __forceinline__ uint32_t from_xor32(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return r[0] ^ r[1] ^ v;
}

// A row's codes and scales, by one wave.  The rounding of every step is fixed (no contraction),
// so that they can be restated bit for bit.  For the 64 channels of each r: K: lanes with
// (lane & 7) < 4 hold the byte at ((lane >> 3) & 3, block, lane & 3) of the slot's K codes; V:
// lanes with (lane & 31) < 16 the byte at (lane & 15, block) of its V codes; the block is 2 r +
// (lane >> 5), and d its scale.
template <int HD, bool IS_K>
__device__ __forceinline__ void kv4_quantize(Kv4Row<HD> &x, int lane, uint8_t (&byte)[HD / 64],
                                             half_t (&scale)[HD / 64]) {
#pragma clang fp contract(off)
  constexpr int R = HD / 64;
  if constexpr (IS_K) {
    if constexpr (HD == 64) {
      const float o = __uint_as_float(from_xor32(__float_as_uint(x.y[0])));
      const float a = x.y[0] * x.c[0], b = o * x.s[0];
      x.y[0] = lane < 32 ? a - b : a + b;
    } else {
#pragma unroll
      for (int r = 0; r < R / 2; ++r) {
        const float a = x.y[r], b = x.y[r + R / 2];
        const float ac = a * x.c[r], bs = b * x.s[r], bc = b * x.c[r], as = a * x.s[r];
        x.y[r] = ac - bs;
        x.y[r + R / 2] = bc + as;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float y = x.y[r], a = fabsf(y), m = max_xor16(max_lanes16(a));
    const uint64_t eq = __ballot(a == m);
    const uint32_t e0 = (uint32_t)eq, e1 = (uint32_t)(eq >> 32);
    // the first of the largest in each block (none where every element is NaN)
    const int i0 = e0 ? __builtin_ctz(e0) : 0, i1 = 32 + (e1 ? __builtin_ctz(e1) : 0);
    const float t0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(y), i0));
    const float t1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(y), i1));
    float d32 = (lane < 32 ? t0 : t1) * -0.125f;
    // the product by itself: fused into the conversion it is added to +0, and -0 is lost
    asm volatile("" : "+v"(d32));
    scale[r] = (half_t)d32;
    const float df = (float)scale[r];
    const float q = df != 0.f ? rintf(y / df) + 8.f : 8.f;
    const uint32_t code = (uint32_t)fminf(fmaxf(q, 0.f), 15.f);
    const uint32_t hi = IS_K ? (uint32_t)__builtin_amdgcn_update_dpp(0, (int)code, 0x104, 0xF, 0xF,
                                                                     true)  // lane + 4
                             : from_xor16(code);
    byte[r] = (uint8_t)(code | (hi << 4));
  }
}

// Quantize a row into slot `slot` of a list.
template <int HD, bool IS_K>
__device__ __forceinline__ void kv4_put_row(uint8_t *list, int slot, Kv4Row<HD> &x, int lane) {
  using L = Kv4<HD>;
  uint8_t byte[HD / 64];
  half_t scale[HD / 64];
  kv4_quantize<HD, IS_K>(x, lane, byte, scale);
  uint8_t *tile = list + (int64_t)(slot / kKv4Tile) * L::TB;
  const int j = slot % kKv4Tile;
#pragma unroll
  for (int r = 0; r < HD / 64; ++r) {
    const int b = 2 * r + (lane >> 5);
    if constexpr (IS_K) {
      if ((lane & 7) < 4)
        tile[j * (HD / 2) + (((lane >> 3) & 3) * L::NB + b) * 4 + (lane & 3)] = byte[r];
    } else {
      if ((lane & 31) < 16)
        tile[L::VO + (j >> 2) * (2 * HD) + ((lane & 15) * L::NB + b) * 4 + (j & 3)] = byte[r];
    }
    if ((lane & 31) == 0)
      *(half_t *)(tile + (IS_K ? L::KS : L::VS) + ((j >> 2) * L::NB + b) * 8 + (j & 3) * 2) =
          scale[r];
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

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

// The value of lane l ^ 16 / l ^ 32 (the two results of a swap are both lanes' values).
__device__ __forceinline__ uint32_t from_xor16(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return r[0] ^ r[1] ^ v;
}
__device__ __forceinline__ uint32_t from_xor32(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return r[0] ^ r[1] ^ v;
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}

// Rows on their way into the cache: lane q of a row's HD / 4 holds its channels 4 q .. 4 q + 3,
// so a wave holds 256 / HD rows, and a block of 32 channels is eight lanes.
template <int HD>
struct Kv4Row {
  static constexpr int LANES = HD / 4;
  float4 y, c, s;  // the values, and for a K row the cos / sin of its lane's channels
  __device__ __forceinline__ void load(const float *__restrict__ x, int q) {
    y = *(const float4 *)(x + 4 * q);
  }
  __device__ __forceinline__ void load_turn(const float *__restrict__ cr,
                                            const float *__restrict__ sr, int q) {
    c = *(const float4 *)(cr + 4 * (q & (LANES / 2 - 1)));
    s = *(const float4 *)(sr + 4 * (q & (LANES / 2 - 1)));
  }
  // Of lane q ^ LANES / 2: the channels that rotate_half pairs with one's own.
  __device__ __forceinline__ static float other(float v) {
    const uint32_t u = __float_as_uint(v);
    return __uint_as_float(HD == 64 ? dpp_u32<0x128>(u) : (HD == 128 ? from_xor16(u) : from_xor32(u)));
  }
};

// A row's code bytes and scales.  The rounding of every step is fixed (no contraction), so that
// they can be restated bit for bit.  `word`: in a K row's even lanes the four bytes at ((q >> 1) &
// 3, block q >> 3) of the slot's K codes; in a V row's lanes with (q & 7) < 4 the bytes (4 (q &
// 3) + 0..3, block q >> 3) of its V codes.  `scale` is the block's, in each of its lanes.
template <int HD>
__device__ __forceinline__ void kv4_quantize(Kv4Row<HD> &x, int q, bool is_k, uint32_t &word,
                                             half_t &scale) {
#pragma clang fp contract(off)
  float y[4] = {x.y.x, x.y.y, x.y.z, x.y.w};
  {
    const float c[4] = {x.c.x, x.c.y, x.c.z, x.c.w}, s[4] = {x.s.x, x.s.y, x.s.z, x.s.w};
    const bool low = q < Kv4Row<HD>::LANES / 2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float o = Kv4Row<HD>::other(y[j]), a = y[j] * c[j], b = o * s[j];
      const float turned = low ? a - b : a + b;
      y[j] = is_k ? turned : y[j];
    }
  }
  float m = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
  m = fmaxf(m, dpp<kDppXor1>(m));
  m = fmaxf(m, dpp<kDppXor2>(m));
  m = fmaxf(m, dpp<kDppHalfMirror>(m));
  // the sign of the first element of that magnitude (none where every element is NaN)
  uint32_t k = 64;
#pragma unroll
  for (int j = 3; j >= 0; --j)
    if (fabsf(y[j]) == m) k = 2 * (4 * (q & 7) + j) + (__float_as_uint(y[j]) >> 31);
  k = min(k, dpp_u32<kDppXor1>(k));
  k = min(k, dpp_u32<kDppXor2>(k));
  k = min(k, dpp_u32<kDppHalfMirror>(k));
  float d32 = __uint_as_float(__float_as_uint(m) | (k << 31)) * -0.125f;
  // the product by itself: fused into the conversion it is added to +0, and -0 is lost
  asm volatile("" : "+v"(d32));
  scale = (half_t)d32;
  const float df = (float)scale, inv = __builtin_amdgcn_rcpf(df);
  // x / d to the nearest integer: by the reciprocal, within 4e-6 of the quotient (at most 16),
  // and by the division itself where that is not enough to tell
  float t[4];
  bool near = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float v = y[j] * inv;
    t[j] = rintf(v);
    near |= fabsf(v - t[j]) > 0.49999f;
  }
  if (__any(near)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = rintf(y[j] / df);
  }
  uint32_t codes = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float v = df != 0.f ? fminf(fmaxf(t[j] + 8.f, 0.f), 15.f) : 8.f;
    codes |= (uint32_t)v << (8 * j);
  }
  // the high nibbles: K channels + 4 (the next lane), V channels + 16 (four lanes on)
  const uint32_t next = dpp_u32<kDppXor1>(codes), four = dpp_u32<0x104>(codes);
  word = codes | ((is_k ? next : four) << 4);
}

// Quantize rows, the lane's of K or V, into slot `slot` of a list.
template <int HD>
__device__ __forceinline__ void kv4_put_row(uint8_t *list, int slot, Kv4Row<HD> &x, int q, bool is_k,
                                            bool store) {
  using L = Kv4<HD>;
  uint32_t word;
  half_t scale;
  kv4_quantize<HD>(x, q, is_k, word, scale);
  if (!store) return;
  uint8_t *tile = list + (int64_t)(slot / kKv4Tile) * L::TB;
  const int j = slot % kKv4Tile, b = q >> 3;
  if (is_k) {
    if (!(q & 1))
      *(uint32_t *)(tile + j * (HD / 2) + (((q >> 1) & 3) * L::NB + b) * 4) = word;
  } else if ((q & 7) < 4) {
    uint8_t *v = tile + L::VO + (j >> 2) * (2 * HD) + (4 * (q & 3) * L::NB + b) * 4 + (j & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i * L::NB * 4] = (uint8_t)(word >> (8 * i));
  }
  if (!(q & 7))
    *(half_t *)(tile + (is_k ? L::KS : L::VS) + ((j >> 2) * L::NB + b) * 8 + (j & 3) * 2) = scale;
}

// whole (without starts): of a sequence whose rows do not all fit, none is stored.
hipError_t launch_kv4_append(const Kv4Cache &c, const float *qkv, int64_t ldq, int64_t n_rows,
                             const int64_t *starts, bool whole, hipStream_t s);
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

// Attention over the 4-bit KV cache.
//
// Query rows of a (sequence, KV head): v = i * group + h for new row i and query head h of
// the group; row v sees slots 0 .. lengths[s] + i.  The slots are split over workgroups;
// each writes, per query row, a record of its partial softmax, and kv4_merge_kernel joins
// them in split order (so the result does not depend on timing).
#include <type_traits>

#include "kv4.hpp"

namespace gguf {

namespace {

// log2(e) / sqrt(head_dim) as two floats: one alone would be off by up to 2^-25, and that times
// a score is the relative error of its probability.
template <int HD>
struct ScoreScale {
  static constexpr double v = 1.4426950408889634074 / (HD == 64 ? 8.0 : (HD == 128 ? 11.313708498984760390 : 16.0));
  static constexpr float hi = (float)v, lo = (float)(v - (double)hi);
};

// A record: sum of p v per channel, then per block of 32 channels the maximum m that its p
// are relative to (in log2 units) and the sum of its p.
template <int HD>
constexpr int record_floats() {
  return HD + 2 * (HD / 32);
}

// The slots in use before the call, or -1 if the sequence takes no part.
__device__ __forceinline__ int kv4_filled(const Kv4Cache &c, int64_t s, int rows) {
  const int64_t n = c.lengths[s], p = c.pos[s];
  return n < 0 || n > c.slots - rows || p < 0 || p > c.rope_rows - rows ? -1 : (int)n;
}

// How the tiles of a list are cut: `per` for each workgroup, `n` of them at most S.  Every
// workgroup of the call gets about the same number, whatever the sequences' lengths: all lists'
// tiles over `wgs` workgroups, in whole turns of a workgroup's W waves, and no fewer than eight:
// they do not make up for a workgroup's start and end (4 x 9000 slots of 256 channels, 8 query
// rows: four 24.8 us, eight 23.5).
constexpr int kLeastTiles = 8;
struct Cut {
  int S, wgs, W;
};
struct Splits {
  int per, n;
};
__device__ __forceinline__ int kv4_tiles(int filled, int rows) {
  return filled < 0 ? 0 : (filled + rows + kKv4Tile - 1) / kKv4Tile;
}
__device__ __forceinline__ Splits kv4_splits(int tiles, int fair, const Cut &k) {
  const int per = (max(max(fair, kLeastTiles), (tiles + k.S - 1) / k.S) + k.W - 1) / k.W * k.W;
  return {per, (tiles + per - 1) / per};
}
// The fair share: a wave's lanes add the sequences.
__device__ __forceinline__ int kv4_fair(const Kv4Cache &c, int rows, const Cut &k) {
  int sum = 0;
  if (c.n_seq == 1) {
    sum = kv4_tiles(kv4_filled(c, 0, rows), rows);
  } else {
    for (int s = threadIdx.x & 63; s < c.n_seq; s += 64) sum += kv4_tiles(kv4_filled(c, s, rows), rows);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    sum = __builtin_amdgcn_readfirstlane(sum);
  }
  return (int)(((int64_t)sum * c.nkv + k.wgs - 1) / k.wgs);
}
// Workgroup `item` of the call: sequences in order, within one the splits in order, each for
// every KV head.  Only the last workgroups of a launch are left without an item, so that the
// dies, which take workgroups in turn, get the same number of items.
struct Item {
  int s, kvh, split, filled;
  Splits sp;
};
__device__ __forceinline__ bool kv4_item(const Kv4Cache &c, int rows, int item, const Cut &k,
                                         Item &it) {
  const int fair = kv4_fair(c, rows, k);
  if (c.n_seq == 1) {
    it.s = 0;
    it.filled = kv4_filled(c, 0, rows);
    it.sp = kv4_splits(kv4_tiles(it.filled, rows), fair, k);
    it.split = item / c.nkv;
    it.kvh = item - it.split * c.nkv;
    return it.filled >= 0 && it.split < it.sp.n;
  }
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
    const int filled = s0 + lane < c.n_seq ? kv4_filled(c, s0 + lane, rows) : -1;
    const Splits sp = kv4_splits(kv4_tiles(filled, rows), fair, k);
    int run = sp.n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(run, o);
      if (lane >= o) run += x;
    }
    const uint64_t hit = __ballot(item < (before + run) * c.nkv);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      it.s = s0 + at;
      it.filled = __builtin_amdgcn_readlane(filled, at);
      it.sp.per = __builtin_amdgcn_readlane(sp.per, at);
      it.sp.n = __builtin_amdgcn_readlane(sp.n, at);
      const int first = before + __builtin_amdgcn_readlane(run, at) - it.sp.n;
      it.split = (item - first * c.nkv) / c.nkv;
      it.kvh = item - first * c.nkv - it.split * c.nkv;
      return true;
    }
    before += __builtin_amdgcn_readlane(run, 63);
  }
  return false;
}

// The stride of a query row's scores: an odd number of 256-byte lines, so that the rows that
// workgroups write side by side do not fall on one memory channel.
__host__ __device__ __forceinline__ int64_t score_stride(int slots) {
  return (int64_t)(((slots + 63) / 64) | 1) * 64;
}

// 4-bit codes as f16 integers: bits 0-3 and 16-19 of w give code - 8 (1024 + code, less 1032),
// bits 4-7 and 20-23 give 16 (code - 8) (1024 + 16 code, less 1152) without a shift.  `magic`
// holds 1024.0 twice in a vector register, so that mask and OR are one instruction.  The
// offset goes before the matrix core: left to the sums (as -8 sum q, or -8 sum w at the end) it
// costs them low bits (scores: 1.0e-6 in log2 units against 4e-7 of a plain f32 product).
template <int SCALE>
__device__ __forceinline__ half2_t codes2(uint32_t w, uint32_t magic) {
  const half2_t c = __builtin_bit_cast(half2_t, (w & (0x000F000Fu * SCALE)) | magic);
  return c - half2_t{(half_t)(1024.f + 8.f * SCALE), (half_t)(1024.f + 8.f * SCALE)};
}
// A word of K: elements 0, 2, 1, 3, then 16 times elements 4, 6, 5, 7.
__device__ __forceinline__ half8_t k_frag(uint32_t w, uint32_t magic) {
  const uint32_t h = w >> 8;
  const half2_t r[4] = {codes2<1>(w, magic), codes2<1>(h, magic), codes2<16>(w, magic),
                        codes2<16>(h, magic)};
  return __builtin_bit_cast(half8_t, r);
}
// Two words of V (h: 8 bits on): slots 0, 2, 1, 3 of both.
template <int SCALE>
__device__ __forceinline__ half8_t v_frag(uint32_t w0, uint32_t h0, uint32_t w1, uint32_t h1,
                                          uint32_t magic) {
  const half2_t r[4] = {codes2<SCALE>(w0, magic), codes2<SCALE>(h0, magic),
                        codes2<SCALE>(w1, magic), codes2<SCALE>(h1, magic)};
  return __builtin_bit_cast(half8_t, r);
}
__device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// x * (float)h in one instruction: a product alone is converted and multiplied in two, and one
// that is added to something would be fused into that.
__device__ __forceinline__ float mul_f16(float x, half_t h) { return fmaf(x, (float)h, 0.f); }

// x and y in f16 parts hi + lo, both to nearest: what is left is under 2^-22 of them.  `minus1` is
// -1 in a scalar register, which has the low parts made in one instruction each.
__device__ __forceinline__ void split_f16(float x, float y, float minus1, half2_t &hi,
                                          half2_t &lo) {
  uint32_t h = __builtin_bit_cast(uint32_t, half2_t{(half_t)x, (half_t)y});
  asm("" : "+v"(h));  // else x and y are each rounded once more for the low parts
  hi = __builtin_bit_cast(half2_t, h);
  lo = half2_t{(half_t)fmaf((float)hi[0], minus1, x), (half_t)fmaf((float)hi[1], minus1, y)};
}

// v plus that of the lane N to the left in its 16, cyclically.
template <int N>
__device__ __forceinline__ float ror16(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xF, 0xF, true));
}
template <int N>
__device__ __forceinline__ float add_ror16(float v) {
  return v + ror16<N>(v);
}

template <int N>
__device__ __forceinline__ float max_ror16(float v) {
  return fmaxf(v, ror16<N>(v));
}

// The one new row of a decode step, in LDS: K and V code bytes and scales.
template <int HD>
struct FreshRow {
  using L = Kv4<HD>;
  static constexpr int NB = L::NB;
  __align__(16) uint8_t code[2][HD / 2];
  half_t scale[2][NB];
  // Made by HD / 4 lanes each (rq) for K (unit 0) and V (unit 1); stored in the cache if `writes`.
  __device__ __forceinline__ void make(const Kv4Cache &c, Kv4Row<HD> &row, int unit, int rq,
                                       uint8_t *base, int64_t list, int slot, int32_t pos,
                                       bool writes) {
    uint32_t word;
    half_t d;
    kv4_quantize<HD>(row, rq, unit == 0, word, d);
    const int j = slot % kKv4Tile, blk = rq >> 3;
    uint8_t *to = base + (int64_t)(slot / kKv4Tile) * L::TB;
    if (unit == 0 && !(rq & 1)) {
      const int at = (((rq >> 1) & 3) * NB + blk) * 4;
      *(uint32_t *)(code[0] + at) = word;
      if (writes) *(uint32_t *)(to + j * (HD / 2) + at) = word;
    } else if (unit == 1 && (rq & 7) < 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (4 * (rq & 3) + i) * NB + blk;
        code[1][at] = (uint8_t)(word >> (8 * i));
        if (writes) to[L::VO + (j >> 2) * (2 * HD) + at * 4 + (j & 3)] = (uint8_t)(word >> (8 * i));
      }
    }
    if (unit < 2 && !(rq & 7)) {
      scale[unit][blk] = d;
      if (writes) *(half_t *)(to + (unit ? L::VS : L::KS) + ((j >> 2) * NB + blk) * 8 + (j & 3) * 2) = d;
    }
    if (writes && unit == 1 && rq == 0) {
      if (c.positions) c.positions[list * c.slots + slot] = pos;
      if (c.weights) c.weights[list * c.slots + slot] = 0.f;
    }
  }
  // Scale of slot j in the four that w holds.  By value: a reference to one of the two words would
  // put registers in memory.
  __device__ __forceinline__ static void put(uint2 &w, int j, half_t d) {
    const int sh = 16 * (j & 1);
    const uint32_t keep = ~(0xFFFFu << sh), n = (uint32_t)__builtin_bit_cast(uint16_t, d) << sh;
    if (j & 2)
      w.y = (w.y & keep) | n;
    else
      w.x = (w.x & keep) | n;
  }
};

// What a wave reads of a tile.  Lane (r = lane % 16, g = lane / 16), halves t = 0, 1: K codes of
// slot 16 t + r, channels 32 b + 8 g + 0..7 of every block b; V codes of slots 16 t + 4 g + 0..3,
// channels 32 b + r and 32 b + 16 + r; scales of those four slots, block r / HPS.
template <int HD>
struct TileRegs {
  static constexpr int NB = HD / 32;
  uint32_t k[2][NB], v[2][NB];
  uint2 ks[2], vs[2];
  __device__ __forceinline__ void load_k(const uint8_t *tile, int r, int g, int b) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      words(tile + (uint32_t)((16 * t + r) * (HD / 2) + g * NB * 4), k[t]);
      const uint8_t *sp = tile + (uint32_t)(Kv4<HD>::KS + ((4 * t + g) * NB + b) * 8);
      ks[t] = *(const uint2 *)sp;
      vs[t] = *(const uint2 *)(sp + 2 * HD);
    }
  }
  __device__ __forceinline__ void load_v(const uint8_t *tile, int r, int g) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      words(tile + (uint32_t)(Kv4<HD>::VO + (4 * t + g) * (2 * HD) + r * NB * 4), v[t]);
    }
  }
  // Slot j's codes from its bytes.
  __device__ __forceinline__ void patch_codes(const FreshRow<HD> &f, int j, int r, int g) {
    const int sh = 8 * (j & 3);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (j == 16 * t + r)
#pragma unroll
        for (int i = 0; i < NB; ++i) k[t][i] = *(const uint32_t *)(f.code[0] + (g * NB + i) * 4);
      if (j >> 2 == 4 * t + g)
#pragma unroll
        for (int i = 0; i < NB; ++i)
          v[t][i] = (v[t][i] & ~(0xFFu << sh)) | ((uint32_t)f.code[1][r * NB + i] << sh);
    }
  }
  __device__ __forceinline__ void patch(const FreshRow<HD> &f, int j, int r, int g, int b) {
    patch_codes(f, j, r, g);
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (j >> 2 == 4 * t + g) {
        FreshRow<HD>::put(ks[t], j, f.scale[0][b]);
        FreshRow<HD>::put(vs[t], j, f.scale[1][b]);
      }
  }
  static __device__ __forceinline__ void words(const uint8_t *p, uint32_t (&w)[NB]) {
    if constexpr (NB == 2) {
      const uint2 x = *(const uint2 *)p;
      w[0] = x.x, w[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < NB / 4; ++i) {
        const uint4 x = ((const uint4 *)p)[i];
        w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
      }
    }
  }
};

// For few query rows.  A workgroup takes one list, one range of its tiles and HPS = 512 / HD
// query rows; its waves take the range's tiles in turn and join at the end.  Nothing but
// registers carries a tile through:
// - Scores: v_mfma_f32_16x16x32_f16 with the slots' codes as A (one K step is one block of 32
//   channels) and the queries as B.  A block's sum has to be multiplied by the slot's scale of
//   that block before the blocks are added, so column HPS b + h of B holds query row h in block
//   b's K step and zero in the others: one accumulator holds every block's sum of HPS rows.
//   Each lane multiplies by its block's scales; rotations within 16 lanes add the blocks,
//   leaving the score in each.
// - Queries are scaled by a power of two per row and enter as two f16 parts (22 bits), twice
//   the MFMAs: the scores are f32-grade.  The operands, three quarters of them zeros at 128
//   channels, are made once per workgroup and read from LDS each turn: in registers they would
//   cost a wave per SIMD.
// - Output: the scores' accumulator layout (lane: slots 4 g + 0..3 of column r) is the A layout
//   of P . V when K index j of lane group g means slot 4 g + j % 4 of half j / 4; V is stored
//   so that a lane's words hold these slots.  Row HPS b + h of A is p * (scale of V's block b)
//   of query row h, so the scales need no pass of their own; only the channels of block b of
//   that row's output are used.  p * scale enters as two f16 parts.
// - Each row's p is 2^(score - m) with a running m, so that p * scale is at most 2^10 when m is
//   set and stays below 2^14 in f16, whatever V's range; where a tile passes that (or p 2^100:
//   scales of zero), m is raised to the largest score + log2 |scale| (the float's bits read as a
//   number, within 0.09) and the sums are scaled down.  That is rare after the first tiles.  A
//   scale of zero counts as 2^-84, so that a slot of zeros far above the others takes no bits
//   from them and p's sum stays a float.
// - K's registers take the next tile as soon as its scores are made, V's after its products:
//   one tile in flight per wave, four waves per SIMD.
// Bound: HBM (9/8 head_dim bytes per slot and list) and, close behind, vector instructions, most
// of them on the codes.  130000 slots of 8 lists, 128 channels, 150 MB: 33-36 us, 4.2-4.5 TB/s with
// the vector unit busy 72 % of the time; short lists are bound by their start (6000 slots: 7.8 us,
// of which 4.5 before the first tile is used).
template <int HD, int W, int WPS>
__global__ __launch_bounds__(64 * W, WPS) void kv4_attention_kernel(Kv4Cache c, Kv4Attn a,
                                                               float *__restrict__ rec,
                                                               float2 *__restrict__ lse,
                                                               float *__restrict__ scores, Cut cut,
                                                               bool store) {
  using L = Kv4<HD>;
  constexpr int NB = L::NB, HPS = 16 / NB, half = HD / 2, RS = record_floats<HD>();
  constexpr float kLift = 10.f, kMostW = 16384.f, kMostP = 0x1p100f;
  __shared__ float lo_[W][512];      // per wave: HPS rows of HD sums
  __shared__ float2 lm[W][16];       // and the 16 rows' (m, sum of p)
  __shared__ half8_t q_[NB][2][64];  // queries: per block, hi and lo part, a B operand
  __shared__ float qc[16];           // per row: log2 units per unit of a score
  __shared__ FreshRow<HD> fresh;
  Item it;
  if (!kv4_item(c, a.rows, blockIdx.x, cut, it)) return;
  it.s = __builtin_amdgcn_readfirstlane(it.s);  // all known uniform from here on
  it.kvh = __builtin_amdgcn_readfirstlane(it.kvh);
  it.split = __builtin_amdgcn_readfirstlane(it.split);
  it.filled = __builtin_amdgcn_readfirstlane(it.filled);
  it.sp.per = __builtin_amdgcn_readfirstlane(it.sp.per);
  it.sp.n = __builtin_amdgcn_readfirstlane(it.sp.n);
  const int64_t s = it.s, list = s * c.nkv + it.kvh;
  const int kvh = it.kvh, grp = c.nh / c.nkv, V = a.rows * grp, filled = it.filled;
  const Splits sp = it.sp;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // known uniform: scalar addresses
  const int b = r / HPS, h = r % HPS;
  const int tile0 = it.split * sp.per, tile1 = min(tile0 + sp.per, kv4_tiles(filled, a.rows));
  uint8_t *base = kv4_list(c.kv, list, c.slots, L::TB);
  const int v0 = blockIdx.z * HPS;
  // the workgroups whose range has the one new row (a call of more rows stores them beforehand)
  // make its bytes in LDS, for the wave whose first tile lacks them; those of the first group of
  // query rows store them
  const bool stores = store && filled / kKv4Tile >= tile0 && filled / kKv4Tile < tile1;
  const float *row0 = a.qkv + s * a.rows * a.ldq;  // the sequence's first row
  const float *kx = row0 + (int64_t)(c.nh + kvh) * HD, *vx = kx + (int64_t)c.nkv * HD;
  const int64_t pos0 = c.pos[s];

  // What comes before the barrier is requested before the tile, since loads return in order:
  // behind a full chip's tiles the queries took 5.6 us (130000 slots).
  float4 xo[2], xp[2], cv[2], sv[2];  // wave 0: the queries, lane (r, g) channels
                                      // 32 b + 8 g + 0..7 of its row
  constexpr int LANES = Kv4Row<HD>::LANES, STORERS = HD == 256 ? 2 : 1;
  Kv4Row<HD> row;  // waves 1 ..: the new row's K (unit 0) and V (1), HD / 4 lanes each
  const int unit = (wave - 1) * (64 / LANES) + lane / LANES, rq = lane % LANES;
  if (wave == 0) {
    const int v = v0 + h, i = v < V ? v / grp : 0;
    const float *x = row0 + i * a.ldq + (int64_t)(kvh * grp + (v < V ? v % grp : 0)) * HD;
    const int e0 = 32 * b + 8 * g, ep = b < NB / 2 ? e0 + half : e0 - half;
    const int64_t p = (pos0 + i) * half + (b < NB / 2 ? e0 : ep);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      xo[j] = *(const float4 *)(x + e0 + 4 * j);
      xp[j] = *(const float4 *)(x + ep + 4 * j);
      cv[j] = *(const float4 *)(c.cs + p + 4 * j);
      sv[j] = *(const float4 *)(c.sn + p + 4 * j);
    }
  } else if (stores && wave < 1 + STORERS && unit < 2) {
    row.load(unit ? vx : kx, rq);
    row.load_turn(c.cs + pos0 * half, c.sn + pos0 * half, rq);
  }
  __builtin_amdgcn_sched_barrier(0);
  TileRegs<HD> d;
  // from the last tile down: the new row's is some wave's first
  int tile = tile1 - 1 - wave;
  if (tile >= tile0) {
    d.load_k(base + (int64_t)tile * L::TB, r, g, b);
    d.load_v(base + (int64_t)tile * L::TB, r, g);
  }
  __builtin_amdgcn_sched_barrier(0);
  if (wave == 0) {
    const bool on = v0 + h < V;  // past the last query row: zeros
    const float sign = b < NB / 2 ? -1.f : 1.f;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float o = (&xo[j >> 2].x)[j & 3], t = (&xp[j >> 2].x)[j & 3];
      const float x = on ? o * (&cv[j >> 2].x)[j & 3] + sign * (t * (&sv[j >> 2].x)[j & 3]) : 0.f;
      y[j] = fmaf(x, ScoreScale<HD>::hi, x * ScoreScale<HD>::lo);
    }
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(y[j]));
    if constexpr (NB > 4) mx = max_ror16<2>(mx);
    if constexpr (NB > 2) mx = max_ror16<4>(mx);
    mx = max_xor32(max_xor16(max_ror16<8>(mx)));
    const int e = stage_exp(mx);
    const float up = pow2f(e);
    half8_t hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // in the codes' order, and those that enter 16-fold over 16
      const int k = (j & 4) | (j & 1) << 1 | (j & 2) >> 1;
      const float t = y[k] * (j < 4 ? up : up * 0.0625f);
      hi[j] = (half_t)t;
      lo[j] = (half_t)(t - (float)hi[j]);
    }
    if (g == 0) qc[r] = pow2f(-e);
    const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      q_[k][0][lane] = b == k ? hi : zero;
      q_[k][1][lane] = b == k ? lo : zero;
    }
  } else if (stores && wave < 1 + STORERS) {
    fresh.make(c, row, unit, rq, base, list, filled, (int32_t)pos0, blockIdx.z == 0);
  }
  __syncthreads();
  const float f = qc[r];  // log2 units per accumulated unit
  const int vis = filled + (v0 + h < V ? (v0 + h) / grp : 0) + 1;  // slots that the row sees
  const int all_see = filled + v0 / grp + 1;  // slots that every row of the workgroup sees

  float4_t acc[2 * NB];
  float m = -INFINITY, l = 0.f;  // p = 2^(score - m)
#pragma unroll
  for (int t = 0; t < 2 * NB; ++t) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};

  uint32_t magic;
  asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(magic));
  float minus1 = -1.f;  // not known to be: x - (float)h stays one fused instruction
  asm volatile("" : "+s"(minus1));
  if (stores && tile == filled / kKv4Tile) d.patch(fresh, filled % kKv4Tile, r, g, b);
  int ql = lane;  // made anew every turn: the queries are read from LDS there, not kept
  for (; tile >= tile0; tile -= W) {
    const uint8_t *next = base + (int64_t)max(tile - W, tile0) * L::TB;  // the last one: unused
    const int slot0 = tile * kKv4Tile + 4 * g;  // of half 0, i = 0
    asm volatile("" : "+v"(ql));
    float y[8];  // scores / f
    {
      float4_t sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const half8_t k0 = k_frag(d.k[0][k], magic), k1 = k_frag(d.k[1][k], magic);
        const half8_t hi = q_[k][0][ql], lo = q_[k][1][ql];
        sc[0] = mfma(k0, hi, sc[0]);
        sc[1] = mfma(k1, hi, sc[1]);
        sc[0] = mfma(k0, lo, sc[0]);
        sc[1] = mfma(k1, lo, sc[1]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const half_t ks = __builtin_bit_cast(half4_t, d.ks[i >> 2])[i & 3];
        float x = mul_f16(sc[i >> 2][i & 3], ks);
        x = add_ror16<8>(x);
        if constexpr (NB > 2) x = add_ror16<4>(x);
        if constexpr (NB > 4) x = add_ror16<2>(x);
        y[i] = x;
      }
    }
    const half4_t dv[2] = {__builtin_bit_cast(half4_t, d.vs[0]), __builtin_bit_cast(half4_t, d.vs[1])};
    d.load_k(next, r, g, b);
    if (scores) {
      float z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = y[i] * f;
      if (r < HPS && v0 + r < V) {
        float *o = scores + (list * V + v0 + r) * score_stride(c.slots) + slot0;
        *(float4 *)o = make_float4(z[0], z[1], z[2], z[3]);
        *(float4 *)(o + 16) = make_float4(z[4], z[5], z[6], z[7]);
      }
    }
    const bool masked = (tile + 1) * kKv4Tile > all_see;
    float p[8], w[8], sum, most;
    auto hidden = [&](int i) { return slot0 + (i < 4 ? i : 12 + i) >= vis; };
    auto weigh = [&]() {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(y[i], f, -m));
        w[i] = mul_f16(p[i], dv[i >> 2][i & 3]);
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (hidden(i)) p[i] = w[i] = 0.f;
      }
      sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      most = fabsf(w[0]);
#pragma unroll
      for (int i = 1; i < 7; i += 2) most = fmaxf(fmaxf(most, fabsf(w[i])), fabsf(w[i + 1]));
      most = fmaxf(most, fabsf(w[7]));
    };
    weigh();
    if (__any(most > kMostW || sum > kMostP)) {
      float n = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t bits = __float_as_uint((float)dv[i >> 2][i & 3]) & 0x7FFFFFFFu;
        const float lg =  // zero: as 2^-84
            fmaf((float)(int)(bits < 0x15800000u ? 0x15800000u : bits), 0x1p-23f, -127.f - kLift);
        if (!masked || !hidden(i)) n = fmaxf(n, fmaf(y[i], f, lg));
      }
      n = max_xor16(n);
      n = max_xor32(n);
      const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - n);
      m = n;
      l *= al;
      float ar[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ar[i] = __shfl(al, 4 * g + i);
#pragma unroll
      for (int t = 0; t < 2 * NB; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] *= ar[i];
      weigh();
    }
    l += sum;
    half2_t hp[4], lp[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // V's pairs: slots (0, 2), (1, 3) of each half
      const int i = (k & 1) + (k >> 1) * 4;
      split_f16(w[i], w[i + 2], minus1, hp[k], lp[k]);
    }
    const half8_t wh = __builtin_bit_cast(half8_t, hp), wl = __builtin_bit_cast(half8_t, lp);
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const uint32_t w0 = d.v[0][k], h0 = w0 >> 8, w1 = d.v[1][k], h1 = w1 >> 8;
      const half8_t va = v_frag<1>(w0, h0, w1, h1, magic);
      const half8_t vb = v_frag<16>(w0, h0, w1, h1, magic);  // channels 16..31 of the block
      acc[2 * k] = mfma(wh, va, acc[2 * k]);
      acc[2 * k + 1] = mfma(wh, vb, acc[2 * k + 1]);
      acc[2 * k] = mfma(wl, va, acc[2 * k]);
      acc[2 * k + 1] = mfma(wl, vb, acc[2 * k + 1]);
    }
    d.load_v(next, r, g);
  }

  // the waves' sums: lane (r, g), register i holds row 4 g + i, channel 16 t + r
  float sum = sum_xor32(sum_xor16(l));
  if (g == 0) lm[wave][r] = make_float2(m, sum);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * g + i, rb = row / HPS;
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t)
      if (rb == t / 2)
        lo_[wave][row % HPS * HD + 16 * t + r] = acc[t][i] * (t & 1 ? 0.0625f : 1.f);
  }
  __syncthreads();
  float *out = rec + (list * cut.S + it.split) * V * RS;
  for (int e = tid; e < 512; e += 64 * W) {
    const int hh = e / HD, ch = e & (HD - 1), row = (ch >> 5) * HPS + hh;
    const int v = v0 + hh;
    if (v >= V) continue;
    float mx = lm[0][row].x, o = 0.f, ls = 0.f;
#pragma unroll
    for (int k = 1; k < W; ++k) mx = fmaxf(mx, lm[k][row].x);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float2 ml = lm[k][row];
      const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
      o = fmaf(w, lo_[k][e], o);
      ls = fmaf(w, ml.y, ls);
    }
    if (sp.n == 1) {  // nothing to join
      a.out[(s * a.rows + v / grp) * a.ldo + (kvh * grp + v % grp) * HD + ch] = o / ls;
      if (lse && ch == 0) lse[list * V + v] = make_float2(mx, 1.f / ls);
    } else {
      out[v * RS + ch] = o;
      if ((ch & 31) == 0) *(float2 *)(out + v * RS + HD + 2 * (ch >> 5)) = make_float2(mx, ls);
    }
  }
}

// Waves of a workgroup of kv4_rows_kernel (measured at plan()).
template <int HD>
constexpr int kRowsWaves = HD == 256 ? 4 : 8;

// The same for many query rows: NS groups of 16, a column each.  Every block's scores are a product
// of their own, multiplied by the slots' scales as they are added, and P times V's scales is made
// for every block.  So a lane holds all blocks' scales of its slots (32 registers at 128 channels
// where the kernel above has 8), but every column is a row of its own: a quarter of the MFMAs and
// exponentials per row at 128 channels, an eighth at 256.
// The largest |p * scale| is bounded by the largest p times the largest |scale| of the lane's
// slots; where m is raised for it, by each slot's own.  m is that of all blocks: p * scale of a
// block whose scales are under 2^-13 of the others' falls below 2^-3, where two f16 parts hold
// fewer bits (2^-25 absolute: 2^-35 of the row's largest).
// Bound: vector instructions (76 % busy, and the matrix cores 21 %), about 150 for a tile's codes
// and 230 for each group of rows (128 channels).  32 rows of 32 / 8 heads over 20000 slots: 47 us,
// 10.5 GFLOP of products in two parts each; the kernel for few rows took about 95.
template <int HD, int NS>
__global__ __launch_bounds__(64 * kRowsWaves<HD>, 2) void kv4_rows_kernel(Kv4Cache c, Kv4Attn a,
                                                          float *__restrict__ rec,
                                                          float2 *__restrict__ lse,
                                                          float *__restrict__ scores, Cut cut,
                                                          bool store) {
  using L = Kv4<HD>;
  constexpr int W = kRowsWaves<HD>, NB = L::NB, half = HD / 2, RS = record_floats<HD>();
  constexpr float kLift = 10.f, kMostW = 16384.f, kMostP = 0x1p100f;
  // Queries (per block, hi and lo part, a B operand) while tiles are read, then the waves' sums, 16
  // rows of HD per group: 64 KB for four waves, 128 for eight, so that eight waves fit a CU.
  __shared__ union {
    half8_t q[NS][NB][2][64];
    float o[W][NS][16 * HD];
  } sh;
  auto &q_ = sh.q;
  auto &lo_ = sh.o;
  __shared__ float2 lm[W][NS][16];             // the rows' (m, sum of p)
  __shared__ float qc[NS][16];                 // per row: log2 units per unit of a score
  __shared__ FreshRow<HD> fresh;
  Item it;
  if (!kv4_item(c, a.rows, blockIdx.x, cut, it)) return;
  it.s = __builtin_amdgcn_readfirstlane(it.s);  // all known uniform from here on
  it.kvh = __builtin_amdgcn_readfirstlane(it.kvh);
  it.split = __builtin_amdgcn_readfirstlane(it.split);
  it.filled = __builtin_amdgcn_readfirstlane(it.filled);
  it.sp.per = __builtin_amdgcn_readfirstlane(it.sp.per);
  it.sp.n = __builtin_amdgcn_readfirstlane(it.sp.n);
  const int64_t s = it.s, list = s * c.nkv + it.kvh;
  const int kvh = it.kvh, grp = c.nh / c.nkv, V = a.rows * grp, filled = it.filled;
  const Splits sp = it.sp;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile0 = it.split * sp.per, tile1 = min(tile0 + sp.per, kv4_tiles(filled, a.rows));
  uint8_t *base = kv4_list(c.kv, list, c.slots, L::TB);
  const int v0 = blockIdx.z * NS * 16;
  const bool stores = store && filled / kKv4Tile >= tile0 && filled / kKv4Tile < tile1;
  const float *row0 = a.qkv + s * a.rows * a.ldq;
  const float *kx = row0 + (int64_t)(c.nh + kvh) * HD, *vx = kx + (int64_t)c.nkv * HD;
  const int64_t pos0 = c.pos[s];
  TileRegs<HD> d;               // codes; the scales of every block apart
  uint2 ks[2][NB], vs[2][NB];   // of slots 16 t + 4 g + 0..3
  auto load_scales = [&](const uint8_t *tile) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int k = 0; k < NB; k += 2) {
        const uint8_t *p = tile + (uint32_t)(L::KS + ((4 * t + g) * NB + k) * 8);
        const uint4 x = *(const uint4 *)p, y = *(const uint4 *)(p + 2 * HD);
        ks[t][k] = make_uint2(x.x, x.y), ks[t][k + 1] = make_uint2(x.z, x.w);
        vs[t][k] = make_uint2(y.x, y.y), vs[t][k + 1] = make_uint2(y.z, y.w);
      }
  };
  auto load_k = [&](const uint8_t *tile) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
      TileRegs<HD>::words(tile + (uint32_t)((16 * t + r) * half + g * NB * 4), d.k[t]);
  };
  // from the last tile down: the new row's is some wave's first
  int tile = tile1 - 1 - wave;
  if (wave < NS) {
    // queries of group `wave`: lane (r, g) holds channels 32 k + 8 g + 0..7 of row r, every block k
    const int v = v0 + wave * 16 + r, i = v < V ? v / grp : 0;
    const float *x = row0 + i * a.ldq + (int64_t)(kvh * grp + (v < V ? v % grp : 0)) * HD + 8 * g;
    const int64_t p = (pos0 + i) * half + 8 * g;
    float y[NB][8], mx = 0.f;
#pragma unroll
    for (int k = 0; k < NB / 2; ++k)
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 x0 = *(const float4 *)(x + 32 * k + j), x1 = *(const float4 *)(x + half + 32 * k + j);
        const float4 cv = *(const float4 *)(c.cs + p + 32 * k + j);
        const float4 sv = *(const float4 *)(c.sn + p + 32 * k + j);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float e = (&x0.x)[n], o = (&x1.x)[n], cc = (&cv.x)[n], ss = (&sv.x)[n];
          const float e1 = e * cc - o * ss, o1 = o * cc + e * ss;
          y[k][j + n] = v < V ? fmaf(e1, ScoreScale<HD>::hi, e1 * ScoreScale<HD>::lo) : 0.f;
          y[k + NB / 2][j + n] = v < V ? fmaf(o1, ScoreScale<HD>::hi, o1 * ScoreScale<HD>::lo) : 0.f;
        }
      }
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(y[k][j]));
    const int e = stage_exp(max_xor32(max_xor16(mx)));
    const float up = pow2f(e);
    if (g == 0) qc[wave][r] = pow2f(-e);
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      half8_t hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // in the codes' order, and those that enter 16-fold over 16
        const float t = y[k][(j & 4) | (j & 1) << 1 | (j & 2) >> 1] * (j < 4 ? up : up * 0.0625f);
        hi[j] = (half_t)t;
        lo[j] = (half_t)(t - (float)hi[j]);
      }
      q_[wave][k][0][lane] = hi;
      q_[wave][k][1][lane] = lo;
    }
  } else if (stores && wave >= NS && wave < NS + (HD == 256 ? 2 : 1)) {
    constexpr int LANES = Kv4Row<HD>::LANES;  // the new row's K (unit 0) and V (1)
    const int unit = (wave - NS) * (64 / LANES) + lane / LANES, rq = lane % LANES;
    Kv4Row<HD> row;
    row.load(unit ? vx : kx, rq);
    row.load_turn(c.cs + pos0 * half, c.sn + pos0 * half, rq);
    fresh.make(c, row, unit, rq, base, list, filled, (int32_t)pos0, blockIdx.z == 0);
  }
  if (tile >= tile0) {
    const uint8_t *p = base + (int64_t)tile * L::TB;
    load_k(p);
    load_scales(p);
    d.load_v(p, r, g);
  }
  __syncthreads();
  if (stores && tile == filled / kKv4Tile) {
    const int j = filled % kKv4Tile;
    d.patch_codes(fresh, j, r, g);
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (j >> 2 == 4 * t + g) {
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          FreshRow<HD>::put(ks[t][k], j, fresh.scale[0][k]);
          FreshRow<HD>::put(vs[t][k], j, fresh.scale[1][k]);
        }
      }
  }
  float f[NS];
  int vis[NS];  // slots that row r of the group sees
#pragma unroll
  for (int u = 0; u < NS; ++u) {
    f[u] = qc[u][r];
    const int v = v0 + u * 16 + r;
    vis[u] = filled + (v < V ? v / grp : 0) + 1;
  }
  const int all_see = filled + v0 / grp + 1, end = filled + a.rows;

  float4_t acc[NS][2 * NB];
  float m[NS], l[NS];  // p = 2^(score - m)
#pragma unroll
  for (int u = 0; u < NS; ++u) {
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t) acc[u][t] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  uint32_t magic;
  asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(magic));
  float minus1 = -1.f;
  asm volatile("" : "+s"(minus1));
  int ql = lane;
  auto at = [](const uint2 &w, int i) { return __builtin_bit_cast(half4_t, w)[i]; };
  for (; tile >= tile0; tile -= W) {
    const uint8_t *next = base + (int64_t)max(tile - W, tile0) * L::TB;  // the last one: unused
    const int slot0 = tile * kKv4Tile + 4 * g;
    const bool masked = (tile + 1) * kKv4Tile > all_see;
    asm volatile("" : "+v"(ql));
    float y[NS][8];  // scores / f
    // the wave that is at its matrix products goes first, the other fills the gaps (window of 32
    // rows over 20000 slots, without weights: 53.3 us without, 51.2 so)
    __builtin_amdgcn_s_setprio(1);
    float4_t sc[2][NS][2];
#pragma unroll
    for (int k = 0; k <= NB; ++k) {
      if (k < NB) {
        const half8_t k0 = k_frag(d.k[0][k], magic), k1 = k_frag(d.k[1][k], magic);
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          const half8_t hi = q_[u][k][0][ql], lo = q_[u][k][1][ql];
          const float4_t z = {0.f, 0.f, 0.f, 0.f};
          sc[k & 1][u][0] = mfma(k0, lo, mfma(k0, hi, z));
          sc[k & 1][u][1] = mfma(k1, lo, mfma(k1, hi, z));
        }
      }
      // a block's products are added while the next one's are made; no further ahead, which would
      // take more registers than there are
      if (k > 0)
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            y[u][i] = fmaf(sc[(k - 1) & 1][u][i >> 2][i & 3], (float)at(ks[i >> 2][k - 1], i & 3),
                           k > 1 ? y[u][i] : 0.f);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    load_k(next);
    if (scores) {
#pragma unroll
      for (int u = 0; u < NS; ++u)
        if (v0 + u * 16 + r < V) {
          float *o = scores + (list * V + v0 + u * 16 + r) * score_stride(c.slots) + slot0;
          *(float4 *)o = make_float4(y[u][0] * f[u], y[u][1] * f[u], y[u][2] * f[u], y[u][3] * f[u]);
          *(float4 *)(o + 16) =
              make_float4(y[u][4] * f[u], y[u][5] * f[u], y[u][6] * f[u], y[u][7] * f[u]);
        }
    }
    if (masked) {  // slots that no row sees hold anything: scales of zero for V
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int n = end - (slot0 + 16 * t);  // of the four, the first n
        const uint32_t x = n > 1 ? ~0u : (n == 1 ? 0xFFFFu : 0u);
        const uint32_t z = n > 3 ? ~0u : (n == 3 ? 0xFFFFu : 0u);
#pragma unroll
        for (int k = 0; k < NB; ++k) vs[t][k].x &= x, vs[t][k].y &= z;
      }
    }
    // the largest |scale| of the lane's slots: f16 magnitudes compare as integers
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = {0, 0};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, vs[t][k].x & 0x7FFF7FFFu));
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, vs[t][k].y & 0x7FFF7FFFu));
      }
    const uint16_t tops = top[0] > top[1] ? top[0] : top[1];
    const float dm = (float)__builtin_bit_cast(half_t, tops);
    float p[NS][8];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      auto hidden = [&](int i) { return slot0 + (i < 4 ? i : 12 + i) >= vis[u]; };
      float sum, most;
      auto weigh = [&]() {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[u][i] = __builtin_amdgcn_exp2f(fmaf(y[u][i], f[u], -m[u]));
        if (masked) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (hidden(i)) p[u][i] = 0.f;
        }
        sum = ((p[u][0] + p[u][1]) + (p[u][2] + p[u][3])) + ((p[u][4] + p[u][5]) + (p[u][6] + p[u][7]));
        most = p[u][0];
#pragma unroll
        for (int i = 1; i < 7; i += 2) most = fmaxf(fmaxf(most, p[u][i]), p[u][i + 1]);
        most = fmaxf(most, p[u][7]) * dm;
      };
      weigh();
      if (__any(!(most <= kMostW) || sum > kMostP)) {
        float n = m[u];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint32_t bits = 0x15800000u;  // zeros: 2^-84
#pragma unroll
          for (int k = 0; k < NB; ++k) {
            const uint32_t x = __float_as_uint((float)at(vs[i >> 2][k], i & 3)) & 0x7FFFFFFFu;
            bits = x > bits ? x : bits;
          }
          const float lg = fmaf((float)(int)bits, 0x1p-23f, -127.f - kLift);
          if (!masked || !hidden(i)) n = fmaxf(n, fmaf(y[u][i], f[u], lg));
        }
        n = max_xor16(n);
        n = max_xor32(n);
        const float al = m[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[u] - n);
        m[u] = n;
        l[u] *= al;
        float ar[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ar[i] = __shfl(al, 4 * g + i);
#pragma unroll
        for (int t = 0; t < 2 * NB; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[u][t][i] *= ar[i];
        weigh();
      }
      l[u] += sum;
    }
    auto products = [&](auto some_hidden) {
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const uint32_t w0 = d.v[0][k], h0 = w0 >> 8, w1 = d.v[1][k], h1 = w1 >> 8;
        const half8_t va = v_frag<1>(w0, h0, w1, h1, magic);
        const half8_t vb = v_frag<16>(w0, h0, w1, h1, magic);
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          half2_t hp[4], lp[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) {  // V's pairs: slots (0, 2), (1, 3) of each half
            const int i = (n & 1) + (n >> 1) * 4, t = n >> 1;
            float wa = mul_f16(p[u][i], at(vs[t][k], i & 3));
            float wb = mul_f16(p[u][i + 2], at(vs[t][k], (i & 3) + 2));
            // a slot that this row does not see may hold any scale, infinite too
            if (some_hidden.value && slot0 + 16 * t + (i & 3) >= vis[u]) wa = 0.f;
            if (some_hidden.value && slot0 + 16 * t + (i & 3) + 2 >= vis[u]) wb = 0.f;
            asm("" : "+v"(wa), "+v"(wb));  // else each is made again as it is rounded
            split_f16(wa, wb, minus1, hp[n], lp[n]);
          }
          const half8_t wh = __builtin_bit_cast(half8_t, hp), wl = __builtin_bit_cast(half8_t, lp);
          acc[u][2 * k] = mfma(wh, va, acc[u][2 * k]);
          acc[u][2 * k + 1] = mfma(wh, vb, acc[u][2 * k + 1]);
          acc[u][2 * k] = mfma(wl, va, acc[u][2 * k]);
          acc[u][2 * k + 1] = mfma(wl, vb, acc[u][2 * k + 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    __builtin_amdgcn_s_setprio(1);
    if (masked)
      products(std::true_type{});
    else
      products(std::false_type{});
    __builtin_amdgcn_s_setprio(0);
    load_scales(next);
    d.load_v(next, r, g);
  }

  __syncthreads();  // the last use of the queries is over
  // the waves' sums: lane (r, g), register i holds row 4 g + i, channel 16 t + r
#pragma unroll
  for (int u = 0; u < NS; ++u) {
    const float sum = sum_xor32(sum_xor16(l[u]));
    if (g == 0) lm[wave][u][r] = make_float2(m[u], sum);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < 2 * NB; ++t)
        lo_[wave][u][(4 * g + i) * HD + 16 * t + r] = acc[u][t][i] * (t & 1 ? 0.0625f : 1.f);
  }
  __syncthreads();
  float *out = rec + (list * cut.S + it.split) * V * RS;
  // four channels per thread: the rows' factors are most of the work
  for (int e = tid; e < NS * 4 * HD; e += 64 * W) {
    const int u = e / (4 * HD), row = e / (HD / 4) % 16, ch = e % (HD / 4) * 4, v = v0 + u * 16 + row;
    if (v >= V) break;
    float mx = lm[0][u][row].x, ls = 0.f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 1; k < W; ++k) mx = fmaxf(mx, lm[k][u][row].x);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float2 ml = lm[k][u][row];
      const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
      const float4_t x = *(const float4_t *)&lo_[k][u][row * HD + ch];
#pragma unroll
      for (int n = 0; n < 4; ++n) o[n] = fmaf(w, x[n], o[n]);
      ls = fmaf(w, ml.y, ls);
    }
    if (sp.n == 1) {  // nothing to join
      float *to = a.out + (s * a.rows + v / grp) * a.ldo + (kvh * grp + v % grp) * HD + ch;
#pragma unroll
      for (int n = 0; n < 4; ++n) to[n] = o[n] / ls;
      if (lse && ch == 0) lse[list * V + v] = make_float2(mx, 1.f / ls);
    } else {
      *(float4_t *)(out + v * RS + ch) = o;
      if ((ch & 31) == 0) *(float2 *)(out + v * RS + HD + 2 * (ch >> 5)) = make_float2(mx, ls);
    }
  }
}

// One workgroup per query row of a list with several splits: their records joined, G groups of
// HD / 4 threads taking every G-th record, then the groups in order.  Eight groups, 16 of 64
// channels (us of a call; 6000 slots of 128 channels 11.2, 16 groups 11.8; 4 x 9000 of 256 with 4
// groups 26.5, 8 25.0, 16 24.9).
template <int HD>
constexpr int kMergeThreads = HD < 128 ? 256 : 2 * HD;
template <int HD>
__global__ __launch_bounds__(kMergeThreads<HD>) void kv4_merge_kernel(Kv4Cache c, Kv4Attn a,
                                                             const float *__restrict__ rec,
                                                             float2 *__restrict__ lse, Cut cut) {
  constexpr int RS = record_floats<HD>(), Q = HD / 4, G = kMergeThreads<HD> / Q;
  __shared__ float4 o_[G][Q];
  __shared__ float2 ml_[G][Q];
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int v = blockIdx.x, grp = c.nh / c.nkv, V = a.rows * grp;
  const int q = threadIdx.x % Q, gi = threadIdx.x / Q;
  const int filled = kv4_filled(c, s, a.rows);
  if (filled < 0) return;
  const Splits sp = kv4_splits(kv4_tiles(filled, a.rows), kv4_fair(c, a.rows, cut), cut);
  if (sp.n == 1) return;
  const float *r = rec + (list * cut.S * V + v) * RS;
  const int64_t step = (int64_t)V * RS;
  const int at = HD + 2 * (q / 8);
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto join = [&](float2 ml, float4 x) {
    const float n = fmaxf(m, ml.x);
    const float wo = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - n);
    const float wn = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - n);
    m = n;
    l = l * wo + ml.y * wn;
    o.x = o.x * wo + x.x * wn;
    o.y = o.y * wo + x.y * wn;
    o.z = o.z * wo + x.z * wn;
    o.w = o.w * wo + x.w * wn;
  };
  for (int k0 = gi; k0 < sp.n; k0 += 4 * G) {
    float2 ml[4];
    float4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // past the last: the last again, unused
      const float *rk = r + (int64_t)min(k0 + j * G, sp.n - 1) * step;
      ml[j] = *(const float2 *)(rk + at);
      x[j] = *(const float4 *)(rk + 4 * q);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k0 + j * G < sp.n) join(ml[j], x[j]);
  }
  o_[gi][q] = o;
  ml_[gi][q] = make_float2(m, l);
  __syncthreads();
  if (gi > 0) return;
  for (int k = 1; k < G; ++k) join(ml_[k][q], o_[k][q]);
  *(float4 *)(a.out + (s * a.rows + v / grp) * a.ldo +
              (int64_t)(list % c.nkv * grp + v % grp) * HD + 4 * q) =
      make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
  if (lse && q == 0) lse[list * V + v] = make_float2(m, 1.f / l);
}

// The attention weights of a list's slots: 64 threads of four slots each times eight shares of
// the query rows, whose scores are taken against the rows' maximum and sum (apart: their
// log-sum-exp in one float would lose the low bits); shares joined in order.  Bound: the scores
// read, 82 MB for 128 query rows over 20000 slots in 8 lists: with four shares 27 us, eight 20,
// sixteen 18.  A call of 16 query rows over 4095 slots in 32 lists: 29.0, 28.3, 29.8.
constexpr int kWeightSlots = 256, kWeightShares = 8;
__global__ __launch_bounds__(64 * kWeightShares) void kv4_weights_kernel(Kv4Cache c, Kv4Attn a,
                                                               const float2 *__restrict__ lse,
                                                               const float *__restrict__ scores) {
  __shared__ float4 part[kWeightShares - 1][64];
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int grp = c.nh / c.nkv, V = a.rows * grp, x = threadIdx.x & 63;
  const int share = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int filled = kv4_filled(c, s, a.rows);
  const int t = blockIdx.x * kWeightSlots + 4 * x;
  if (filled < 0 || (int)(blockIdx.x * kWeightSlots) >= filled + a.rows) return;
  const int64_t step = score_stride(c.slots);
  const float2 *e = lse + list * V;
  const float *sc = scores + list * V * step + t;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (t < filled + a.rows) {
    if (t + 3 <= filled) {  // every row sees the four slots
#pragma unroll 8
      for (int v = share; v < V; v += kWeightShares) {
        const float4 y = *(const float4 *)(sc + v * step);
        const float2 z = e[v];
        sum.x = fmaf(__builtin_amdgcn_exp2f(y.x - z.x), z.y, sum.x);
        sum.y = fmaf(__builtin_amdgcn_exp2f(y.y - z.x), z.y, sum.y);
        sum.z = fmaf(__builtin_amdgcn_exp2f(y.z - z.x), z.y, sum.z);
        sum.w = fmaf(__builtin_amdgcn_exp2f(y.w - z.x), z.y, sum.w);
      }
    } else {
      for (int v = share; v < V; v += kWeightShares) {
        const int last = filled + v / grp;  // the last slot that row v sees
        const float4 y = *(const float4 *)(sc + v * step);
        const float2 z = e[v];
        if (t <= last) sum.x = fmaf(__builtin_amdgcn_exp2f(y.x - z.x), z.y, sum.x);
        if (t + 1 <= last) sum.y = fmaf(__builtin_amdgcn_exp2f(y.y - z.x), z.y, sum.y);
        if (t + 2 <= last) sum.z = fmaf(__builtin_amdgcn_exp2f(y.z - z.x), z.y, sum.z);
        if (t + 3 <= last) sum.w = fmaf(__builtin_amdgcn_exp2f(y.w - z.x), z.y, sum.w);
      }
    }
  }
  if (share) part[share - 1][x] = sum;
  __syncthreads();
  if (share) return;
#pragma unroll
  for (int k = 0; k < kWeightShares - 1; ++k) {
    const float4 y = part[k][x];
    sum.x += y.x, sum.y += y.y, sum.z += y.z, sum.w += y.w;
  }
  const float w[4] = {sum.x, sum.y, sum.z, sum.w};
  float *to = c.weights + list * c.slots + t;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (t + k < filled + a.rows) to[k] = a.weights_mode == 2 ? to[k] + w[k] : w[k];
}

// How a call is cut: kv4_rows_kernel with nsub groups of 16 query rows per workgroup (dense), or
// kv4_attention_kernel with HPS rows; W waves per workgroup, `wgs` workgroups at a time on the
// GPU for each set of rows, a list in S of them at most.
struct Plan {
  int V, nsub, nz;
  bool dense;
  Cut cut;
  int64_t lists;
};
Plan plan(int rows, int n_seq, int nh, int nkv, int hd, int slots) {
  Plan p;
  const int hps = 512 / hd;
  p.V = rows * (nh / nkv);
  // The two kernels, V query rows per list (us of a replayed call, caches warm, V of 8 and less one
  // row per sequence; kv4_attention_kernel in as many groups as it takes / kv4_rows_kernel; 8 KV
  // heads, 2 of 256 channels):
  //                                    V 4          V 5          V 8          V 16         V 128
  //   64,  one sequence,  300 slots    6.2 / 6.6    6.4 / 6.6    6.5 / 6.6    8.6 / 8.8   13.9 / 11.3
  //        one sequence, 20000        13.8 / 12.5  13.9 / 12.7  14.2 / 12.8  18.5 / 15.6  56.3 / 31.6
  //        16 sequences,  4095        20.3 / 21.1  20.4 / 20.8  21.1 / 21.0  36.2 / 26.6   142 / 91.8
  //   128, one sequence,  300          7.4 / 8.4    7.4 / 8.5    7.5 / 8.5   12.6 / 11.0  16.0 / 15.1
  //        one sequence, 20000        16.2 / 15.5  18.1 / 15.5  18.4 / 15.8  30.9 / 18.8   139 / 46.2
  //        16 sequences,  4095        24.4 / 27.6  39.1 / 27.8  39.8 / 28.1  71.1 / 34.0   333 / 135
  //   256, one sequence,  300          9.5 / 14.6   9.5 / 14.9   9.6 / 15.0  11.9 / 18.1  21.4 / 18.5
  //        one sequence, 20000        15.6 / 17.5  16.2 / 17.7  18.3 / 18.1  26.7 / 21.9   194 / 39.1
  //        16 sequences,  4095        22.9 / 22.1  40.0 / 22.4  32.6 / 22.7  53.5 / 28.1   330 / 89.7
  // The rule follows the batches, where there is most to win.  It costs a lone sequence of few slots
  // up to 1 us at 128 channels and 6 at 256 from V = 5 on, and one of 20000 slots of 64 channels 1.3
  // at V = 4.
  p.dense = p.V > 4;
  const int group = p.dense ? 16 : hps;
  p.nsub = p.dense && p.V > 16 && hd < 256 ? 2 : 1;
  p.nz = (p.V + p.nsub * group - 1) / (p.nsub * group);
  p.lists = (int64_t)n_seq * nkv;
  // Waves per workgroup and workgroups at a time (us; 32 / 8 heads of 128).  Few rows: many lists
  // of different lengths balance better in small workgroups (16 sequences of up to 4095 slots:
  // 8 x 512 25.6, 4 x 768 21.7); few lists leave fewer records with large ones (6000 slots: 11.1
  // against 13.1; 130000: 42.2 against 42.7).  Of 256 channels and with many rows a kernel takes
  // up to 256 registers: two waves per SIMD, with many rows as one workgroup per CU (32 rows of
  // 20000 slots: 51.8 with two, 50.0 with one), but of 256 channels as two (4 x 9000 slots, 16 /
  // 2 heads: 23.8 against 25.0).
  const bool many = p.lists * p.nz >= 32;
  int resident;
  if (p.dense) {
    p.cut.W = hd == 256 ? 4 : 8, resident = hd == 256 ? 512 : 256;
  } else if (hd == 256) {
    p.cut.W = 8, resident = 256;
  } else {
    p.cut.W = many ? 4 : 8, resident = many ? 768 : 512;
  }
  p.cut.wgs = (resident + p.nz - 1) / p.nz;
  // a list of two turns is not cut: one launch, and nothing to join
  const int64_t tiles = slots / kKv4Tile;
  const int64_t most = tiles <= 2 * p.cut.W ? 1 : (tiles + kLeastTiles - 1) / kLeastTiles;
  // sequences of different lengths: up to four times the workgroups that equal ones would take
  const int64_t want = (4 * p.cut.wgs + p.lists - 1) / p.lists;
  p.cut.S = (int)(want < most ? want : most);
  return p;
}

// Work: records (several splits), then per query row its (m, 1 / sum of p) and its scores (weights).
int64_t record_bytes(const Plan &p, int hd) {
  return p.cut.S > 1 ? p.lists * p.cut.S * p.V * (int64_t)(hd + hd / 16) * 4 : 0;
}
int64_t lse_bytes(const Plan &p) { return (p.lists * p.V * 8 + 15) / 16 * 16; }

template <int HD>
hipError_t launch(const Kv4Cache &c, const Kv4Attn &a, hipStream_t s) {
  const Plan p = plan(a.rows, c.n_seq, c.nh, c.nkv, HD, c.slots);
  float *rec = (float *)a.work, *scores = nullptr;
  float2 *lse = nullptr;
  if (a.weights_mode) {
    lse = (float2 *)((char *)a.work + record_bytes(p, HD));
    scores = (float *)((char *)lse + lse_bytes(p));
  }
  const bool inside = a.store && a.rows == 1;  // the one row is stored by the workgroups
  if (a.store && !inside) {
    const hipError_t e =
        launch_kv4_append(c, a.qkv, a.ldq, (int64_t)c.n_seq * a.rows, nullptr, true, s);
    if (e != hipSuccess) return e;
  }
  // No call has more items than wgs + lists (every list but for its last workgroup gets whole
  // shares).  A multiple of the dies: one item's groups of rows meet in one L2.
  const int64_t most = p.lists * p.cut.S, items = most < p.cut.wgs + p.lists ? most : p.cut.wgs + p.lists;
  const dim3 grid((unsigned)((items + 7) / 8 * 8), 1, (unsigned)p.nz), block(64 * p.cut.W);
  auto go = [&](auto *kernel) {
    hipLaunchKernelGGL(kernel, grid, block, 0, s, c, a, rec, lse, scores, p.cut, inside);
  };
  if (p.dense) {
    if constexpr (HD < 256) {
      if (p.nsub == 2)
        go(kv4_rows_kernel<HD, 2>);
      else
        go(kv4_rows_kernel<HD, 1>);
    } else {
      go(kv4_rows_kernel<HD, 1>);
    }
  } else if constexpr (HD == 256) {
    go(kv4_attention_kernel<HD, 8, 2>);
  } else if (p.cut.W == 4) {
    go(kv4_attention_kernel<HD, 4, 4>);
  } else {
    go(kv4_attention_kernel<HD, 8, 4>);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.cut.S > 1) {
    hipLaunchKernelGGL(kv4_merge_kernel<HD>, dim3((unsigned)p.V, (unsigned)p.lists),
                       dim3(kMergeThreads<HD>), 0, s, c, a, rec, lse, p.cut);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (!a.weights_mode) return hipSuccess;
  hipLaunchKernelGGL(kv4_weights_kernel,
                     dim3((unsigned)((c.slots + kWeightSlots - 1) / kWeightSlots), (unsigned)p.lists),
                     dim3(64 * kWeightShares), 0, s, c, a, lse, scores);
  return hipGetLastError();
}

}  // namespace

int64_t kv4_attention_work_bytes(int rows, bool weights, int n_seq, int nh, int nkv, int hd,
                                 int slots) {
  const Plan p = plan(rows, n_seq, nh, nkv, hd, slots);
  return record_bytes(p, hd) + 16 + (weights ? lse_bytes(p) + p.lists * p.V * score_stride(slots) * 4 : 0);
}

hipError_t launch_kv4_attention(const Kv4Cache &c, const Kv4Attn &a, hipStream_t s) {
  if (c.hd == 64) return launch<64>(c, a, s);
  if (c.hd == 128) return launch<128>(c, a, s);
  return launch<256>(c, a, s);
}

}  // namespace gguf

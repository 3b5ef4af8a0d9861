// Attention over the 4-bit KV cache.
//
// Query rows of a (sequence, KV head): v = i * group + h for new row i and query head h of
// the group; row v sees slots 0 .. lengths[s] + i.  The slots are split over workgroups;
// each writes, per query row, a record of its partial softmax, and kv4_merge_kernel joins
// them in split order (so the result does not depend on timing).
#include "kv4.hpp"

namespace gguf {

namespace {

constexpr int kThreads = 256;

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
  return n < 0 || n + rows > c.slots || p < 0 || p + rows > c.rope_rows ? -1 : (int)n;
}

// How the tiles of a list are cut: `per` for each workgroup, `n` of them at most S.  Every
// workgroup of the call gets about the same number, whatever the sequences' lengths: all lists'
// tiles over `wgs` workgroups, in whole turns of a workgroup's W waves.
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
  const int per = (max(max(fair, 1), (tiles + k.S - 1) / k.S) + k.W - 1) / k.W * k.W;
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
  // Slot j of the tile from its bytes and scales.
  __device__ __forceinline__ void patch(const uint8_t (&fresh)[2][HD / 2],
                                        const half_t (&fscale)[2][NB], int j, int r, int g, int b) {
    const int sh = 8 * (j & 3), ss = 16 * (j & 1);
    const uint32_t kd = __builtin_bit_cast(uint16_t, fscale[0][b]);
    const uint32_t vd = __builtin_bit_cast(uint16_t, fscale[1][b]);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (j == 16 * t + r)
#pragma unroll
        for (int i = 0; i < NB; ++i) k[t][i] = *(const uint32_t *)(fresh[0] + (g * NB + i) * 4);
      if (j >> 2 == 4 * t + g) {
#pragma unroll
        for (int i = 0; i < NB; ++i)
          v[t][i] = (v[t][i] & ~(0xFFu << sh)) | ((uint32_t)fresh[1][r * NB + i] << sh);
        // by value: a reference to one of two words would put the registers in memory
        const uint32_t keep = ~(0xFFFFu << ss), kn = kd << ss, vn = vd << ss;
        if (j & 2) {
          ks[t].y = (ks[t].y & keep) | kn;
          vs[t].y = (vs[t].y & keep) | vn;
        } else {
          ks[t].x = (ks[t].x & keep) | kn;
          vs[t].x = (vs[t].x & keep) | vn;
        }
      }
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

// A workgroup takes one list, one range of its tiles and NSUB groups of HPS = 512 / HD query
// rows; its waves take the range's tiles in turn and join at the end.  Nothing but registers
// carries a tile through:
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
//   set and stays below 2^14 in f16, whatever V's range; where a tile passes that (or p 2^40:
//   scales near zero), m is raised to the largest score + log2 |scale| (the float's bits read as
//   a number, within 0.09) and the sums are scaled down.  That is rare after the first tiles.
// - K's registers take the next tile as soon as its scores are made, V's after its products:
//   one tile in flight per wave, four waves per SIMD.
// Bound: HBM, 9/8 head_dim bytes per slot and list.
template <int HD, int NSUB, int W, int WPS>
__global__ __launch_bounds__(64 * W, WPS) void kv4_attention_kernel(Kv4Cache c, Kv4Attn a,
                                                               float *__restrict__ rec,
                                                               float2 *__restrict__ lse,
                                                               float *__restrict__ scores, Cut cut,
                                                               bool store) {
  using L = Kv4<HD>;
  constexpr int NB = L::NB, HPS = 16 / NB, half = HD / 2, RS = record_floats<HD>();
  constexpr float kLift = 10.f, kMostW = 16384.f, kMostP = 0x1p40f;
  __shared__ float lo_[W][NSUB][512];          // per wave and group: HPS rows of HD sums
  __shared__ float2 lm[W][NSUB][16];           // and the 16 rows' (m, sum of p)
  __shared__ half8_t q_[NSUB][NB][2][64];      // queries: per block, hi and lo part, a B operand
  __shared__ float qc[NSUB][16];               // per row: log2 units per unit of a score
  __shared__ __align__(16) uint8_t fresh[2][half];  // the stored row's K and V code bytes,
  __shared__ half_t fscale[2][NB];                  // and scales
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
  const int v0 = blockIdx.z * NSUB * HPS;
  // the workgroups whose range has the one new row (a call of more rows stores them beforehand)
  // make its bytes in LDS, for the wave whose first tile lacks them; those of the first group of
  // query rows store them
  const bool stores = store && filled / kKv4Tile >= tile0 && filled / kKv4Tile < tile1;
  const float *row0 = a.qkv + s * a.rows * a.ldq;  // the sequence's first row
  const float *kx = row0 + (int64_t)(c.nh + kvh) * HD, *vx = kx + (int64_t)c.nkv * HD;
  const int64_t pos0 = c.pos[s];

  // What comes before the barrier is requested before the tile, since loads return in order:
  // behind a full chip's tiles the queries took 5.6 us (130000 slots).
  float4 xo[2], xp[2], cv[2], sv[2];  // wave < NSUB: the queries of group `wave`: lane (r, g)
                                      // holds channels 32 b + 8 g + 0..7 of its row
  constexpr int LANES = Kv4Row<HD>::LANES, STORERS = HD == 256 ? 2 : 1;
  Kv4Row<HD> row;  // waves NSUB ..: the new row's K (unit 0) and V (1), HD / 4 lanes each
  const int unit = (wave - NSUB) * (64 / LANES) + lane / LANES, rq = lane % LANES;
  if (wave < NSUB) {
    const int v = v0 + wave * HPS + h, i = v < V ? v / grp : 0;
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
  } else if (stores && wave < NSUB + STORERS && unit < 2) {
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
  if (wave < NSUB) {
    const bool on = v0 + wave * HPS + h < V;  // past the last query row: zeros
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
    if (g == 0) qc[wave][r] = pow2f(-e);
    const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      q_[wave][k][0][lane] = b == k ? hi : zero;
      q_[wave][k][1][lane] = b == k ? lo : zero;
    }
  } else if (stores && wave < NSUB + STORERS) {
    uint32_t word;
    half_t scale;
    kv4_quantize<HD>(row, rq, unit == 0, word, scale);
    const int j = filled % kKv4Tile, blk = rq >> 3;
    uint8_t *to = base + (int64_t)(filled / kKv4Tile) * L::TB;
    const bool writes = blockIdx.z == 0;
    if (unit == 0 && !(rq & 1)) {
      const int at = (((rq >> 1) & 3) * NB + blk) * 4;
      *(uint32_t *)(fresh[0] + at) = word;
      if (writes) *(uint32_t *)(to + j * half + at) = word;
    } else if (unit == 1 && (rq & 7) < 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = (4 * (rq & 3) + i) * NB + blk;
        fresh[1][at] = (uint8_t)(word >> (8 * i));
        if (writes) to[L::VO + (j >> 2) * (2 * HD) + at * 4 + (j & 3)] = (uint8_t)(word >> (8 * i));
      }
    }
    if (unit < 2 && !(rq & 7)) {
      fscale[unit][blk] = scale;
      if (writes)
        *(half_t *)(to + (unit ? L::VS : L::KS) + ((j >> 2) * NB + blk) * 8 + (j & 3) * 2) = scale;
    }
    if (writes && unit == 1 && rq == 0) {
      if (c.positions) c.positions[list * c.slots + filled] = (int32_t)pos0;
      if (c.weights) c.weights[list * c.slots + filled] = 0.f;
    }
  }
  __syncthreads();
  float f[NSUB];            // log2 units per accumulated unit
  int vis[NSUB];            // slots that the row sees
#pragma unroll
  for (int u = 0; u < NSUB; ++u) {
    f[u] = qc[u][r];
    const int v = v0 + u * HPS + h;
    vis[u] = filled + (v < V ? v / grp : 0) + 1;
  }
  const int all_see = filled + v0 / grp + 1;  // slots that every row of the workgroup sees

  float4_t acc[NSUB][2 * NB];
  float m[NSUB], l[NSUB];  // p = 2^(score - m)
#pragma unroll
  for (int u = 0; u < NSUB; ++u) {
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t) acc[u][t] = float4_t{0.f, 0.f, 0.f, 0.f};
  }

  uint32_t magic;
  asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(magic));
  float minus1 = -1.f;  // not known to be: x - (float)h stays one fused instruction
  asm volatile("" : "+s"(minus1));
  if (stores && tile == filled / kKv4Tile) d.patch(fresh, fscale, filled % kKv4Tile, r, g, b);
  int ql = lane;  // made anew every turn: the queries are read from LDS there, not kept
  for (; tile >= tile0; tile -= W) {
    const uint8_t *next = base + (int64_t)max(tile - W, tile0) * L::TB;  // the last one: unused
    const int slot0 = tile * kKv4Tile + 4 * g;  // of half 0, i = 0
    asm volatile("" : "+v"(ql));
    float y[NSUB][8];  // scores / f
    {
      float4_t sc[NSUB][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int u = 0; u < NSUB; ++u) sc[u][t] = float4_t{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const half8_t k0 = k_frag(d.k[0][k], magic), k1 = k_frag(d.k[1][k], magic);
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
          const half8_t hi = q_[u][k][0][ql], lo = q_[u][k][1][ql];
          sc[u][0] = mfma(k0, hi, sc[u][0]);
          sc[u][1] = mfma(k1, hi, sc[u][1]);
          sc[u][0] = mfma(k0, lo, sc[u][0]);
          sc[u][1] = mfma(k1, lo, sc[u][1]);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const half_t ks = __builtin_bit_cast(half4_t, d.ks[i >> 2])[i & 3];
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
          float x = mul_f16(sc[u][i >> 2][i & 3], ks);
          x = add_ror16<8>(x);
          if constexpr (NB > 2) x = add_ror16<4>(x);
          if constexpr (NB > 4) x = add_ror16<2>(x);
          y[u][i] = x;
        }
      }
    }
    const half4_t dv[2] = {__builtin_bit_cast(half4_t, d.vs[0]), __builtin_bit_cast(half4_t, d.vs[1])};
    d.load_k(next, r, g, b);
    if (scores) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = y[u][i] * f[u];
        if (r < HPS && v0 + u * HPS + r < V) {
          float *o = scores + (list * V + v0 + u * HPS + r) * score_stride(c.slots) + slot0;
          *(float4 *)o = make_float4(z[0], z[1], z[2], z[3]);
          *(float4 *)(o + 16) =
              make_float4(z[4], z[5], z[6], z[7]);
        }
      }
    }
    const bool masked = (tile + 1) * kKv4Tile > all_see;
    half8_t wh[NSUB], wl[NSUB];
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      float p[8], w[8], sum, most;
      // the first slot past those that the row sees, from slot0: hides i from there on (unrolled
      // turns share nothing of this but where a tile is masked)
      auto hidden = [&](int i) { return slot0 + (i < 4 ? i : 12 + i) >= vis[u]; };
      auto weigh = [&]() {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(y[u][i], f[u], -m[u]));
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
        float n = m[u];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t bits = __float_as_uint((float)dv[i >> 2][i & 3]) & 0x7FFFFFFFu;
          const float lg =  // of at least 2^-24
              fmaf((float)(int)(bits < 0x33800000u ? 0x33800000u : bits), 0x1p-23f, -127.f - kLift);
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
      half2_t hp[4], lp[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // V's pairs: slots (0, 2), (1, 3) of each half
        const int i = (k & 1) + (k >> 1) * 4;
        hp[k] = half2_t{(half_t)w[i], (half_t)w[i + 2]};
        lp[k] = half2_t{(half_t)fmaf((float)hp[k][0], minus1, w[i]),
                        (half_t)fmaf((float)hp[k][1], minus1, w[i + 2])};
      }
      wh[u] = __builtin_bit_cast(half8_t, hp);
      wl[u] = __builtin_bit_cast(half8_t, lp);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const uint32_t w0 = d.v[0][k], h0 = w0 >> 8, w1 = d.v[1][k], h1 = w1 >> 8;
      const half8_t va = v_frag<1>(w0, h0, w1, h1, magic);
      const half8_t vb = v_frag<16>(w0, h0, w1, h1, magic);  // channels 16..31 of the block
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        acc[u][2 * k] = mfma(wh[u], va, acc[u][2 * k]);
        acc[u][2 * k + 1] = mfma(wh[u], vb, acc[u][2 * k + 1]);
        acc[u][2 * k] = mfma(wl[u], va, acc[u][2 * k]);
        acc[u][2 * k + 1] = mfma(wl[u], vb, acc[u][2 * k + 1]);
      }
    }
    d.load_v(next, r, g);
  }

  // the waves' sums: lane (r, g), register i holds row 4 g + i, channel 16 t + r
#pragma unroll
  for (int u = 0; u < NSUB; ++u) {
    float sum = sum_xor32(sum_xor16(l[u]));
    if (g == 0) lm[wave][u][r] = make_float2(m[u], sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 4 * g + i, rb = row / HPS;
#pragma unroll
      for (int t = 0; t < 2 * NB; ++t)
        if (rb == t / 2)
          lo_[wave][u][row % HPS * HD + 16 * t + r] = acc[u][t][i] * (t & 1 ? 0.0625f : 1.f);
    }
  }
  __syncthreads();
  float *out = rec + (list * cut.S + it.split) * V * RS;
  for (int e = tid; e < NSUB * 512; e += 64 * W) {
    const int u = e >> 9, hh = (e & 511) / HD, ch = e & (HD - 1), row = (ch >> 5) * HPS + hh;
    const int v = v0 + u * HPS + hh;
    if (v >= V) continue;
    float mx = lm[0][u][row].x, o = 0.f, ls = 0.f;
#pragma unroll
    for (int k = 1; k < W; ++k) mx = fmaxf(mx, lm[k][u][row].x);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float2 ml = lm[k][u][row];
      const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
      o = fmaf(w, lo_[k][u][e & 511], o);
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

// One workgroup per query row of a list with several splits: their records joined, groups of
// HD / 4 threads taking every G-th record, then the groups in order.
template <int HD>
__global__ __launch_bounds__(kThreads) void kv4_merge_kernel(Kv4Cache c, Kv4Attn a,
                                                             const float *__restrict__ rec,
                                                             float2 *__restrict__ lse, Cut cut) {
  constexpr int RS = record_floats<HD>(), Q = HD / 4, G = kThreads / Q;
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

// The attention weights of a list's slots: 64 threads of four slots each times four shares of
// the query rows, whose scores are taken against the rows' maximum and sum (apart: their
// log-sum-exp in one float would lose the low bits); shares joined in order.
constexpr int kWeightSlots = 256;
__global__ __launch_bounds__(kThreads) void kv4_weights_kernel(Kv4Cache c, Kv4Attn a,
                                                               const float2 *__restrict__ lse,
                                                               const float *__restrict__ scores) {
  __shared__ float4 part[3][64];
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
      for (int v = share; v < V; v += 4) {
        const float4 y = *(const float4 *)(sc + v * step);
        const float2 z = e[v];
        sum.x = fmaf(__builtin_amdgcn_exp2f(y.x - z.x), z.y, sum.x);
        sum.y = fmaf(__builtin_amdgcn_exp2f(y.y - z.x), z.y, sum.y);
        sum.z = fmaf(__builtin_amdgcn_exp2f(y.z - z.x), z.y, sum.z);
        sum.w = fmaf(__builtin_amdgcn_exp2f(y.w - z.x), z.y, sum.w);
      }
    } else {
      for (int v = share; v < V; v += 4) {
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
  for (int k = 0; k < 3; ++k) {
    const float4 y = part[k][x];
    sum.x += y.x, sum.y += y.y, sum.z += y.z, sum.w += y.w;
  }
  const float w[4] = {sum.x, sum.y, sum.z, sum.w};
  float *to = c.weights + list * c.slots + t;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (t + k < filled + a.rows) to[k] = a.weights_mode == 2 ? to[k] + w[k] : w[k];
}

// How a call is cut: NSUB groups of HPS query rows per workgroup of W waves, `wgs` workgroups
// at a time on the GPU for each group of rows, a list in S of them at most.
struct Plan {
  int V, nsub, nz;
  Cut cut;
  int64_t lists;
};
Plan plan(int rows, int n_seq, int nh, int nkv, int hd, int slots) {
  Plan p;
  const int hps = 512 / hd;
  p.V = rows * (nh / nkv);
  p.nsub = hd < 256 && p.V > hps ? 2 : 1;
  p.nz = (p.V + p.nsub * hps - 1) / (p.nsub * hps);
  p.lists = (int64_t)n_seq * nkv;
  // Waves per workgroup and workgroups at a time, measured (us; 32 / 8 heads of 128 unless said):
  // many lists of different lengths balance better in small workgroups (16 sequences of up to
  // 4095 slots: 8 x 512 24.8, 4 x 768 21.2); few lists leave fewer records with large ones (6000
  // slots: 11.1 against 12.7; 130000: 40.2 against 40.8).  Two groups of rows take 182 registers:
  // two workgroups of four waves (32 rows over 20000 slots: 4 x 512 133, 8 x 512 142, 8 x 256 218,
  // where ten of the 256 CUs get two); 256 channels 160 (4 sequences of 9000 slots, 16 / 2 heads:
  // 8 x 256 32.3, 4 x 768 34.2).
  const bool many = p.lists * p.nz >= 32;
  int resident;
  if (p.nsub == 2) {
    p.cut.W = 4, resident = 512;
  } else if (hd == 256) {
    p.cut.W = 8, resident = 256;
  } else {
    p.cut.W = many ? 4 : 8, resident = many ? 768 : 512;
  }
  p.cut.wgs = (resident + p.nz - 1) / p.nz;
  // a list is not cut below two turns of a workgroup's waves: one launch, and nothing to join
  const int64_t tiles = slots / kKv4Tile, most = tiles <= 2 * p.cut.W ? 1 : (tiles + p.cut.W - 1) / p.cut.W;
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
        launch_kv4_append(c, a.qkv, a.ldq, (int64_t)c.n_seq * a.rows, nullptr, s);
    if (e != hipSuccess) return e;
  }
  // No call has more items than wgs + lists (every list but for its last workgroup gets whole
  // shares).  A multiple of the dies: one item's groups of rows meet in one L2.
  const int64_t most = p.lists * p.cut.S, items = most < p.cut.wgs + p.lists ? most : p.cut.wgs + p.lists;
  const dim3 grid((unsigned)((items + 7) / 8 * 8), 1, (unsigned)p.nz), block(64 * p.cut.W);
  auto go = [&](auto *kernel) {
    hipLaunchKernelGGL(kernel, grid, block, 0, s, c, a, rec, lse, scores, p.cut, inside);
  };
  if constexpr (HD == 256)
    go(kv4_attention_kernel<HD, 1, 8, 2>);
  else if (p.nsub == 2)
    go(kv4_attention_kernel<HD, 2, 4, 2>);
  else if (p.cut.W == 4)
    go(kv4_attention_kernel<HD, 1, 4, 4>);
  else
    go(kv4_attention_kernel<HD, 1, 8, 4>);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.cut.S > 1) {
    hipLaunchKernelGGL(kv4_merge_kernel<HD>, dim3((unsigned)p.V, (unsigned)p.lists), dim3(kThreads),
                       0, s, c, a, rec, lse, p.cut);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (!a.weights_mode) return hipSuccess;
  hipLaunchKernelGGL(kv4_weights_kernel,
                     dim3((unsigned)((c.slots + kWeightSlots - 1) / kWeightSlots), (unsigned)p.lists),
                     dim3(kThreads), 0, s, c, a, lse, scores);
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

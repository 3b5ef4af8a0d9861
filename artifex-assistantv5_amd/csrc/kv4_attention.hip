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
constexpr float kLog2e = 1.4426950408889634f;

// A record: sum of p v per channel, then per block of 32 channels the maximum m that its p
// are relative to (in log2 units) and the sum of its p.
template <int HD>
constexpr int record_floats() {
  return HD + 2 * (HD / 32);
}

// The splits of a sequence that sees `vis` slots: `per` tiles each (whole turns of the W waves
// of a workgroup), `n` of them.
struct Splits {
  int per, n;
};
__device__ __forceinline__ Splits kv4_splits(int vis, int S, int W) {
  const int tiles = (vis + kKv4Tile - 1) / kKv4Tile;
  int per = (tiles + S - 1) / S;
  per = (per + W - 1) / W * W;
  return {per, (tiles + per - 1) / per};
}

// The slots in use before the call, or -1 if the sequence takes no part.
__device__ __forceinline__ int kv4_filled(const Kv4Cache &c, int64_t s, int rows) {
  const int64_t n = c.lengths[s], p = c.pos[s];
  return n < 0 || n + rows > c.slots || p < 0 || p + rows > c.rope_rows ? -1 : (int)n;
}

// Eight 4-bit codes (element 0..3 in the low nibbles of bytes 0..3, 4..7 in the high ones) as
// f16 integers 0..15: a byte below 16 read as E4M3 is code * 2^-9, exactly.
__device__ __forceinline__ half8_t k_codes(uint32_t w) {
  const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
  const uint32_t r[4] = {
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true))};
  return __builtin_bit_cast(half8_t, r);
}
// Codes in bits 0-3 and 16-19 of w as f16 integers code - 8 (1024 + code, less 1032); `magic`
// holds 1024.0 twice in a vector register, so that mask and OR are one instruction.
__device__ __forceinline__ half2_t v_codes(uint32_t w, uint32_t magic) {
  const half2_t c = __builtin_bit_cast(half2_t, (w & 0x000F000Fu) | magic);
  return c - half2_t{(half_t)1032.f, (half_t)1032.f};
}
__device__ __forceinline__ half8_t v_frag(uint32_t w0, uint32_t w1, uint32_t magic) {
  const half2_t r[4] = {v_codes(w0, magic), v_codes(w0 >> 8, magic), v_codes(w1, magic),
                        v_codes(w1 >> 8, magic)};
  return __builtin_bit_cast(half8_t, r);
}
__device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// v plus that of the lane N to the left in its 16, cyclically.
template <int N>
__device__ __forceinline__ float add_ror16(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xF, 0xF, true));
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
      ks[t] = *(const uint2 *)(tile + (uint32_t)(Kv4<HD>::KS + ((4 * t + g) * NB + b) * 8));
    }
  }
  __device__ __forceinline__ void load_v(const uint8_t *tile, int r, int g, int b) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      words(tile + (uint32_t)(Kv4<HD>::VO + (4 * t + g) * (2 * HD) + r * NB * 4), v[t]);
      vs[t] = *(const uint2 *)(tile + (uint32_t)(Kv4<HD>::VS + ((4 * t + g) * NB + b) * 8));
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
//   Its offset of 8 per code is the accumulator's initial value.  Each lane multiplies by its
//   block's scales; rotations within 16 lanes add the blocks, leaving the score in each.
// - Queries are scaled by a power of two per row and enter as two f16 parts (22 bits), twice
//   the MFMAs: the scores are f32-grade.  The operands, three quarters of them zeros at 128
//   channels, are made once per workgroup and read from LDS each turn: in registers they would
//   cost a wave per SIMD.
// - Output: the scores' accumulator layout (lane: slots 4 g + 0..3 of column r) is the A layout
//   of P . V when K index j of lane group g means slot 4 g + j % 4 of half j / 4; V is stored
//   so that a lane's words hold these slots.  Row HPS b + h of A is p * (scale of V's block b)
//   of query row h, so the scales need no pass of their own; only the channels of block b of
//   that row's output are used.  p * scale enters as two f16 parts.  V's codes enter as
//   code - 8, exactly: an offset taken off at the end would cost the sums their low bits.
// - Each row's p is 2^(score - m) with a running m, so that p * scale is at most 2^10 when m is
//   set and stays below 2^14 in f16, whatever V's range; where a tile passes that (or p 2^40:
//   scales near zero), m is raised to the largest score + log2 |scale| (the float's bits read as
//   a number, within 0.09) and the sums are scaled down.  That is rare after the first tiles.
// - K's registers take the next tile as soon as its scores are made, V's after its products:
//   one tile in flight per wave, four waves per SIMD.
// Bound: HBM, 9/8 head_dim bytes per slot and list.
template <int HD, int NSUB, int W>
__global__ __launch_bounds__(64 * W) void kv4_attention_kernel(Kv4Cache c, Kv4Attn a,
                                                               float *__restrict__ rec,
                                                               float *__restrict__ lse,
                                                               float *__restrict__ scores, int S,
                                                               bool store) {
  using L = Kv4<HD>;
  constexpr int NB = L::NB, HPS = 16 / NB, half = HD / 2, RS = record_floats<HD>();
  constexpr float kLift = 10.f, kMostW = 16384.f, kMostP = 0x1p40f;
  __shared__ float lo_[W][NSUB][512];          // per wave and group: HPS rows of HD sums
  __shared__ float2 lm[W][NSUB][16];           // and the 16 rows' (m, sum of p)
  __shared__ half8_t q_[NSUB][NB][2][64];      // queries: per block, hi and lo part, a B operand
  __shared__ float2 qc[NSUB][16];              // per row: initial value, log2 units per unit
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int kvh = (int)(list - s * c.nkv), grp = c.nh / c.nkv, V = a.rows * grp;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // known uniform: scalar addresses
  const int b = r / HPS, h = r % HPS;
  const int filled = kv4_filled(c, s, a.rows);
  if (filled < 0) return;
  const Splits sp = kv4_splits(filled + a.rows, S, W);
  if ((int)blockIdx.x >= sp.n) return;
  const int tile0 = blockIdx.x * sp.per;
  const int tile1 = min(tile0 + sp.per, (filled + a.rows + kKv4Tile - 1) / kKv4Tile);
  uint8_t *base = kv4_list(c.kv, list, c.slots, L::TB);
  const int v0 = blockIdx.z * NSUB * HPS;
  // the workgroup whose range has the one new row stores it (a call of more rows stores them
  // beforehand) and reads its tiles afterwards; the others request theirs now
  const bool stores = store && filled / kKv4Tile >= tile0 && filled / kKv4Tile < tile1;
  TileRegs<HD> d;
  int tile = tile0 + wave;
  if (!stores && tile < tile1) {
    d.load_k(base + (int64_t)tile * L::TB, r, g, b);
    d.load_v(base + (int64_t)tile * L::TB, r, g, b);
  }
  if (wave < NSUB) {
    // queries of group `wave`: lane (r, g) holds channels 32 b + 8 g + 0..7 of its row
    const int v = v0 + wave * HPS + h, i = v < V ? v / grp : 0;
    const float *x = a.qkv + (s * a.rows + i) * a.ldq + (int64_t)(kvh * grp + v - v / grp * grp) * HD;
    const int e0 = 32 * b + 8 * g, ep = b < NB / 2 ? e0 + half : e0 - half;
    const int64_t p = (c.pos[s] + i) * half + (b < NB / 2 ? e0 : ep);
    const float sign = b < NB / 2 ? -1.f : 1.f;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const float4 xo = v < V ? *(const float4 *)(x + e0 + j) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 xp = v < V ? *(const float4 *)(x + ep + j) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float4 cv = *(const float4 *)(c.cs + p + j), sv = *(const float4 *)(c.sn + p + j);
      y[j] = xo.x * cv.x + sign * (xp.x * sv.x);
      y[j + 1] = xo.y * cv.y + sign * (xp.y * sv.y);
      y[j + 2] = xo.z * cv.z + sign * (xp.z * sv.z);
      y[j + 3] = xo.w * cv.w + sign * (xp.w * sv.w);
    }
    float mx = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fabsf(y[j]));
#pragma unroll
    for (int o = HPS; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    const int e = stage_exp(mx);
    const float up = pow2f(e);
    half8_t hi, lo;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float t = y[j] * up;
      hi[j] = (half_t)t;
      lo[j] = (half_t)(t - (float)hi[j]);
      sum += (float)hi[j] + (float)lo[j];
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (g == 0) qc[wave][r] = make_float2(-8.f * sum, pow2f(-e) * (kLog2e / sqrtf((float)HD)));
    const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      q_[wave][k][0][lane] = b == k ? hi : zero;
      q_[wave][k][1][lane] = b == k ? lo : zero;
    }
  } else if (stores && wave < NSUB + 3) {
    const float *x = a.qkv + s * a.ldq + (int64_t)(c.nh + kvh) * HD;
    const int64_t p = c.pos[s];
    if (wave == NSUB) {
      kv4_store_row<HD, true>(base, filled, x, c.cs + p * half, c.sn + p * half, lane);
    } else if (wave == NSUB + 1) {
      kv4_store_row<HD, false>(base, filled, x + (int64_t)c.nkv * HD, nullptr, nullptr, lane);
    } else if (lane == 0) {
      if (c.positions) c.positions[list * c.slots + filled] = (int32_t)p;
      if (c.weights) c.weights[list * c.slots + filled] = 0.f;
    }
  }
  __syncthreads();
  if (stores && tile < tile1) {
    d.load_k(base + (int64_t)tile * L::TB, r, g, b);
    d.load_v(base + (int64_t)tile * L::TB, r, g, b);
  }
  float q0[NSUB], f[NSUB];  // the accumulators' initial value; log2 units per accumulated unit
  int vis[NSUB];            // slots that the row sees
#pragma unroll
  for (int u = 0; u < NSUB; ++u) {
    q0[u] = qc[u][r].x;
    f[u] = qc[u][r].y;
    const int v = v0 + u * HPS + h;
    vis[u] = filled + (v < V ? v / grp : 0) + 1;
  }
  const int all_see = filled + v0 / grp + 1;  // slots that every row of the workgroup sees

  float4_t acc[NSUB][2 * NB];
  float m[NSUB], l[NSUB];  // m: p = 2^(score - m)
#pragma unroll
  for (int u = 0; u < NSUB; ++u) {
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t) acc[u][t] = float4_t{0.f, 0.f, 0.f, 0.f};
  }

  uint32_t magic;
  asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(magic));
  int ql = lane;  // made anew every turn: the queries are read from LDS there, not kept
  for (; tile < tile1; tile += W) {
    const uint8_t *next = base + (int64_t)min(tile + W, tile1 - 1) * L::TB;  // the last one: unused
    const int slot0 = tile * kKv4Tile + 4 * g;  // of half 0, i = 0
    asm volatile("" : "+v"(ql));
    float y[NSUB][8];  // scores / f
    {
      float4_t sc[NSUB][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int u = 0; u < NSUB; ++u) sc[u][t] = float4_t{q0[u], q0[u], q0[u], q0[u]};
      }
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const half8_t k0 = k_codes(d.k[0][k]), k1 = k_codes(d.k[1][k]);
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
        const float ks = (float)__builtin_bit_cast(half4_t, d.ks[i >> 2])[i & 3];
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
          float x = sc[u][i >> 2][i & 3] * ks;
          if constexpr (NB > 1) x = add_ror16<8>(x);
          if constexpr (NB > 2) x = add_ror16<4>(x);
          if constexpr (NB > 4) x = add_ror16<2>(x);
          y[u][i] = x;
        }
      }
    }
    d.load_k(next, r, g, b);
    if (scores) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u)
        if (r < HPS && v0 + u * HPS + r < V) {
          float *o = scores + (list * V + v0 + u * HPS + r) * c.slots + slot0;
          *(float4 *)o = make_float4(y[u][0] * f[u], y[u][1] * f[u], y[u][2] * f[u], y[u][3] * f[u]);
          *(float4 *)(o + 16) =
              make_float4(y[u][4] * f[u], y[u][5] * f[u], y[u][6] * f[u], y[u][7] * f[u]);
        }
    }
    const bool masked = (tile + 1) * kKv4Tile > all_see;
    half8_t wh[NSUB], wl[NSUB];
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      float p[8], w[8];
      float most_w, most_p;
      auto weigh = [&]() {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(y[u][i], f[u], -m[u]));
          w[i] = p[i] * (float)__builtin_bit_cast(half4_t, d.vs[i >> 2])[i & 3];
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (slot0 + (i < 4 ? i : 12 + i) >= vis[u]) p[i] = w[i] = 0.f;
        }
        most_w = fmaxf(fabsf(w[0]), fabsf(w[1]));
        most_p = fmaxf(p[0], p[1]);
#pragma unroll
        for (int i = 2; i < 8; i += 2) {
          most_w = fmaxf(fmaxf(most_w, fabsf(w[i])), fabsf(w[i + 1]));
          most_p = fmaxf(fmaxf(most_p, p[i]), p[i + 1]);
        }
      };
      weigh();
      if (__any(most_w > kMostW || most_p > kMostP)) {
        float n = m[u];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t bits =
              __float_as_uint((float)__builtin_bit_cast(half4_t, d.vs[i >> 2])[i & 3]) & 0x7FFFFFFFu;
          const float lg =  // of at least 2^-24
              fmaf((float)(int)(bits < 0x33800000u ? 0x33800000u : bits), 0x1p-23f, -127.f - kLift);
          if (!masked || slot0 + (i < 4 ? i : 12 + i) < vis[u])
            n = fmaxf(n, fmaf(y[u][i], f[u], lg));
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
#pragma unroll
      for (int i = 0; i < 8; ++i) l[u] += p[i];
      half2_t hp[4], lp[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // V's pairs: slots (0, 2), (1, 3) of each half
        const int i = (k & 1) + (k >> 1) * 4;
        hp[k] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(w[i], w[i + 2]));
        lp[k] = __builtin_bit_cast(half2_t,
                                   __builtin_amdgcn_cvt_pkrtz(fmaf((float)hp[k][0], -1.f, w[i]),
                                                              fmaf((float)hp[k][1], -1.f, w[i + 2])));
      }
      wh[u] = __builtin_bit_cast(half8_t, hp);
      wl[u] = __builtin_bit_cast(half8_t, lp);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const half8_t va = v_frag(d.v[0][k], d.v[1][k], magic);
      const half8_t vb = v_frag(d.v[0][k] >> 4, d.v[1][k] >> 4, magic);
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        acc[u][2 * k] = mfma(wh[u], va, acc[u][2 * k]);
        acc[u][2 * k + 1] = mfma(wh[u], vb, acc[u][2 * k + 1]);
        acc[u][2 * k] = mfma(wl[u], va, acc[u][2 * k]);
        acc[u][2 * k + 1] = mfma(wl[u], vb, acc[u][2 * k + 1]);
      }
    }
    d.load_v(next, r, g, b);
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
        if (rb == t / 2) lo_[wave][u][row % HPS * HD + 16 * t + r] = acc[u][t][i];
    }
  }
  __syncthreads();
  float *out = rec + (list * S + blockIdx.x) * V * RS;
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
      if (lse && ch == 0) lse[list * V + v] = mx + log2f(ls);
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
                                                             float *__restrict__ lse, int S, int W) {
  constexpr int RS = record_floats<HD>(), Q = HD / 4, G = kThreads / Q;
  __shared__ float4 o_[G][Q];
  __shared__ float2 ml_[G][Q];
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int v = blockIdx.x, grp = c.nh / c.nkv, V = a.rows * grp;
  const int q = threadIdx.x % Q, gi = threadIdx.x / Q;
  const int filled = kv4_filled(c, s, a.rows);
  if (filled < 0) return;
  const Splits sp = kv4_splits(filled + a.rows, S, W);
  if (sp.n == 1) return;
  const float *r = rec + (list * S * V + v) * RS;
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
  if (lse && q == 0) lse[list * V + v] = m + log2f(l);
}

// The attention weights of a list's slots, a thread per slot: the scores of every query row
// against the row's log-sum-exp.
__global__ __launch_bounds__(kThreads) void kv4_weights_kernel(Kv4Cache c, Kv4Attn a,
                                                               const float *__restrict__ lse,
                                                               const float *__restrict__ scores) {
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int grp = c.nh / c.nkv, V = a.rows * grp;
  const int filled = kv4_filled(c, s, a.rows);
  const int t = blockIdx.x * kThreads + threadIdx.x;
  if (filled < 0 || t >= filled + a.rows) return;
  const float *e = lse + list * V, *x = scores + list * V * c.slots + t;
  float sum = 0.f;
#pragma unroll 8
  for (int v = 0; v < V; ++v)
    if (t <= filled + v / grp) sum += __builtin_amdgcn_exp2f(x[(int64_t)v * c.slots] - e[v]);
  float *w = c.weights + list * c.slots + t;
  *w = a.weights_mode == 2 ? *w + sum : sum;
}

// How a call is cut: NSUB groups of HPS query rows per workgroup of W waves, S splits at most.
struct Plan {
  int V, nsub, W, nz, S;
  int64_t lists;
};
Plan plan(int rows, int n_seq, int nh, int nkv, int hd, int slots) {
  Plan p;
  const int hps = 512 / hd;
  p.V = rows * (nh / nkv);
  p.nsub = hd < 256 && p.V > hps ? 2 : 1;
  p.W = hd < 256 && p.nsub == 1 ? 16 : 8;
  p.nz = (p.V + p.nsub * hps - 1) / (p.nsub * hps);
  p.lists = (int64_t)n_seq * nkv;
  const int64_t most = (slots / kKv4Tile + p.W - 1) / p.W;
  const int64_t want = (4096 / p.W + p.lists * p.nz - 1) / (p.lists * p.nz);
  p.S = (int)(want < most ? want : most);
  return p;
}

// Work: records (several splits), then per query row its log-sum-exp and its scores (weights).
int64_t record_bytes(const Plan &p, int hd) {
  return p.S > 1 ? p.lists * p.S * p.V * (int64_t)(hd + hd / 16) * 4 : 0;
}
int64_t lse_bytes(const Plan &p) { return (p.lists * p.V * 4 + 15) / 16 * 16; }

template <int HD>
hipError_t launch(const Kv4Cache &c, const Kv4Attn &a, hipStream_t s) {
  const Plan p = plan(a.rows, c.n_seq, c.nh, c.nkv, HD, c.slots);
  float *rec = (float *)a.work, *lse = nullptr, *scores = nullptr;
  if (a.weights_mode) {
    lse = (float *)((char *)a.work + record_bytes(p, HD));
    scores = (float *)((char *)lse + lse_bytes(p));
  }
  const bool inside = a.store && a.rows == 1 && p.nz == 1;  // one workgroup stores the one row
  if (a.store && !inside) {
    const hipError_t e =
        launch_kv4_append(c, a.qkv, a.ldq, (int64_t)c.n_seq * a.rows, nullptr, s);
    if (e != hipSuccess) return e;
  }
  const dim3 grid((unsigned)p.S, (unsigned)p.lists, (unsigned)p.nz), block(64 * p.W);
  if constexpr (HD == 256) {
    hipLaunchKernelGGL((kv4_attention_kernel<HD, 1, 8>), grid, block, 0, s, c, a, rec, lse, scores,
                       p.S, inside);
  } else if (p.nsub == 2) {
    hipLaunchKernelGGL((kv4_attention_kernel<HD, 2, 8>), grid, block, 0, s, c, a, rec, lse, scores,
                       p.S, inside);
  } else {
    hipLaunchKernelGGL((kv4_attention_kernel<HD, 1, 16>), grid, block, 0, s, c, a, rec, lse, scores,
                       p.S, inside);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.S > 1) {
    hipLaunchKernelGGL(kv4_merge_kernel<HD>, dim3((unsigned)p.V, (unsigned)p.lists), dim3(kThreads),
                       0, s, c, a, rec, lse, p.S, p.W);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (!a.weights_mode) return hipSuccess;
  hipLaunchKernelGGL(kv4_weights_kernel,
                     dim3((unsigned)((c.slots + kThreads - 1) / kThreads), (unsigned)p.lists),
                     dim3(kThreads), 0, s, c, a, lse, scores);
  return hipGetLastError();
}

}  // namespace

int64_t kv4_attention_work_bytes(int rows, bool weights, int n_seq, int nh, int nkv, int hd,
                                 int slots) {
  const Plan p = plan(rows, n_seq, nh, nkv, hd, slots);
  return record_bytes(p, hd) + 16 + (weights ? lse_bytes(p) + p.lists * p.V * (int64_t)slots * 4 : 0);
}

hipError_t launch_kv4_attention(const Kv4Cache &c, const Kv4Attn &a, hipStream_t s) {
  if (c.hd == 64) return launch<64>(c, a, s);
  if (c.hd == 128) return launch<128>(c, a, s);
  return launch<256>(c, a, s);
}

}  // namespace gguf

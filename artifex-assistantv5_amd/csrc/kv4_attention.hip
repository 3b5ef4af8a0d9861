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

// The splits of a sequence that sees `vis` slots: `per` tiles each, `n` of them.
struct Splits {
  int per, n;
};
__device__ __forceinline__ Splits kv4_splits(int vis, int S) {
  const int tiles = (vis + kKv4Tile - 1) / kKv4Tile;
  int per = (tiles + S - 1) / S;
  per = (per + 3) / 4 * 4;
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
// Codes in bits 0-3 and 16-19 of w as f16 integers code - 8 (1024 + code, less 1032).
__device__ __forceinline__ half2_t v_codes(uint32_t w) {
  const half2_t c = __builtin_bit_cast(half2_t, (w & 0x000F000Fu) | 0x64006400u);
  return c - half2_t{(half_t)1032.f, (half_t)1032.f};
}
__device__ __forceinline__ half8_t v_frag(uint32_t w0, uint32_t w1) {
  const half2_t r[4] = {v_codes(w0), v_codes(w0 >> 8), v_codes(w1), v_codes(w1 >> 8)};
  return __builtin_bit_cast(half8_t, r);
}
__device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// v plus that of the lane N to the left in its 16, cyclically.
template <int N>
__device__ __forceinline__ float add_ror16(float v) {
  return v + dpp<0x120 + N>(v);
}

// What a wave reads of a tile.  Lane (r = lane % 16, g = lane / 16), halves t = 0, 1: K codes of
// slot 16 t + r, channels 32 b + 8 g + 0..7 of every block b; V codes of slots 16 t + 4 g + 0..3,
// channels 32 b + r and 32 b + 16 + r; scales of those four slots, block r / HPS.
template <int HD>
struct TileRegs {
  static constexpr int NB = HD / 32;
  uint32_t k[2][NB], v[2][NB];
  uint2 ks[2], vs[2];
  __device__ __forceinline__ void load(const uint8_t *tile, int r, int g, int b) {
    using L = Kv4<HD>;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t *kp = tile + (16 * t + r) * (HD / 2) + g * NB * 4;
      const uint8_t *vp = tile + L::VO + (4 * t + g) * (2 * HD) + r * NB * 4;
      words(kp, k[t]);
      words(vp, v[t]);
      const uint8_t *sp = tile + L::KS + ((4 * t + g) * NB + b) * 8;
      ks[t] = *(const uint2 *)sp;
      vs[t] = *(const uint2 *)(sp + 2 * HD);
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
//   the MFMAs: the scores are f32-grade.
// - Output: the scores' accumulator layout (lane: slots 4 g + 0..3 of column r) is the A layout
//   of P . V when K index j of lane group g means slot 4 g + j % 4 of half j / 4; V is stored
//   so that a lane's words hold these slots.  Row HPS b + h of A is p * (scale of V's block b)
//   of query row h, so the scales need no pass of their own; only the channels of block b of
//   that row's output are used.  p * scale enters as two f16 parts.  V's codes enter as
//   code - 8, exactly: an offset taken off at the end would cost the sums their low bits.
// - Each row's p is relative to a running maximum of score + log2 |scale| (the float's bits
//   read as a number, within 0.09), so p * scale stays below 2^14 in f16 whatever V's range;
//   the maximum is raised, and sums rescaled, only where it is passed by 4.
// Bound: HBM, 9/8 head_dim bytes per slot and list.
template <int HD, int NSUB>
__global__ __launch_bounds__(kThreads) void kv4_attention_kernel(Kv4Cache c, Kv4Attn a,
                                                                 float *__restrict__ rec,
                                                                 float *__restrict__ scores, int S,
                                                                 bool store) {
  using L = Kv4<HD>;
  constexpr int NB = L::NB, HPS = 16 / NB, half = HD / 2, RS = record_floats<HD>();
  constexpr float kLift = 10.f, kSlack = 4.f;
  __shared__ float lo_[4][NSUB][512];          // per wave and group: HPS rows of HD sums
  __shared__ float2 lm[4][NSUB][16];           // and the 16 rows' (maximum, sum of p)
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int kvh = (int)(list - s * c.nkv), grp = c.nh / c.nkv, V = a.rows * grp;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
  const int b = r / HPS, h = r % HPS;
  const int filled = kv4_filled(c, s, a.rows);
  if (filled < 0) return;
  const Splits sp = kv4_splits(filled + a.rows, S);
  if ((int)blockIdx.x >= sp.n) return;
  const int tile0 = blockIdx.x * sp.per;
  const int tile1 = min(tile0 + sp.per, (filled + a.rows + kKv4Tile - 1) / kKv4Tile);
  uint8_t *base = kv4_list(c.kv, list, c.slots, L::TB);
  if (store && filled / kKv4Tile >= tile0 && filled / kKv4Tile < tile1) {
    // the one new row (a call of more rows stores them beforehand)
    const float *x = a.qkv + s * a.ldq + (int64_t)(c.nh + kvh) * HD;
    const int64_t p = c.pos[s];
    if (wave == 0)
      kv4_store_row<HD, true>(base, filled, x, c.cs + p * half, c.sn + p * half, lane);
    else if (wave == 1)
      kv4_store_row<HD, false>(base, filled, x + (int64_t)c.nkv * HD, nullptr, nullptr, lane);
    else if (tid == 128) {
      if (c.positions) c.positions[list * c.slots + filled] = (int32_t)p;
      if (c.weights) c.weights[list * c.slots + filled] = 0.f;
    }
    __syncthreads();
  }

  // queries: lane (r, g) holds channels 32 b + 8 g + 0..7 of its row
  half8_t qh[NSUB][NB], ql[NSUB][NB];
  float q0[NSUB], f[NSUB];  // the accumulators' initial value; log2 units per accumulated unit
  int vis[NSUB];            // slots that the row sees
  const int v0 = blockIdx.z * NSUB * HPS;
#pragma unroll
  for (int u = 0; u < NSUB; ++u) {
    const int v = v0 + u * HPS + h, i = v < V ? v / grp : 0;
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
    q0[u] = -8.f * sum;
    f[u] = pow2f(-e) * (kLog2e / sqrtf((float)HD));
    vis[u] = filled + i + 1;
    const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      qh[u][k] = b == k ? hi : zero;
      ql[u][k] = b == k ? lo : zero;
    }
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

  TileRegs<HD> cur, nxt;
  int tile = tile0 + wave;
  if (tile < tile1) cur.load(base + (int64_t)tile * L::TB, r, g, b);
  for (; tile < tile1; tile += 4) {
    if (tile + 4 < tile1) nxt.load(base + (int64_t)(tile + 4) * L::TB, r, g, b);
    const int slot0 = tile * kKv4Tile + 4 * g;  // of half 0, i = 0
    const bool masked = (tile + 1) * kKv4Tile > all_see;
    float4_t sc[NSUB][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int u = 0; u < NSUB; ++u) sc[u][t] = float4_t{q0[u], q0[u], q0[u], q0[u]};
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const half8_t kc = k_codes(cur.k[t][k]);
#pragma unroll
        for (int u = 0; u < NSUB; ++u) {
          sc[u][t] = mfma(kc, qh[u][k], sc[u][t]);
          sc[u][t] = mfma(kc, ql[u][k], sc[u][t]);
        }
      }
    }
    float dv[8], lg[8];  // V's scales of this lane's block, and log2 of their magnitudes
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const half4_t d = __builtin_bit_cast(half4_t, cur.vs[t]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = (float)d[i];
        dv[4 * t + i] = x;
        const uint32_t bits = __float_as_uint(x) & 0x7FFFFFFFu;  // at least 2^-24
        lg[4 * t + i] = fmaf((float)(int)(bits < 0x33800000u ? 0x33800000u : bits), 0x1p-23f, -127.f);
      }
    }
    half8_t wh[NSUB], wl[NSUB];
#pragma unroll
    for (int u = 0; u < NSUB; ++u) {
      float x[8], top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const half4_t d = __builtin_bit_cast(half4_t, cur.ks[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y = sc[u][t][i] * (float)d[i];
          if constexpr (NB > 1) y = add_ror16<8>(y);
          if constexpr (NB > 2) y = add_ror16<4>(y);
          if constexpr (NB > 4) y = add_ror16<2>(y);
          x[4 * t + i] = y * f[u];
        }
        if (scores && r < HPS && v0 + u * HPS + r < V)
          *(float4 *)(scores + (list * V + v0 + u * HPS + r) * c.slots + slot0 + 16 * t) =
              make_float4(x[4 * t], x[4 * t + 1], x[4 * t + 2], x[4 * t + 3]);
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (slot0 + (i < 4 ? i : 12 + i) >= vis[u]) x[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i] == -INFINITY ? -INFINITY : x[i] + lg[i]);
      if (__any(top - kLift > m[u] + kSlack)) {
        float n = fmaxf(top - kLift, m[u]);
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
      }
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = x[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x[i] - m[u]);
        l[u] += p;
        w[i] = x[i] == -INFINITY ? 0.f : p * dv[i];
      }
      half2_t hp[4], lp[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // V's pairs: slots (0, 2), (1, 3) of each half
        const int i = (k & 1) + (k >> 1) * 4;
        hp[k] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(w[i], w[i + 2]));
        lp[k] = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(w[i] - (float)hp[k][0],
                                                                       w[i + 2] - (float)hp[k][1]));
      }
      wh[u] = __builtin_bit_cast(half8_t, hp);
      wl[u] = __builtin_bit_cast(half8_t, lp);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const half8_t va = v_frag(cur.v[0][k], cur.v[1][k]);
      const half8_t vb = v_frag(cur.v[0][k] >> 4, cur.v[1][k] >> 4);
#pragma unroll
      for (int u = 0; u < NSUB; ++u) {
        acc[u][2 * k] = mfma(wh[u], va, acc[u][2 * k]);
        acc[u][2 * k + 1] = mfma(wh[u], vb, acc[u][2 * k + 1]);
        acc[u][2 * k] = mfma(wl[u], va, acc[u][2 * k]);
        acc[u][2 * k + 1] = mfma(wl[u], vb, acc[u][2 * k + 1]);
      }
    }
    cur = nxt;
  }

  // the four waves' sums: lane (r, g), register i holds row 4 g + i, channel 16 t + r
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
  for (int e = tid; e < NSUB * 512; e += kThreads) {
    const int u = e >> 9, hh = (e & 511) / HD, ch = e & (HD - 1), row = (ch >> 5) * HPS + hh;
    const int v = v0 + u * HPS + hh;
    if (v >= V) continue;
    float mx = lm[0][u][row].x, o = 0.f, ls = 0.f;
#pragma unroll
    for (int k = 1; k < 4; ++k) mx = fmaxf(mx, lm[k][u][row].x);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 ml = lm[k][u][row];
      const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
      o = fmaf(w, lo_[k][u][e & 511], o);
      ls = fmaf(w, ml.y, ls);
    }
    out[v * RS + ch] = o;
    if ((ch & 31) == 0) *(float2 *)(out + v * RS + HD + 2 * (ch >> 5)) = make_float2(mx, ls);
  }
}

// One workgroup per query row: the records joined in split order.
template <int HD>
__global__ __launch_bounds__(HD) void kv4_merge_kernel(Kv4Cache c, Kv4Attn a,
                                                       const float *__restrict__ rec, int S) {
  constexpr int RS = record_floats<HD>();
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int v = blockIdx.x, grp = c.nh / c.nkv, V = a.rows * grp, ch = threadIdx.x;
  const int filled = kv4_filled(c, s, a.rows);
  if (filled < 0) return;
  const Splits sp = kv4_splits(filled + a.rows, S);
  const float *r = rec + (list * S * V + v) * RS;
  const int64_t step = (int64_t)V * RS;
  const int ml = HD + 2 * (ch >> 5);
  float m = -INFINITY;
  for (int k = 0; k < sp.n; ++k) m = fmaxf(m, r[k * step + ml]);
  float l = 0.f, o = 0.f;
  for (int k = 0; k < sp.n; ++k) {
    const float mk = r[k * step + ml];
    const float w = mk == -INFINITY ? 0.f : exp2f(mk - m);
    l = fmaf(w, r[k * step + ml + 1], l);
    o = fmaf(w, r[k * step + ch], o);
  }
  a.out[(s * a.rows + v / grp) * a.ldo + (list % c.nkv * grp + v % grp) * HD + ch] = o / l;
}

// The attention weights of a list's slots, a thread per slot: scores of every query row
// against the row's log-sum-exp (from block 0 of its records).
template <int HD>
__global__ __launch_bounds__(kThreads) void kv4_weights_kernel(Kv4Cache c, Kv4Attn a,
                                                               const float *__restrict__ rec,
                                                               const float *__restrict__ scores,
                                                               int S) {
  constexpr int RS = record_floats<HD>();
  __shared__ float lse[kThreads];
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int grp = c.nh / c.nkv, V = a.rows * grp, tid = threadIdx.x;
  const int filled = kv4_filled(c, s, a.rows);
  const int t = blockIdx.x * kThreads + tid;
  if (filled < 0 || (int)(blockIdx.x * kThreads) >= filled + a.rows) return;
  const Splits sp = kv4_splits(filled + a.rows, S);
  float sum = 0.f;
  for (int v0 = 0; v0 < V; v0 += kThreads) {
    __syncthreads();
    if (v0 + tid < V) {
      const float *r = rec + (list * S * V + v0 + tid) * RS + HD;
      const int64_t step = (int64_t)V * RS;
      float m = -INFINITY, l = 0.f;
      for (int k = 0; k < sp.n; ++k) m = fmaxf(m, r[k * step]);
      for (int k = 0; k < sp.n; ++k) {
        const float mk = r[k * step];
        l = fmaf(mk == -INFINITY ? 0.f : exp2f(mk - m), r[k * step + 1], l);
      }
      lse[tid] = m + log2f(l);
    }
    __syncthreads();
    for (int v = v0; v < min(V, v0 + kThreads); ++v)
      if (t <= filled + v / grp) sum += exp2f(scores[(list * V + v) * c.slots + t] - lse[v - v0]);
  }
  if (t < filled + a.rows) {
    float *w = c.weights + list * c.slots + t;
    *w = a.weights_mode == 2 ? *w + sum : sum;
  }
}

int splits(int64_t lists, int slots) {
  const int64_t most = (slots + 127) / 128;
  const int64_t want = (768 + lists - 1) / lists;
  return (int)(want < most ? want : most);
}

int64_t record_bytes(int64_t lists, int V, int hd, int S) {
  return lists * S * V * (int64_t)(hd + hd / 16) * 4;
}

template <int HD>
hipError_t launch(const Kv4Cache &c, const Kv4Attn &a, hipStream_t s) {
  const int64_t lists = (int64_t)c.n_seq * c.nkv;
  const int V = a.rows * (c.nh / c.nkv), S = splits(lists, c.slots);
  float *rec = (float *)a.work;
  float *scores =
      a.weights_mode ? (float *)((char *)a.work + record_bytes(lists, V, HD, S)) : nullptr;
  constexpr int HPS = 512 / HD, NSUB = HD == 256 ? 1 : 2;
  const bool two = NSUB == 2 && V > HPS;
  const int rows = two ? 2 * HPS : HPS, nz = (V + rows - 1) / rows;
  const bool inside = a.store && a.rows == 1 && nz == 1;  // one workgroup stores the one row
  if (a.store && !inside) {
    const hipError_t e =
        launch_kv4_append(c, a.qkv, a.ldq, (int64_t)c.n_seq * a.rows, nullptr, s);
    if (e != hipSuccess) return e;
  }
  const dim3 grid((unsigned)S, (unsigned)lists, (unsigned)nz);
  if (two)
    hipLaunchKernelGGL((kv4_attention_kernel<HD, NSUB>), grid, dim3(kThreads), 0, s, c, a, rec,
                       scores, S, inside);
  else
    hipLaunchKernelGGL((kv4_attention_kernel<HD, 1>), grid, dim3(kThreads), 0, s, c, a, rec, scores,
                       S, inside);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kv4_merge_kernel<HD>, dim3((unsigned)V, (unsigned)lists), dim3(HD), 0, s, c, a,
                     rec, S);
  e = hipGetLastError();
  if (e != hipSuccess || !a.weights_mode) return e;
  hipLaunchKernelGGL(kv4_weights_kernel<HD>,
                     dim3((unsigned)((c.slots + kThreads - 1) / kThreads), (unsigned)lists),
                     dim3(kThreads), 0, s, c, a, rec, scores, S);
  return hipGetLastError();
}

}  // namespace

int64_t kv4_attention_work_bytes(int rows, bool weights, int n_seq, int nh, int nkv, int hd,
                                 int slots) {
  const int64_t lists = (int64_t)n_seq * nkv;
  const int V = rows * (nh / nkv);
  const int64_t r = record_bytes(lists, V, hd, splits(lists, slots));
  return r + (weights ? lists * V * slots * 4 : 0);
}

hipError_t launch_kv4_attention(const Kv4Cache &c, const Kv4Attn &a, hipStream_t s) {
  if (c.hd == 64) return launch<64>(c, a, s);
  if (c.hd == 128) return launch<128>(c, a, s);
  return launch<256>(c, a, s);
}

}  // namespace gguf

// Attention of one new row per sequence over the KV cache in pages.
//
// The slots of a (sequence, KV head) are split over workgroups; each writes, per query head, a
// record of its partial softmax, and paged_merge_kernel joins them in split order (so the result
// does not depend on timing).
#include <type_traits>

#include "paged.hpp"

namespace gguf {

namespace {

constexpr int kUnit = 32;  // slots that a wave takes at a time

// log2(e) / sqrt(head_dim) as two floats: one alone would be off by up to 2^-25, and that times
// a score is the relative error of its probability.
template <int HD>
struct ScoreScale {
  static constexpr double v = 1.4426950408889634074 / (HD == 64 ? 8.0 : (HD == 128 ? 11.313708498984760390 : 16.0));
  static constexpr float hi = (float)v, lo = (float)(v - (double)hi);
};

// A record: sum of p v per channel, then the maximum m that its p are relative to (in log2 units)
// and the sum of its p.
template <int HD>
constexpr int record_floats() {
  return HD + 4;
}

// The slots in use before the call, or -1 if the sequence takes no part (or 0 .. if only the page
// of its new row can tell).
__device__ __forceinline__ int filled_of(const PagedCache &c, int64_t s) {
  const int64_t n = steady(c.lengths + s);
  return n < 0 || n >= paged_end(c, s) ? -1 : (int)n;
}
// The page of the new row, or -1.
__device__ __forceinline__ int32_t page_of(const PagedCache &c, int64_t s, int slot) {
  const int32_t p = steady(c.tables + s * c.columns + (slot >> c.shift));
  return (uint32_t)p < (uint32_t)c.n_pages ? p : -1;
}

// How the units of a list are cut: `per` for each workgroup, `n` of them at most S.  Every workgroup
// of the call gets about the same number: all lists' units over `wgs` workgroups, in whole turns of a
// workgroup's W waves, and no fewer than eight.  But for S, which goes by the number of lists (`plan`):
// a sequence much longer than the others is on S workgroups a list, each with more than the others'.
// 130000 slots beside 31 sequences of 300 take 174 us, alone 97.
constexpr int kLeastUnits = 8;
struct Cut {
  int S, wgs, W;
};
struct Splits {
  int per, n;
};
__device__ __forceinline__ int units_of(int filled) {
  return filled < 0 ? 0 : filled / kUnit + 1;
}
__device__ __forceinline__ Splits splits_of(int units, int fair, const Cut &k) {
  const int most = (max(max(fair, kLeastUnits), (units + k.S - 1) / k.S) + k.W - 1) / k.W * k.W;
  const int n = (units + most - 1) / most;
  // alike, in whole turns: the last one is not left with a few units
  const int per = n > 1 ? ((units + n - 1) / n + k.W - 1) / k.W * k.W : most;
  return {per, (units + per - 1) / per};
}
// The fair share: a wave's lanes add the sequences.
__device__ __forceinline__ int fair_share(const PagedCache &c, const Cut &k) {
  int sum = 0;
  if (c.n_seq == 1) {
    sum = units_of(filled_of(c, 0));
  } else {
    for (int s = threadIdx.x & 63; s < c.n_seq; s += 64) sum += units_of(filled_of(c, s));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    sum = __builtin_amdgcn_readfirstlane(sum);
  }
  return (int)(((int64_t)sum * c.nkv + k.wgs - 1) / k.wgs);
}
// Workgroup `item` of the call: sequences in order, within one the splits in order, each for
// every KV head.
struct Item {
  int s, kvh, split, filled;
  Splits sp;
};
__device__ __forceinline__ bool item_of(const PagedCache &c, int item, const Cut &k, Item &it) {
  const int fair = fair_share(c, k);
  if (c.n_seq == 1) {
    it.s = 0;
    it.filled = filled_of(c, 0);
    it.sp = splits_of(units_of(it.filled), fair, k);
    it.split = item / c.nkv;
    it.kvh = item - it.split * c.nkv;
    return it.filled >= 0 && it.split < it.sp.n;
  }
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
    const int filled = s0 + lane < c.n_seq ? filled_of(c, s0 + lane) : -1;
    const Splits sp = splits_of(units_of(filled), fair, k);
    const int run = lanes_before(sp.n);
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

__device__ __forceinline__ float4_t mfma(uint4 a, uint4 b, float4_t c, std::false_type) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a),
                                                __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ float4_t mfma(uint4 a, uint4 b, float4_t c, std::true_type) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8_t, a),
                                                 __builtin_bit_cast(bhalf8_t, b), c, 0, 0, 0);
}

// 16 bytes; STREAM: past the caches (`plan` says when).  No other wave of the list reads them; those of
// sequences that share the page do.
template <bool STREAM>
__device__ __forceinline__ uint4 load16(const uint16_t *p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  if (STREAM) return __builtin_bit_cast(uint4, __builtin_nontemporal_load((const u32x4 *)p));
  return *(const uint4 *)p;
}

// That of the lane N to the left in its 16, cyclically.
template <int N>
__device__ __forceinline__ float ror16(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xF, 0xF, true));
}

// Eight values as a matrix operand's lane.  Column r of the matrix cores' 16 holds query head r % C,
// part r / C of its values: f16 parts hi + lo, 22 bits; bf16 parts hi + mid + lo, 24 bits, where C = 8
// leaves lo for a second operand.
template <bool BF, int C>
struct Parts {
  static constexpr int N = BF && C == 8 ? 2 : 1;  // operands
  uint4 w[N];
  __device__ __forceinline__ void make(const float (&x)[8], int part) {
    if constexpr (!BF) {
      half8_t h;
      const float sel = part ? -1.f : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const half_t hi = (half_t)x[i];
        h[i] = (half_t)fmaf((float)hi, sel, x[i]);
      }
      w[0] = __builtin_bit_cast(uint4, h);
    } else {
      bhalf8_t a, b;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bhalf_t hi = (bhalf_t)x[i];
        const float rest = x[i] - (float)hi;
        const bhalf_t mid = (bhalf_t)rest;
        const float last = rest - (float)mid;
        if constexpr (C == 8) {
          a[i] = part ? mid : hi;
          b[i] = (bhalf_t)(part ? 0.f : last);
        } else {
          a[i] = (bhalf_t)(part == 0 ? x[i] : (part == 1 ? rest : (part == 2 ? last : 0.f)));
        }
      }
      w[0] = __builtin_bit_cast(uint4, a);
      if constexpr (C == 8) w[N - 1] = __builtin_bit_cast(uint4, b);
    }
  }
};
// The sum of a head's parts, in each of its columns.
template <bool BF, int C>
__device__ __forceinline__ float all_parts(float v) {
  v += ror16<8>(v);
  if constexpr (BF && C == 4) v += ror16<4>(v);
  return v;
}

// A workgroup takes one list and one range of its units of 32 slots; its waves take the range's
// units in turn and join at the end.  Nothing but registers carries a unit through:
// - Scores: v_mfma_f32_16x16x32 with the slots' K rows as A and the queries as B, each head's parts
//   in columns of their own (Parts), which rotations within 16 lanes add.  Row m of A's half t holds
//   slot 8 (m / 4) + 4 t + m % 4, so that lane (r, g) = (lane % 16, lane / 16) of the accumulators
//   has the scores of slots 8 g .. 8 g + 7.
// - Output: that is the B layout of V . P^T, with V's channels as A, 16 bytes of a block's channel
//   a lane; a lane's accumulators are of one head, and its p's scale is its own.
// - p = 2^(score - m) with a running m, raised where a p would pass 2^15: to the largest score
//   less 10, so that p's f16 parts keep 22 bits down to 2^-13 of the largest.
// - K's registers take the next unit as soon as its scores are made, V's after its products: 16 KB
//   of 128 channels in flight per wave, three waves per SIMD.
// Bound: HBM (4 head_dim bytes per slot and list) where lists are long: 130000 slots of 8 lists, 128
// channels, 533 MB: 89 us, 6.0 TB/s (a 1 GB copy reads and writes 4.7 together); 32 sequences of 37 ..
// 8191 slots, 475 MB: 98, 4.8 TB/s, the uneven ends of their lists.  A short list waits for its chain of
// loads (length, page, rows): 300 slots 9.0 us.
template <int HD, bool BF, int C, int W, int WPS, bool STREAM>
__global__ __launch_bounds__(64 * W, WPS) void paged_attention_kernel(PagedCache c, PagedAttn a,
                                                                      float *__restrict__ rec,
                                                                      Cut cut) {
  constexpr int NB = HD / 32, CT = HD / 16, RS = record_floats<HD>(), half = HD / 2;
  constexpr int NP = Parts<BF, C>::N;
  constexpr bool kInLds = HD == 256;  // the queries are read again each turn
  constexpr std::bool_constant<BF> bf{};
  constexpr float kLift = 10.f, kMost = 15.f;
  __shared__ __align__(16) float o_[W][8][HD];  // per wave and head its sums
  __shared__ float2 ml_[W][8];
  __shared__ uint4 q_[NB][NP][64];  // queries: per block and operand
  __shared__ float qc[16];
  __shared__ __align__(16) uint16_t fresh[2][HD];  // the new row's K and V
  Item it;
  if (!item_of(c, blockIdx.x, cut, it)) return;
  it.s = __builtin_amdgcn_readfirstlane(it.s);  // all known uniform from here on
  it.kvh = __builtin_amdgcn_readfirstlane(it.kvh);
  it.split = __builtin_amdgcn_readfirstlane(it.split);
  it.filled = __builtin_amdgcn_readfirstlane(it.filled);
  it.sp.per = __builtin_amdgcn_readfirstlane(it.sp.per);
  it.sp.n = __builtin_amdgcn_readfirstlane(it.sp.n);
  const int64_t s = it.s;
  const int kvh = it.kvh, grp = c.nh / c.nkv, filled = it.filled;
  const Splits sp = it.sp;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int32_t *table = c.tables + s * c.columns;
  const int32_t own_page = page_of(c, s, filled);
  if (own_page < 0) return;
  const int unit0 = it.split * sp.per, unit1 = min(unit0 + sp.per, units_of(filled));
  const bool stores = filled / kUnit < unit1;  // the last range has the new row
  const float *row = a.qkv + s * a.ldq;

  // the two pages of a unit's blocks, and where their lists begin
  const int to_block = c.shift - 4, in_page = (c.page >> 4) - 1;
  auto ids = [&](int unit, int &p0, int &p1) {
    const int b0 = 2 * unit, b1 = b0 + 1;
    p0 = steady(table + min(b0 >> to_block, c.columns - 1));
    p1 = steady(table + min(b1 >> to_block, c.columns - 1));
  };
  auto known = [&](int p) { return (uint32_t)p < (uint32_t)c.n_pages; };
  const int64_t page_values = (int64_t)2 * c.nkv * c.page * HD;
  const int row_in = 8 * ((r >> 2) & 1) + (r & 3);  // of K's half t: + 4 t
  const int list_k = kvh * c.page * HD, list_v = (c.nkv + kvh) * c.page * HD;
  uint4 kf[2][NB], vf[CT];
  auto load_k = [&](int unit, int p0, int p1) {
    const int b = 2 * unit + (r >> 3);
    const int64_t p = r >> 3 ? (known(p1) ? p1 : 0) : (known(p0) ? p0 : 0);
    const uint16_t *k = c.kv + p * page_values + (list_k + ((b & in_page) * 16 + row_in) * HD + 8 * g);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < NB; ++i) kf[t][i] = load16<STREAM>(k + 4 * t * HD + 32 * i);
  };
  auto load_v = [&](int unit, int p0, int p1) {
    const int b = 2 * unit + (g >> 1);
    const int64_t p = g >> 1 ? (known(p1) ? p1 : 0) : (known(p0) ? p0 : 0);
    const uint16_t *v =
        c.kv + p * page_values + (list_v + (b & in_page) * 16 * HD + 16 * r + 8 * (g & 1));
#pragma unroll
    for (int i = 0; i < CT; ++i) vf[i] = load16<STREAM>(v + 256 * i);
  };

  // What comes before the barrier is requested before the unit, since loads return in order.  The
  // first wave makes the queries: lane (r, g) channels 32 i + 8 g + 0 .. 7 of head r % C, whose RoPE
  // partners are the same lane's of block i +- NB / 2.  The second one makes the new row, for its
  // page and for the workgroup.
  constexpr int LANES = Kv4Row<HD>::LANES, SIDE = 64 / LANES, N = (2 + SIDE - 1) / SIDE;
  const int h = r % C, rq = lane % LANES;
  const float *cr = c.cs + (int64_t)filled * half, *sr = c.sn + (int64_t)filled * half;
  float4 xq[2 * NB], cq[NB], sq[NB];
  Kv4Row<HD> own[N];
  auto request = [&]() {
    const float *x = row + (int64_t)(kvh * grp + (h < grp ? h : 0)) * HD + 8 * g;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) xq[i] = *(const float4 *)(x + 32 * (i >> 1) + 4 * (i & 1));
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      cq[i] = *(const float4 *)(cr + 8 * g + 32 * (i >> 1) + 4 * (i & 1));
      sq[i] = *(const float4 *)(sr + 8 * g + 32 * (i >> 1) + 4 * (i & 1));
    }
  };
  constexpr bool kFirst = HD < 256;  // of 256 channels there are no registers for both
  if (kFirst && wave == 0) request();
  if (stores && wave == 1) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int u = min(n * SIDE + lane / LANES, 1);
      own[n].load(row + (int64_t)(c.nh + u * c.nkv + kvh) * HD, rq);
      own[n].load_turn(cr, sr, rq);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  // from the last unit down: the new row's is some wave's first
  int unit = unit1 - 1 - wave, p0 = 0, p1 = 0, n0 = 0, n1 = 0;
  auto begin = [&]() {
    if (unit < unit0) return;
    ids(unit, p0, p1);
    load_k(unit, p0, p1);
    load_v(unit, p0, p1);
    ids(max(unit - W, unit0), n0, n1);
  };
  if (kFirst) begin();
  __builtin_amdgcn_sched_barrier(0);
  if (wave == 0) {
    if (!kFirst) request();
    auto at = [](const float4 *w, int i) { return (&w[i >> 2].x)[i & 3]; };
    float y[NB][8], mx = 0.f;
#pragma unroll
    for (int i = 0; i < NB / 2; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x1 = at(xq, 8 * i + j), x2 = at(xq, 8 * (i + NB / 2) + j);
        const float cv = at(cq, 8 * i + j), sv = at(sq, 8 * i + j);
        const float a1 = h < grp ? x1 * cv - x2 * sv : 0.f, a2 = h < grp ? x2 * cv + x1 * sv : 0.f;
        y[i][j] = fmaf(a1, ScoreScale<HD>::hi, a1 * ScoreScale<HD>::lo);
        y[i + NB / 2][j] = fmaf(a2, ScoreScale<HD>::hi, a2 * ScoreScale<HD>::lo);
        mx = fmaxf(mx, fmaxf(fabsf(y[i][j]), fabsf(y[i + NB / 2][j])));
      }
    mx = max_xor32(max_xor16(mx));
    const int e = BF ? 0 : stage_exp(mx);
    const float up = pow2f(e);
    if (g == 0) qc[r] = pow2f(-e);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) y[i][j] *= up;
      Parts<BF, C> w;
      w.make(y[i], r / C);
#pragma unroll
      for (int k = 0; k < NP; ++k) q_[i][k][lane] = w.w[k];
    }
  } else if (stores && wave == 1) {
    const int j = filled & (c.page - 1);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int u = n * SIDE + lane / LANES;
      float y[4];
      paged_turn<HD>(own[n], rq, u == 0, y);
      const uint2 w = paged_round<BF>(y);
      if (u == 0) {
        *(uint2 *)(fresh[0] + 4 * rq) = w;
        *(uint2 *)(c.kv + paged_k_at(c, own_page, kvh, j) + 4 * rq) = w;
      } else if (u == 1) {
        *(uint2 *)(fresh[1] + 4 * rq) = w;
        uint16_t *v = c.kv + paged_v_at(c, own_page, kvh, j) + 64 * rq;
        v[0] = (uint16_t)w.x;
        v[16] = (uint16_t)(w.x >> 16);
        v[32] = (uint16_t)w.y;
        v[48] = (uint16_t)(w.y >> 16);
      }
    }
  }
  if (!kFirst) begin();
  __syncthreads();
  uint4 qf[kInLds ? 1 : NB][NP];
  if (!kInLds)
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int k = 0; k < NP; ++k) qf[i][k] = q_[i][k][lane];
  const float f = qc[r];  // log2 units per unit of an accumulated score
  if (stores && unit == filled / kUnit) {
    const int j = filled % kUnit, in = j & 15;
    if (j >> 4 == r >> 3) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (in == row_in + 4 * t)
#pragma unroll
          for (int i = 0; i < NB; ++i) kf[t][i] = *(const uint4 *)(fresh[0] + 32 * i + 8 * g);
    }
    if (j >> 3 == g) {
      const int e = j & 7, sh = 16 * (e & 1);
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        const uint32_t x = (uint32_t)fresh[1][16 * i + r] << sh, keep = ~(0xFFFFu << sh);
        if (e < 2) vf[i].x = (vf[i].x & keep) | x;
        else if (e < 4) vf[i].y = (vf[i].y & keep) | x;
        else if (e < 6) vf[i].z = (vf[i].z & keep) | x;
        else vf[i].w = (vf[i].w & keep) | x;
      }
    }
  }

  int ql = lane;  // made anew every turn: the queries are read from LDS there, not kept
  float4_t acc[CT];
  float m = -INFINITY, l = 0.f;  // p = 2^(score - m)
#pragma unroll
  for (int i = 0; i < CT; ++i) acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
  for (; unit >= unit0; unit -= W) {
    if (kInLds) asm volatile("" : "+v"(ql));
    float y[8];
    {
      float4_t sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int k = NP - 1; k >= 0; --k) {
          const uint4 q = kInLds ? q_[i][k][ql] : qf[kInLds ? 0 : i][k];
          sc[0] = mfma(kf[0][i], q, sc[0], bf);
          sc[1] = mfma(kf[1][i], q, sc[1], bf);
        }
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = all_parts<BF, C>(sc[j >> 2][j & 3]);
    }
    const int next = max(unit - W, unit0);  // the last one: unused
    load_k(next, n0, n1);
    // slots that are not seen: past the new row, or without a page
    const bool masked = (unit + 1) * kUnit > filled + 1 || !known(p0) || !known(p1);
    const int seen = known(g >> 1 ? p1 : p0) ? filled + 1 - (unit * kUnit + 8 * g) : 0;  // of the lane's
    if (masked) {
#pragma unroll
      for (int i = 0; i < CT; ++i) {  // whatever they hold must not meet a p of zero
        uint32_t x[4] = {vf[i].x, vf[i].y, vf[i].z, vf[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x[k] = seen >= 2 * k + 2 ? x[k] : (seen == 2 * k + 1 ? x[k] & 0xFFFFu : 0u);
        vf[i] = make_uint4(x[0], x[1], x[2], x[3]);
      }
    }
    float p[8], sum;
    auto weigh = [&]() {
      bool over = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float t = fmaf(y[j], f, -m);
        if (masked && j >= seen) t = -INFINITY;
        over |= !(t <= kMost);
        p[j] = __builtin_amdgcn_exp2f(t);
      }
      sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      return over;
    };
    if (__any(weigh())) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!masked || j < seen) top = fmaxf(top, y[j] * f);
      top = max_xor32(max_xor16(top)) - kLift;
      const float n = fmaxf(m, top);
      const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - n);
      if (n != -INFINITY) {  // else nothing has been seen yet
        m = n;
        l *= al;
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[i][k] *= al;
      }
      weigh();
    }
    l += sum;
    Parts<BF, C> pf;
    pf.make(p, r / C);
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int k = NP - 1; k >= 0; --k) acc[i] = mfma(vf[i], pf.w[k], acc[i], bf);
    load_v(next, n0, n1);
    p0 = n0;
    p1 = n1;
    ids(max(next - W, unit0), n0, n1);
  }

  // the waves' sums: lane (r, g), register k of i: channel 16 i + 4 g + k, head r % C
  const float ls = sum_xor32(sum_xor16(l));
  if (g == 0 && r < C) ml_[wave][r] = make_float2(m, ls);
#pragma unroll
  for (int i = 0; i < CT; ++i) {
    float4_t x = acc[i];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = all_parts<BF, C>(x[k]);
    if (r < grp) *(float4_t *)&o_[wave][r][16 * i + 4 * g] = x;
  }
  __syncthreads();
  for (int e = tid; e < grp * (HD / 4); e += 64 * W) {
    const int h = e / (HD / 4), ch = e % (HD / 4) * 4;
    float mx = ml_[0][h].x, sum = 0.f;
    float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 1; k < W; ++k) mx = fmaxf(mx, ml_[k][h].x);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float2 ml = ml_[k][h];
      const float w = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mx);
      const float4_t x = *(const float4_t *)&o_[k][h][ch];
#pragma unroll
      for (int n = 0; n < 4; ++n) o[n] = fmaf(w, x[n], o[n]);
      sum = fmaf(w, ml.y, sum);
    }
    if (sp.n == 1) {  // nothing to join
      float *to = a.out + s * a.ldo + (int64_t)(kvh * grp + h) * HD + ch;
      *(float4 *)to = make_float4(o[0] / sum, o[1] / sum, o[2] / sum, o[3] / sum);
    } else {
      float *to = rec + (((s * c.nkv + kvh) * cut.S + it.split) * grp + h) * RS;
      *(float4_t *)(to + ch) = o;
      if (ch == 0) *(float2 *)(to + HD) = make_float2(mx, sum);
    }
  }
}

// One workgroup per query head of a list with several splits: their records joined, G groups of
// HD / 4 threads taking every G-th record, then the groups in order.  96 records of each of 32 heads
// 6.1 us, three of each of 1024 5.1.
template <int HD>
constexpr int kMergeThreads = HD < 128 ? 256 : 2 * HD;
template <int HD>
__global__ __launch_bounds__(kMergeThreads<HD>) void paged_merge_kernel(PagedCache c, PagedAttn a,
                                                                        const float *__restrict__ rec,
                                                                        Cut cut) {
  constexpr int RS = record_floats<HD>(), Q = HD / 4, G = kMergeThreads<HD> / Q;
  __shared__ float4 o_[G][Q];
  __shared__ float2 ml_[G][Q];
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int h = blockIdx.x, grp = c.nh / c.nkv;
  const int q = threadIdx.x % Q, gi = threadIdx.x / Q;
  const int filled = filled_of(c, s);
  if (filled < 0 || page_of(c, s, filled) < 0) return;
  const Splits sp = splits_of(units_of(filled), fair_share(c, cut), cut);
  if (sp.n == 1) return;
  const float *r = rec + (list * cut.S * grp + h) * RS;
  const int64_t step = (int64_t)grp * RS;
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
      ml[j] = *(const float2 *)(rk + HD);
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
  *(float4 *)(a.out + s * a.ldo + (int64_t)(list % c.nkv * grp + h) * HD + 4 * q) =
      make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
}

// How a call is cut: W waves per workgroup, `wgs` workgroups at a time on the GPU, a list in S of
// them at most.
struct Plan {
  Cut cut;
  int64_t lists;
  bool stream;
};
Plan plan(int page, int64_t columns, int n_seq, int nkv, int hd) {
  Plan p;
  p.lists = (int64_t)n_seq * nkv;
  const int64_t units = (columns * page + kUnit - 1) / kUnit;
  // a list of two turns is not cut: one launch, and nothing to join.  What counts is what a table holds,
  // which the host knows: 300 slots 8.9 us of a table of 512 slots, 11.3 of one of 2048.
  const bool whole = units <= 16;
  // (300 slots: 4 waves and the join's launch 7.8 + 2.9 us, 8 waves 9.0)
  p.cut.W = whole && units > 8 ? 8 : 4;
  // Workgroups at a time, as many as fit (us, 32 sequences of 37 .. 8191 slots / 32 of 4000 / 130000
  // slots): 512 109 / 101 / 99, 768 104 / 104 / 100, 1024 105 / 106 / 104, 1536 106 / 116 / 115.
  p.cut.wgs = hd == 256 ? 512 : 768;
  const int64_t most = whole ? 1 : (units + kLeastUnits - 1) / kLeastUnits;
  // sequences of different lengths: up to four times the workgroups that equal ones would take
  const int64_t want = (4 * p.cut.wgs + p.lists - 1) / p.lists;
  p.cut.S = (int)(want < most ? want : most);
  // Tables of more than the last cache holds (256 MB) are read past the caches (us, 8 lists a sequence,
  // cached / past them): 130000 slots 101 / 93, 32 sequences of 4000 103 / 96.  What the caches still
  // hold from the call before is read faster from there: a list of 6000 slots 11.6 / 13.9.  That goes
  // for large tables with little in them, and with pages that sequences share, too, which the rule does
  // not see: 32 sequences of 300 slots 17.8 / 21.1, 16 and 32 of 8100 of which 8000 are shared 50 / 61
  // and 85 / 109.
  p.stream = p.lists * columns * page * hd * 4 > (int64_t)256 << 20;
  return p;
}

template <int HD, bool BF, int C>
hipError_t launch(const PagedCache &c, const PagedAttn &a, hipStream_t s) {
  const Plan p = plan(c.page, c.columns, c.n_seq, c.nkv, HD);
  float *rec = (float *)a.work;
  // No call has more items than wgs + lists (every list but for its last workgroup gets whole
  // shares).
  const int64_t most = p.lists * p.cut.S, items = most < p.cut.wgs + p.lists ? most : p.cut.wgs + p.lists;
  const dim3 grid((unsigned)items), block(64 * p.cut.W);
  constexpr int WPS = HD == 256 ? 2 : 3;
  auto go = [&](auto *kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, c, a, rec, p.cut); };
  if (p.cut.W == 8)
    go(paged_attention_kernel<HD, BF, C, 8, 2, false>);
  else if (p.stream)
    go(paged_attention_kernel<HD, BF, C, 4, WPS, true>);
  else
    go(paged_attention_kernel<HD, BF, C, 4, WPS, false>);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.cut.S == 1) return e;
  hipLaunchKernelGGL(paged_merge_kernel<HD>, dim3((unsigned)(c.nh / c.nkv), (unsigned)p.lists),
                     dim3(kMergeThreads<HD>), 0, s, c, a, rec, p.cut);
  return hipGetLastError();
}
template <int HD>
hipError_t launch(const PagedCache &c, const PagedAttn &a, hipStream_t s) {
  if (!c.bf16) return launch<HD, false, 8>(c, a, s);
  return c.nh / c.nkv <= 4 ? launch<HD, true, 4>(c, a, s) : launch<HD, true, 8>(c, a, s);
}

}  // namespace

int64_t paged_attention_work_bytes(int page, int64_t columns, int n_seq, int nh, int nkv, int hd) {
  const Plan p = plan(page, columns, n_seq, nkv, hd);
  return (p.cut.S > 1 ? p.lists * p.cut.S * (nh / nkv) * (int64_t)(hd + 4) * 4 : 0) + 16;
}

hipError_t launch_paged_attention(const PagedCache &c, const PagedAttn &a, hipStream_t s) {
  if (c.hd == 64) return launch<64>(c, a, s);
  if (c.hd == 128) return launch<128>(c, a, s);
  return launch<256>(c, a, s);
}

}  // namespace gguf

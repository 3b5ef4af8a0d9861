// The 4-bit KV cache: storing rows, reading them back, eviction.
#include <type_traits>

#include "kv4.hpp"

namespace gguf {

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// Storing rows: a wave takes one row and N units (K or V of a KV head, 256 / HD of them side by
// side); four neighbouring rows per workgroup, which mostly share the four slots that V's words
// hold, so that their bytes meet in one L2.  Bound: vector instructions, then the chain of loads
// that finds a row's place.  3716 packed rows of five sequences, 8 heads of 128: a channel per
// lane 16.8 us (300 instructions for K and V of a head), four channels per lane 13.9, with the
// vector unit busy 73 % of the time; the 565000 writes that reach the L2, most of them V's bytes,
// leave it as 87000.
// ---------------------------------------------------------------------------
template <int HD, int N>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(Kv4Cache c,
                                                              const float *__restrict__ qkv,
                                                              int64_t ldq, uint32_t n_rows,
                                                              const int64_t *__restrict__ starts,
                                                              bool whole) {
  constexpr int LANES = Kv4Row<HD>::LANES, SIDE = 64 / LANES;
  const int lane = threadIdx.x & 63, q = lane % LANES;
  const uint32_t r = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (r >= n_rows) return;
  // unit u: KV head u / 2, K or V; in qkv after the queries all of K, then all of V
  const int u0 = blockIdx.y * N * SIDE + lane / LANES, units = 2 * c.nkv;
  const float *x = qkv + r * ldq + (int64_t)c.nh * HD;
  Kv4Row<HD> row[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {  // past the last unit: the last again, not stored
    const int u = min(u0 + i * SIDE, units - 1);
    row[i].load(x + (int64_t)((u & 1) * c.nkv + (u >> 1)) * HD, q);
  }
  uint32_t s;
  int64_t i, last;  // the row of s, and the one that has to fit for it to be stored
  if (starts) {
    if (r < starts[0] || r >= starts[c.n_seq]) return;
    uint32_t lo = 0, hi = c.n_seq;  // starts[lo] <= r < starts[hi]
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) >> 1;
      if (starts[mid] <= r)
        lo = mid;
      else
        hi = mid;
    }
    s = lo;
    if (starts[lo] < -(int64_t)c.slots) return;  // r would be behind every slot, and i not fit 64 bits
    last = i = r - starts[lo];
  } else {
    const uint32_t per = n_rows / (uint32_t)c.n_seq;
    s = r / per;
    i = r - s * per;
    last = whole ? per - 1 : i;
  }
  const int64_t n = c.lengths[s], p0 = c.pos[s], slot = n + i, p = p0 + i;
  if (n < 0 || n >= c.slots - last || p0 < 0 || p0 >= c.rope_rows - last) return;
  row[0].load_turn(c.cs + p * (HD / 2), c.sn + p * (HD / 2), q);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int u = u0 + k * SIDE;
    const int64_t list = (int64_t)s * c.nkv + (u >> 1);
    row[k].c = row[0].c;
    row[k].s = row[0].s;
    kv4_put_row<HD>(kv4_list(c.kv, list, c.slots, Kv4<HD>::TB), (int)slot, row[k], q, !(u & 1),
                    u < units);
    if (u < units && (u & 1) && q == 0) {
      if (c.positions) c.positions[list * c.slots + slot] = (int32_t)p;
      if (c.weights) c.weights[list * c.slots + slot] = 0.f;
    }
  }
}

// ---------------------------------------------------------------------------
// Reading rows back: a workgroup per tile of 32 slots.  Bound: the f32 rows written; 40 lists of
// up to 2000 rows of 128 channels, with the rows' storing before: 31.5 us with a float of V per
// lane, 30.0 with four, 29.4 past the caches (which hold no call's rows); 96 short lists 10.2,
// 9.6, 8.8.
// ---------------------------------------------------------------------------
template <int HD>
__global__ __launch_bounds__(kThreads) void kv4_load_kernel(const uint8_t *__restrict__ kv,
                                                            const int64_t *__restrict__ lengths,
                                                            float *__restrict__ ko,
                                                            float *__restrict__ vo,
                                                            int64_t out_slots, int n_seq, int nkv,
                                                            int slots) {
  using L = Kv4<HD>;
  constexpr int NB = L::NB;
  const int64_t list = blockIdx.y;
  const int t0 = blockIdx.x * kKv4Tile, tid = threadIdx.x;
  const int64_t n64 = lengths[list / nkv % n_seq];
  const int64_t n = n64 < out_slots ? n64 : out_slots;
  if (t0 >= n || n64 > slots) return;
  const int tn = (int)(n - t0);
  const uint8_t *tile = kv4_list((uint8_t *)kv, list, slots, L::TB) + (int64_t)blockIdx.x * L::TB;
  float *kr = ko + (list * out_slots + t0) * HD, *vr = vo + (list * out_slots + t0) * HD;
  for (int w = tid; w < 32 * 4 * NB; w += kThreads) {  // a word of K codes: 8 channels of a slot
    const int j = w / (4 * NB), b = w / 4 % NB, g = w & 3;  // rows are written from end to end
    if (j >= tn) continue;
    const uint32_t q = *(const uint32_t *)(tile + j * (HD / 2) + (g * NB + b) * 4);
    const float d = (float)*(const half_t *)(tile + L::KS + ((j >> 2) * NB + b) * 8 + (j & 3) * 2);
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = d * (float)((int)((q >> (8 * i)) & 15u) - 8);
      y[i + 4] = d * (float)((int)((q >> (8 * i + 4)) & 15u) - 8);
    }
    float *o = kr + (int64_t)j * HD + 32 * b + 8 * g;
    __builtin_nontemporal_store(float4_t{y[0], y[1], y[2], y[3]}, (float4_t *)o);
    __builtin_nontemporal_store(float4_t{y[4], y[5], y[6], y[7]}, (float4_t *)(o + 4));
  }
  for (int w = tid; w < 8 * 4 * NB; w += kThreads) {  // four words of V codes: 4 slots, 8 channels
    const int q4 = w / (4 * NB), b = w / 4 % NB, n = 4 * (w & 3);
    const uint8_t *v = tile + L::VO + q4 * (2 * HD) + (n * NB + b) * 4;
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = *(const uint32_t *)(v + i * (NB * 4));
    const half4_t d = *(const half4_t *)(tile + L::VS + (q4 * NB + b) * 8);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int j = 4 * q4 + s;
      if (j < tn) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] = (float)d[s] * (float)((int)((q[i] >> (8 * s)) & 15u) - 8);
          y[i + 4] = (float)d[s] * (float)((int)((q[i] >> (8 * s + 4)) & 15u) - 8);
        }
        float *o = vr + (int64_t)j * HD + 32 * b + n;
        __builtin_nontemporal_store(float4_t{y[0], y[1], y[2], y[3]}, (float4_t *)o);
        __builtin_nontemporal_store(float4_t{y[4], y[5], y[6], y[7]}, (float4_t *)(o + 16));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Eviction: which slots stay, then the moves.
// ---------------------------------------------------------------------------
constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

// The order of the slots: larger is kept first.  NaN is 0, -0 equals +0, and a protected slot is
// above every weight, infinite ones too.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t p, int32_t from, int32_t sinks) {
  const bool first = (p >= from) | (p < sinks);  // selects, no branches
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return first ? ~0u : (w == w ? k : 0u);
}

// Work: per list the number of moves, then the slots given up below `keep` (holes) and the
// kept ones from `keep` on, both ascending.
__device__ __forceinline__ int32_t *evict_holes(void *work, int64_t lists, int64_t list, int half) {
  return (int32_t *)work + (lists + 3) / 4 * 4 + list * 2 * half;
}

// v plus those of the lanes below it: in rows of 16 by DPP shifts, then the rows' ends.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int row_sums(int v) {
  v = dpp_add<0x111, 0xF>(v);
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  return dpp_add<0x118, 0xF>(v);
}
__device__ __forceinline__ int wave_sums(int v) {
  v = dpp_add<0x142, 0xA>(row_sums(v));  // lane 15 to row 1, 47 to row 3
  return dpp_add<0x143, 0xC>(v);         // lane 31 to rows 2 and 3
}
// The sum of v over the threads below this one, and over all of them.  Calls that follow each
// other without a barrier between take different `part`s.
__device__ __forceinline__ int block_before(int v, int *part, int &all) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int run = wave_sums(v);
  if (lane == 63) part[wave] = run;
  __syncthreads();
  static_assert(kSelWaves == 16);
  const int x = row_sums(part[lane & 15]);
  all = __builtin_amdgcn_readlane(x, 15);
  return run - v + (wave ? __builtin_amdgcn_readlane(x, wave - 1) : 0);
}

// The same number, not known to be: what is computed from it is computed where it is used, and
// not kept for all the turns of an unrolled loop.
__device__ __forceinline__ int again(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// x of the eight lanes (aligned) that this one is of, or-ed.
__device__ __forceinline__ uint32_t or8(uint32_t x) {
  x |= __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, true);   // lane ^ 1
  x |= __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, true);   // lane ^ 2
  x |= __builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, true);  // 7 - lane: the other four
  return x;
}

// One workgroup per list; a turn takes 4096 slots, four neighbouring ones per thread, and the
// keys of T turns stay in registers (a longer list is read again, segment by segment, for every
// pass).
// - The keep-th largest key by digits of 11, 11 and 10 bits: a histogram in LDS (four copies
//   for the first digit, where most keys share a few bins), then a scan from the top.  Where
//   some of the keys equal to it go, their ranks decide (ranked).
// - Ranks: the turns' four bits per thread (stays, equals) become a bitmap in LDS, of which each
//   thread takes its segment's next 4 T slots: counts are bit counts, one scan of the workgroup
//   gives all ranks.  The lists of slots are put together in LDS and written in order.
// Bound: one CU's loads and vector instructions, and for short lists the chain of barriers.  48
// lists of up to 61000 slots, with their moves: 75.5 us with ranks counted turn by turn by ballots,
// 53.4 with bitmaps, 51.6 with scans by DPP instead of shuffles; 32 lists of 2049 slots 15.0, 13.4,
// 11.2.
template <int T>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(Kv4Cache c, Kv4Evict e, int half) {
  constexpr int kBins = 2048, kTurn = 4 * kSelThreads, kSeg = T * kTurn, kMine = 4 * T;
  using Bits = std::conditional_t<T == 16, uint64_t, uint32_t>;  // of a thread's kMine slots
  __shared__ __align__(16) union {
    int hist[6][kBins];  // the first digit in four copies, the others
    struct {
      uint32_t map[2][kSeg / 32];  // stays, equals: a bit per slot of the segment
      uint16_t slot[kSeg];         // its holes, then its moves
    };
  } sh;
  __shared__ int part[2][kSelWaves], found[3];
  auto &hist = sh.hist;
  const int64_t list = blockIdx.x, lists = gridDim.x;
  const int64_t s = list / c.nkv % c.n_seq;
  const int64_t n64 = c.lengths[s];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int32_t *count = (int32_t *)e.work + list;
  const float *w = e.weights + list * c.slots;
  const int32_t *p = e.positions + list * c.slots;
  float *wo = e.weights_out + list * c.slots;
  int32_t *po = e.positions_out + list * c.slots;
  const bool cut = n64 > e.keep && n64 >= e.trigger && n64 <= c.slots;
  const int n = (int)(n64 < 0 ? 0 : (n64 < c.slots ? n64 : c.slots)), keep = (int)e.keep;
  if (!cut) {
    if (tid == 0) *count = 0;
    for (int i = tid; i < n; i += kSelThreads) {
      if (wo != w) wo[i] = w[i];
      if (po != p) po[i] = p[i];
    }
    return;
  }
  // positions are below 2^31 - 1 (the tables' rows); pos may be anything, so it is limited first
  const int64_t pos = c.pos[s], most = (int64_t)INT32_MAX + e.recent;
  const int64_t least = (int64_t)INT32_MIN + e.recent;
  const int32_t from = (int32_t)((pos < least ? least : (pos > most ? most : pos)) - e.recent);
  const int32_t sinks = (int32_t)e.sinks;
  uint32_t key[4 * T];
  int held = -1;  // the segment in `key`
  auto read = [&](int s0) {
    if (held == s0) return;
    held = s0;
    const int at = 4 * again(threadIdx.x);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const int i = s0 + t * kTurn + at;
      const int f = i < n ? i : 0;  // past the list: its first slots, not counted below
      const float4 x = *(const float4 *)(w + f);
      const int4 q = *(const int4 *)(p + f);
      key[4 * t] = evict_key(x.x, q.x, from, sinks);
      key[4 * t + 1] = evict_key(x.y, q.y, from, sinks);
      key[4 * t + 2] = evict_key(x.z, q.z, from, sinks);
      key[4 * t + 3] = evict_key(x.w, q.w, from, sinks);
      if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // 8 loads of a wave in flight at a time
    }
  };
#pragma unroll
  for (int i = 0; i < 6 * kBins / kSelThreads; ++i) ((int *)hist)[i * kSelThreads + tid] = 0;
  __syncthreads();
  uint32_t prefix = 0;
  int need = keep, alike = 0;  // of `alike` keys that share the prefix, `need` stay
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
    for (int s0 = 0; s0 < n; s0 += kSeg) {
      read(s0);
      const int at = 4 * again(threadIdx.x);
      int *h = hist[pass == 0 ? wave & 3 : pass + 3];
#pragma unroll
      for (int t = 0; t < T; ++t) {
        if (s0 + t * kTurn >= n) break;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t k = key[4 * t + j];
          if ((s0 + t * kTurn + at + j < n) &
              (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits))))
            atomicAdd(&h[(k >> shift) & ((1u << bits) - 1u)], 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();
    // bins from the top, two per thread: the first whose running count reaches `need`
    const int b0 = kBins - 1 - 2 * tid;
    const int *h = hist[pass == 0 ? 0 : pass + 3];
    int h0 = h[b0], h1 = h[b0 - 1];
    if (pass == 0) {
      h0 += hist[1][b0] + hist[2][b0] + hist[3][b0];
      h1 += hist[1][b0 - 1] + hist[2][b0 - 1] + hist[3][b0 - 1];
    }
    int all;
    const int before = block_before(h0 + h1, part[pass & 1], all);
    if (before < need && before + h0 >= need) {
      found[0] = b0;
      found[1] = need - before;
      found[2] = h0;
    } else if (before + h0 < need && before + h0 + h1 >= need) {
      found[0] = b0 - 1;
      found[1] = need - before - h0;
      found[2] = h1;
    }
    __syncthreads();
    prefix |= (uint32_t)__builtin_amdgcn_readfirstlane(found[0]) << shift;
    need = __builtin_amdgcn_readfirstlane(found[1]);
    alike = __builtin_amdgcn_readfirstlane(found[2]);
  }
  const bool ranked = need < alike;
  int32_t *holes = evict_holes(e.work, lists, list, half), *late = holes + half;
  const uint32_t lim = ranked ? prefix : prefix - 1;  // not ranked: all keys from `prefix` stay
  auto take = [&](const uint32_t *map) -> Bits {
    if constexpr (T == 16) return ((const uint64_t *)map)[tid];
    if constexpr (T == 4) return ((const uint16_t *)map)[tid];
    return map[tid >> 3] >> (4 * (tid & 7)) & 15u;
  };
  auto lowest = [](int k) -> Bits {  // k bits
    return k <= 0 ? 0 : (k >= kMine ? (Bits)(~(Bits)0 >> (8 * sizeof(Bits) - kMine)) : ((Bits)1 << k) - 1);
  };
  auto bits = [](Bits x) { return (int)__popcll(x); };
  int ties = 0, nh = 0, nl = 0;  // of the segments before
  for (int s0 = 0; s0 < n; s0 += kSeg) {
    read(s0);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      uint32_t over = 0, same = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        over |= key[4 * t + j] > lim ? 1u << j : 0u;
        same |= key[4 * t + j] == prefix ? 1u << j : 0u;
      }
      over = or8(over << (4 * (lane & 7)));
      if (ranked) same = or8(same << (4 * (lane & 7)));
      if ((lane & 7) == 0) {
        sh.map[0][t * (kTurn / 32) + (tid >> 3)] = over;
        if (ranked) sh.map[1][t * (kTurn / 32) + (tid >> 3)] = same;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    const int at = s0 + kMine * tid;
    const Bits in = lowest(n - at), low = lowest(keep - at);
    Bits stays = take(sh.map[0]) & in;
    int all, moves;
    if (ranked) {
      Bits same = take(sh.map[1]) & in;
      const int some = bits(same), k = need - ties - block_before(some, part[1], all);
      ties += all;
      if (k < some) {  // the first k of them
        Bits rest = same;
        for (int i = 0; i < k; ++i) rest &= rest - 1;
        same ^= rest;
      }
      stays |= same;
    }
    // a hole: a slot below `keep` that goes; a move: one from `keep` on that stays
    Bits hole = in & low & ~stays, move = stays & ~low;
    int rh = block_before(bits(hole), part[0], all);
    int rm = block_before(bits(move), part[1], moves) + all;
    for (; hole; hole &= hole - 1) sh.slot[rh++] = (uint16_t)(kMine * tid + __builtin_ctzll(hole));
    for (; move; move &= move - 1) sh.slot[rm++] = (uint16_t)(kMine * tid + __builtin_ctzll(move));
    __syncthreads();
    for (int i = tid; i < all; i += kSelThreads) holes[nh + i] = s0 + sh.slot[i];
    for (int i = tid; i < moves; i += kSelThreads) late[nl + i] = s0 + sh.slot[all + i];
    nh += all;
    nl += moves;
  }
  // what stays below `keep`; the holes among them are written by the moves
  if (wo != w || po != p)
    for (int i = tid; i < keep; i += kSelThreads) {
      if (wo != w) wo[i] = w[i];
      if (po != p) po[i] = p[i];
    }
  if (tid == 0) *count = nl;
}

// A wave takes 16 moves at a time, slot late[i] to slot holes[i]: all their loads are issued
// before the first store (a slot from `keep` on is never written, so the order of the waves
// does not matter).  V's bytes are four apart, a lane takes one; K goes in 16 bytes a lane.
// Bound: the lines that a slot's bytes lie in, 640 bytes read at 128 channels for its 144.  256
// lists of 15999 slots cut to 2000, about 1750 moves each: 72 us, 400 MB, 5.5 TB/s.
template <int HD>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(Kv4Cache c, Kv4Evict e, int half) {
  using L = Kv4<HD>;
  constexpr int NB = L::NB, M = 16;
  constexpr int VN = M * HD / 2 / 64, KN = (M * NB + 63) / 64, SN = M * 2 * NB / 64;
  const int64_t list = blockIdx.y, lists = gridDim.y;
  const int lane = threadIdx.x & 63;
  if (blockIdx.x == 0 && threadIdx.x == 0 && list < (int64_t)c.n_seq * c.nkv && list % c.nkv == 0) {
    const int64_t s = list / c.nkv, n = c.lengths[s];
    e.lengths_out[s] = n > e.keep && n >= e.trigger && n <= c.slots ? e.keep : n;
  }
  const int count = ((const int32_t *)e.work)[list];
  const int32_t *holes = evict_holes(e.work, lists, list, half), *late = holes + half;
  uint8_t *base = kv4_list(c.kv, list, c.slots, L::TB);
  const float *wi = e.weights + list * c.slots;
  const int32_t *pi = e.positions + list * c.slots;
  // byte offset of the tile of slot x, and of a slot within the V codes and the scales
  auto tile = [](int x) { return (uint32_t)(x / kKv4Tile) * (uint32_t)L::TB; };
  for (int i0 = (blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * M; i0 < count;
       i0 += gridDim.x * (kThreads / 64) * M) {
    const int nm = min(M, count - i0), at = i0 + min(lane & (M - 1), nm - 1);
    const int dst = holes[at], src = late[at];  // past the last move: the last one again
    uint8_t v[VN];
    uint4 k[KN];
    uint16_t sc[SN];
#pragma unroll
    for (int j = 0; j < VN; ++j) {
      const int x = j * 64 + lane, f = __shfl(src, x / (HD / 2)), b = x % (HD / 2);
      v[j] = base[tile(f) + L::VO + (f % kKv4Tile >> 2) * (2 * HD) + b * 4 + (f & 3)];
    }
#pragma unroll
    for (int j = 0; j < KN; ++j) {
      const int x = j * 64 + lane, f = __shfl(src, x / NB % M);
      k[j] = *(const uint4 *)(base + tile(f) + f % kKv4Tile * (HD / 2) + x % NB * 16);
    }
#pragma unroll
    for (int j = 0; j < SN; ++j) {
      const int x = j * 64 + lane, f = __shfl(src, x / (2 * NB)), b = x % (2 * NB);
      sc[j] = *(const uint16_t *)(base + tile(f) + (b < NB ? L::KS : L::VS) +
                                  ((f % kKv4Tile >> 2) * NB + b % NB) * 8 + (f & 3) * 2);
    }
    const float wv = wi[src];
    const int32_t pv = pi[src];
#pragma unroll
    for (int j = 0; j < VN; ++j) {
      const int x = j * 64 + lane, t = __shfl(dst, x / (HD / 2)), b = x % (HD / 2);
      if (x / (HD / 2) < nm)
        base[tile(t) + L::VO + (t % kKv4Tile >> 2) * (2 * HD) + b * 4 + (t & 3)] = v[j];
    }
#pragma unroll
    for (int j = 0; j < KN; ++j) {
      const int x = j * 64 + lane, t = __shfl(dst, x / NB % M);
      if (x / NB < nm) *(uint4 *)(base + tile(t) + t % kKv4Tile * (HD / 2) + x % NB * 16) = k[j];
    }
#pragma unroll
    for (int j = 0; j < SN; ++j) {
      const int x = j * 64 + lane, t = __shfl(dst, x / (2 * NB)), b = x % (2 * NB);
      if (x / (2 * NB) < nm)
        *(uint16_t *)(base + tile(t) + (b < NB ? L::KS : L::VS) +
                      ((t % kKv4Tile >> 2) * NB + b % NB) * 8 + (t & 3) * 2) = sc[j];
    }
    if (lane < nm) {
      e.weights_out[list * c.slots + dst] = wv;
      e.positions_out[list * c.slots + dst] = pv;
    }
  }
}

}  // namespace

#define KV4_DISPATCH(hd, call)      \
  switch (hd) {                     \
    case 64: {                      \
      constexpr int HD = 64;        \
      call;                         \
      break;                        \
    }                               \
    case 128: {                     \
      constexpr int HD = 128;       \
      call;                         \
      break;                        \
    }                               \
    default: {                      \
      constexpr int HD = 256;       \
      call;                         \
    }                               \
  }

hipError_t launch_kv4_append(const Kv4Cache &c, const float *qkv, int64_t ldq, int64_t n_rows,
                             const int64_t *starts, bool whole, hipStream_t s) {
  // few rows: as many waves as there are units; many: fewer waves with more in flight
  const int n = n_rows * c.nkv >= 8192 ? 4 : 1, per = n * (256 / c.hd);
  const dim3 grid((unsigned)((n_rows + 3) / 4), (unsigned)((2 * c.nkv + per - 1) / per));
  KV4_DISPATCH(c.hd, if (n == 4) hipLaunchKernelGGL((kv4_append_kernel<HD, 4>), grid,
                                                    dim3(kThreads), 0, s, c, qkv, ldq,
                                                    (uint32_t)n_rows, starts, whole);
               else hipLaunchKernelGGL((kv4_append_kernel<HD, 1>), grid, dim3(kThreads), 0, s, c,
                                       qkv, ldq, (uint32_t)n_rows, starts, whole));
  return hipGetLastError();
}

hipError_t launch_kv4_load(const uint8_t *kv, const int64_t *lengths, float *k, float *v,
                           int64_t out_slots, int n_layers, int n_seq, int nkv, int hd, int slots,
                           hipStream_t s) {
  const int64_t most = out_slots < slots ? out_slots : slots;
  const dim3 grid((unsigned)((most + kKv4Tile - 1) / kKv4Tile), (unsigned)(n_layers * n_seq * nkv));
  KV4_DISPATCH(hd, hipLaunchKernelGGL(kv4_load_kernel<HD>, grid, dim3(kThreads), 0, s, kv, lengths,
                                      k, v, out_slots, n_seq, nkv, slots));
  return hipGetLastError();
}

int64_t kv4_evict_work_bytes(int64_t lists, int slots) {
  return 4 * ((lists + 3) / 4 * 4 + lists * slots);
}

hipError_t launch_kv4_evict(const Kv4Cache &c, const Kv4Evict &e, hipStream_t s) {
  const int64_t lists = (int64_t)e.n_layers * c.n_seq * c.nkv;
  const int half = c.slots / 2;  // at most min(keep, slots - keep) slots move
  const dim3 sel((unsigned)lists), st(kSelThreads);
  if (c.slots <= 4 * kSelThreads)
    hipLaunchKernelGGL(evict_select_kernel<1>, sel, st, 0, s, c, e, half);
  else if (c.slots <= 16 * kSelThreads)
    hipLaunchKernelGGL(evict_select_kernel<4>, sel, st, 0, s, c, e, half);
  else
    hipLaunchKernelGGL(evict_select_kernel<16>, sel, st, 0, s, c, e, half);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int64_t most = e.keep < c.slots - e.keep ? e.keep : c.slots - e.keep;
  int64_t bx = (most + 63) / 64;  // four waves of 16 moves
  bx = bx < 1 ? 1 : (bx > 1024 ? 1024 : bx);
  const dim3 grid((unsigned)bx, (unsigned)lists);
  KV4_DISPATCH(c.hd, hipLaunchKernelGGL(evict_move_kernel<HD>, grid, dim3(kThreads), 0, s, c, e,
                                        half));
  return hipGetLastError();
}

}  // namespace gguf

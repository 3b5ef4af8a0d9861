// The KV cache in pages: storing rows, reading them back, and the pages themselves (forks, room
// for new rows, compaction).
#include <type_traits>

#include "paged.hpp"

namespace gguf {

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// Storing rows: a wave takes one row and 256 / HD units (K or V of a KV head) side by side.  Bound: the
// chain of loads that finds a row's place; 146 rows of six sequences, 4 heads of 64, 3.6 us.
// ---------------------------------------------------------------------------
template <int HD, bool BF>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(PagedCache c,
                                                                const float *__restrict__ qkv,
                                                                int64_t ldq, uint32_t n_rows,
                                                                const int64_t *__restrict__ starts) {
  constexpr int LANES = Kv4Row<HD>::LANES, SIDE = 64 / LANES;
  const int lane = threadIdx.x & 63, q = lane % LANES;
  const uint32_t r = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (r >= n_rows) return;
  // unit u: KV head u / 2, K or V; in qkv after the queries all of K, then all of V
  const int u = blockIdx.y * SIDE + lane / LANES, units = 2 * c.nkv;
  const int ul = min(u, units - 1);  // past the last unit: the last again, not stored
  Kv4Row<HD> row;
  row.load(qkv + r * ldq + (int64_t)(c.nh + (ul & 1) * c.nkv + (ul >> 1)) * HD, q);
  uint32_t s;
  int64_t i;  // the row of s
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
    // so far back that r lies behind every slot: and i need not fit 64 bits
    if (starts[lo] < -((int64_t)c.columns << c.shift)) return;
    i = r - starts[lo];
  } else {
    const uint32_t per = n_rows / (uint32_t)c.n_seq;
    s = r / per;
    i = r - s * per;
  }
  const int64_t n = c.lengths[s], end = paged_end(c, s);
  if (n < 0 || n >= end - i) return;
  const int slot = (int)(n + i), j = slot & (c.page - 1);
  const int32_t page = c.tables[(int64_t)s * c.columns + (slot >> c.shift)];
  if ((uint32_t)page >= (uint32_t)c.n_pages) return;
  row.load_turn(c.cs + (int64_t)slot * (HD / 2), c.sn + (int64_t)slot * (HD / 2), q);
  float y[4];
  paged_turn<HD>(row, q, !(u & 1), y);
  if (u >= units) return;
  const uint2 w = paged_round<BF>(y);
  if (!(u & 1)) {
    *(uint2 *)(c.kv + paged_k_at(c, page, u >> 1, j) + 4 * q) = w;
  } else {
    uint16_t *v = c.kv + paged_v_at(c, page, u >> 1, j) + 64 * q;
    v[0] = (uint16_t)w.x;
    v[16] = (uint16_t)(w.x >> 16);
    v[32] = (uint16_t)w.y;
    v[48] = (uint16_t)(w.y >> 16);
  }
}

// ---------------------------------------------------------------------------
// Storing prompts: a wave takes the rows of one block of 16 slots, K or V of one KV head.  V's 16
// slots of a channel are 32 bytes, which a lane has from its loads of the 16 rows; K's rows go as
// they come.  Bound: the chain that finds a block's rows and page, then their bytes, since one
// generation of waves takes them all; 3714 rows of five sequences, 8 heads of 128, 46 MB: 13 us, 3.5 TB/s
// (the page looked up before the rows are requested, and K's row by row: 15; a wave for K and V both
// 17, V's values one by one 26).
// ---------------------------------------------------------------------------
// The rows of sequence s that are stored: rows first .. first + n - 1 of qkv in slots from `slot` on.
struct Stretch {
  int first, n, slot;
  __device__ __forceinline__ int blocks() const {
    return n > 0 ? ((slot + n - 1) >> 4) - (slot >> 4) + 1 : 0;
  }
};
__device__ __forceinline__ Stretch stretch_of(const PagedCache &c, int s, int64_t n_rows,
                                              const int64_t *starts) {
  const int64_t per = starts ? 0 : n_rows / c.n_seq;
  const int64_t from = starts ? starts[s] : s * per, to = starts ? starts[s + 1] : from + per;
  const int64_t held = c.lengths[s], end = paged_end(c, s);
  // so far back that all its rows lie behind every slot: and differences need not fit 64 bits
  if (held < 0 || held >= end || from >= n_rows || from < -((int64_t)c.columns << c.shift))
    return {0, 0, 0};
  const int64_t first = from < 0 ? 0 : from, last = to < n_rows ? (to < 0 ? 0 : to) : n_rows;
  const int64_t slot = held + (first - from), room = end - slot;
  const int64_t n = last - first < room ? last - first : room;
  return {(int)first, n > 0 ? (int)n : 0, (int)slot};
}

template <int HD, bool BF>
__global__ __launch_bounds__(kThreads) void paged_append_blocks_kernel(
    PagedCache c, const float *__restrict__ qkv, int64_t ldq, int64_t n_rows,
    const int64_t *__restrict__ starts) {
  constexpr int LANES = Kv4Row<HD>::LANES, SIDE = 64 / LANES, CH = HD / 64;
  const int lane = threadIdx.x & 63, q = lane % LANES;
  const int u = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6)), h = u >> 1;
  if (h >= c.nkv) return;
  // block blockIdx.x of the call: sequences in order
  int s = -1, block = 0;
  Stretch x{0, 0, 0};
  for (int s0 = 0, before = 0; s0 < c.n_seq; s0 += 64) {
    const Stretch mine = s0 + lane < c.n_seq ? stretch_of(c, s0 + lane, n_rows, starts) : Stretch{0, 0, 0};
    const int n = mine.blocks(), run = before + lanes_before(n);
    const uint64_t hit = __ballot((int)blockIdx.x < run);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      s = s0 + at;
      block = blockIdx.x - (__builtin_amdgcn_readlane(run, at) - __builtin_amdgcn_readlane(n, at));
      x = {__builtin_amdgcn_readlane(mine.first, at), __builtin_amdgcn_readlane(mine.n, at),
           __builtin_amdgcn_readlane(mine.slot, at)};
      break;
    }
    before = __builtin_amdgcn_readlane(run, 63);
  }
  if (s < 0) return;
  const int slot0 = (x.slot & ~15) + 16 * block;     // of the block
  const int j0 = max(x.slot - slot0, 0), j1 = min(x.slot + x.n - slot0, 16);  // its slots
  const int32_t page = c.tables[(int64_t)s * c.columns + (slot0 >> c.shift)];  // needed by the stores
  const float *rows = qkv + (int64_t)(x.first + (slot0 - x.slot)) * ldq + (int64_t)c.nh * HD;  // of slot0
  const int j_in = slot0 & (c.page - 1);
  if (!(u & 1)) {  // K: 64 / LANES rows at a time
    const float *k = rows + (int64_t)h * HD;
    constexpr int N = 16 / SIDE < 8 ? 16 / SIDE : 8;  // rows of a lane in flight
#pragma unroll
    for (int i0 = 0; i0 < 16; i0 += N * SIDE) {
      Kv4Row<HD> row[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = min(max(i0 + i * SIDE + lane / LANES, j0), j1 - 1);
        row[i].load(k + at * ldq, q);
        row[i].load_turn(c.cs + (int64_t)(slot0 + at) * (HD / 2), c.sn + (int64_t)(slot0 + at) * (HD / 2), q);
      }
      __builtin_amdgcn_sched_barrier(0);
      if ((uint32_t)page >= (uint32_t)c.n_pages) return;
      uint16_t *ko = c.kv + paged_k_at(c, page, h, j_in) + 4 * q;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = i0 + i * SIDE + lane / LANES;
        float t[4];
        paged_turn<HD>(row[i], q, true, t);
        const uint2 w = paged_round<BF>(t);
        if (j >= j0 && j < j1) *(uint2 *)(ko + j * HD) = w;
      }
    }
    return;
  }
  // V: lane's channels CH lane .. of the 16 rows (past the ends: the nearest, not stored)
  const float *v = rows + (int64_t)(c.nkv + h) * HD + CH * lane;
  float y[16][CH];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float *src = v + (int64_t)min(max(j, j0), j1 - 1) * ldq;
    if constexpr (CH == 1) {
      y[j][0] = *src;
    } else if constexpr (CH == 2) {
      const float2 w = *(const float2 *)src;
      y[j][0] = w.x, y[j][1] = w.y;
    } else {
      const float4 w = *(const float4 *)src;
      y[j][0] = w.x, y[j][1] = w.y, y[j][2] = w.z, y[j][3] = w.w;
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  if ((uint32_t)page >= (uint32_t)c.n_pages) return;
  uint16_t *vo = c.kv + paged_v_at(c, page, h, j_in) + 16 * CH * lane;
#pragma unroll
  for (int e = 0; e < CH; ++e) {
    uint2 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float four[4] = {y[4 * i][e], y[4 * i + 1][e], y[4 * i + 2][e], y[4 * i + 3][e]};
      w[i] = paged_round<BF>(four);
    }
    if (j0 == 0 && j1 == 16) {
      *(uint4 *)(vo + 16 * e) = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
      *(uint4 *)(vo + 16 * e + 8) = make_uint4(w[2].x, w[2].y, w[3].x, w[3].y);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j >= j0 && j < j1)
          vo[16 * e + j] = (uint16_t)((j & 2 ? w[j >> 2].y : w[j >> 2].x) >> (16 * (j & 1)));
    }
  }
}

template <bool BF>
__device__ __forceinline__ float paged_value(uint32_t bits16) {
  if (BF) return __uint_as_float(bits16 << 16);
  return (float)__builtin_bit_cast(half_t, (uint16_t)bits16);
}

// ---------------------------------------------------------------------------
// Reading rows back: a workgroup per block of 16 slots of a KV head.  Bound: the f32 rows written, past
// the caches, which hold no call's rows; 6104 slots of 8 heads of 128, 75 MB: 14.7 us, 5.1 TB/s.
// ---------------------------------------------------------------------------
template <int HD, bool BF>
__global__ __launch_bounds__(HD) void paged_load_kernel(PagedCache c, float *__restrict__ ko,
                                                        float *__restrict__ vo, int64_t out_slots) {
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int h = (int)(list % c.nkv), t0 = blockIdx.x * kPageBlock, tid = threadIdx.x;
  const int64_t n64 = c.lengths[s], n = n64 < out_slots ? n64 : out_slots;
  if (t0 >= n) return;
  const int32_t page = c.tables[s * c.columns + (t0 >> c.shift)];
  if ((uint32_t)page >= (uint32_t)c.n_pages) return;
  const int tn = (int)(n - t0 < kPageBlock ? n - t0 : kPageBlock), j0 = t0 & (c.page - 1);
  const uint16_t *kr = c.kv + paged_k_at(c, page, h, j0);
  float *ro = ko + (list * out_slots + t0) * HD;
  for (int w = tid; w < 2 * HD; w += HD) {  // eight channels of a slot
    if (w / (HD / 8) >= tn) break;
    const uint4 x = *(const uint4 *)(kr + 8 * w);
    float *o = ro + 8 * w;
    const uint32_t q[4] = {x.x, x.y, x.z, x.w};
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = paged_value<BF>(q[i >> 1] >> (16 * (i & 1)) & 0xFFFFu);
    __builtin_nontemporal_store(float4_t{y[0], y[1], y[2], y[3]}, (float4_t *)o);
    __builtin_nontemporal_store(float4_t{y[4], y[5], y[6], y[7]}, (float4_t *)(o + 4));
  }
  // a channel's 16 slots per thread: what a wave writes of a slot is one run
  const uint16_t *vr = c.kv + paged_v_at(c, page, h, j0) + 16 * tid;
  const uint4 a = *(const uint4 *)vr, b = *(const uint4 *)(vr + 8);
  const uint32_t q[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  float *o = vo + (list * out_slots + t0) * HD + tid;
#pragma unroll
  for (int j = 0; j < kPageBlock; ++j)
    if (j < tn)
      __builtin_nontemporal_store(paged_value<BF>(q[j >> 1] >> (16 * (j & 1)) & 0xFFFFu), o + j * HD);
}

// ---------------------------------------------------------------------------
// Forks.  A workgroup takes `stripe` columns of every table: it reads all of them before it writes
// any, so that the tables may be their own output.  Pages that a sequence had before are not counted
// again, so that a common beginning costs no atomics.  Bound: a launch and the chain of loads, copies
// and atomics; 16 tables of 66 columns 3.4 us, four of 14 1.9, in one workgroup with the counts' copy.
// ---------------------------------------------------------------------------
constexpr int kForkThreads = 1024, kForkWords = 16384;

__global__ __launch_bounds__(kForkThreads) void paged_copy_refs_kernel(
    const int32_t *__restrict__ refs, int32_t *__restrict__ refs_out, int n_pages) {
  const int i = blockIdx.x * kForkThreads + threadIdx.x;
  if (i < n_pages) refs_out[i] = refs[i];
}

__global__ __launch_bounds__(kForkThreads) void paged_fork_kernel(
    const int32_t *tables, const int64_t *lengths, const int32_t *refs, const int64_t *parents,
    int32_t *tables_out, int64_t *lengths_out, int32_t *refs_out, int n_pages, int columns,
    int n_seq, int stripe, bool copy_refs) {
  __shared__ union {
    int32_t old[kForkWords];
    int64_t len[kForkWords / 2];
  } sh;
  const int tid = threadIdx.x;
  if (copy_refs)  // one workgroup does all
    for (int i = tid; i < n_pages; i += kForkThreads) refs_out[i] = refs[i];
  for (int c0 = blockIdx.x * stripe; c0 < columns; c0 += gridDim.x * stripe) {
    const int w = min(stripe, columns - c0), all = w * n_seq;
    __syncthreads();
    for (int i = tid; i < all; i += kForkThreads)
      sh.old[i] = tables[(int64_t)(i / w) * columns + c0 + i % w];
    __syncthreads();
    for (int i = tid; i < all; i += kForkThreads) {
      const int s = i / w, x = i % w;
      const int64_t parent = parents[s];
      const int32_t was = sh.old[i];
      const int32_t now = parent >= 0 && parent < n_seq ? sh.old[(int)parent * w + x] : -1;
      tables_out[(int64_t)s * columns + c0 + x] = now;
      if (now == was) continue;
      if ((uint32_t)was < (uint32_t)n_pages) atomicSub(&refs_out[was], 1);
      if ((uint32_t)now < (uint32_t)n_pages) atomicAdd(&refs_out[now], 1);
    }
  }
  if (blockIdx.x) return;
  __syncthreads();
  for (int s = tid; s < n_seq; s += kForkThreads) sh.len[s] = lengths[s];
  __syncthreads();
  for (int s = tid; s < n_seq; s += kForkThreads) {
    const int64_t parent = parents[s];
    lengths_out[s] = parent >= 0 && parent < n_seq ? sh.len[parent] : 0;
  }
}

// ---------------------------------------------------------------------------
// Room for new rows.  One workgroup walks the entries (sequence, column) in order, 1024 at a
// time: what an entry needs follows from refs, which the entries before it have brought up to
// date, and from the entries of its own turn that hold the same page.  The n-th need takes the
// n-th free page.  A second launch copies the pages.  Bound: the chain of barriers and loads, 5.8 us
// for 16 sequences, 4.9 for four.
// ---------------------------------------------------------------------------
constexpr int kGrowThreads = 1024, kGrowWaves = kGrowThreads / 64;
constexpr int kGrowSeqs = 4096;

struct GrowJob {
  int32_t src, dst, blocks, pad;
};

// The sum of v over the threads below this one, and over all of them.
__device__ __forceinline__ int sum_before(int v, int *part, int &all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int run = lanes_before(v);
  __syncthreads();
  if (lane == 63) part[wave] = run;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kGrowWaves; ++w) {
    before += w < wave ? part[w] : 0;
    all += part[w];
  }
  return before + run - v;
}

// Of the M pages from i0 on (below n), those whose refs are as asked: a bit each.  A thread of the
// kernels below takes one, 16 of a pool of more than four turns: 40000 pages are then three turns.
constexpr int kFewPages = 4 * kGrowThreads;
template <int M, typename F>
__device__ __forceinline__ uint32_t pages_by(const int32_t *refs, int i0, int n, F is) {
  uint32_t mask = 0;
  if constexpr (M == 1) {
    if (i0 < n) mask = is(refs[i0]);
  } else if (i0 + M <= n) {
    int4 v[M / 4];
#pragma unroll
    for (int j = 0; j < M / 4; ++j) v[j] = *(const int4 *)(refs + i0 + 4 * j);
#pragma unroll
    for (int j = 0; j < M / 4; ++j)
      mask |= (uint32_t)(is(v[j].x) | is(v[j].y) << 1 | is(v[j].z) << 2 | is(v[j].w) << 3) << (4 * j);
  } else {
    for (int j = 0; i0 + j < n; ++j) mask |= (uint32_t)is(refs[i0 + j]) << j;
  }
  return mask;
}

// refs as the atomics of earlier turns left it (they act behind the first cache).
__device__ __forceinline__ int32_t current(const int32_t *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int M>
__global__ __launch_bounds__(kGrowThreads) void paged_grow_kernel(PagedPool c, int32_t *tables,
                                                                  const int64_t *lengths,
                                                                  int32_t *refs,
                                                                  const int64_t *rows,
                                                                  int64_t *room, GrowJob *jobs) {
  __shared__ int ends[kGrowSeqs];        // entries of the sequences up to this one
  __shared__ int32_t held[kGrowThreads];  // the turn's pages that others hold too, -1: none
  __shared__ int32_t free_[kGrowThreads];
  __shared__ int copy_[kGrowThreads];  // which of the turn's needs a copy is, -1: no copy
  __shared__ int part[kGrowWaves];
  const int tid = threadIdx.x;
  const int64_t slots = (int64_t)c.columns << c.shift;
  int total = 0;
  for (int s0 = 0; s0 < c.n_seq; s0 += kGrowThreads) {
    const int s = s0 + tid;
    int count = 0;
    if (s < c.n_seq) {
      const int64_t n = lengths[s], m = rows[s];
      int64_t to = n < 0 ? 0 : n;
      if (n >= 0 && n < slots && m > 0) {
        const int64_t last = m > slots - n ? slots - 1 : n + m - 1;
        count = (int)((last >> c.shift) - (n >> c.shift)) + 1;
        to = ((last >> c.shift) + 1) << c.shift;
      }
      room[s] = to;
      jobs[s].blocks = 0;
    }
    int all;
    const int before = sum_before(count, part, all);
    if (s < c.n_seq) ends[s] = total + before + count;
    total += all;
  }
  __syncthreads();
  int at = 0;  // no page below is free
  for (int e0 = 0; e0 < total; e0 += kGrowThreads) {
    const int e = e0 + tid;
    int s = 0, column = 0, refcount = 0;
    int32_t p = -1;
    bool first = false;
    if (e < total) {
      int lo = 0, hi = c.n_seq - 1;  // the first sequence with e < ends[s]
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (e < ends[mid])
          hi = mid;
        else
          lo = mid + 1;
      }
      s = lo;
      const int k = e - (s ? ends[s - 1] : 0);
      first = k == 0;
      column = (int)(lengths[s] >> c.shift) + k;
      p = tables[(int64_t)s * c.columns + column];
      if ((uint32_t)p >= (uint32_t)c.n_pages)
        p = -1;
      else
        refcount = current(&refs[p]);
    }
    __syncthreads();
    held[tid] = refcount > 1 ? p : -1;
    __syncthreads();
    int earlier = 0;  // entries of this turn that leave the same page first
    if (refcount > 1)
      for (int j = 0; j < tid; ++j) earlier += held[j] == p;
    const bool copies = refcount - earlier > 1;
    const bool needs = e < total && (p < 0 || copies);
    int wanted;
    const int k = sum_before(needs, part, wanted);
    copy_[tid] = copies ? k : -1;
    // the first free pages, in order: as many as are wanted, or all that there are
    int got = 0;
    if (wanted) {
      if (e0) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");  // not as the turn before read them
      while (at < c.n_pages) {
        const int i0 = at + tid * M;
        uint32_t mask = pages_by<M>(refs, i0, c.n_pages, [](int32_t n) { return n <= 0; });
        int found;
        int rank = got + sum_before(__popc(mask), part, found);
        for (; mask && rank < wanted; mask &= mask - 1) free_[rank++] = i0 + __builtin_ctz(mask);
        if (got + found >= wanted) break;  // (the others of these pages are for the next turn)
        got += found;
        at += kGrowThreads * M;
      }
      if (at < c.n_pages) got = wanted;
      __syncthreads();
    }
    // an entry that keeps its page since the others leave it: if they all could
    bool fails = needs && k >= got;
    if (refcount > 1 && !copies && k > got)
      for (int j = 0; j < tid; ++j) fails |= held[j] == p && copy_[j] >= got;
    if (fails) {
      const int64_t n = lengths[s], start = (int64_t)column << c.shift;
      atomicMin((long long *)&room[s], (long long)(start < n ? n : start));
    } else if (needs) {
      const int32_t f = free_[k];
      tables[(int64_t)s * c.columns + column] = f;
      refs[f] = 1;
      if (copies) {
        atomicSub(&refs[p], 1);
        const int filled = (int)(lengths[s] & (c.page - 1));
        if (first && filled) {
          jobs[s].src = p;
          jobs[s].dst = f;
          jobs[s].blocks = (filled + kPageBlock - 1) / kPageBlock;
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // refs are what the next turn goes by
    __syncthreads();
  }
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kFlight = 4, kPiece = kFlight * kThreads;  // 16-byte units of a thread in flight, of a piece

// Pieces y, y + 4 .. of sequence x's copy in layer z.  Bound: the copies, 29 MB of 16 sequences of
// which seven copy a page in 32 layers, 9 us (a unit of a thread in flight: the same).
__global__ __launch_bounds__(kThreads) void paged_grow_copy_kernel(PagedPool c,
                                                                   const GrowJob *__restrict__ jobs) {
  const GrowJob j = jobs[blockIdx.x];
  if (!j.blocks) return;
  const int64_t layer = (int64_t)blockIdx.z * c.n_pages;
  const u32x4 *src = (const u32x4 *)(c.kv + (layer + j.src) * c.page_values);
  u32x4 *dst = (u32x4 *)(c.kv + (layer + j.dst) * c.page_values);
  // of each KV head's K and V the first blocks
  const uint32_t per = (uint32_t)(c.head_values / 8), n = per / (c.page / kPageBlock) * j.blocks;
  const uint32_t units = (uint32_t)(c.page_values / c.head_values) * n;
  for (uint32_t u0 = blockIdx.y * kPiece; u0 < units; u0 += gridDim.y * kPiece) {
    uint32_t at[kFlight];
    u32x4 v[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {  // past the end: the last again, not stored
      const uint32_t u = min(u0 + i * kThreads + threadIdx.x, units - 1);
      at[i] = u / n * per + u % n;
      v[i] = src[at[i]];
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i)
      if (u0 + i * kThreads + threadIdx.x < units) dst[at[i]] = v[i];
  }
}

// ---------------------------------------------------------------------------
// Compaction: a workgroup finds the moves, the second launch makes them: 236 pages of 4 MB in 32
// layers, 2.0 GB read and written in 386 us, 5.1 TB/s; 74 pages of four layers 2.8 + 4.4 us.
// ---------------------------------------------------------------------------
struct CompactWork {
  int32_t *count, *to, *src, *dst;  // moves; where each page goes; the moves
};
__host__ __device__ __forceinline__ CompactWork compact_work(void *work, int n_pages) {
  int32_t *w = (int32_t *)work;
  const int64_t half = n_pages / 2 + 1;
  return {w, w + 4, w + 4 + n_pages, w + 4 + n_pages + half};
}

template <int M>
__global__ __launch_bounds__(kGrowThreads) void paged_compact_plan_kernel(
    PagedPool c, const int32_t *refs, int32_t *refs_out, int64_t *live, CompactWork w) {
  __shared__ int part[kGrowWaves];
  const int tid = threadIdx.x;
  auto used = [](int32_t r) { return r > 0; };
  int mine = 0, n;
  for (int i0 = tid * M; i0 < c.n_pages; i0 += kGrowThreads * M)
    mine += __popc(pages_by<M>(refs, i0, c.n_pages, used));
  sum_before(mine, part, n);
  int holes = 0, moves = 0;
  for (int i1 = 0; i1 < c.n_pages; i1 += kGrowThreads * M) {
    const int i0 = i1 + tid * M, below = min(max(n - i0, 0), M), in = min(max(c.n_pages - i0, 0), M);
    const uint32_t mask = i0 < c.n_pages ? pages_by<M>(refs, i0, c.n_pages, used) : 0u;
    const uint32_t low = (1u << below) - 1u;
    uint32_t hole = ~mask & low, move = mask & ~low;  // (n is at most the number of pages)
    int all;
    const int k = sum_before(__popc(hole) | __popc(move) << 16, part, all);
    int h = holes + (k & 0xFFFF), m = moves + (k >> 16);
    for (; hole; hole &= hole - 1) w.dst[h++] = i0 + __builtin_ctz(hole);
    for (; move; move &= move - 1) w.src[m++] = i0 + __builtin_ctz(move);
    holes += all & 0xFFFF;
    moves += all >> 16;
    for (int j = 0; j < in; ++j) {
      w.to[i0 + j] = i0 + j;
      if (refs_out != refs) refs_out[i0 + j] = refs[i0 + j];
    }
  }
  __syncthreads();
  for (int k = tid; k < moves; k += kGrowThreads) {
    const int32_t from = w.src[k], to = w.dst[k], r = refs[from];
    w.to[from] = to;
    refs_out[to] = r;
    refs_out[from] = 0;
  }
  if (tid == 0) {
    *w.count = moves;
    *live = n;
  }
}

// The moves of layer y in 16 KB pieces, and the tables.
__global__ __launch_bounds__(kThreads) void paged_compact_move_kernel(
    PagedPool c, const int32_t *tables, int32_t *tables_out, CompactWork w) {
  const int64_t entries = (int64_t)c.n_seq * c.columns;
  const int64_t wgs = (int64_t)gridDim.x * gridDim.y, wg = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  for (int64_t i = wg * kThreads + threadIdx.x; i < entries; i += wgs * kThreads) {
    const int32_t p = tables[i];
    tables_out[i] = (uint32_t)p < (uint32_t)c.n_pages ? w.to[p] : p;
  }
  const int moves = *w.count;
  const int64_t units = c.page_values / 8, layer = (int64_t)blockIdx.y * c.n_pages;
  const int pieces = (int)((units + kPiece - 1) / kPiece);
  u32x4 *kv = (u32x4 *)c.kv;
  for (int64_t x = blockIdx.x; x < (int64_t)moves * pieces; x += gridDim.x) {
    const int m = (int)(x / pieces), at = (int)(x % pieces) * kPiece + threadIdx.x;
    const u32x4 *src = kv + (layer + w.src[m]) * units;
    u32x4 *dst = kv + (layer + w.dst[m]) * units;
    u32x4 v[kFlight];  // past the end: the last again, not stored
#pragma unroll
    for (int i = 0; i < kFlight; ++i) v[i] = __builtin_nontemporal_load(src + min(at + i * kThreads, (int)units - 1));
#pragma unroll
    for (int i = 0; i < kFlight; ++i)
      if (at + i * kThreads < units) __builtin_nontemporal_store(v[i], dst + at + i * kThreads);
  }
}

}  // namespace

#define PAGED_DISPATCH(c, call)                     \
  do {                                              \
    auto with_type = [&](auto bf) {                 \
      constexpr bool BF = decltype(bf)::value;      \
      if (c.hd == 64) {                             \
        constexpr int HD = 64;                      \
        call;                                       \
      } else if (c.hd == 128) {                     \
        constexpr int HD = 128;                     \
        call;                                       \
      } else {                                      \
        constexpr int HD = 256;                     \
        call;                                       \
      }                                             \
    };                                              \
    if (c.bf16)                                     \
      with_type(std::true_type{});                  \
    else                                            \
      with_type(std::false_type{});                 \
  } while (0)

hipError_t launch_paged_append(const PagedCache &c, const float *qkv, int64_t ldq, int64_t n_rows,
                               const int64_t *starts, hipStream_t s) {
  // By blocks where the sequences' rows fill some, and there are enough of them (us, a row at a time /
  // by blocks): 8 heads of 128, four sequences of 64, 128 and 512 rows 4.9 / 5.5, 6.8 / 5.9 and 16 / 8.5,
  // 3714 rows of five 26 / 13; 4 heads of 64, four of 128, 256 and 512 rows 4.0 / 4.4, 4.8 / 4.4 and
  // 6.7 / 5.0; one head of 256, where the border is lower, four of 256 and 512 5.0 / 5.6 and 7.0 / 5.8.
  // Many sequences of one block each are the rule's worst: 32 of 16 rows, 8 heads of 128, 7.1 / 9.0.
  if (n_rows >= 16 * (int64_t)c.n_seq && n_rows * c.nkv >= 4096) {
    const dim3 blocks((unsigned)(n_rows / 16 + 2 * c.n_seq), (unsigned)((2 * c.nkv + 3) / 4));
    PAGED_DISPATCH(c, hipLaunchKernelGGL((paged_append_blocks_kernel<HD, BF>), blocks, dim3(kThreads),
                                         0, s, c, qkv, ldq, n_rows, starts));
    return hipGetLastError();
  }
  const int per = 256 / c.hd;
  const dim3 grid((unsigned)((n_rows + 3) / 4), (unsigned)((2 * c.nkv + per - 1) / per));
  PAGED_DISPATCH(c, hipLaunchKernelGGL((paged_append_kernel<HD, BF>), grid, dim3(kThreads), 0, s, c,
                                       qkv, ldq, (uint32_t)n_rows, starts));
  return hipGetLastError();
}

hipError_t launch_paged_load(const PagedCache &c, float *k, float *v, int64_t out_slots,
                             hipStream_t s) {
  const int64_t slots = (int64_t)c.columns << c.shift, most = out_slots < slots ? out_slots : slots;
  const dim3 grid((unsigned)((most + kPageBlock - 1) / kPageBlock), (unsigned)(c.n_seq * c.nkv));
  PAGED_DISPATCH(c, hipLaunchKernelGGL((paged_load_kernel<HD, BF>), grid, dim3(HD), 0, s, c, k, v,
                                       out_slots));
  return hipGetLastError();
}

hipError_t launch_paged_fork(const int32_t *tables, const int64_t *lengths, const int32_t *refs,
                             const int64_t *parents, int32_t *tables_out, int64_t *lengths_out,
                             int32_t *refs_out, int n_pages, int columns, int n_seq, hipStream_t s) {
  const int most = kForkWords / n_seq;
  const bool other = refs_out != refs;
  const bool one = other && n_pages <= 8 * kForkThreads && columns <= 4 * most;
  if (other && !one) {
    hipLaunchKernelGGL(paged_copy_refs_kernel, dim3((n_pages + kForkThreads - 1) / kForkThreads),
                       dim3(kForkThreads), 0, s, refs, refs_out, n_pages);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  int stripe = one ? most : (columns + 255) / 256;
  stripe = stripe < 1 ? 1 : (stripe > most ? most : stripe);
  const int wgs = one ? 1 : (columns + stripe - 1) / stripe;
  hipLaunchKernelGGL(paged_fork_kernel, dim3(wgs < 4096 ? wgs : 4096), dim3(kForkThreads), 0, s,
                     tables, lengths, refs, parents, tables_out, lengths_out, refs_out, n_pages,
                     columns, n_seq, stripe, one);
  return hipGetLastError();
}

int64_t paged_grow_work_bytes(int n_seq) { return (int64_t)n_seq * sizeof(GrowJob); }

hipError_t launch_paged_grow(const PagedPool &c, int32_t *tables, const int64_t *lengths,
                             int32_t *refs, const int64_t *rows, int64_t *room, void *work,
                             hipStream_t s) {
  GrowJob *jobs = (GrowJob *)work;
  auto plan = [&](auto *kernel) {
    hipLaunchKernelGGL(kernel, dim3(1), dim3(kGrowThreads), 0, s, c, tables, lengths, refs, rows, room,
                       jobs);
  };
  if (c.n_pages <= kFewPages)
    plan(paged_grow_kernel<1>);
  else
    plan(paged_grow_kernel<16>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(paged_grow_copy_kernel, dim3(c.n_seq, 4, c.n_layers), dim3(kThreads), 0, s, c,
                     jobs);
  return hipGetLastError();
}

int64_t paged_compact_work_bytes(int64_t n_pages) { return 4 * (4 + n_pages + 2 * (n_pages / 2 + 1)); }

hipError_t launch_paged_compact(const PagedPool &c, const int32_t *tables, const int32_t *refs,
                                int32_t *tables_out, int32_t *refs_out, int64_t *live, void *work,
                                hipStream_t s) {
  const CompactWork w = compact_work(work, c.n_pages);
  auto plan = [&](auto *kernel) {
    hipLaunchKernelGGL(kernel, dim3(1), dim3(kGrowThreads), 0, s, c, refs, refs_out, live, w);
  };
  if (c.n_pages <= kFewPages)
    plan(paged_compact_plan_kernel<1>);
  else
    plan(paged_compact_plan_kernel<16>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  int x = 2048 / c.n_layers;
  x = x < 1 ? 1 : x;
  hipLaunchKernelGGL(paged_compact_move_kernel, dim3(x, c.n_layers), dim3(kThreads), 0, s, c, tables,
                     tables_out, w);
  return hipGetLastError();
}

}  // namespace gguf

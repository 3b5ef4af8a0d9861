// The 4-bit KV cache: storing rows, reading them back, eviction.
#include "kv4.hpp"

namespace gguf {

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// Storing rows: a wave per (row, KV head, K or V).
// ---------------------------------------------------------------------------
template <int HD>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(Kv4Cache c,
                                                              const float *__restrict__ qkv,
                                                              int64_t ldq, int64_t n_rows,
                                                              const int64_t *__restrict__ starts) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int64_t r = unit / (2 * c.nkv);
  if (r >= n_rows) return;
  const int hv = (int)(unit - r * 2 * c.nkv), h = hv >> 1;
  int64_t s, i;
  if (starts) {
    if (r < starts[0] || r >= starts[c.n_seq]) return;
    int lo = 0, hi = c.n_seq;  // starts[lo] <= r < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= r)
        lo = mid;
      else
        hi = mid;
    }
    s = lo;
    i = r - starts[lo];
  } else {
    const int64_t per = n_rows / c.n_seq;
    s = r / per;
    i = r - s * per;
  }
  const int64_t slot = c.lengths[s] + i, p = c.pos[s] + i;
  if (slot < 0 || slot >= c.slots || p < 0 || p >= c.rope_rows) return;
  const int64_t list = s * c.nkv + h;
  uint8_t *base = kv4_list(c.kv, list, c.slots, Kv4<HD>::TB);
  const float *x = qkv + r * ldq + (int64_t)(c.nh + (hv & 1) * c.nkv + h) * HD;
  if (hv & 1) {
    kv4_store_row<HD, false>(base, (int)slot, x, nullptr, nullptr, lane);
    if (lane == 0) {
      if (c.positions) c.positions[list * c.slots + slot] = (int32_t)p;
      if (c.weights) c.weights[list * c.slots + slot] = 0.f;
    }
  } else {
    kv4_store_row<HD, true>(base, (int)slot, x, c.cs + p * (HD / 2), c.sn + p * (HD / 2), lane);
  }
}

// ---------------------------------------------------------------------------
// Reading rows back: a workgroup per tile of 32 slots.
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
    const int j = w / (4 * NB), gb = w % (4 * NB), g = gb / NB, b = gb % NB;
    if (j >= tn) continue;
    const uint32_t q = *(const uint32_t *)(tile + j * (HD / 2) + gb * 4);
    const float d = (float)*(const half_t *)(tile + L::KS + ((j >> 2) * NB + b) * 8 + (j & 3) * 2);
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = d * (float)((int)((q >> (8 * i)) & 15u) - 8);
      y[i + 4] = d * (float)((int)((q >> (8 * i + 4)) & 15u) - 8);
    }
    float4 *o = (float4 *)(kr + (int64_t)j * HD + 32 * b + 8 * g);
    o[0] = make_float4(y[0], y[1], y[2], y[3]);
    o[1] = make_float4(y[4], y[5], y[6], y[7]);
  }
  for (int w = tid; w < 8 * 16 * NB; w += kThreads) {  // a word of V codes: 4 slots, 2 channels
    const int q4 = w / (16 * NB), b = w / 16 % NB, n16 = w & 15;
    const uint32_t q = *(const uint32_t *)(tile + L::VO + q4 * (2 * HD) + (n16 * NB + b) * 4);
    const half4_t d = *(const half4_t *)(tile + L::VS + (q4 * NB + b) * 8);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int j = 4 * q4 + s;
      if (j < tn) {
        float *o = vr + (int64_t)j * HD + 32 * b + n16;
        o[0] = (float)d[s] * (float)((int)((q >> (8 * s)) & 15u) - 8);
        o[16] = (float)d[s] * (float)((int)((q >> (8 * s + 4)) & 15u) - 8);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Eviction: which slots stay, then the moves.
// ---------------------------------------------------------------------------
constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

// The order of the slots: larger is kept first.  NaN is 0, -0 equals +0.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t p, int64_t from, int64_t sinks) {
  if (p >= from || p < sinks) w = INFINITY;
  if (!(w == w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Work: per list the number of moves, then the slots given up below `keep` (holes) and the
// kept ones from `keep` on, both ascending.
__device__ __forceinline__ int32_t *evict_holes(void *work, int64_t lists, int64_t list, int half) {
  return (int32_t *)work + (lists + 3) / 4 * 4 + list * 2 * half;
}

// Sum over the workgroup of one bit per thread below this thread; `all` gets the total.
__device__ __forceinline__ int block_rank(bool bit, int *part, int &all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t m = __ballot(bit);
  __syncthreads();
  if (lane == 0) part[wave] = __popcll(m);
  __syncthreads();
  int before = 0;
  all = 0;
  for (int w = 0; w < kSelWaves; ++w) {
    before += w < wave ? part[w] : 0;
    all += part[w];
  }
  return before + __popcll(m & ((1ull << lane) - 1ull));
}

// One workgroup per list: the keep-th largest key by four 8-bit digits (a histogram each),
// then one pass in slot order that writes the lists.
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(Kv4Cache c, Kv4Evict e, int half) {
  __shared__ int hist[256], part[kSelWaves], found[2];
  const int64_t list = blockIdx.x, lists = gridDim.x;
  const int64_t s = list / c.nkv % c.n_seq;
  const int64_t n64 = c.lengths[s];
  const int tid = threadIdx.x;
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
  const int64_t from = c.pos[s] - e.recent;
  uint32_t prefix = 0;
  int need = keep;  // of the keys that share the prefix, this many stay
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSelThreads) {
      const uint32_t k = evict_key(w[i], p[i], from, e.sinks);
      if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid < 64) {  // the digit: from the top, the first whose running count reaches `need`
      int h[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += h[i] = hist[255 - (4 * tid + i)];
      int run = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(run, o);
        if (tid >= o) run += v;
      }
      int before = run - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < need && before + h[i] >= need) {
          found[0] = 255 - (4 * tid + i);
          found[1] = need - before;
        }
        before += h[i];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    need = found[1];
    __syncthreads();
  }
  int32_t *holes = evict_holes(e.work, lists, list, half), *late = holes + half;
  int ties = 0, nh = 0, nl = 0;
  for (int i0 = 0; i0 < n; i0 += kSelThreads) {
    const int i = i0 + tid;
    const bool in = i < n;
    const float wi = in ? w[i] : 0.f;
    const int32_t pi = in ? p[i] : 0;
    const uint32_t k = in ? evict_key(wi, pi, from, e.sinks) : 0u;
    int all;
    const int rank = ties + block_rank(in && k == prefix, part, all);
    ties += all;
    const bool stays = in && (k > prefix || (k == prefix && rank < need));
    const bool hole = in && !stays && i < keep, moves = stays && i >= keep;
    const int hr = nh + block_rank(hole, part, all);
    nh += all;
    if (hole) holes[hr] = i;
    const int lr = nl + block_rank(moves, part, all);
    nl += all;
    if (moves) late[lr] = i;
    if (stays && i < keep) {
      if (wo != w) wo[i] = wi;
      if (po != p) po[i] = pi;
    }
  }
  if (tid == 0) *count = nl;
}

// One wave per move: the bytes of slot `late[i]` to slot `holes[i]`.
template <int HD>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(Kv4Cache c, Kv4Evict e, int half) {
  using L = Kv4<HD>;
  constexpr int NB = L::NB;
  const int64_t list = blockIdx.y, lists = gridDim.y;
  const int lane = threadIdx.x & 63;
  if (blockIdx.x == 0 && threadIdx.x == 0 && list < (int64_t)c.n_seq * c.nkv && list % c.nkv == 0) {
    const int64_t s = list / c.nkv, n = c.lengths[s];
    e.lengths_out[s] = n > e.keep && n >= e.trigger && n <= c.slots ? e.keep : n;
  }
  const int count = ((const int32_t *)e.work)[list];
  const int32_t *holes = evict_holes(e.work, lists, list, half), *late = holes + half;
  uint8_t *base = kv4_list(c.kv, list, c.slots, L::TB);
  for (int i = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); i < count;
       i += gridDim.x * (kThreads / 64)) {
    const int dst = holes[i], src = late[i];
    uint8_t *to = base + (int64_t)(dst / kKv4Tile) * L::TB;
    const uint8_t *from = base + (int64_t)(src / kKv4Tile) * L::TB;
    const int jd = dst % kKv4Tile, js = src % kKv4Tile;
    if (lane < HD / 8)
      ((uint32_t *)(to + jd * (HD / 2)))[lane] = ((const uint32_t *)(from + js * (HD / 2)))[lane];
    for (int b = lane; b < HD / 2; b += 64)
      to[L::VO + (jd >> 2) * (2 * HD) + b * 4 + (jd & 3)] =
          from[L::VO + (js >> 2) * (2 * HD) + b * 4 + (js & 3)];
    if (lane < 2 * NB) {
      const int o = (lane < NB ? L::KS : L::VS) + (lane % NB) * 8;
      *(half_t *)(to + o + (jd >> 2) * NB * 8 + (jd & 3) * 2) =
          *(const half_t *)(from + o + (js >> 2) * NB * 8 + (js & 3) * 2);
    }
    if (lane == 0) {
      e.weights_out[list * c.slots + dst] = e.weights[list * c.slots + src];
      e.positions_out[list * c.slots + dst] = e.positions[list * c.slots + src];
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
                             const int64_t *starts, hipStream_t s) {
  const int64_t units = n_rows * c.nkv * 2;
  const dim3 grid((unsigned)((units + kThreads / 64 - 1) / (kThreads / 64)));
  KV4_DISPATCH(c.hd, hipLaunchKernelGGL(kv4_append_kernel<HD>, grid, dim3(kThreads), 0, s, c, qkv,
                                        ldq, n_rows, starts));
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
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)lists), dim3(kSelThreads), 0, s, c, e,
                     half);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  const int64_t most = e.keep < c.slots - e.keep ? e.keep : c.slots - e.keep;
  int64_t bx = (most + 3) / 4;
  bx = bx < 1 ? 1 : (bx > 1024 ? 1024 : bx);
  const dim3 grid((unsigned)bx, (unsigned)lists);
  KV4_DISPATCH(c.hd, hipLaunchKernelGGL(evict_move_kernel<HD>, grid, dim3(kThreads), 0, s, c, e,
                                        half));
  return hipGetLastError();
}

}  // namespace gguf

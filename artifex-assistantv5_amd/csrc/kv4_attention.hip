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

template <int HD>
__global__ __launch_bounds__(kThreads) void kv4_attention_kernel(Kv4Cache c, Kv4Attn a,
                                                                 float *__restrict__ rec,
                                                                 float *__restrict__ scores, int S) {
  using L = Kv4<HD>;
  constexpr int NB = L::NB, half = HD / 2, P = kThreads / HD;
  __shared__ float q[HD], p_[kThreads], red[4], part[kThreads];
  const int64_t list = blockIdx.y, s = list / c.nkv;
  const int v = blockIdx.z, grp = c.nh / c.nkv, V = a.rows * grp, tid = threadIdx.x;
  const int filled = kv4_filled(c, s, a.rows);
  if (filled < 0) return;
  const Splits sp = kv4_splits(filled + a.rows, S);
  if ((int)blockIdx.x >= sp.n) return;
  const int i = v / grp, vis = filled + i + 1;
  const int t0 = blockIdx.x * sp.per * kKv4Tile;
  const int t1 = min(vis, t0 + sp.per * kKv4Tile);
  const uint8_t *base = kv4_list(c.kv, list, c.slots, L::TB);
  const float *x = a.qkv + (s * a.rows + i) * a.ldq + (list % c.nkv * grp + v % grp) * HD;
  const float *cr = c.cs + (c.pos[s] + i) * half, *sr = c.sn + (c.pos[s] + i) * half;
  const float scale = kLog2e / sqrtf((float)HD);
  for (int e = tid; e < half; e += kThreads) {
    q[e] = (x[e] * cr[e] - x[e + half] * sr[e]) * scale;
    q[e + half] = (x[e + half] * cr[e] + x[e] * sr[e]) * scale;
  }
  __syncthreads();
  const int ch = tid % HD, pt = tid / HD, vb = ch >> 5, vn = ch & 15, vs = ch & 16 ? 4 : 0;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int b0 = t0; b0 < t1; b0 += kThreads) {
    const int t = b0 + tid, j = t % kKv4Tile;
    float sc = -INFINITY;
    if (t < t1) {
      const uint8_t *tile = base + (int64_t)(t / kKv4Tile) * L::TB;
      sc = 0.f;
      for (int b = 0; b < NB; ++b) {
        float dot = 0.f;
        for (int g = 0; g < 4; ++g) {
          const uint32_t w = *(const uint32_t *)(tile + j * half + (g * NB + b) * 4);
          for (int k = 0; k < 4; ++k) {
            dot += (float)((int)((w >> (8 * k)) & 15u) - 8) * q[32 * b + 8 * g + k];
            dot += (float)((int)((w >> (8 * k + 4)) & 15u) - 8) * q[32 * b + 8 * g + 4 + k];
          }
        }
        sc += (float)*(const half_t *)(tile + L::KS + ((j >> 2) * NB + b) * 8 + (j & 3) * 2) * dot;
      }
      if (scores) scores[(list * V + v) * c.slots + t] = sc;
    }
    float mx = sc;
    for (int d = 32; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mn = fmaxf(m, mx), alpha = m == -INFINITY ? 0.f : exp2f(m - mn);
    const float p = t < t1 ? exp2f(sc - mn) : 0.f;
    p_[tid] = p;
    l = l * alpha + p;
    o *= alpha;
    m = mn;
    __syncthreads();
    for (int u = pt; u < min(kThreads, t1 - b0); u += P) {
      const int tt = b0 + u, jj = tt % kKv4Tile;
      const uint8_t *tile = base + (int64_t)(tt / kKv4Tile) * L::TB;
      const int code =
          (tile[L::VO + (jj >> 2) * (2 * HD) + (vn * NB + vb) * 4 + (jj & 3)] >> vs) & 15;
      const float d =
          (float)*(const half_t *)(tile + L::VS + ((jj >> 2) * NB + vb) * 8 + (jj & 3) * 2);
      o += p_[u] * (d * (float)(code - 8));
    }
  }
  for (int d = 32; d > 0; d >>= 1) l += __shfl_xor(l, d);
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = l;
  part[tid] = o;
  __syncthreads();
  constexpr int RS = record_floats<HD>();
  float *r = rec + ((list * S + blockIdx.x) * V + v) * RS;
  if (tid < HD) {
    float sum = part[tid];
    for (int k = 1; k < P; ++k) sum += part[tid + k * HD];
    r[tid] = sum;
  }
  if (tid < NB) {
    r[HD + 2 * tid] = m;
    r[HD + 2 * tid + 1] = red[0] + red[1] + red[2] + red[3];
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
  if (a.store) {
    const hipError_t e =
        launch_kv4_append(c, a.qkv, a.ldq, (int64_t)c.n_seq * a.rows, nullptr, s);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kv4_attention_kernel<HD>, dim3((unsigned)S, (unsigned)lists, (unsigned)V),
                     dim3(kThreads), 0, s, c, a, rec, scores, S);
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

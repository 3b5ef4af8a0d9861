// Sampling a token per row of logits (gguf_hip_sample.h).
#include "paged.hpp"

namespace gguf {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;
constexpr double kOne = 0x1p43;  // a weight of 1

// Larger is drawn earlier; -0 is +0, NaN and -inf are 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x > -INFINITY ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

struct Row {
  double scale;  // log2(e) / temperature
  float top;     // the largest logit
};
// w as a fraction, and in multiples of 2^-43.
__device__ __forceinline__ double weight(const Row &r, uint32_t key) {
  const float x = key_value(key);
  if (x == r.top) return 1.0;  // infinite ones too
  const double d = (double)x - (double)r.top;
  return key && d > -INFINITY ? exp2(d * r.scale) : 0.0;
}
__device__ __forceinline__ uint64_t fixed(double w) { return (uint64_t)__double2ll_rn(w * kOne); }

template <typename T>
__device__ __forceinline__ T block_sum(T v, T *red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  T all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) all += red[w];
  return all;
}

// One workgroup per row.
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ uint32_t count[kBins];
  __shared__ unsigned long long mass[kBins], red[kWaves];
  __shared__ uint32_t redk[kWaves];
  __shared__ uint32_t found_bin, found_count;
  __shared__ unsigned long long found_before, found_n;
  __shared__ int result;
  const int row = blockIdx.x, tid = threadIdx.x;
  const float *x = a.logits + row * a.ld;
  const int n = a.vocab;
  uint32_t top = 0;
  for (int i = tid; i < n; i += kThreads) top = max(top, order_key(x[i]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  if ((tid & 63) == 0) redk[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = max(top, redk[w]);
  const float t = a.temperature ? a.temperature[row] : a.temperature_all;
  const int32_t top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  const float min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  float u = a.u[row];
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  if (!top) {
    if (tid == 0) {
      a.out[row] = 0;
      if (a.probs) a.probs[row] = 0.f;
    }
    return;
  }
  const bool greedy = !(t > 0.f);
  const Row r{1.4426950408889634074 / (double)t, key_value(top)};

  // The key at which a running sum, from the largest key down, reaches a target: digits of 11, 11
  // and 10 bits.  by_count: reaches `want` tokens; else the first sum for which `enough`.  Gives the
  // key, the tokens and the mass above it, and how many tokens have the key.
  struct Place {
    uint32_t key, above, same;
    uint64_t before;
  };
  auto locate = [&](bool by_count, uint32_t want, auto enough) {
    Place p{0, 0, 0, 0};
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
      for (int b = tid; b < kBins; b += kThreads) count[b] = 0, mass[b] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const uint32_t k = order_key(x[i]);
        if (pass == 0 || (k >> (shift + bits)) == (p.key >> (shift + bits))) {
          const uint32_t b = (k >> shift) & ((1u << bits) - 1u);
          atomicAdd(&count[b], 1u);
          const uint64_t w = fixed(weight(r, k));
          if (w) atomicAdd(&mass[b], (unsigned long long)w);
        }
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t c = p.above;
        uint64_t m = p.before;
        int b = (1 << bits) - 1;
        for (; b > 0; --b) {
          if (by_count ? c + count[b] >= want : (count[b] && enough(m + mass[b]))) break;
          c += count[b];
          m += mass[b];
        }
        found_bin = b;
        found_count = c;
        found_before = m;
        found_n = count[b];
      }
      __syncthreads();
      p.key |= found_bin << shift;
      p.above = found_count;
      p.before = found_before;
      p.same = (uint32_t)found_n;
      __syncthreads();
    }
    return p;
  };
  // the first of `same` equal tokens at which it is enough
  auto rank_of = [&](const Place &p, auto enough) {
    const uint64_t w = fixed(weight(r, p.key));
    uint32_t lo = 1, hi = p.same < 1 ? 1 : p.same;
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (enough(p.before + mid * w))
        hi = mid;
      else
        lo = mid + 1;
    }
    return lo;
  };
  uint64_t total;
  {
    uint64_t sum = 0, large = 0;
    for (int i = tid; i < n; i += kThreads) {
      const double w = weight(r, order_key(x[i]));
      const uint64_t f = fixed(w);
      sum += f;
      if (w >= (double)min_p) large += f;
    }
    total = block_sum<unsigned long long>(sum, red);
    large = block_sum<unsigned long long>(large, red);
    if (!(min_p > 0.f)) large = total;
    if (top_k > 0 && top_k < n) {
      const Place p = locate(true, (uint32_t)top_k, [](uint64_t) { return false; });
      total = p.before + ((uint32_t)top_k - p.above) * fixed(weight(r, p.key));
    }
    if (top_p < 1.f) {
      const double want = (double)top_p * (double)total;
      auto enough = [&](uint64_t m) { return (double)m >= want; };
      const Place p = locate(false, 0, enough);
      const uint64_t kept = p.before + rank_of(p, enough) * fixed(weight(r, p.key));
      total = kept < total ? kept : total;
    }
    total = large < total ? large : total;
    const uint64_t one = (uint64_t)kOne;
    total = total < one ? one : total;
  }
  const double want = (double)u * (double)total;
  auto enough = [&](uint64_t m) { return (double)m > want; };
  Place p{top, 0, 1, 0};
  uint32_t rank = 1;
  if (!greedy) {
    p = locate(false, 0, enough);
    rank = rank_of(p, enough);
  }
  // the rank-th token with that key, by index
  uint32_t before = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + tid;
    const bool same = i < n && order_key(x[i]) == p.key;
    const uint64_t mask = __ballot(same);
    __syncthreads();
    if ((tid & 63) == 0) redk[tid >> 6] = __popcll(mask);
    __syncthreads();
    uint32_t at = before, all = before;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      at += w < (tid >> 6) ? redk[w] : 0;
      all += redk[w];
    }
    at += __popcll(mask & (((uint64_t)1 << (tid & 63)) - 1)) + 1;
    if (same && at == rank) result = i;
    before = all;
    if (before >= rank) break;
  }
  __syncthreads();
  if (tid == 0) {
    a.out[row] = result;
    if (a.probs)
      a.probs[row] = greedy ? 1.f : (float)((double)fixed(weight(r, p.key)) / (double)total);
  }
}

}  // namespace

int64_t sample_work_bytes(int64_t rows, int64_t vocab) { return 16; }

hipError_t launch_sample(const SampleArgs &a, hipStream_t s) {
  hipLaunchKernelGGL(sample_kernel, dim3(a.rows), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace gguf

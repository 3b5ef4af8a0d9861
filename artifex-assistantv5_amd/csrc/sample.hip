// Sampling a token per row of logits (gguf_hip_sample.h).
//
// A row is cut into chunks.  Its tokens' weights are sorted into bins by their exponent, evenly over
// the row's range, largest first; a running sum over the bins tells in which bin a limit or the
// draw falls, and only that bin's tokens are put in order.  Three launches:
//   top      each chunk's largest and smallest logit
//   bins     each chunk's bins: their tokens' indices in the order of the bins, and their masses
//   draw     a workgroup per row: the chunks' bins added up, the limits, the draw
// All sums are of 64-bit integers, so that neither the chunks nor timing matter.
#include "paged.hpp"

namespace gguf {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 512;    // the last one holds the tokens of weight 0
constexpr int kSorted = 4096;  // tokens that a workgroup puts in order
constexpr int kChunks = 64;
constexpr double kOne = 0x1p43;  // a weight of 1
constexpr double kNothing = 44.5;  // 2^-kNothing of it rounds to 0

// Larger is drawn earlier; -0 is +0, NaN and -inf are 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x > -INFINITY ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// A token's place: larger first, of equal logits the lower index.
__device__ __forceinline__ uint64_t place(uint32_t key, uint32_t index) {
  return (uint64_t)key << 32 | (uint32_t)~index;
}

// 2^y of y <= 0 to within 2^-50: 2^f, |f| <= 1/2, by its Taylor series to ln(2)^11 f^11 / 11!, whose
// rest is below 6e-15.
__device__ __forceinline__ double pow2(double y) {
  const double n = __builtin_rint(y), f = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800;
  p = fma(p, f, 1.0 / 3628800);
  p = fma(p, f, 1.0 / 362880);
  p = fma(p, f, 1.0 / 40320);
  p = fma(p, f, 1.0 / 5040);
  p = fma(p, f, 1.0 / 720);
  p = fma(p, f, 1.0 / 120);
  p = fma(p, f, 1.0 / 24);
  p = fma(p, f, 1.0 / 6);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return __builtin_ldexp(p, (int)n);
}

struct Row {
  double scale;  // log2(e) / temperature
  float top;     // the largest logit
};
// log2 of a token's weight, -inf for none.
__device__ __forceinline__ double exponent(const Row &r, uint32_t key) {
  const float x = key_value(key);
  if (x == r.top) return 0.0;  // infinite ones too
  const double d = ((double)x - (double)r.top) * r.scale;
  return key && d > -INFINITY ? d : -INFINITY;
}
__device__ __forceinline__ double weight(double e) { return e > -1000.0 ? pow2(e) : 0.0; }
// In multiples of 2^-43: below 2^52, adding 2^52 leaves the nearest integer in the low bits.
__device__ __forceinline__ uint64_t fixed(double w) {
  return (uint64_t)__double_as_longlong(fma(w, kOne, 0x1p52)) & 0xFFFFFFFFFFFFFull;
}
__device__ __forceinline__ uint64_t mass_of(const Row &r, uint32_t key) {
  return fixed(weight(exponent(r, key)));
}

template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_max(T v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const T w = __shfl_xor(v, o);
    v = w > v ? w : v;
  }
  return v;
}
// v and those of the threads below; `part` holds a value per wave.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T w = __shfl_up(v, o);
    if (lane >= o) v += w;
  }
  __syncthreads();
  if (lane == 63) part[wave] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves - 1; ++w) v += w < wave ? part[w] : 0;
  return v;
}

// The workspace: per row and chunk the place of its first token and the inverse of its smallest
// key; the ends of its bins; their masses; the mass that min_p keeps; its tokens in the order of
// the bins (indices within the chunk).
struct Work {
  uint64_t *first, *mass, *large;
  uint32_t *least;
  uint16_t *ends, *order;
};
struct Cut {
  int chunk, chunks;  // tokens of a chunk, chunks of a row
};
Cut cut_of(int64_t rows, int64_t vocab) {
  // small chunks while they do not fill the chip
  const bool small = vocab <= 4 * kThreads * kChunks && rows * vocab < (int64_t)4 * kThreads * 1024;
  Cut c;
  c.chunk = (small ? 4 : 16) * kThreads;
  c.chunks = (int)((vocab + c.chunk - 1) / c.chunk);
  return c;
}
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }
int64_t place_work(char *base, int64_t rows, const Cut &c, Work &w) {
  const int64_t lists = rows * c.chunks;
  char *p = base;
  auto take = [&](int64_t bytes) {
    char *q = p;
    p += round16(bytes);
    return q;
  };
  w.first = (uint64_t *)take(lists * 8);
  w.large = (uint64_t *)take(lists * 8);
  w.mass = (uint64_t *)take(lists * kBins * 8);
  w.least = (uint32_t *)take(lists * 4);
  w.ends = (uint16_t *)take(lists * kBins * 2);
  w.order = (uint16_t *)take(lists * c.chunk * 2);
  return p - base;
}

template <int T>
__global__ __launch_bounds__(kThreads) void sample_top_kernel(SampleArgs a, Work w) {
  __shared__ uint64_t part[kWaves];
  __shared__ uint32_t partl[kWaves];
  const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * T * kThreads;
  const float *x = a.logits + row * a.ld;
  uint64_t first = 0;
  uint32_t least = 0;
#pragma unroll
  for (int j = 0; j < T; ++j) {
    const int i = i0 + j * kThreads + tid;
    const uint32_t k = i < a.vocab ? order_key(x[i]) : 0u;
    const uint64_t p = place(k, i);
    first = k && p > first ? p : first;
    least = k && ~k > least ? ~k : least;
  }
  first = wave_max(first);
  least = wave_max(least);
  if ((tid & 63) == 0) part[tid >> 6] = first, partl[tid >> 6] = least;
  __syncthreads();
  if (tid) return;
  for (int v = 1; v < kWaves; ++v) {
    first = part[v] > first ? part[v] : first;
    least = partl[v] > least ? partl[v] : least;
  }
  const int64_t list = (int64_t)row * gridDim.x + blockIdx.x;
  w.first[list] = first;
  w.least[list] = least;
}

// What the row's workgroups make of the first launch: the row's largest logit, and its bins' width.
struct Bins {
  Row r;
  double per;      // bins per unit of -exponent
  uint64_t first;  // the row's first token
  float t;
};
__device__ __forceinline__ Bins bins_of(const SampleArgs &a, const Work &w, int row, int chunks) {
  const int lane = threadIdx.x & 63;
  const int64_t list = (int64_t)row * chunks + lane;
  Bins b;
  b.first = wave_max(lane < chunks ? w.first[list] : (uint64_t)0);
  const uint32_t least = wave_max(lane < chunks ? w.least[list] : 0u);
  b.t = a.temperature ? a.temperature[row] : a.temperature_all;
  b.r.scale = 1.4426950408889634074 / (double)b.t;
  b.r.top = key_value((uint32_t)(b.first >> 32));
  double range = -exponent(b.r, ~least);
  range = range < kNothing ? range : kNothing;
  b.per = range > 0.0 ? (kBins - 1) / range : 0.0;
  return b;
}
__device__ __forceinline__ int bin_of(const Bins &b, double e, uint64_t mass) {
  if (!mass) return kBins - 1;
  const int k = (int)(-e * b.per);
  return k < kBins - 2 ? k : kBins - 2;
}

template <int T>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleArgs a, Work w, int chunks) {
  __shared__ uint32_t count[kBins];
  __shared__ unsigned long long mass[kBins];
  __shared__ uint32_t part[kWaves];
  __shared__ uint64_t partm[kWaves];
  const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * T * kThreads;
  const Bins b = bins_of(a, w, row, chunks);
  if (!b.first || !(b.t > 0.f)) return;  // nothing to draw, or no draw
  const float *x = a.logits + row * a.ld;
  const float min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  for (int k = tid; k < kBins; k += kThreads) count[k] = 0, mass[k] = 0;
  __syncthreads();
  uint32_t rank[T];  // bin and place in it
  uint64_t large = 0;
#pragma unroll
  for (int j = 0; j < T; ++j) {
    const int i = i0 + j * kThreads + tid;
    if (i >= a.vocab) break;
    const double e = exponent(b.r, order_key(x[i])), v = weight(e);
    const uint64_t m = fixed(v);
    const int k = bin_of(b, e, m);
    rank[j] = atomicAdd(&count[k], 1u) | (uint32_t)k << 16;
    if (m) atomicAdd(&mass[k], (unsigned long long)m);
    if (v >= (double)min_p) large += m;
  }
  __syncthreads();
  const int64_t list = (int64_t)row * chunks + blockIdx.x;
  const uint32_t n = tid < kBins ? count[tid] : 0u, end = block_scan(n, part);
  if (tid < kBins) {
    count[tid] = end - n;
    w.ends[list * kBins + tid] = (uint16_t)end;
    w.mass[list * kBins + tid] = mass[tid];
  }
  large = wave_sum(large);
  if ((tid & 63) == 0) partm[tid >> 6] = large;
  __syncthreads();
  if (tid == 0) {
    for (int v = 1; v < kWaves; ++v) large += partm[v];
    w.large[list] = large;
  }
  uint16_t *order = w.order + list * (T * kThreads);
#pragma unroll
  for (int j = 0; j < T; ++j) {
    if (i0 + j * kThreads + tid >= a.vocab) break;
    order[count[rank[j] >> 16] + (rank[j] & 0xFFFFu)] = (uint16_t)(j * kThreads + tid);
  }
}

// A row's tokens by digits of their places, one workgroup reading the whole row again for each:
// where more tokens share a bin than a workgroup sorts (many equal logits).  The place of the first
// token, in order, at which the running count reaches `want` (by_count) or its running mass is
// `enough`, and the running mass with it.
struct Found {
  uint64_t place, mass;
};
template <typename F>
__device__ Found find_by_digits(const SampleArgs &a, int row, const Row &r, bool by_count,
                                uint32_t want, F enough, uint32_t *count, unsigned long long *mass,
                                uint32_t *part, uint64_t *partm, Found *found) {
  const float *x = a.logits + row * a.ld;
  const int tid = threadIdx.x;
  uint64_t prefix = 0, above_m = 0;
  uint32_t above = 0;
  __shared__ uint32_t s_above;
  // 64 bits in digits of 9 from the top; the last one has one bit
  for (int shift = 55; shift > -9; shift -= 9) {
    const int sh = shift < 0 ? 0 : shift, bits = shift < 0 ? 9 + shift : 9;
    for (int k = tid; k < kBins; k += kThreads) count[k] = 0, mass[k] = 0;
    __syncthreads();
    for (int i = tid; i < a.vocab; i += kThreads) {
      const uint32_t key = order_key(x[i]);
      const uint64_t p = place(key, i);
      if (sh + bits < 64 && (p >> (sh + bits)) != (prefix >> (sh + bits))) continue;
      const int k = (int)(p >> sh) & ((1 << bits) - 1);
      atomicAdd(&count[k], 1u);
      const uint64_t m = mass_of(r, key);
      if (m) atomicAdd(&mass[k], (unsigned long long)m);
    }
    __syncthreads();
    // digits from the largest down, one per thread
    const int k = (1 << bits) - 1 - tid;
    const uint32_t c = k >= 0 ? count[k] : 0u;
    const uint64_t m = k >= 0 ? mass[k] : 0;
    const uint32_t ce = above + block_scan(c, part);
    const uint64_t me = above_m + block_scan(m, partm);
    const bool now = by_count ? ce >= want : enough(me), before = by_count ? ce - c >= want : enough(me - m);
    if (k >= 0 && c && now && !before) {
      found->place = prefix | (uint64_t)k << sh;
      found->mass = me - m;
      s_above = ce - c;
    }
    __syncthreads();
    prefix = found->place;
    above_m = found->mass;
    above = s_above;
    __syncthreads();
  }
  return {prefix, above_m + mass_of(r, (uint32_t)(prefix >> 32))};
}

__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs a, Work w, Cut cut) {
  __shared__ uint32_t count[kBins];              // tokens up to the end of a bin
  __shared__ unsigned long long mass[kBins];     // and their mass
  __shared__ __align__(16) uint64_t list[kSorted];
  __shared__ uint32_t counts[kBins], part[kWaves], begin[kChunks], base[kChunks + 1];
  __shared__ unsigned long long masses[kBins];
  __shared__ uint64_t partm[kWaves];
  __shared__ Found found;
  __shared__ int found_bin;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, chunks = cut.chunks;
  const float *x = a.logits + row * a.ld;
  const Bins b = bins_of(a, w, row, chunks);
  if (!b.first || !(b.t > 0.f)) {
    if (tid == 0) {
      a.out[row] = b.first ? (uint32_t)~(uint32_t)b.first : 0;
      if (a.probs) a.probs[row] = b.first ? 1.f : 0.f;
    }
    return;
  }
  const int32_t top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  const float min_p = a.min_p ? a.min_p[row] : a.min_p_all;
  float u = a.u[row];
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  const int64_t lists = (int64_t)row * chunks;

  // the row's bins: half of the threads take every other chunk
  {
    const int k = tid % kBins, half = tid / kBins;
    uint32_t c = 0;
    uint64_t m = 0;
#pragma unroll 4
    for (int l = half; l < chunks; l += 2) {
      const uint16_t *e = w.ends + (lists + l) * kBins + k;
      c += k ? e[0] - e[-1] : e[0];
      m += w.mass[(lists + l) * kBins + k];
    }
    if (half) counts[k] = c, masses[k] = m;
    __syncthreads();
    if (!half) c += counts[k], m += masses[k];
    else c = 0, m = 0;
    const uint32_t ce = block_scan(c, part);
    const uint64_t me = block_scan(m, partm);
    if (!half) count[k] = ce, mass[k] = me;
    __syncthreads();
  }
  uint64_t large = wave_sum(lane < chunks ? w.large[lists + lane] : (uint64_t)0);

  // the first bin at whose end it is enough; of none, the last
  auto bin_where = [&](auto enough) {
    if (tid == 0) found_bin = kBins - 1;
    __syncthreads();
    if (tid < kBins && enough(count[tid], (uint64_t)mass[tid]) &&
        !(tid && enough(count[tid - 1], (uint64_t)mass[tid - 1])))
      found_bin = tid;
    __syncthreads();
    const int k = found_bin;
    __syncthreads();
    return k;
  };
  // The tokens of bins k0 .. k1 in order, each thread with four neighbours' places and the running
  // masses at their ends.  False: more than fit.
  int sorted = 0;
  uint64_t run[kSorted / kThreads];
  uint64_t run0;
  auto sort_bins = [&](int k0, int k1) {
    const uint32_t before = k0 ? count[k0 - 1] : 0, n = count[k1] - before;
    if (n > kSorted) return false;
    if (tid < 64) {
      uint32_t from = 0, len = 0;
      if (lane < chunks) {
        const uint16_t *e = w.ends + (lists + lane) * kBins;
        from = k0 ? e[k0 - 1] : 0;
        len = e[k1] - from;
      }
      uint32_t end = len;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(end, o);
        if (lane >= o) end += v;
      }
      begin[lane] = from;
      base[lane] = end - len;
      if (lane == 63) base[64] = end;
    }
    int size = 64;
    while (size < (int)n) size <<= 1;
    __syncthreads();
    for (int j = tid; j < size; j += kThreads) {
      uint64_t p = 0;
      if (j < (int)n) {
        int lo = 0, hi = chunks - 1;  // the last chunk with base <= j
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if ((int)base[mid] <= j)
            lo = mid;
          else
            hi = mid - 1;
        }
        const uint32_t i =
            lo * cut.chunk + w.order[(lists + lo) * cut.chunk + begin[lo] + j - base[lo]];
        p = place(order_key(x[i]), i);
      }
      list[j] = p;
    }
    for (int k = 2; k <= size; k <<= 1)
      for (int s = k >> 1; s > 0; s >>= 1) {
        __syncthreads();
        for (int q = tid; q < size / 2; q += kThreads) {
          const int i = 2 * q - (q & (s - 1)), l = i + s;
          const uint64_t p = list[i], r = list[l];
          if ((p < r) == ((i & k) == 0)) list[i] = r, list[l] = p;
        }
      }
    __syncthreads();
    sorted = (int)n;
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < kSorted / kThreads; ++j) {
      const int i = tid * (kSorted / kThreads) + j;
      sum += i < sorted ? mass_of(b.r, (uint32_t)(list[i] >> 32)) : 0;
      run[j] = sum;
    }
    const uint64_t end = block_scan(sum, partm) + (k0 ? mass[k0 - 1] : 0);
    run0 = end - sum;
    return true;
  };
  // the first sorted token at which it is enough
  auto token_where = [&](uint32_t before, auto enough) {
#pragma unroll
    for (int j = 0; j < kSorted / kThreads; ++j) {
      const int i = tid * (kSorted / kThreads) + j;
      if (i < sorted && enough(before + i + 1, run0 + run[j]) &&
          !enough(before + i, run0 + (j ? run[j - 1] : 0))) {
        found.place = list[i];
        found.mass = run0 + run[j];
      }
    }
    __syncthreads();
    const Found f = found;
    __syncthreads();
    return f;
  };
  // The first token of the row at which it is enough, of bin k.  `all`: the sorted tokens are the
  // first of the row, this one among them.
  bool all = false;
  auto find = [&](bool by_count, uint32_t want, auto enough_mass) {
    auto enough = [&](uint32_t c, uint64_t m) { return by_count ? c >= want : enough_mass(m); };
    if (all) return token_where(0, enough);
    const int k = bin_where(enough);
    if (count[k] <= kSorted / 4 && sort_bins(0, k)) {
      all = true;
      return token_where(0, enough);
    }
    if (sort_bins(k, k)) return token_where(k ? count[k - 1] : 0, enough);
    const Found f = find_by_digits(a, row, b.r, by_count, want, enough_mass, counts, masses, part,
                                   partm, &found);
    return f;
  };

  const uint64_t whole = mass[kBins - 1];
  uint64_t total = whole;
  if (!(min_p > 0.f)) large = whole;
  auto never = [](uint64_t) { return false; };
  // (a first run down to tokens of weight zero keeps all mass)
  if (top_k > 0 && (uint32_t)top_k < count[kBins - 2]) total = find(true, (uint32_t)top_k, never).mass;
  if (top_p < 1.f) {
    const double want = fmax((double)top_p * (double)total, 1.0);  // the first token has 2^43
    const uint64_t kept = find(false, 0, [&](uint64_t m) { return (double)m >= want; }).mass;
    total = kept < total ? kept : total;
  }
  total = large < total ? large : total;
  total = total < (uint64_t)kOne ? (uint64_t)kOne : total;
  const double want = (double)u * (double)total;
  const Found f = find(false, 0, [&](uint64_t m) { return (double)m > want; });
  if (tid == 0) {
    a.out[row] = (uint32_t)~(uint32_t)f.place;
    if (a.probs) a.probs[row] = (float)((double)mass_of(b.r, (uint32_t)(f.place >> 32)) / (double)total);
  }
}

}  // namespace

int64_t sample_work_bytes(int64_t rows, int64_t vocab) {
  // of the two cuts the larger, so that a workspace serves fewer rows too
  Work w;
  int64_t most = 16;
  for (int per : {4, 16}) {
    Cut c{per * kThreads, (int)((vocab + per * kThreads - 1) / (per * kThreads))};
    if (c.chunks > kChunks) continue;
    const int64_t n = place_work(nullptr, rows, c, w);
    most = n > most ? n : most;
  }
  return most;
}

hipError_t launch_sample(const SampleArgs &a, hipStream_t s) {
  const Cut c = cut_of(a.rows, a.vocab);
  Work w;
  place_work((char *)a.work, a.rows, c, w);
  const dim3 grid(c.chunks, a.rows), block(kThreads);
  const bool small = c.chunk == 4 * kThreads;
  if (small)
    hipLaunchKernelGGL(sample_top_kernel<4>, grid, block, 0, s, a, w);
  else
    hipLaunchKernelGGL(sample_top_kernel<16>, grid, block, 0, s, a, w);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (small)
    hipLaunchKernelGGL(sample_bins_kernel<4>, grid, block, 0, s, a, w, c.chunks);
  else
    hipLaunchKernelGGL(sample_bins_kernel<16>, grid, block, 0, s, a, w, c.chunks);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sample_draw_kernel, dim3(a.rows), block, 0, s, a, w, c);
  return hipGetLastError();
}

}  // namespace gguf

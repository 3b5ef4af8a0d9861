// Sampling a token per row of logits (gguf_hip_sample.h).
//
// A row is cut into chunks.  Its tokens' weights are sorted into bins by their exponent, evenly over
// the row's range, largest first; a running sum over the bins tells in which bin a limit or the
// draw falls, and only that bin's tokens are put in order.  Three launches:
//   top      each chunk's largest and smallest logit
//   bins     each chunk's bins: their tokens' indices in the order of the bins, and their masses
//   draw     a workgroup per row: the chunks' bins added up, the limits, the draw
// All sums are of 64-bit integers, so that neither the chunks nor timing matter.
//
// One row of 151936 tokens: 3.1 + 5.0 + 11.9 us, launches and chains of loads and barriers.  48 rows, of
// which 16 without top_k: 7 (29 MB, 4.1 TB/s) + 15.5 (the vector unit, most of it in 64 bits) + 19 (two
// bins put in order, one workgroup per row).
#include "paged.hpp"

namespace gguf {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 512;     // the last one for tokens of weight 0, which are in none
constexpr int kSorted = 4096;  // tokens that a workgroup puts in order
constexpr int kRanked = 256;   // up to so many by counting, for each, those before it
constexpr int kFewest = 512;   // a top_k of up to so many needs no bins' masses
constexpr int kChunks = 64;
constexpr double kOne = 0x1p43;     // a weight of 1
constexpr double kNothing = -44.0 * 32;  // the exponent (below) from which on a weight is 0

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

// A row's weights: exponents are log2 of a token's weight, in units of 1 / 32; kLeast and below
// (nothing to draw, too) is a weight of 0 in the sums.
constexpr double kLeast = -60.0 * 32;
struct Row {
  double scale;  // 32 log2(e) / temperature
  float top;     // the largest logit
};
__device__ __forceinline__ double exponent(const Row &r, uint32_t key) {
  const float x = key_value(key);  // of key 0 a NaN
  const double d = x == r.top ? 0.0 : ((double)x - (double)r.top) * r.scale;  // infinite ones too
  return d > kLeast ? d : kLeast;
}
// 2^(y / 32): by a table (in LDS) of 2^(j / 32) and the Taylor series of 2^(f / 32), |f| <= 1/2, to its
// fifth power, whose rest is below 3e-15.  The coefficients are held in scalar registers.
struct Powers {
  const double *table;
  double c5 = 1.0 / 120, c4 = 1.0 / 24, c3 = 1.0 / 6, c2 = 0.5, ln = 0.69314718055994530942 / 32;
  __device__ __forceinline__ explicit Powers(const double *t) : table(t) {
    asm volatile("" : "+s"(c5), "+s"(c4), "+s"(c3), "+s"(c2), "+s"(ln));
  }
  // by all threads, before a barrier
  static __device__ __forceinline__ void fill(double *table) {
    if (threadIdx.x < 32) table[threadIdx.x] = exp2(threadIdx.x / 32.0);
  }
  __device__ __forceinline__ double operator()(double y) const {
    const double n = __builtin_rint(y), f = (y - n) * ln;
    const int k = (int)n;
    const uint64_t t = (uint64_t)__double_as_longlong(table[k & 31]);
    const double at = __longlong_as_double((long long)(t + ((uint64_t)(uint32_t)(k >> 5) << 52)));
    double p = fma(c5, f, c4);
    p = fma(p, f, c3);
    p = fma(p, f, c2);
    p = fma(p, f, 1.0);
    return fma(at * f, p, at);
  }
};
// A weight in multiples of 2^-43: below 2^52, adding 2^52 leaves the nearest integer in the low bits.
__device__ __forceinline__ uint64_t fixed(double w) {
  return (uint64_t)__double_as_longlong(fma(w, kOne, 0x1p52)) & 0xFFFFFFFFFFFFFull;
}
__device__ __forceinline__ uint64_t mass_of(const Row &r, const Powers &pow2, uint32_t key) {
  return fixed(pow2(exponent(r, key)));
}

// Sums and maxima over lanes by DPP shifts within rows of 16, then the rows' ends.  A lane without a
// source gets zero, which neither adds nor is larger.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T shifted(T v) {
  if constexpr (sizeof(T) == 8) {
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xF, false);
    return (T)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
  } else {
    return (T)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
  }
}
template <typename T>
__device__ __forceinline__ T of_lane(T v, int lane) {
  if constexpr (sizeof(T) == 8) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
    return (T)((uint64_t)hi << 32 | lo);
  } else {
    return (T)__builtin_amdgcn_readlane((int)v, lane);
  }
}
template <typename T>
__device__ __forceinline__ T row_sums(T v) {
  v += shifted<0x111, 0xF>(v);
  v += shifted<0x112, 0xF>(v);
  v += shifted<0x114, 0xF>(v);
  return v + shifted<0x118, 0xF>(v);
}
// v and those of the lanes below
template <typename T>
__device__ __forceinline__ T wave_sums(T v) {
  v = row_sums(v);
  v += shifted<0x142, 0xA>(v);  // lane 15 to row 1, 47 to row 3
  return v + shifted<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
  return of_lane(wave_sums(v), 63);
}
template <typename T>
__device__ __forceinline__ T wave_max(T v) {
  auto larger = [](T x, T y) { return x > y ? x : y; };
  v = larger(v, shifted<0x111, 0xF>(v));
  v = larger(v, shifted<0x112, 0xF>(v));
  v = larger(v, shifted<0x114, 0xF>(v));
  v = larger(v, shifted<0x118, 0xF>(v));
  v = larger(v, shifted<0x142, 0xA>(v));
  v = larger(v, shifted<0x143, 0xC>(v));
  return of_lane(v, 63);
}
// v and those of the threads below; `part` holds a value per wave.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *part) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  v = wave_sums(v);
  __syncthreads();
  if (lane == 63) part[wave] = v;
  __syncthreads();
  static_assert(kWaves == 16);
  const T before = row_sums(part[lane & 15]);
  return wave ? v + of_lane(before, wave - 1) : v;
}

// The workspace: per row and chunk the place of its first token and the inverse of its smallest
// key; the mass that min_p keeps; its bins; its tokens in their order (indices within the chunk).
struct Bin {
  uint16_t count, end;  // of the chunk's tokens in the order of the bins
};
struct Work {
  uint64_t *first, *large, *mass;
  Bin *bin;
  uint32_t *least;
  uint16_t *order;
};
struct Cut {
  int chunk, chunks;  // tokens of a chunk, chunks of a row
};
// Small chunks while they do not fill the chip (us of a replayed call of 48 rows of 151936 tokens:
// 16 tokens a thread 40.4, eight 43.4).
constexpr int64_t kSmall = 4 * kThreads * 1024;  // tokens of a call
Cut cut(int64_t vocab, bool small) {
  const int chunk = (small ? 4 : 16) * kThreads;
  return {chunk, (int)((vocab + chunk - 1) / chunk)};
}
Cut cut_of(int64_t rows, int64_t vocab) {
  return cut(vocab, vocab <= 4 * kThreads * kChunks && rows * vocab < kSmall);
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
  w.bin = (Bin *)take(lists * kBins * sizeof(Bin));
  w.least = (uint32_t *)take(lists * 4);
  w.order = (uint16_t *)take(lists * c.chunk * 2);
  return p - base;
}

template <int T>
__global__ __launch_bounds__(kThreads) void sample_top_kernel(SampleArgs a, Work w) {
  __shared__ uint64_t part[kWaves];
  __shared__ uint32_t partl[kWaves];
  const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * T * kThreads;
  const float *x = a.logits + row * a.ld;
  float high = -INFINITY, low = INFINITY;  // of those above -inf
  int at = 0;
#pragma unroll
  for (int j = 0; j < T; ++j) {
    const int i = min(i0 + j * kThreads + tid, a.vocab - 1);  // past the end: the last again
    const float y = x[i];
    at = y > high ? i : at;
    high = y > high ? y : high;
    low = y > -INFINITY && y < low ? y : low;
  }
  uint64_t first = high > -INFINITY ? place(order_key(high), at) : 0;
  uint32_t least = high > -INFINITY ? ~order_key(low) : 0u;
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
struct Chunk {  // what the first launch left of a lane's chunk
  uint64_t first;
  uint32_t least;
};
__device__ __forceinline__ Chunk chunk_of(const Work &w, int row, int chunks) {
  const int64_t list = (int64_t)row * chunks + min((int)(threadIdx.x & 63), chunks - 1);
  return {w.first[list], w.least[list]};
}
__device__ __forceinline__ Bins bins_of(const SampleArgs &a, int row, const Chunk &c) {
  Bins b;
  b.t = a.temperature ? steady(a.temperature + row) : a.temperature_all;
  b.first = wave_max(c.first);
  const uint32_t least = wave_max(c.least);
  b.r.scale = 32 * 1.4426950408889634074 / (double)b.t;
  b.r.top = key_value((uint32_t)(b.first >> 32));
  const double range = fmin(-exponent(b.r, ~least), -kNothing);
  b.per = range > 0.0 ? (kBins - 1) / range : 0.0;
  return b;
}
// Where the first top_k tokens are all that counts, their masses are taken from them alone.
__device__ __forceinline__ bool few(int32_t top_k) { return top_k > 0 && top_k <= kFewest; }

template <int T>
__global__ __launch_bounds__(kThreads, 8) void sample_bins_kernel(SampleArgs a, Work w, int chunks) {
  __shared__ uint32_t count[kBins];
  __shared__ unsigned long long mass[kBins];
  __shared__ uint32_t part[kWaves];
  __shared__ uint64_t partm[kWaves];
  __shared__ __align__(16) uint16_t order[T * kThreads];
  __shared__ uint32_t wanted, fewest;
  __shared__ double table[32];
  const int row = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * T * kThreads;
  const float *x = a.logits + row * a.ld;
  constexpr int L = T < 8 ? T : 8;  // tokens of a thread in flight
  float y[L];
  auto load = [&](int j0) {
#pragma unroll
    for (int j = 0; j < L; ++j) y[j] = x[min(i0 + (j0 + j) * kThreads + tid, a.vocab - 1)];
  };
  const Chunk own = chunk_of(w, row, chunks);
  load(0);
  const float min_p = a.min_p ? steady(a.min_p + row) : a.min_p_all;
  const int32_t top_k = a.top_k ? steady(a.top_k + row) : a.top_k_all;
  const bool counts_only = few(top_k);
  for (int k = tid; k < kBins; k += kThreads) count[k] = 0, mass[k] = 0;
  if (tid == 0) fewest = ~0u;
  Powers::fill(table);
  const Powers pow2(table);
  const Bins b = bins_of(a, row, own);
  if (!b.first || !(b.t > 0.f)) return;  // nothing to draw, or no draw
  __syncthreads();
  uint32_t rank[T];  // bin and place in it; a token of weight 0 has none
  uint64_t large = 0;
  const bool endless = b.r.top == INFINITY;
  const double top = endless ? 0.0 : (double)b.r.top;
#pragma unroll
  for (int j = 0; j < T; ++j) {
    if (j && j % L == 0) load(j);
    if (j % L == 0 && endless)  // as logits of 0 and of less than any
#pragma unroll
      for (int l = 0; l < L; ++l) y[l] = y[l] == INFINITY ? 0.f : -INFINITY;
    const double e = ((double)y[j % L] - top) * b.r.scale;  // as `exponent`
    rank[j] = ~0u;
    if (!(e > kNothing) || i0 + j * kThreads + tid >= a.vocab) continue;
    const int k = min((int)(-e * b.per), kBins - 2);
    rank[j] = atomicAdd(&count[k], 1u) | (uint32_t)k << 16;
    if (counts_only) continue;
    const double v = pow2(e);
    const uint64_t m = fixed(v);
    if (m) atomicAdd(&mass[k], (unsigned long long)m);
    if (v >= (double)min_p) large += m;
  }
  __syncthreads();
  const int64_t list = (int64_t)row * chunks + blockIdx.x;
  const uint32_t n = tid < kBins ? count[tid] : 0u, end = block_scan(n, part);
  // those that may be asked for: not the tokens of weight zero, of the first top_k the chunk's own
  if (tid == kBins - 2) wanted = end;
  if (counts_only && tid < kBins - 1 && end >= top_k && end - n < top_k) fewest = end;
  if (tid < kBins) {
    count[tid] = end - n;
    w.bin[list * kBins + tid] = {(uint16_t)n, (uint16_t)end};
    if (!counts_only) w.mass[list * kBins + tid] = mass[tid];
  }
  large = wave_sum(large);
  if ((tid & 63) == 0) partm[tid >> 6] = large;
  __syncthreads();
  if (tid == 0) {
    for (int v = 1; v < kWaves; ++v) large += partm[v];
    w.large[list] = large;
  }
  // put together here: written one by one, the indices took most of the kernel's time
#pragma unroll
  for (int j = 0; j < T; ++j) {
    if (rank[j] == ~0u) continue;
    order[count[rank[j] >> 16] + (rank[j] & 0xFFFFu)] = (uint16_t)(j * kThreads + tid);
  }
  __syncthreads();
  const uint32_t last = min(wanted, fewest);
  uint4 *to = (uint4 *)(w.order + list * (T * kThreads));
  for (uint32_t q = tid; 8 * q < last; q += kThreads) to[q] = ((const uint4 *)order)[q];
}

// A row's tokens by digits of their places, one workgroup reading the whole row again for each:
// where more tokens share a bin than a workgroup sorts.  Those are many equal logits, or a row whose
// range is wide for its temperature, so that its bins are: of 151936 normal logits at temperature 2, 30 %
// masked with -1e4, 310 us (48 rows 343; masked with -inf 29 and 43, at temperature 1 32 and 58).  The
// place of the first token, in order, at which it is enough, and the running mass with it.
struct Found {
  uint64_t place, mass;
};
// When it is enough: `count` tokens, or (count 0) a mass of `mass`, or of more than that.
struct Goal {
  uint32_t count;
  bool more;
  double mass;
  __device__ __forceinline__ bool operator()(uint32_t c, uint64_t m) const {
    return count ? c >= count : (more ? (double)m > mass : (double)m >= mass);
  }
};
__device__ Found find_by_digits(const SampleArgs &a, int row, const Row &r, const Powers &pow2,
                                const Goal &enough,
                                uint32_t *count, unsigned long long *mass, uint32_t *part,
                                uint64_t *partm, Found *found) {
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
      const uint64_t m = mass_of(r, pow2, key);
      if (m) atomicAdd(&mass[k], (unsigned long long)m);
    }
    __syncthreads();
    // digits from the largest down, one per thread
    const int k = (1 << bits) - 1 - tid;
    const uint32_t c = k >= 0 ? count[k] : 0u;
    const uint64_t m = k >= 0 ? mass[k] : 0;
    const uint32_t ce = above + block_scan(c, part);
    const uint64_t me = above_m + block_scan(m, partm);
    if (k >= 0 && c && enough(ce, me) && !enough(ce - c, me - m)) {
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
  return {prefix, above_m + mass_of(r, pow2, (uint32_t)(prefix >> 32))};
}

// Tokens in order: those of a run of bins, or of a part of one.
struct Sorted {
  uint32_t before;      // tokens of the row before them
  uint64_t mass_before;
  int n;
};

__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs a, Work w, Cut cut) {
  __shared__ uint32_t count[kBins];              // tokens up to the end of a bin
  __shared__ unsigned long long mass[kBins];     // and their mass
  __shared__ __align__(16) uint64_t list[kSorted], next[kSorted];
  __shared__ uint32_t counts[kBins], part[kWaves], begin[kChunks], base[kChunks + 1];
  __shared__ unsigned long long masses[kBins];
  __shared__ uint64_t partm[kWaves];
  __shared__ Found found;
  __shared__ int found_bin;
  __shared__ uint32_t appended;
  __shared__ double table[32];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, chunks = cut.chunks;
  const float *x = a.logits + row * a.ld;
  const int64_t lists = (int64_t)row * chunks;
  const int32_t top_k = a.top_k ? steady(a.top_k + row) : a.top_k_all;
  const float top_p = a.top_p ? steady(a.top_p + row) : a.top_p_all;
  const float min_p = a.min_p ? steady(a.min_p + row) : a.min_p_all;
  float u = steady(a.u + row);
  u = u > 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
  Powers::fill(table);
  const Powers pow2(table);
  // the row's bins: half of the threads take every other chunk
  const Chunk own = chunk_of(w, row, chunks);
  uint64_t large = w.large[lists + min(lane, chunks - 1)];
  uint32_t c = 0;
  uint64_t m = 0;
  {
    const int64_t at = lists * kBins + tid % kBins;
    const uint32_t *bin = (const uint32_t *)w.bin + at;
    const uint64_t *mass = w.mass + at;
    constexpr int L = 8;  // chunks in flight
    for (int l0 = tid / kBins; l0 < chunks; l0 += 2 * L) {
      uint32_t cl[L];
      uint64_t ml[L] = {};
#pragma unroll
      for (int j = 0; j < L; ++j) cl[j] = bin[min(l0 + 2 * j, chunks - 1) * kBins] & 0xFFFFu;
      if (!few(top_k))
#pragma unroll
        for (int j = 0; j < L; ++j) ml[j] = mass[min(l0 + 2 * j, chunks - 1) * kBins];
#pragma unroll
      for (int j = 0; j < L; ++j) {
        c += l0 + 2 * j < chunks ? cl[j] : 0;
        m += l0 + 2 * j < chunks ? ml[j] : 0;
      }
    }
  }
  const Bins b = bins_of(a, row, own);
  if (!b.first || !(b.t > 0.f)) {  // the bins have not been made
    if (tid == 0) {
      a.out[row] = b.first ? (uint32_t)~(uint32_t)b.first : 0;
      if (a.probs) a.probs[row] = b.first ? 1.f : 0.f;
    }
    return;
  }
  if (tid >= kBins) counts[tid - kBins] = c, masses[tid - kBins] = m;
  __syncthreads();
  c = tid < kBins ? c + counts[tid] : 0;
  m = tid < kBins ? m + masses[tid] : 0;
  const uint32_t ce = block_scan(c, part);
  const uint64_t me = block_scan(m, partm);
  if (tid < kBins) count[tid] = ce, mass[tid] = me;
  large = wave_sum(lane < chunks ? large : (uint64_t)0);
  __syncthreads();

  // the first of the bins (sums up to their ends) at which it is enough; of none, the last
  auto bin_where = [&](const uint32_t *cs, const unsigned long long *ms, uint32_t c0, uint64_t m0,
                       const Goal &enough) {
    if (tid == 0) found_bin = kBins - 1;
    __syncthreads();
    if (tid < kBins && enough(c0 + cs[tid], m0 + ms[tid]) &&
        !(tid && enough(c0 + cs[tid - 1], m0 + ms[tid - 1])))
      found_bin = tid;
    __syncthreads();
    return found_bin;
  };
  // The n tokens of bins k0 .. k1 (n <= kSorted) into `list`, in no order.
  auto gather = [&](int k0, int k1, uint32_t n) {
    if (tid < 64) {
      uint32_t from = 0, len = 0;
      if (lane < chunks) {
        const Bin *bin = w.bin + (lists + lane) * kBins;
        const Bin v = bin[k1], v0 = bin[k0];
        from = v0.end - v0.count;
        len = v.end - from;
      }
      const uint32_t end = wave_sums(len);
      begin[lane] = from;
      base[lane] = end - len;
    }
    __syncthreads();
    for (uint32_t j = tid; j < n; j += kThreads) {
      int lo = 0, hi = chunks - 1;  // the last chunk with base <= j
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (base[mid] <= j)
          lo = mid;
        else
          hi = mid - 1;
      }
      const uint32_t i = lo * cut.chunk + w.order[(lists + lo) * cut.chunk + begin[lo] + j - base[lo]];
      list[j] = place(order_key(x[i]), i);
    }
    __syncthreads();
  };
  // the first n tokens of `list` put in order
  auto sort = [&](int n) {
    if (n <= kRanked) {
      uint64_t p = 0;
      int rank = 0;
      if (tid < n) {
        p = list[tid];
#pragma unroll 16
        for (int j = 0; j < n; ++j) rank += list[j] > p;
      }
      __syncthreads();
      if (tid < n) list[rank] = p;
      __syncthreads();
      return;
    }
    int size = 2 * kRanked;
    while (size < n) size <<= 1;
    for (int j = n + tid; j < size; j += kThreads) list[j] = 0;
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
  };
  // each thread's four neighbours of the sorted tokens: the running masses at their ends
  constexpr int kEach = kSorted / kThreads;
  Sorted in{0, 0, 0};
  uint64_t run[kEach], run0 = 0;
  auto masses_of = [&](const Sorted &of) {
    in = of;
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = tid + j * kThreads;
      if (i < in.n) next[i] = mass_of(b.r, pow2, (uint32_t)(list[i] >> 32));
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = tid * kEach + j;
      sum += i < in.n ? next[i] : 0;
      run[j] = sum;
    }
    run0 = block_scan(sum, partm) + in.mass_before - sum;
  };
  // the first sorted token at which it is enough
  auto token_where = [&](const Goal &enough) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = tid * kEach + j;
      if (i < in.n && enough(in.before + i + 1, run0 + run[j]) &&
          !enough(in.before + i, run0 + (j ? run[j - 1] : 0))) {
        found.place = list[i];
        found.mass = run0 + run[j];
      }
    }
    __syncthreads();
    const Found f = found;
    __syncthreads();
    return f;
  };
  // Of the n tokens in `list`, from (c0, m0) on, more than are sorted by counting: those that share
  // the bin, by their logits' bits, in which it is enough.
  auto narrow = [&](const Sorted &of, const Goal &enough) {
    uint32_t lo = ~0u, hi = 0;
    for (int j = tid; j < of.n; j += kThreads) {
      const uint32_t k = (uint32_t)(list[j] >> 32);
      lo = k < lo ? k : lo;
      hi = k > hi ? k : hi;
    }
    lo = ~wave_max(~lo);
    hi = wave_max(hi);
    if (lane == 0) part[tid >> 6] = lo, partm[tid >> 6] = hi;
    if (tid < kBins) counts[tid] = 0, masses[tid] = 0;
    if (tid == 0) appended = 0;
    __syncthreads();
    for (int v = 0; v < kWaves; ++v) {
      lo = part[v] < lo ? part[v] : lo;
      hi = (uint32_t)partm[v] > hi ? (uint32_t)partm[v] : hi;
    }
    const uint32_t per = (hi - lo) / kBins + 1;  // keys of a bin
    for (int j = tid; j < of.n; j += kThreads) {
      const uint32_t key = (uint32_t)(list[j] >> 32), k = (hi - key) / per;
      atomicAdd(&counts[k], 1u);
      atomicAdd(&masses[k], (unsigned long long)mass_of(b.r, pow2, key));
    }
    __syncthreads();
    const uint32_t cs = tid < kBins ? counts[tid] : 0;
    const uint64_t ms = tid < kBins ? masses[tid] : 0;
    const uint32_t ce = block_scan(cs, part);
    const uint64_t me = block_scan(ms, partm);
    if (tid < kBins) counts[tid] = ce, masses[tid] = me;
    __syncthreads();
    const int k = bin_where(counts, masses, of.before, of.mass_before, enough);
    const int n = (int)(counts[k] - (k ? counts[k - 1] : 0));
    const Sorted to{of.before + (k ? counts[k - 1] : 0), of.mass_before + (k ? masses[k - 1] : 0), n};
    for (int j = tid; j < of.n; j += kThreads) {
      const uint64_t p = list[j];
      if ((int)((hi - (uint32_t)(p >> 32)) / per) == k) next[atomicAdd(&appended, 1u)] = p;
    }
    __syncthreads();
    for (int j = tid; j < n; j += kThreads) list[j] = next[j];
    __syncthreads();
    return to;
  };
  // The first token of the row at which it is enough.  `all`: the sorted tokens are the first of the
  // row, this one among them.
  bool all = false, by_digits = false;
  auto find = [&](const Goal &enough) {
    if (!all) {
      const int k = by_digits ? 0 : bin_where(count, mass, 0, 0, enough);
      const uint32_t before = k ? count[k - 1] : 0;
      all = !by_digits && (count[k] <= kRanked || (few(top_k) && count[k] <= kSorted));
      Sorted of{before, k ? (uint64_t)mass[k - 1] : 0, (int)(count[k] - before)};
      if (all) of = {0, 0, (int)count[k]};
      // (where the bins have no masses, those before this one are not known without `all`)
      if (by_digits || of.n > kSorted || (few(top_k) && !all))
        return find_by_digits(a, row, b.r, pow2, enough, counts, masses, part, partm, &found);
      gather(all ? 0 : k, k, of.n);
      if (!all && of.n > kRanked) of = narrow(of, enough);
      sort(of.n);
      masses_of(of);
    }
    return token_where(enough);
  };

  uint64_t total = mass[kBins - 1];
  const uint32_t most = count[kBins - 2];  // tokens of a weight above zero: a run of them keeps all mass
  Found f{0, 0};
#pragma unroll 1
  for (int goal = 0; goal < 3; ++goal) {  // top_k, top_p, the draw
    Goal enough{0, false, 0.0};
    if (goal == 0) {
      if (!few(top_k) && (top_k <= 0 || (uint32_t)top_k >= most)) continue;
      enough.count = min((uint32_t)top_k, most);
    } else if (goal == 1) {
      if (!(top_p < 1.f)) continue;
      enough.mass = fmax((double)top_p * (double)total, 1.0);  // the first token has 2^43
    } else {
      if (min_p > 0.f) {
        if (few(top_k)) {  // not known yet: of the kept ones, or of all
          large = 0;
          const int n = all ? in.n : a.vocab;
          for (int i = tid; i < n; i += kThreads) {
            const double v = pow2(exponent(b.r, all ? (uint32_t)(list[i] >> 32) : order_key(x[i])));
            if (v >= (double)min_p) large += fixed(v);
          }
          large = wave_sum(large);
          __syncthreads();
          if (lane == 0) partm[tid >> 6] = large;
          __syncthreads();
          large = 0;
          for (int v = 0; v < kWaves; ++v) large += partm[v];
        }
        total = large < total ? large : total;
        total = total < (uint64_t)kOne ? (uint64_t)kOne : total;
      }
      enough.more = true;
      enough.mass = (double)u * (double)total;
    }
    f = find(enough);
    if (goal == 0) {
      total = f.mass;
      by_digits = few(top_k) && !all;  // the bins' masses have not been made
    } else if (goal == 1) {
      total = f.mass < total ? f.mass : total;
    }
  }
  if (tid == 0) {
    a.out[row] = (uint32_t)~(uint32_t)f.place;
    if (a.probs) a.probs[row] = (float)((double)mass_of(b.r, pow2, (uint32_t)(f.place >> 32)) / (double)total);
  }
}

}  // namespace

int64_t sample_work_bytes(int64_t rows, int64_t vocab) {
  // a workspace serves fewer rows too: those that are cut into small chunks, and all of them
  Work w;
  const int64_t few = (kSmall - 1) / vocab < rows ? (kSmall - 1) / vocab : rows;
  const int64_t a = place_work(nullptr, few, cut_of(few, vocab), w);
  const int64_t b = place_work(nullptr, rows, cut_of(rows, vocab), w);
  return (a > b ? a : b) + 16;
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

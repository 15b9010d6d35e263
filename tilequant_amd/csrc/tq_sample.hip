// tq_sample.hip -- drawing one token per row of logits with temperature, top-k, top-p and min-p, gfx950.
//
// Row z[0 .. V), settings T, k, p, m and one number u in [0, 1).  Tokens are taken in the order of descending z, equal
// ones by ascending index; w_i = exp((z_i - z_max) / T).
//   top-k   keeps the first k (k <= 0 or k >= V: all); W_k is the mass (sum of w) of what it keeps;
//   top-p   keeps token i of those while the mass before it is < p W_k (p >= 1: all);
//   min-p   keeps those with w_i >= m;                    the first token is always kept.
//   The answer is the first kept token, in that order, whose inclusive mass is > u W, W the mass of the kept.
// Every rule keeps a prefix of the order, so a row needs only: the prefix mass at a rank, and the first rank whose prefix
// mass passes a target.  NaN counts as -infinity, which is never drawn; +infinity leaves only the infinite ones, equally
// likely.  T <= 0 (or NaN), or a row with nothing to draw: torch.argmax's answer (NaN first, then the lowest index).
//
// Which token a number u falls on has to be the same whatever the order of summation, and the steps of the cumulative
// distribution are as small as a token's probability (1e-6 and less), so masses are exact integers: w is computed in
// fp64 and rounded to a multiple of 2^-40 (tokens below 2^-41 of the likeliest count as 0), and sums are 64-bit.
//
// One workgroup of 1024 threads per row.  The row is read two or more times (the second time from the caches); the
// choice of path is by the row's settings:
//   list   k <= 512, or min-p alone: a bound that at least k logits reach comes from the threads' maxima; the logits
//          above it (a few more than k) are sorted in LDS, and all rules are applied there.
//   bins   otherwise: one pass adds every token's count and mass to 128 bins of 0.3 octaves of w, then only the tokens of
//          the bins where a target falls are sorted.  Bins are 128 columns wide, and a lane adds to the column of its
//          number: no bank conflicts, no two lanes of a wave at one address.  A bin with more tokens than the list holds
//          is divided by key until it fits or holds one value, whose ties are counted in index order.
#include "tq_common.h"

namespace tq {

constexpr int kSampThreads = 1024;
constexpr int kSampWaves = kSampThreads / kWave;
constexpr int kSampBins = 128;
constexpr int kSampCols = 128;
constexpr int kSampList = 8192;        // entries of the sorted list: 8 bytes of key and index, 8 of prefix mass
constexpr int kSampTopK = 512;         // largest k of the list path: half the threads' maxima
constexpr int kSampBoundBins = 512;
constexpr int kSampMaxVocab = 500000;  // a column's count has 12 bits: 1024 threads deal at most 4095 tokens to a column
constexpr int kSampWhole = 2048;       // the bins down to the last one needed are sorted together up to this many tokens
constexpr uint64_t kSampCount = 1ull << 52;    // one token in a column's word: count above bit 52, mass below

struct SampleArgs {
  const void* x;
  int64_t ld;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature0, top_p0, min_p0;
  int top_k0;
  int64_t* out;
  int rows, vocab;
};

struct F32In {
  using T = float;
  static constexpr int kVec = 4;
  __device__ static inline void unpack(u32x4 w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  }
};
template <class XT>
struct H16In {
  using T = uint16_t;
  static constexpr int kVec = 8;
  __device__ static inline void unpack(u32x4 w, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = XT::to_f32((uint16_t)(w[i] & 0xffffu));
      f[2 * i + 1] = XT::to_f32((uint16_t)(w[i] >> 16));
    }
  }
};

// Unsigned order of the bits = order of the numbers (both zeros the same, no NaN).
__device__ inline uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);
  return b ^ ((int32_t)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ inline float of_key(uint32_t k) { return __uint_as_float(k ^ ((int32_t)k < 0 ? 0x80000000u : 0xffffffffu)); }

// 2^x for x in [-42, 0]: the Taylor series of e^(f ln 2), |f| <= 1/2, to degree 11 (6e-15 relative).
__device__ inline double exp2_small(double x) {
  const double n = __builtin_rint(x);
  const double f = (x - n) * 0.693147180559945309417;
  double r = 1.0 / 39916800.0;
  r = fma(r, f, 1.0 / 3628800.0);
  r = fma(r, f, 1.0 / 362880.0);
  r = fma(r, f, 1.0 / 40320.0);
  r = fma(r, f, 1.0 / 5040.0);
  r = fma(r, f, 1.0 / 720.0);
  r = fma(r, f, 1.0 / 120.0);
  r = fma(r, f, 1.0 / 24.0);
  r = fma(r, f, 1.0 / 6.0);
  r = fma(r, f, 0.5);
  r = fma(r, f, 1.0);
  r = fma(r, f, 1.0);
  return __builtin_ldexp(r, (int)n);
}

// The row as its settings see it.
struct SampleRow {
  float top;       // z_max
  bool infinite;   // z_max is +infinity: z becomes 0 there and -infinity elsewhere (top is 0 then)
  double c;        // log2(e) / T
  __device__ inline float see(float z) const {   // NaN -> -infinity
    if (infinite) return z == INFINITY ? 0.0f : -INFINITY;
    return z == z ? z : -INFINITY;
  }
  __device__ inline double x(float z) const { return z == -INFINITY ? -1e30 : ((double)z - (double)top) * c; }
  __device__ inline double weight(float z) const {
    const double v = x(z);
    return v < -42.0 ? 0.0 : exp2_small(v);
  }
  // the weight in 2^-40: adding 2^12 leaves it in the low bits of the mantissa, rounded to nearest
  __device__ static inline uint64_t mass(double w) {
    return __builtin_bit_cast(uint64_t, w + 4096.0) & (kSampCount - 1);
  }
  __device__ static inline int bin(double v) { return min((int)(v * -3.0), kSampBins - 1); }
};

struct SampleShared {
  float red_f[kSampWaves];
  uint64_t red_u[kSampWaves];
  int red_i[kSampWaves];
  uint32_t bound[kSampBoundBins];
  uint32_t bin_count[kSampBins];
  uint64_t bin_mass[kSampBins];      // then: before each bin
  uint32_t bin_before[kSampBins];
  uint64_t mass_before[kSampBins];
  int n_list, found, found_index;
  uint32_t lo, hi;
  uint64_t found_before, found_mass;
};

__device__ inline float block_max_f(float v, float* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[threadIdx.x & (kSampWaves - 1)];
#pragma unroll
  for (int o = kSampWaves / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  return v;
}
__device__ inline uint64_t block_sum(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[threadIdx.x & (kSampWaves - 1)];
#pragma unroll
  for (int o = kSampWaves / 2; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  return v;
}
// sum of v over the threads before this one
__device__ inline uint64_t block_before(uint64_t v, uint64_t* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t inc = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint64_t y = __shfl_up(inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == kWave - 1) red[wave] = inc;
  __syncthreads();
  uint64_t before = inc - v;
  for (int w = 0; w < wave; ++w) before += red[w];
  __syncthreads();
  return before;
}

// f(z, i) for the vectors vec0, vec0 + step, .. of the row: 16-byte aligned loads from the one that holds the row's first
// element on; what they hold beside the row is given as -infinity with an index out of range.
template <class IN, class F>
__device__ inline void sweep(const typename IN::T* row, int vocab, int vec0, int vec1, int step, F f) {
  constexpr int V = IN::kVec;
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(typename IN::T));
  const u32x4* base = reinterpret_cast<const u32x4*>(row - off);
  constexpr int kBatch = 4;
  for (int j0 = vec0; j0 < vec1; j0 += step * kBatch) {
    u32x4 w[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) w[b] = base[min(j0 + b * step, vec1 - 1)];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int j = j0 + b * step;
      float z[V];
      IN::unpack(w[b], z);
      const int i0 = j * V - off;
      if (i0 < 0 || i0 + V > vocab || j >= vec1) {
#pragma unroll
        for (int e = 0; e < V; ++e) z[e] = (j < vec1 && i0 + e >= 0 && i0 + e < vocab) ? z[e] : -INFINITY;
      }
      f(z, i0);
    }
  }
}
template <class IN>
__device__ inline int row_vectors(const typename IN::T* row, int vocab) {
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(typename IN::T));
  return (off + vocab + IN::kVec - 1) / IN::kVec;
}

// torch.argmax: NaN first, then the largest, the lowest index among equals.
template <class IN>
__device__ inline int argmax_row(const typename IN::T* row, int vocab, SampleShared& sh) {
  float best = -INFINITY;
  int at = 0x7fffffff;
  sweep<IN>(row, vocab, threadIdx.x, row_vectors<IN>(row, vocab), kSampThreads, [&](const auto& z, int i0) {
#pragma unroll
    for (int e = 0; e < IN::kVec; ++e) {
      const int i = i0 + e;
      if (i < 0 || i >= vocab) continue;
      const float v = z[e] == z[e] ? z[e] : INFINITY;
      const bool nan = z[e] != z[e], had = best != best;
      const bool better = at == 0x7fffffff || (nan && !had) || (!had && !nan && v > best);
      if (better) {   // a thread's indexes ascend: the first of equals stays
        best = z[e];
        at = i;
      }
    }
  });
  const auto pick = [](float& v, int& i, float v2, int i2) {
    const bool n1 = v != v, n2 = v2 != v2;
    const bool take = n1 != n2 ? n2 : (n1 || v == v2) ? i2 < i : v2 > v;
    if (take) {
      v = v2;
      i = i2;
    }
  };
#pragma unroll
  for (int o = 32; o; o >>= 1) pick(best, at, __shfl_xor(best, o), __shfl_xor(at, o));
  if ((threadIdx.x & 63) == 0) {
    sh.red_f[threadIdx.x >> 6] = best;
    sh.red_i[threadIdx.x >> 6] = at;
  }
  __syncthreads();
  best = sh.red_f[0];
  at = sh.red_i[0];
  for (int w = 1; w < kSampWaves; ++w) pick(best, at, sh.red_f[w], sh.red_i[w]);
  __syncthreads();
  return at;
}

// ---- the sorted list ------------------------------------------------------------
// list[i] = (~key) << 32 | index: ascending order is the order of the tokens.  n entries at any place; afterwards sorted.
__device__ inline void sort_list(uint64_t* list, uint64_t* spare, int n) {
  const int t = threadIdx.x;
  if (n <= 256) {   // by rank: four threads per entry, each against a quarter of the others
    const int e = t >> 2, part = t & 3;
    uint64_t mine = ~0ull;
    int rank = 0;
    if (e < n) {
      mine = list[e];
      for (int j = part; j < n; j += 4) rank += list[j] < mine;
    }
    rank += __shfl_xor(rank, 1);
    rank += __shfl_xor(rank, 2);
    if (e < n && part == 0) spare[rank] = mine;
    __syncthreads();
    if (t < n) list[t] = spare[t];
    __syncthreads();
    return;
  }
  int size = 512;
  while (size < n) size <<= 1;
  for (int i = n + t; i < size; i += kSampThreads) list[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j; j >>= 1) {
      for (int i = t; i < size / 2; i += kSampThreads) {
        const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
        const uint64_t x = list[a], y = list[b];
        if ((x > y) == ((a & k) == 0)) {
          list[a] = y;
          list[b] = x;
        }
      }
      __syncthreads();
    }
}

// prefix[i] = mass of the entries 0 .. i
__device__ inline void sum_list(const uint64_t* list, uint64_t* prefix, int n, const SampleRow& r, SampleShared& sh) {
  const int per = (n + kSampThreads - 1) / kSampThreads, i0 = threadIdx.x * per, i1 = min(i0 + per, n);
  uint64_t sum = 0;
  for (int i = i0; i < i1; ++i) {
    sum += SampleRow::mass(r.weight(of_key(~(uint32_t)(list[i] >> 32))));
    prefix[i] = sum;
  }
  const uint64_t before = block_before(sum, sh.red_u);
  for (int i = i0; i < i1; ++i) prefix[i] += before;
  __syncthreads();
}

// First entry whose inclusive mass (with `base` before the list) is > target, or >= it; n if none.
__device__ inline int first_past(const uint64_t* prefix, int n, uint64_t base, double target, bool or_equal) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    const double s = (double)(base + prefix[mid]);
    if (or_equal ? s >= target : s > target) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Adds the row's tokens that `take(z, key)` accepts to the list.  The list holds kSampList entries; sh.n_list is their number
// also where it is more.
template <class IN, class F>
__device__ inline void collect(const typename IN::T* row, int vocab, const SampleRow& r, uint64_t* list, SampleShared& sh,
                               F take) {
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  sweep<IN>(row, vocab, threadIdx.x, row_vectors<IN>(row, vocab), kSampThreads, [&](const auto& z, int i0) {
#pragma unroll
    for (int e = 0; e < IN::kVec; ++e) {
      const float v = r.see(z[e]);
      if (v != -INFINITY && take(v)) {
        const int at = atomicAdd(&sh.n_list, 1);
        if (at < kSampList) list[at] = (uint64_t)~key_of(v) << 32 | (uint32_t)(i0 + e);
      }
    }
  });
  __syncthreads();
}

// Applies the rules to a sorted list that is the whole beginning of the order.  w_k: the mass top-p is a part of, or
// ~0 for that of the list's first k.
__device__ inline int draw_from_list(const uint64_t* list, const uint64_t* prefix, int n, int k, double p, double m, double u,
                                     uint64_t w_k, const SampleRow& r) {
  int kept = k > 0 ? min(k, n) : n;
  if (p < 1.0) {
    const double all = (double)(w_k == ~0ull ? prefix[kept - 1] : w_k);
    kept = min(kept, first_past(prefix, kept, 0, p * all, true) + 1);
  }
  if (m > 0.0) {   // weights descend
    int lo = 0, hi = kept;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (r.weight(of_key(~(uint32_t)(list[mid] >> 32))) >= m) lo = mid + 1;
      else hi = mid;
    }
    kept = lo;
  }
  kept = max(kept, 1);
  const int at = min(first_past(prefix, kept, 0, u * (double)prefix[kept - 1], false), kept - 1);
  return (int)(uint32_t)list[at];
}

// ---- bins -----------------------------------------------------------------------
// Counts and masses of up to kSampBins bins over the tokens for which bin_of(z, x) >= 0; prefix sums in sh.
template <class IN, class F>
__device__ inline void fill_bins(const typename IN::T* row, int vocab, const SampleRow& r, uint64_t* cells, SampleShared& sh,
                                 F bin_of) {
  const int t = threadIdx.x;
  for (int i = t; i < kSampBins * kSampCols; i += kSampThreads) cells[i] = 0;
  __syncthreads();
  uint64_t* mine = cells + (t & (kSampCols - 1));
  sweep<IN>(row, vocab, t, row_vectors<IN>(row, vocab), kSampThreads, [&](const auto& z, int) {
#pragma unroll
    for (int e = 0; e < IN::kVec; ++e) {
      const float v = r.see(z[e]);
      const double x = r.x(v);
      if (x >= -42.0) {
        const double w = exp2_small(x);
        const int b = bin_of(v, x, w);
        if (b >= 0) atomicAdd((unsigned long long*)&mine[b * kSampCols], (unsigned long long)(SampleRow::mass(w) + kSampCount));
      }
    }
  });
  __syncthreads();
  {
    const int b = t >> 3, part = t & 7;
    uint64_t mass = 0;
    uint32_t count = 0;
    for (int i = 0; i < kSampCols / 8; ++i) {
      const uint64_t c = cells[b * kSampCols + part + 8 * i];
      mass += c & (kSampCount - 1);
      count += (uint32_t)(c >> 52);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      mass += __shfl_xor(mass, o);
      count += __shfl_xor(count, o);
    }
    if (part == 0) {
      sh.bin_count[b] = count;
      sh.bin_mass[b] = mass;
    }
  }
  __syncthreads();
  if (t < kWave) {   // prefix sums: lane takes bins 2 t and 2 t + 1
    const uint32_t c0 = sh.bin_count[2 * t], c1 = sh.bin_count[2 * t + 1];
    const uint64_t m0 = sh.bin_mass[2 * t], m1 = sh.bin_mass[2 * t + 1];
    uint32_t c = c0 + c1;
    uint64_t m = m0 + m1;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t cy = __shfl_up(c, o);
      const uint64_t my = __shfl_up(m, o);
      if (t >= o) {
        c += cy;
        m += my;
      }
    }
    sh.bin_before[2 * t] = c - c0 - c1;
    sh.bin_before[2 * t + 1] = c - c1;
    sh.mass_before[2 * t] = m - m0 - m1;
    sh.mass_before[2 * t + 1] = m - m1;
  }
  __syncthreads();
}

// What a search stops at: the token of a rank (0-based), or the first whose inclusive mass passes a target.
struct Search {
  bool by_rank, or_equal;
  int64_t rank;
  double target;
};
struct Found {
  int64_t rank;      // of the token
  int index;         // in the vocabulary
  uint64_t through;  // mass of the tokens up to it, itself included
};

// The bin of a search among those of the last fill_bins (base: what lies before bin 0); the last that holds a token if none.
__device__ inline int bin_of_search(const Search& s, const SampleShared& sh, int64_t base_count, uint64_t base_mass) {
  const int lane = threadIdx.x & 63;   // bins 2 lane and 2 lane + 1
  bool some[2], past[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = 2 * lane + i;
    some[i] = sh.bin_count[b] != 0;
    const int64_t c = base_count + sh.bin_before[b] + sh.bin_count[b];
    const double m = (double)(base_mass + sh.mass_before[b] + sh.bin_mass[b]);
    past[i] = some[i] && (s.by_rank ? c > s.rank : s.or_equal ? m >= s.target : m > s.target);
  }
  const uint64_t first = __ballot(past[0] || past[1]), even = __ballot(past[0]);
  if (first) {
    const int l = __builtin_ctzll(first);
    return 2 * l + ((even >> l) & 1 ? 0 : 1);
  }
  const uint64_t any = __ballot(some[0] || some[1]), odd = __ballot(some[1]);
  if (!any) return 0;
  const int l = 63 - __builtin_clzll(any);
  return 2 * l + ((odd >> l) & 1 ? 1 : 0);
}

// The search's token within the tokens `in(z, x)` accepts, `count` of them, after base_count tokens of base_mass.
template <class IN, class F>
__device__ inline Found search_in(const typename IN::T* row, int vocab, const SampleRow& r, uint64_t* list, uint64_t* prefix,
                                  SampleShared& sh, const Search& s, int64_t base_count, uint64_t base_mass, uint32_t count,
                                  F in) {
  const int t = threadIdx.x;
  uint32_t lo = 0, hi = 0xffffffffu;   // keys
  if (count > kSampList) {
    if (t == 0) {
      sh.lo = 0xffffffffu;
      sh.hi = 0;
    }
    __syncthreads();
    uint32_t a = 0xffffffffu, b = 0;
    sweep<IN>(row, vocab, t, row_vectors<IN>(row, vocab), kSampThreads, [&](const auto& z, int) {
#pragma unroll
      for (int e = 0; e < IN::kVec; ++e) {
        const float v = r.see(z[e]);
        if (v != -INFINITY && in(v)) {
          a = min(a, key_of(v));
          b = max(b, key_of(v));
        }
      }
    });
    atomicMin(&sh.lo, a);
    atomicMax(&sh.hi, b);
    __syncthreads();
    lo = sh.lo;
    hi = sh.hi;
    __syncthreads();
    while (count > kSampList && lo != hi) {   // the range shrinks 64-fold or more each time
      int shift = 0;
      while (((hi - lo) >> shift) >= kSampBins) ++shift;
      fill_bins<IN>(row, vocab, r, list, sh, [&](float v, double, double) {
        const uint32_t k = key_of(v);
        return k >= lo && k <= hi && in(v) ? (int)((hi - k) >> shift) : -1;
      });
      const int b = bin_of_search(s, sh, base_count, base_mass);
      base_count += sh.bin_before[b];
      base_mass += sh.mass_before[b];
      count = sh.bin_count[b];
      hi -= (uint32_t)b << shift;
      const uint32_t width = (1u << shift) - 1;
      lo = hi - lo > width ? hi - width : lo;
      __syncthreads();   // the next fill writes the bins
    }
  }
  if (count > kSampList) {   // one value: its ties in index order
    const uint64_t each = SampleRow::mass(r.weight(of_key(lo)));
    int64_t j;
    if (s.by_rank) j = s.rank - base_count;
    else {
      int64_t a = 0, b = count - 1;
      while (a < b) {
        const int64_t mid = (a + b) >> 1;
        const double m = (double)(base_mass + (uint64_t)(mid + 1) * each);
        if (s.or_equal ? m >= s.target : m > s.target) b = mid;
        else a = mid + 1;
      }
      j = a;
    }
    j = min(max(j, (int64_t)0), (int64_t)count - 1);
    // each thread counts a stretch of the row; the one that holds the j-th tie names it
    const int nvec = row_vectors<IN>(row, vocab), per = (nvec + kSampThreads - 1) / kSampThreads;
    const int v0 = min(t * per, nvec), v1 = min(v0 + per, nvec);
    uint32_t n = 0;
    const auto tie = [&](float z) {
      const float v = r.see(z);
      return v != -INFINITY && key_of(v) == lo && in(v);
    };
    sweep<IN>(row, vocab, v0, v1, 1, [&](const auto& z, int) {
#pragma unroll
      for (int e = 0; e < IN::kVec; ++e) n += tie(z[e]);
    });
    int64_t before = (int64_t)block_before(n, sh.red_u);
    if (before <= j && j < before + n)
      sweep<IN>(row, vocab, v0, v1, 1, [&](const auto& z, int i0) {
#pragma unroll
        for (int e = 0; e < IN::kVec; ++e)
          if (tie(z[e]) && before++ == j) sh.found_index = i0 + e;
      });
    __syncthreads();
    const Found f{base_count + j, sh.found_index, base_mass + (uint64_t)(j + 1) * each};
    __syncthreads();
    return f;
  }
  collect<IN>(row, vocab, r, list, sh, [&](float v) {
    const uint32_t k = key_of(v);
    return k >= lo && k <= hi && in(v);
  });
  const int n = min(sh.n_list, kSampList);
  sort_list(list, prefix, n);
  sum_list(list, prefix, n, r, sh);
  int at = s.by_rank ? (int)min(s.rank - base_count, (int64_t)n - 1) : first_past(prefix, n, base_mass, s.target, s.or_equal);
  at = max(min(at, n - 1), 0);
  const Found f{base_count + at, (int)(uint32_t)list[at], base_mass + prefix[at]};
  __syncthreads();   // the list is written again
  return f;
}

template <class IN>
__device__ inline int draw_from_bins(const typename IN::T* row, int vocab, const SampleRow& r, uint64_t* cells,
                                     SampleShared& sh, int k, double p, double m, double u) {
  uint64_t* list = cells;                 // the list takes the cells' place after they are summed up
  uint64_t* prefix = cells + kSampList;
  uint64_t above = 0, above_mass = 0;     // tokens with w >= m, of this thread
  fill_bins<IN>(row, vocab, r, cells, sh, [&](float, double x, double w) {
    if (w >= m) {
      above += 1;
      above_mass += SampleRow::mass(w);
    }
    return SampleRow::bin(x);
  });
  const int64_t total = (int64_t)sh.bin_before[kSampBins - 1] + sh.bin_count[kSampBins - 1];
  const uint64_t total_mass = sh.mass_before[kSampBins - 1] + sh.bin_mass[kSampBins - 1];
  int64_t kept = total;
  uint64_t kept_mass = total_mass;
  const auto in_bin = [&](int b) { return [&r, b](float v) { const double x = r.x(v); return x >= -42.0 && SampleRow::bin(x) == b; }; };
  const auto run = [&](const Search& s) {
    const int b = bin_of_search(s, sh, 0, 0);
    return search_in<IN>(row, vocab, r, list, prefix, sh, s, sh.bin_before[b], sh.mass_before[b], sh.bin_count[b], in_bin(b));
  };
  // the bins of the row, kept over searches that fill them again
  __shared__ uint32_t count0[kSampBins], before0[kSampBins];
  __shared__ uint64_t mass0[kSampBins], mbefore0[kSampBins];
  if (threadIdx.x < kSampBins) {
    count0[threadIdx.x] = sh.bin_count[threadIdx.x];
    before0[threadIdx.x] = sh.bin_before[threadIdx.x];
    mass0[threadIdx.x] = sh.bin_mass[threadIdx.x];
    mbefore0[threadIdx.x] = sh.mass_before[threadIdx.x];
  }
  const auto restore = [&] {
    __syncthreads();
    if (threadIdx.x < kSampBins) {
      sh.bin_count[threadIdx.x] = count0[threadIdx.x];
      sh.bin_before[threadIdx.x] = before0[threadIdx.x];
      sh.bin_mass[threadIdx.x] = mass0[threadIdx.x];
      sh.mass_before[threadIdx.x] = mbefore0[threadIdx.x];
    }
    __syncthreads();
  };
  uint64_t w_k = total_mass;
  if (k > 0 && k < total) {
    const Found f = run(Search{true, false, k - 1, 0.0});
    kept = k;
    w_k = kept_mass = f.through;
    restore();
  }
  if (p < 1.0) {
    const Search s{false, true, 0, p * (double)w_k};
    const int b = bin_of_search(s, sh, 0, 0);
    const int64_t n = (int64_t)sh.bin_before[b] + sh.bin_count[b];
    if (n <= kSampWhole) {   // all that can be kept, at once
      const auto upto = [&r, b](float v) { const double x = r.x(v); return x >= -42.0 && SampleRow::bin(x) <= b; };
      collect<IN>(row, vocab, r, list, sh, upto);
      const int got = min(sh.n_list, kSampList);
      sort_list(list, prefix, got);
      sum_list(list, prefix, got, r, sh);
      return draw_from_list(list, prefix, got, k > 0 ? (int)min(kept, (int64_t)got) : 0, p, m, u, w_k, r);
    }
    const Found f = run(s);
    if (f.rank + 1 < kept) {
      kept = f.rank + 1;
      kept_mass = f.through;
    }
    restore();
  }
  if (m > 0.0) {
    const uint64_t n = block_sum(above, sh.red_u), s = block_sum(above_mass, sh.red_u);
    if ((int64_t)n < kept && n > 0) {
      kept = (int64_t)n;
      kept_mass = s;
    }
    // nothing is that likely (m > 1): the first token alone
    if (n == 0) return run(Search{true, false, 0, 0.0}).index;
  }
  const Found f = run(Search{false, false, 0, u * (double)kept_mass});
  if (f.rank < kept) return f.index;
  restore();
  return run(Search{true, false, kept - 1, 0.0}).index;   // u of 1 or more: the last that is kept
}

template <class IN>
__global__ void __launch_bounds__(kSampThreads)
sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint64_t cells[];   // bins, or list and prefix
  __shared__ SampleShared sh;
  const int t = threadIdx.x, b = blockIdx.x;
  const typename IN::T* row = static_cast<const typename IN::T*>(a.x) + (int64_t)b * a.ld;
  const float T = a.temperature ? a.temperature[b] : a.temperature0;
  int k = a.top_k ? a.top_k[b] : a.top_k0;
  const double p = a.top_p ? a.top_p[b] : a.top_p0;
  const double m = a.min_p ? a.min_p[b] : a.min_p0;
  const double u = a.u[b];
  const auto answer = [&](int i) {
    if (t == 0) a.out[b] = i;
  };
  if (!(T > 0.0f)) return answer(argmax_row<IN>(row, a.vocab, sh));

  float mine = -INFINITY;
  sweep<IN>(row, a.vocab, t, row_vectors<IN>(row, a.vocab), kSampThreads, [&](const auto& z, int) {
#pragma unroll
    for (int e = 0; e < IN::kVec; ++e) mine = fmaxf(mine, z[e]);   // passes over NaN
  });
  SampleRow r;
  r.top = block_max_f(mine, sh.red_f);
  if (r.top == -INFINITY) return answer(argmax_row<IN>(row, a.vocab, sh));
  r.infinite = r.top == INFINITY;
  if (r.infinite) {
    r.top = 0.0f;
    mine = mine == INFINITY ? 0.0f : -INFINITY;
  }
  r.c = 1.4426950408889634074 / (double)T;
  if (k <= 0 || k >= a.vocab) k = 0;

  uint64_t* list = cells;
  uint64_t* prefix = cells + kSampList;
  float bound = INFINITY;   // the list path's: logits from here on
  if (k > 0 && k <= kSampTopK) {
    // the k-th largest of the threads' maxima, to a bin of (top - the smallest of them) / kSampBoundBins
    const float low = -block_max_f(mine == -INFINITY ? -INFINITY : -mine, sh.red_f);
    const float s = r.top > low ? (float)kSampBoundBins / (r.top - low) : 0.0f;
    const int bin = mine == -INFINITY ? kSampBoundBins : min((int)((r.top - mine) * s), kSampBoundBins - 1);
    for (int i = t; i < kSampBoundBins; i += kSampThreads) sh.bound[i] = 0;
    __syncthreads();
    if (bin < kSampBoundBins) atomicAdd(&sh.bound[bin], 1u);
    __syncthreads();
    if (t < kWave) {
      uint32_t c[kSampBoundBins / kWave], sum = 0;
#pragma unroll
      for (int i = 0; i < kSampBoundBins / kWave; ++i) sum += c[i] = sh.bound[t * (kSampBoundBins / kWave) + i];
      uint32_t inc = sum;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t y = __shfl_up(inc, o);
        if (t >= o) inc += y;
      }
      uint32_t before = inc - sum;
      if (t == kWave - 1) sh.found = inc < (uint32_t)k ? kSampBoundBins : sh.found;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < kSampBoundBins / kWave; ++i) {
        if (before < (uint32_t)k && before + c[i] >= (uint32_t)k) sh.found = t * (kSampBoundBins / kWave) + i;
        before += c[i];
      }
    }
    __syncthreads();
    // the smallest of the maxima in the bins down to that one: at least k logits are as large
    const int last = sh.found;
    bound = -block_max_f(bin <= last && bin < kSampBoundBins ? -mine : -INFINITY, sh.red_f);
    if (last == kSampBoundBins) bound = -INFINITY;   // fewer than k threads have one to show: all logits
  } else if (k == 0 && p >= 1.0 && m > 0.0) {
    // min-p alone: w >= m, a little below it for the rounding of the bound itself
    const double z = (double)r.top + (m < 1.0 ? ((double)__builtin_amdgcn_logf((float)m) - 1e-4) / r.c : 0.0);
    bound = fminf((float)(z - fabs(z) * 1e-6), r.top);
  }
  if (bound <= r.top) {
    collect<IN>(row, a.vocab, r, list, sh, [&](float v) { return v >= bound; });
    const int n = sh.n_list;
    if (n <= kSampList && n > 0) {
      sort_list(list, prefix, n);
      sum_list(list, prefix, n, r, sh);
      return answer(draw_from_list(list, prefix, n, k, p, m, u, ~0ull, r));
    }
    __syncthreads();
  }
  answer(draw_from_bins<IN>(row, a.vocab, r, cells, sh, k, p, m, u));
}

}  // namespace tq

using namespace tq;

extern "C" int tq_sample_tokens(const void* logits, int64_t logits_stride, int dtype, int rows, int vocab,
                                const float* uniform, const float* temperature, float temperature_all,
                                const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all,
                                const float* min_p, float min_p_all, int64_t* tokens, void* stream) {
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_FP16 && dtype != TQ_DTYPE_FP32) return TQ_ERR_DTYPE;
  if (rows < 0 || vocab <= 0 || vocab > kSampMaxVocab || (rows > 1 && logits_stride < vocab)) return TQ_ERR_ARG;
  if (rows == 0) return TQ_OK;
  if (!logits || !uniform || !tokens) return TQ_ERR_ARG;
  const size_t size = dtype == TQ_DTYPE_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return TQ_ERR_ALIGN;
  const SampleArgs a{logits, logits_stride, uniform, temperature, top_k, top_p, min_p, temperature_all, top_p_all,
                     min_p_all, top_k_all, tokens, rows, vocab};
  constexpr size_t lds = (size_t)kSampBins * kSampCols * sizeof(uint64_t);
  static_assert((size_t)kSampList * 16 == lds, "list and prefix take the bins' place");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == TQ_DTYPE_BF16) {
    TQ_RETURN_IF_HIP_ERROR((allow_lds<sample_kernel<H16In<Bf16>>>(lds)));
    hipLaunchKernelGGL(sample_kernel<H16In<Bf16>>, dim3(rows), dim3(kSampThreads), lds, s, a);
  } else if (dtype == TQ_DTYPE_FP16) {
    TQ_RETURN_IF_HIP_ERROR((allow_lds<sample_kernel<H16In<Fp16>>>(lds)));
    hipLaunchKernelGGL(sample_kernel<H16In<Fp16>>, dim3(rows), dim3(kSampThreads), lds, s, a);
  } else {
    TQ_RETURN_IF_HIP_ERROR((allow_lds<sample_kernel<F32In>>(lds)));
    hipLaunchKernelGGL(sample_kernel<F32In>, dim3(rows), dim3(kSampThreads), lds, s, a);
  }
  return (int)hipGetLastError();
}

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
// fp64 and rounded to a multiple of 2^-39 (tokens below 2^-40 of the likeliest count as 0), and sums are 64-bit.
//
// Two ways through a row, by its settings:
//   list   k <= 512, or min-p alone: a bound that at least k logits reach comes from the threads' maxima; the logits
//          above it (a few more than k) are sorted in LDS, and all rules are applied there.
//   bins   otherwise: one pass adds every token's count and mass to 252 bins of 1/6 octave of w, then only the tokens of
//          the bins where a target falls are looked at: they are narrowed down by key and index until at most 256 are
//          left to sort.  Bins have 16 or more columns, and a lane adds to the column of its number, which keeps the lanes
//          that meet at one address few.
// Short rows take one launch of one workgroup per row.  Others are cut in C chunks, and there are up to four:
// maxima of every chunk; the chunk's list or bins, now that the row's maximum is known; the tokens of the bins that the
// row's searches can end in, which the bins' sums tell, gathered; and one workgroup per row that finishes from the list
// in LDS.  Masses being integers, C does not change the answer.
// Bounds, and what the four take at a vocabulary of 128256 (us): 256 fp32 rows of mixed settings 32 + 37 + 29 + 25, the
// passes bound by memory (131 MB each at most, 4.1 TB/s in the first), the last by its slowest row's chain of steps; 64
// bf16 rows, top-p alone 6 + 18 + 21 + 24, the weights in fp64 and again the steps; one row with top-k 3 + 8 + 2 + 5.  One
// workgroup per row throughout took 254 / 202 / 21.
#include "tq_common.h"

#include <float.h>

namespace tq {

constexpr int kSampThreads = 512;      // of the workgroup that finishes a row
constexpr int kSampWaves = kSampThreads / kWave;
constexpr int kSampBins = 256;
constexpr int kSampCols = 64;
constexpr int kChunkThreads = 256;     // of a chunk's workgroup
constexpr int kChunkCols = 16;
constexpr int kChunkList = 2048;       // list entries that one chunk may hand over
constexpr int kMaxima = 2048;          // maxima of a row, at most
constexpr int kSampList = 8192;        // entries of the sorted list: 8 bytes of key and index, 8 of prefix mass
constexpr int kSampTopK = 512;         // largest k of the list path
constexpr int kSampSort = 512;         // entries sorted by rank, an entry a thread at most
constexpr int kSampEnd = 256;          // a search's last entries: a turn more costs as much as sorting twice as many
constexpr int kSampBoundBins = 512;
constexpr int kSampMaxVocab = 500000;  // a column's count has 13 bits: at most 8191 tokens of a row per column
constexpr int kChunkMost = 120000;     // tokens of a chunk, for the same reason
constexpr int kSampWhole = 512;        // the bins down to the last one needed are sorted together up to this many tokens
constexpr uint64_t kSampCount = 1ull << 51;    // one token in a column's word: count from bit 51 on, mass below

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
  // the split form's workspace, per row
  int chunks;
  int per;              // maxima per chunk: of groups of kChunkThreads / per threads
  int list_cap;
  float* maxima;        // [chunks * per]; of a greedy row [chunks]: its best logits
  int32_t* best;        // [chunks]: and where they are
  uint64_t* bin_mass;   // [chunks][kSampBins]
  uint64_t* list;       // [list_cap]
  uint64_t* above_mass; // [chunks]: mass and number of the tokens with w >= m
  uint32_t* above;
  uint32_t* bin_count;  // [chunks][kSampBins]
  uint32_t* n_list;     // [1]
  float* top;           // [1]: the row's maximum, where it is not greedy
  uint64_t* row_mass;   // [kSampBins + 2]: the row's bins, above_mass and above
  uint32_t* row_count;  // [kSampBins]
};

struct F32In {
  using T = float;
  static constexpr int kVec = 4;
  static constexpr int kLow = 0;   // low bits of a logit's key that are the same for all of one sign
  __device__ static inline float shift(u32x4& w) {   // the first element, the others one place down
    const float f = __uint_as_float(w[0]);
    w[0] = w[1];
    w[1] = w[2];
    w[2] = w[3];
    return f;
  }
  __device__ static inline void unpack(u32x4 w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  }
};
template <class XT>
struct H16In {
  using T = uint16_t;
  static constexpr int kVec = 8;
  static constexpr int kLow = std::is_same<XT, Bf16>::value ? 16 : 13;
  __device__ static inline float shift(u32x4& w) {
    const float f = XT::to_f32((uint16_t)(w[0] & 0xffffu));
    w[0] = (w[0] >> 16) | (w[1] << 16);
    w[1] = (w[1] >> 16) | (w[2] << 16);
    w[2] = (w[2] >> 16) | (w[3] << 16);
    w[3] >>= 16;
    return f;
  }
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

// 2^x for x in [-42, 0]: the Taylor series of e^(f ln 2), |f| <= 1/2, to degree 11 (6e-15 relative).  Its coefficients are
// made scalar operands: held in vector registers, each step would begin with a copy of one.
__device__ __forceinline__ double in_scalar(double c) {
  asm("" : "+s"(c));
  return c;
}
__device__ __forceinline__ double exp2_small(double x) {
  const double n = __builtin_rint(x);
  const double f = (x - n) * 0.693147180559945309417;
  double r = in_scalar(1.0 / 39916800.0);
  r = fma(r, f, in_scalar(1.0 / 3628800.0));
  r = fma(r, f, in_scalar(1.0 / 362880.0));
  r = fma(r, f, in_scalar(1.0 / 40320.0));
  r = fma(r, f, in_scalar(1.0 / 5040.0));
  r = fma(r, f, in_scalar(1.0 / 720.0));
  r = fma(r, f, in_scalar(1.0 / 120.0));
  r = fma(r, f, in_scalar(1.0 / 24.0));
  r = fma(r, f, in_scalar(1.0 / 6.0));
  r = fma(r, f, 0.5);
  r = fma(r, f, 1.0);
  r = fma(r, f, 1.0);
  return __builtin_ldexp(r, (int)n);
}

// A row's settings.
struct SampleSettings {
  float T;
  int k;         // 0: all
  double p, m;
  float u;
  // Every load is made, from the numbers u where a setting has no vector, so that all go out together: a branch each
  // would be a round trip to memory each.
  __device__ __forceinline__ SampleSettings(const SampleArgs& a, int b) {
    const float* any = a.u;
    const float tv = (a.temperature ? a.temperature : any)[b], pv = (a.top_p ? a.top_p : any)[b];
    const float mv = (a.min_p ? a.min_p : any)[b];
    const int kv = (a.top_k ? a.top_k : reinterpret_cast<const int32_t*>(any))[b];
    u = any[b];
    T = a.temperature ? tv : a.temperature0;
    k = a.top_k ? kv : a.top_k0;
    if (k <= 0 || k >= a.vocab) k = 0;
    p = a.top_p ? pv : a.top_p0;
    m = a.min_p ? mv : a.min_p0;
  }
  __device__ bool greedy() const { return !(T > 0.0f); }
  __device__ bool by_list() const { return (k > 0 && k <= kSampTopK) || (k == 0 && p >= 1.0 && m > 0.0); }
};

// The row as its settings see it.
struct SampleRow {
  float top;             // z_max
  bool infinite;         // z_max is +infinity: z becomes 0 there and -infinity elsewhere (top is 0 then)
  double c, top64;       // log2 w = (z - z_max) c, c = log2(e) / T; the difference first: z c alone may be huge
  float half_top, step;  // 6 log2(w) = -(half_top - z / 2) step, which does not overflow
  __device__ SampleRow(float z_max, float T) {   // the same in all lanes: kept in scalar registers
    z_max = uniform(z_max);
    infinite = z_max == INFINITY;
    top = infinite ? 0.0f : z_max;
    c = uniform(1.4426950408889634074 / (double)T);
    top64 = uniform((double)top);
    half_top = uniform(0.5f * top);
    step = uniform((float)fmin(12.0 * c, 3.0e38));
  }
  __device__ static inline float uniform(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }
  __device__ static inline double uniform(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)b), hi = __builtin_amdgcn_readfirstlane((int)(b >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  }
  __device__ inline float see(float z) const { return !infinite ? z : z == INFINITY ? 0.0f : -INFINITY; }
  // The place among the bins: bin i holds place in [i, i + 1).  Ascends as z descends; from 252 on (w < 2^-42) a token
  // counts as nothing, and for NaN and -infinity no comparison holds.
  __device__ inline float place(float z) const { return fmaf(z, -0.5f, half_top) * step; }
  __device__ static inline bool alive(float place) { return place < 252.0f; }
  __device__ inline double log2_weight(float z) const { return ((double)z - top64) * c; }
  __device__ inline double weight(float z) const { return alive(place(z)) ? exp2_small(log2_weight(z)) : 0.0; }
  // the weight in 2^-39: adding 2^13 leaves it in the low bits of the mantissa, rounded to nearest
  __device__ static inline uint64_t mass(double w) {
    return __builtin_bit_cast(uint64_t, w + 8192.0) & (kSampCount - 1);
  }
};

// Bins and what lies before each.
template <int N>
struct Bins {
  uint64_t mass[N], mass_before[N];
  uint32_t count[N], before[N];
};
constexpr int kWorkBins = 64;          // of a turn that narrows a search down

struct SampleShared {
  float red_f[kSampWaves];
  uint64_t red_u[kSampWaves];
  int red_i[kSampWaves];
  union {
    uint32_t bound[kSampBoundBins];   // while the list's bound is looked for
    Bins<kSampBins> row;
  };
  int n_list, n_work, found;
};

template <int NT = kSampThreads>
__device__ inline float block_max_f(float v, float* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[threadIdx.x & (NT / kWave - 1)];
#pragma unroll
  for (int o = NT / kWave / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  return v;
}
template <int NT = kSampThreads>
__device__ inline uint64_t block_sum(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[threadIdx.x & (NT / kWave - 1)];
#pragma unroll
  for (int o = NT / kWave / 2; o; o >>= 1) v += __shfl_xor(v, o);
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
// element on; what they hold beside the row is given as -infinity with an index out of range.  kBatch vectors are loaded
// while the batch before is looked at.
template <class IN, int kBatch, class F>
__device__ __forceinline__ void sweep(const typename IN::T* row, int vocab, int vec0, int vec1, int step, F f) {
  constexpr int V = IN::kVec;
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(typename IN::T));
  const u32x4* base = reinterpret_cast<const u32x4*>(row - off);
  if (vec0 >= vec1) return;
  u32x4 next[kBatch];
#pragma unroll
  for (int b = 0; b < kBatch; ++b) next[b] = base[min(vec0 + b * step, vec1 - 1)];
#pragma unroll 1
  for (int j0 = vec0; j0 < vec1; j0 += step * kBatch) {
    u32x4 w[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      w[b] = next[b];
      next[b] = base[min(j0 + (kBatch + b) * step, vec1 - 1)];
    }
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
// The same, token by token: f(z, i) with z = -infinity where i is not of the row.  A vector's elements go through one copy of
// f, shifted down to the first register in turn: for the passes that few rows take, so that their code stays small.
template <class IN, class F>
__device__ __forceinline__ void each_token(const typename IN::T* row, int vocab, int vec0, int vec1, int step, F f) {
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(typename IN::T));
  const u32x4* base = reinterpret_cast<const u32x4*>(row - off);
  if (vec0 >= vec1) return;
  u32x4 next = base[vec0];
#pragma unroll 1
  for (int j = vec0; j < vec1; j += step) {
    u32x4 w = next;
    next = base[min(j + step, vec1 - 1)];
    int i = j * IN::kVec - off;
#pragma unroll 1
    for (int e = 0; e < IN::kVec; ++e, ++i) {
      f((uint32_t)i < (uint32_t)vocab ? IN::shift(w) : (IN::shift(w), -INFINITY), i);
    }
  }
}
template <class IN>
__device__ inline int row_vectors(const typename IN::T* row, int vocab) {
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(typename IN::T));
  return (off + vocab + IN::kVec - 1) / IN::kVec;
}

// torch.argmax: NaN first, then the largest, the lowest index among equals.
struct Best {
  float v;
  int i;
  __device__ inline void pick(float v2, int i2) {
    const bool n1 = v != v, n2 = v2 != v2;
    if (n1 != n2 ? n2 : (n1 || v == v2) ? i2 < i : v2 > v) {
      v = v2;
      i = i2;
    }
  }
};
template <int NT>
__device__ __forceinline__ Best block_best(Best b, SampleShared& sh) {
#pragma unroll
  for (int o = 32; o; o >>= 1) b.pick(__shfl_xor(b.v, o), __shfl_xor(b.i, o));
  if ((threadIdx.x & 63) == 0) {
    sh.red_f[threadIdx.x >> 6] = b.v;
    sh.red_i[threadIdx.x >> 6] = b.i;
  }
  __syncthreads();
  b = Best{sh.red_f[0], sh.red_i[0]};
  for (int w = 1; w < NT / kWave; ++w) b.pick(sh.red_f[w], sh.red_i[w]);
  __syncthreads();
  return b;
}
template <class IN, int NT>
__device__ __forceinline__ Best argmax_row(const typename IN::T* row, int vocab, int v0, int v1, SampleShared& sh) {
  Best best{-INFINITY, 0x7fffffff};
  sweep<IN, 2>(row, vocab, v0 + (int)threadIdx.x, v1, NT, [&](const auto& z, int i0) {
    // a thread's indexes ascend, so only a larger logit or a first NaN changes its best; the first token always does
    float most = z[0];
    bool look = z[0] != z[0];
#pragma unroll
    for (int e = 1; e < IN::kVec; ++e) {
      most = fmaxf(most, z[e]);
      look |= z[e] != z[e];
    }
    if (look || most > best.v || best.i == 0x7fffffff) {
#pragma unroll
      for (int e = 0; e < IN::kVec; ++e)
        if (i0 + e >= 0 && i0 + e < vocab) best.pick(z[e], i0 + e);
    }
  });
  return block_best<NT>(best, sh);
}

// ---- the sorted list ------------------------------------------------------------
// A token's place in the order as one number: (~key) << 32 | index ascends with it.
__device__ inline uint64_t entry_of(float z, int i) { return (uint64_t)~key_of(z) << 32 | (uint32_t)i; }
__device__ inline float logit_of(uint64_t entry) { return of_key(~(uint32_t)(entry >> 32)); }

// Sorts n entries; up to kSampSort by rank (kSampThreads / n threads per entry, up to 4, each against a part of the
// others, through spare), more in a bitonic network.
__device__ __forceinline__ void sort_small(uint64_t* list, uint64_t* spare, int n) {
  const int t = threadIdx.x;
  const int parts = n <= kSampThreads / 4 ? 4 : n <= kSampThreads / 2 ? 2 : 1;
  const int e = t / parts, part = t & (parts - 1);
  uint64_t mine = ~0ull;
  int rank = 0;
  if (e < n) {
    mine = list[e];
#pragma unroll 8
    for (int j = part; j < n; j += parts) rank += list[j] < mine;
  }
  for (int o = 1; o < parts; o <<= 1) rank += __shfl_xor(rank, o);
  if (e < n && part == 0) spare[rank] = mine;
  __syncthreads();
  if (t < n) list[t] = spare[t];
  __syncthreads();
}
__device__ __forceinline__ void sort_list(uint64_t* list, uint64_t* spare, int n) {
  if (n <= kSampSort) return sort_small(list, spare, n);
  const int t = threadIdx.x;
  int size = 2 * kSampSort;
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
__device__ __forceinline__ void sum_list(const uint64_t* list, uint64_t* prefix, int n, const SampleRow& r,
                                         SampleShared& sh) {
  const int per = (n + kSampThreads - 1) / kSampThreads, i0 = threadIdx.x * per, i1 = min(i0 + per, n);
  uint64_t sum = 0;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    sum += SampleRow::mass(r.weight(logit_of(list[i])));
    prefix[i] = sum;
  }
  const uint64_t before = block_before(sum, sh.red_u);
#pragma unroll 1
  for (int i = i0; i < i1; ++i) prefix[i] += before;
  __syncthreads();
}

// What a search stops at: the token of a rank (0-based), or the first whose inclusive mass passes a target.
// Masses are whole numbers: one is > target from floor(target) + 1 on, >= target from ceil(target) on.
struct Search {
  bool by_rank;
  int64_t rank;
  uint64_t least;   // the mass from which on a search for a mass stops
  __device__ static inline Search of_rank(int64_t rank) { return Search{true, rank, 0}; }
  // masses are below 2^58 (500000 tokens); a target beyond, of a number far above 1, is as good as 2^62
  __device__ static inline double in_range(double target) { return fmin(fmax(target, 0.0), 0x1p62); }
  __device__ static inline Search over(double target) { return Search{false, 0, (uint64_t)in_range(target) + 1}; }
  __device__ static inline Search from(double target) { return Search{false, 0, (uint64_t)ceil(in_range(target))}; }
  __device__ inline bool past(int64_t count, uint64_t mass) const {   // of the tokens up to and with some token
    return by_rank ? count > rank : mass >= least;
  }
};
// First entry where the inclusive mass (with `base` before the list) is least or more; n if none.
__device__ inline int first_past(const uint64_t* prefix, int n, uint64_t base, uint64_t least) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (base + prefix[mid] >= least) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Puts the row's tokens that `take(z, entry)` accepts in the list, which holds kSampList; sh.n_list is their number also
// where it is more.
template <class IN, class F>
__device__ __forceinline__ void collect(const typename IN::T* row, int vocab, const SampleRow& r, uint64_t* list,
                                        SampleShared& sh, F take) {
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  each_token<IN>(row, vocab, threadIdx.x, row_vectors<IN>(row, vocab), kSampThreads, [&](float z, int i) {
    const float v = r.see(z);
    const uint64_t entry = entry_of(v, i);
    if (take(v, entry)) {
      const int at = atomicAdd(&sh.n_list, 1);
      if (at < kSampList) list[at] = entry;
    }
  });
  __syncthreads();
}

// Applies the rules to a sorted list that is the whole beginning of the order.  w_k: the mass top-p is a part of, or
// ~0 for that of the list's first k.
__device__ __forceinline__ int draw_from_list(const uint64_t* list, const uint64_t* prefix, int n, int k, double p, double m,
                                              double u, uint64_t w_k, const SampleRow& r) {
  int kept = k > 0 ? min(k, n) : n;
  if (p < 1.0) {
    const double all = (double)(w_k == ~0ull ? prefix[kept - 1] : w_k);
    kept = min(kept, first_past(prefix, kept, 0, Search::from(p * all).least) + 1);
  }
  if (m > 0.0) {   // weights descend
    int lo = 0, hi = kept;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (r.weight(logit_of(list[mid])) >= m) lo = mid + 1;
      else hi = mid;
    }
    kept = lo;
  }
  kept = max(kept, 1);
  const int at = min(first_past(prefix, kept, 0, Search::over(u * (double)prefix[kept - 1]).least), kept - 1);
  return (int)(uint32_t)list[at];
}

// ---- bins -----------------------------------------------------------------------
// A token's word for its bin's cell.
__device__ inline void add_to_cell(uint64_t* cell, double w) {
  atomicAdd((unsigned long long*)cell, (unsigned long long)(SampleRow::mass(w) + kSampCount));
}

// Counts and masses of the bins, their columns summed up, by kSampThreads / BINS threads each, 4 at most.
template <int BINS>
__device__ __forceinline__ void sum_cells(const uint64_t* cells, int cols, Bins<BINS>& out) {
  const int t = threadIdx.x;
  constexpr int kParts = kSampThreads / BINS < 4 ? kSampThreads / BINS : 4;
  if (t < BINS * kParts) {
    const int b = t / kParts, part = t % kParts;
    uint64_t mass = 0;
    uint32_t count = 0;
#pragma unroll 4
    for (int i = 0; i < cols / kParts; ++i) {
      const uint64_t c = cells[b * cols + ((part + kParts * (i + b)) & (cols - 1))];
      mass += c & (kSampCount - 1);
      count += (uint32_t)(c >> 51);
    }
#pragma unroll
    for (int o = 1; o < kParts; o <<= 1) {
      mass += __shfl_xor(mass, o);
      count += __shfl_xor(count, o);
    }
    if (part == 0) {
      out.count[b] = count;
      out.mass[b] = mass;
    }
  }
  __syncthreads();
}
template <int BINS>
__device__ __forceinline__ void before_bins(Bins<BINS>& b) {
  constexpr int kPer = BINS / kWave;
  const int t = threadIdx.x;
  if (t < kWave) {
    uint32_t c = 0;
    uint64_t m = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      c += b.count[kPer * t + i];
      m += b.mass[kPer * t + i];
    }
    const uint32_t c_own = c;
    const uint64_t m_own = m;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t cy = __shfl_up(c, o);
      const uint64_t my = __shfl_up(m, o);
      if (t >= o) {
        c += cy;
        m += my;
      }
    }
    c -= c_own;
    m -= m_own;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      b.before[kPer * t + i] = c;
      b.mass_before[kPer * t + i] = m;
      c += b.count[kPer * t + i];
      m += b.mass[kPer * t + i];
    }
  }
  __syncthreads();
}

struct Found {
  int64_t rank;      // of the token
  int index;         // in the vocabulary
  uint64_t through;  // mass of the tokens up to it, itself included
};

// The bin where a search stops (base: what lies before bin 0), or the last that holds a token; every wave finds it.
template <int BINS>
__device__ __forceinline__ int bin_of_search(const Search& s, const Bins<BINS>& bins, int64_t base_count,
                                             uint64_t base_mass) {
  constexpr int kPer = BINS / kWave;
  const int lane = threadIdx.x & 63;   // bins kPer lane ..
  int first = -1, last = -1;           // of this lane's: past, holding a token
#pragma unroll
  for (int i = kPer - 1; i >= 0; --i) {
    const int b = kPer * lane + i;
    if (bins.count[b] == 0) continue;
    if (last < 0) last = b;
    if (s.past(base_count + bins.before[b] + bins.count[b], base_mass + bins.mass_before[b] + bins.mass[b])) first = b;
  }
  const uint64_t p = __ballot(first >= 0), h = __ballot(last >= 0);
  if (p) return __builtin_amdgcn_readlane(first, __builtin_ctzll(p));
  return h ? __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(h)) : 0;
}

// The bins of a whole row; above, above_mass: number and mass of the tokens with w >= m.
template <class IN>
__device__ __forceinline__ void fill_bins(const typename IN::T* row, int vocab, const SampleRow& r, double m, uint64_t* cells,
                                          SampleShared& sh, uint64_t& above, uint64_t& above_mass) {
  const int t = threadIdx.x;
  for (int i = t; i < kSampBins * kSampCols; i += kSampThreads) cells[i] = 0;
  __syncthreads();
  uint64_t* mine = cells + (t & (kSampCols - 1));
  uint64_t n = 0, mass = 0;
  each_token<IN>(row, vocab, t, row_vectors<IN>(row, vocab), kSampThreads, [&](float z, int) {
    const float v = r.see(z), place = r.place(v);
    if (SampleRow::alive(place)) {
      const double w = exp2_small(r.log2_weight(v));
      if (w >= m) {
        n += 1;
        mass += SampleRow::mass(w);
      }
      add_to_cell(&mine[(int)place * kSampCols], w);
    }
  });
  __syncthreads();
  sum_cells(cells, kSampCols, sh.row);
  before_bins(sh.row);
  above = block_sum(n, sh.red_u);
  above_mass = block_sum(mass, sh.red_u);
}

// Where a search stops in the row, its bins being known.  The tokens of the bin are narrowed down, 64 ranges of their
// order (key, then index) at a time: over the row while they are more than the list holds, then in the list, until at
// most kSampEnd are left, which are sorted.  Each turn divides the range of the numbers by 32 or more.  The numbers
// leave out what does not vary, the low bits of a 16-bit logit's key and the high ones of the index: of a bin's several
// thousand bf16 tokens, many of them equal, one turn leaves few enough (with 64-bit numbers five turns, 3.6 us each).
// gathered: the list holds that many tokens, all of the bin among them, and stays as it is; or -1.
template <class IN>
__device__ __forceinline__ Found search_row(const typename IN::T* row, int vocab, const SampleRow& r, uint64_t* cells,
                                            SampleShared& sh, const Search& s, int gathered) {
  __shared__ Bins<kWorkBins> turn_bins;
  const int t = threadIdx.x;
  uint64_t* list = cells;
  uint64_t* work = cells + kSampList;   // the turns' cells; then the last entries, a copy and their prefix masses
  constexpr int kRowCols = 128;         // a column counts up to 8191 tokens: of the whole row, and of the list
  constexpr int kListCols = 32;
  static_assert(kWorkBins * kRowCols == kSampList && 3 * kSampEnd <= kSampList, "what the second half holds");
  const int b = bin_of_search(s, sh.row, 0, 0);
  const float from = (float)b, to = (float)(b + 1);
  int64_t base_count = sh.row.before[b];
  uint64_t base_mass = sh.row.mass_before[b];
  int count = (int)sh.row.count[b], whole = max(gathered, 0);
  const int index_bits = 32 - __builtin_clz((uint32_t)vocab);
  const uint64_t index_mask = (1ull << index_bits) - 1;
  const auto number = [&](uint64_t entry) {
    return (entry >> (32 + IN::kLow)) << index_bits | (entry & index_mask);
  };
  // the range of the order that the bin takes up, a little wide: place says what is in it
  uint64_t first = 0, last = number(~0ull);
  const float upper = 2.0f * (r.half_top - from / r.step), lower = 2.0f * (r.half_top - to / r.step);
  const float slack = 1e-5f * (fabsf(upper) + fabsf(lower) + fabsf(r.top));
  if (upper + slack < FLT_MAX && lower - slack > -FLT_MAX) {
    first = number((uint64_t)~key_of(upper + slack) << 32);
    last = number((uint64_t)~key_of(lower - slack) << 32 | 0xffffffffull);
  }
  bool listed = gathered >= 0;
  const auto in = [&](float v, uint64_t x) {
    const float place = r.place(v);
    return place >= from && place < to && x >= first && x <= last;
  };
  for (int turn = 0; turn < 20; ++turn) {   // up to 51 bits, 5 or more a turn, and one turn to list them
    if (!listed && count <= kSampList) {
      collect<IN>(row, vocab, r, list, sh, [&](float v, uint64_t e) { return in(v, number(e)); });
      whole = min(sh.n_list, kSampList);
      listed = true;
    }
    if (listed && count <= kSampEnd) break;
    const uint64_t range = last - first;
    const int shift = max(0, 58 - (int)__builtin_clzll(range | 1));
    const int cols = listed ? kListCols : kRowCols;
    for (int i = t; i < kWorkBins * cols; i += kSampThreads) work[i] = 0;
    __syncthreads();
    uint64_t* mine = work + (t & (cols - 1));
    if (listed) {
#pragma unroll 1
      for (int i = t; i < whole; i += kSampThreads) {
        const uint64_t e = list[i], x = number(e);
        const float v = logit_of(e);
        if (in(v, x)) add_to_cell(&mine[(int)((x - first) >> shift) * cols], r.weight(v));
      }
    } else {
      each_token<IN>(row, vocab, t, row_vectors<IN>(row, vocab), kSampThreads, [&](float z, int i) {
        const float v = r.see(z);
        const uint64_t x = number(entry_of(v, i));
        if (in(v, x)) add_to_cell(&mine[(int)((x - first) >> shift) * cols], r.weight(v));
      });
    }
    __syncthreads();
    sum_cells(work, cols, turn_bins);
    before_bins(turn_bins);
    const int w = bin_of_search(s, turn_bins, base_count, base_mass);
    base_count += turn_bins.before[w];
    base_mass += turn_bins.mass_before[w];
    count = (int)turn_bins.count[w];
    first += (uint64_t)w << shift;
    const uint64_t end = first + ((1ull << shift) - 1);
    last = end < last ? end : last;
    __syncthreads();   // the next turn writes the bins
  }
  __syncthreads();   // every thread has read the list's length
  if (t == 0) sh.n_work = 0;
  __syncthreads();
  for (int i = t; i < whole; i += kSampThreads) {
    const uint64_t e = list[i];
    if (in(logit_of(e), number(e))) {
      const int at = atomicAdd(&sh.n_work, 1);
      if (at < kSampEnd) work[at] = e;
    }
  }
  __syncthreads();
  const int n = max(1, min(sh.n_work, kSampEnd));
  uint64_t* prefix = work + 2 * kSampEnd;
  sort_small(work, work + kSampEnd, n);
  sum_list(work, prefix, n, r, sh);
  int at = s.by_rank ? (int)(s.rank - base_count) : first_past(prefix, n, base_mass, s.least);
  at = max(min(at, n - 1), 0);
  const Found f{base_count + at, (int)(uint32_t)work[at], base_mass + prefix[at]};
  __syncthreads();   // the work half is written again
  return f;
}

// Whether what top-p can keep is few enough to be sorted at once, and the bin it ends in at the latest (w_most: the most
// that top-k can have left it).
__device__ __forceinline__ bool sort_whole(const SampleSettings& set, const Bins<kSampBins>& bins, double w_most, int& end) {
  if (!(set.p < 1.0)) return false;
  end = bin_of_search(Search::from(set.p * w_most), bins, 0, 0);
  return (int64_t)bins.before[end] + bins.count[end] <= kSampWhole;
}

// The places that a row's searches can end in, from its bins: the bin where top-k ends, those where top-p can end
// whatever top-k keeps of its bin, and those where the number can fall.
struct Needed {
  float from[3], to[3];
  __device__ inline void range(int i, int b0, int b1) {
    from[i] = (float)b0;
    to[i] = (float)(b1 + 1);
  }
  __device__ inline bool has(float place) const {
    return (place >= from[0] && place < to[0]) || (place >= from[1] && place < to[1]) || (place >= from[2] && place < to[2]);
  }
  __device__ __forceinline__ Needed(const SampleSettings& set, const Bins<kSampBins>& bins, uint64_t above,
                                    uint64_t above_mass) {
#pragma unroll
    for (int i = 0; i < 3; ++i) range(i, -1, -2);   // nothing
    const int64_t total = (int64_t)bins.before[kSampBins - 1] + bins.count[kSampBins - 1];
    uint64_t lo = bins.mass_before[kSampBins - 1] + bins.mass[kSampBins - 1], hi = lo;   // the mass of what is kept
    if (set.k > 0 && set.k < total) {
      const int b = bin_of_search(Search::of_rank(set.k - 1), bins, 0, 0);
      range(0, b, b);
      lo = bins.mass_before[b];
      hi = lo + bins.mass[b];
    }
    int end;
    if (sort_whole(set, bins, (double)hi, end)) {
      range(1, 0, end);
      return;
    }
    if (set.p < 1.0) {
      const int b = lo == hi ? end : bin_of_search(Search::from(set.p * (double)lo), bins, 0, 0);
      range(1, b, end);
      const uint64_t through = bins.mass_before[end] + bins.mass[end];
      lo = bins.mass_before[b] < lo ? bins.mass_before[b] : lo;
      hi = through < hi ? through : hi;
    }
    if (set.m > 0.0 && above > 0) {
      lo = above_mass < lo ? above_mass : lo;
      hi = above_mass < hi ? above_mass : hi;
    }
    const bool none = set.m > 0.0 && above == 0;   // the first token alone
    const int b0 = bin_of_search(none ? Search::of_rank(0) : Search::over((double)set.u * (double)lo), bins, 0, 0);
    const int b1 = hi == lo ? b0 : bin_of_search(Search::over((double)set.u * (double)hi), bins, 0, 0);
    range(2, b0, none ? b0 : b1);
  }
};

// The answer of a row whose bins are in sh.row.  gathered: tokens in the list (Needed's), or -1.
template <class IN>
__device__ __forceinline__ int draw_from_bins(const typename IN::T* row, int vocab, const SampleRow& r, uint64_t* cells,
                                              SampleShared& sh, const SampleSettings& set, uint64_t above,
                                              uint64_t above_mass, int gathered) {
  const int64_t total = (int64_t)sh.row.before[kSampBins - 1] + sh.row.count[kSampBins - 1];
  const uint64_t total_mass = sh.row.mass_before[kSampBins - 1] + sh.row.mass[kSampBins - 1];
  int64_t kept = total;
  uint64_t kept_mass = total_mass, w_k = total_mass;
  double w_most = (double)total_mass;
  int answer = 0;
#pragma unroll 1
  for (int stage = 0; stage < 4; ++stage) {   // what top-k keeps, what top-p keeps, the number, the last that is kept
    Search s = Search::of_rank(0);
    if (stage == 0) {
      if (!(set.k > 0 && set.k < total)) continue;
      s.rank = set.k - 1;
      const int b = bin_of_search(s, sh.row, 0, 0);
      w_most = (double)(sh.row.mass_before[b] + sh.row.mass[b]);
    } else if (stage == 1) {
      if (!(set.p < 1.0)) continue;
      s = Search::from(set.p * (double)w_k);
      int end;
      if (sort_whole(set, sh.row, w_most, end)) {
        const float to = (float)(end + 1);
        if (gathered < 0) {
          collect<IN>(row, vocab, r, cells, sh, [&](float v, uint64_t) { return r.place(v) < to; });
        } else {   // the list without what is only top-k's
          uint64_t* work = cells + kSampList;
          if (threadIdx.x == 0) sh.n_list = 0;
          __syncthreads();
          for (int i = threadIdx.x; i < gathered; i += kSampThreads)
            if (r.place(logit_of(cells[i])) < to) work[atomicAdd(&sh.n_list, 1)] = cells[i];
          __syncthreads();
          cells = work;
        }
        const int n = max(1, min(sh.n_list, kSampWhole));
        sort_list(cells, cells + kSampWhole, n);
        sum_list(cells, cells + kSampWhole, n, r, sh);
        const int k = set.k > 0 ? (int)(kept < n ? kept : n) : 0;
        return draw_from_list(cells, cells + kSampWhole, n, k, set.p, set.m, set.u, w_k, r);
      }
    } else if (stage == 2) {
      if (set.m > 0.0 && (int64_t)above < kept) {
        kept = above > 0 ? (int64_t)above : 1;
        kept_mass = above_mass;
      }
      // where nothing is likely enough the first token alone is kept
      if (!(set.m > 0.0 && above == 0)) s = Search::over((double)set.u * (double)kept_mass);
    } else {
      s.rank = kept - 1;   // a number of 1 or more
      gathered = -1;
    }
    const Found f = search_row<IN>(row, vocab, r, cells, sh, s, gathered);
    if (stage == 0) {
      kept = set.k;
      w_k = kept_mass = f.through;
    } else if (stage == 1) {
      if (f.rank + 1 < kept) {
        kept = f.rank + 1;
        kept_mass = f.through;
      }
    } else {
      answer = f.index;
      if (f.rank < kept) break;
    }
  }
  return answer;
}

// The list path's bound: logits from here on make the list.  each(f) calls f on all of this thread's maxima.
template <int NT, class F>
__device__ inline float list_bound(const SampleSettings& set, const SampleRow& r, SampleShared& sh, F each) {
  if (set.k == 0) {   // min-p alone: w >= m, a little below it for the rounding of the bound itself
    const double z = (double)r.top + (set.m < 1.0 ? ((double)__builtin_amdgcn_logf((float)set.m) - 1e-4) / r.c : 0.0);
    return fmaxf(fminf((float)(z - fabs(z) * 1e-6), r.top), -FLT_MAX);
  }
  // the k-th largest of the threads' maxima, to a bin of (top - the smallest of them) / kSampBoundBins
  float neg = -INFINITY;
  each([&](float z) { neg = fmaxf(neg, z == -INFINITY ? -INFINITY : -z); });
  const float low = -block_max_f<NT>(neg, sh.red_f);
  const float half = 0.5f * r.top - 0.5f * low;   // does not overflow
  const float s = half > 0.0f ? fminf((float)kSampBoundBins / half, 3.0e38f) : 0.0f;
  const auto bin_of = [&](float z) { return min((int)((0.5f * r.top - 0.5f * z) * s), kSampBoundBins - 1); };
  for (int i = threadIdx.x; i < kSampBoundBins; i += NT) sh.bound[i] = 0;
  __syncthreads();
  each([&](float z) {
    if (z != -INFINITY) atomicAdd(&sh.bound[bin_of(z)], 1u);
  });
  __syncthreads();
  const int t = threadIdx.x;
  const uint32_t k = (uint32_t)set.k;
  if (t < kWave) {
    constexpr int kPer = kSampBoundBins / kWave;
    uint32_t c[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += c[i] = sh.bound[t * kPer + i];
    uint32_t inc = sum;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t y = __shfl_up(inc, o);
      if (t >= o) inc += y;
    }
    uint32_t before = inc - sum;
    if (t == kWave - 1 && inc < k) sh.found = kSampBoundBins;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (before < k && before + c[i] >= k) sh.found = t * kPer + i;
      before += c[i];
    }
  }
  __syncthreads();
  // the smallest of the maxima in the bins down to that one: at least k logits are as large
  const int last = sh.found;
  float mine = -INFINITY;
  each([&](float z) {
    if (z != -INFINITY && bin_of(z) <= last) mine = fmaxf(mine, -z);
  });
  const float bound = -block_max_f<NT>(mine, sh.red_f);
  return last == kSampBoundBins ? -FLT_MAX : bound;   // fewer than k threads have one to show: all logits
}

template <class IN>
__global__ void __launch_bounds__(kSampThreads)
sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint64_t cells[];   // bins, or list and prefix
  __shared__ SampleShared sh;
  const int t = threadIdx.x, b = blockIdx.x;
  const typename IN::T* row = static_cast<const typename IN::T*>(a.x) + (int64_t)b * a.ld;
  const SampleSettings set(a, b);
  float mine = -INFINITY, top = -INFINITY;
  if (!set.greedy()) {
    sweep<IN, 4>(row, a.vocab, t, row_vectors<IN>(row, a.vocab), kSampThreads, [&](const auto& z, int) {
#pragma unroll
      for (int e = 0; e < IN::kVec; ++e) mine = fmaxf(mine, z[e]);   // passes over NaN
    });
    top = block_max_f(mine, sh.red_f);
  }
  int token = -1;
  if (top == -INFINITY) {
    token = argmax_row<IN, kSampThreads>(row, a.vocab, 0, row_vectors<IN>(row, a.vocab), sh).i;
  } else {
    const SampleRow r(top, set.T);
    mine = r.see(mine);
    if (set.by_list()) {
      const float bound = list_bound<kSampThreads>(set, r, sh, [&](auto f) { f(mine); });
      collect<IN>(row, a.vocab, r, cells, sh, [&](float v, uint64_t) { return v >= bound; });
      const int n = sh.n_list;
      if (n <= kSampList) {
        sort_list(cells, cells + kSampList, n);
        sum_list(cells, cells + kSampList, n, r, sh);
        token = draw_from_list(cells, cells + kSampList, n, set.k, set.p, set.m, set.u, ~0ull, r);
      }
      __syncthreads();
    }
    if (token < 0) {
      uint64_t above, above_mass;
      fill_bins<IN>(row, a.vocab, r, set.m, cells, sh, above, above_mass);
      token = draw_from_bins<IN>(row, a.vocab, r, cells, sh, set, above, above_mass, -1);
    }
  }
  if (t == 0) a.out[b] = token;
}

// ---- the split form ----------------------------------------------------------------
__device__ inline void chunk_range(int nvec, int chunks, int chunk, int& v0, int& v1) {
  const int per = (nvec + chunks - 1) / chunks;
  v0 = min(chunk * per, nvec);
  v1 = min(v0 + per, nvec);
}

template <class IN>
__global__ void __launch_bounds__(kChunkThreads)
sample_max_kernel(SampleArgs a) {
  const int b = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
  const typename IN::T* row = static_cast<const typename IN::T*>(a.x) + (int64_t)b * a.ld;
  int v0, v1;
  chunk_range(row_vectors<IN>(row, a.vocab), a.chunks, c, v0, v1);
  float* maxima = a.maxima + (int64_t)b * a.chunks * a.per;
  if (c == 0 && t == 0) a.n_list[b] = 0;
  if (SampleSettings(a, b).greedy()) {
    __shared__ SampleShared sh;
    const Best best = argmax_row<IN, kChunkThreads>(row, a.vocab, v0, v1, sh);
    if (t == 0) {
      maxima[c] = best.v;
      a.best[(int64_t)b * a.chunks + c] = best.i;
    }
    return;
  }
  float mine = -INFINITY;
  sweep<IN, 4>(row, a.vocab, v0 + t, v1, kChunkThreads, [&](const auto& z, int) {
#pragma unroll
    for (int e = 0; e < IN::kVec; ++e) mine = fmaxf(mine, z[e]);
  });
  const int group = kChunkThreads / a.per;   // 1 .. 32 neighbours
  for (int o = 1; o < group; o <<= 1) mine = fmaxf(mine, __shfl_xor(mine, o));
  if ((t & (group - 1)) == 0) maxima[c * a.per + t / group] = mine;
}

// The maxima of a row in registers, and the largest.
template <int NT>
struct RowMaxima {
  static constexpr int kMine = (kMaxima + NT - 1) / NT;
  float z[kMine];
  __device__ __forceinline__ float load(const SampleArgs& a, int b, SampleShared& sh) {
    const int n = a.chunks * a.per;
    const float* from = a.maxima + (int64_t)b * n;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int j = (int)threadIdx.x + i * NT;
      z[i] = j < n ? from[j] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) top = fmaxf(top, z[i]);
    return block_max_f<NT>(top, sh.red_f);
  }
};

// The chunk's tokens that `take` accepts, through LDS to the row's list.
template <class IN, class F>
__device__ __forceinline__ void hand_over(const SampleArgs& a, int b, const typename IN::T* row, int v0, int v1,
                                          const SampleRow& r, uint64_t* list, SampleShared& sh, F take) {
  const int t = threadIdx.x;
  if (t == 0) sh.n_list = 0;
  __syncthreads();
  sweep<IN, 1>(row, a.vocab, v0 + t, v1, kChunkThreads, [&](const auto& z, int i0) {
    uint32_t taken = 0;
#pragma unroll
    for (int e = 0; e < IN::kVec; ++e) taken |= take(r.see(z[e])) ? 1u << e : 0u;
    if (taken) {   // places for all of the vector's at once
      int at = atomicAdd(&sh.n_list, __builtin_popcount(taken));
#pragma unroll
      for (int e = 0; e < IN::kVec; ++e) {
        if (!(taken >> e & 1u)) continue;
        if (at < kChunkList) list[at] = entry_of(r.see(z[e]), i0 + e);
        ++at;
      }
    }
  });
  __syncthreads();
  // more than fit here: a number that no list holds
  const int n = sh.n_list;
  if (t == 0) sh.n_work = (int)min(atomicAdd(&a.n_list[b], n <= kChunkList ? (uint32_t)n : 1u << 20), 1u << 24);
  __syncthreads();
  const int at = sh.n_work;
  if (n > kChunkList || at + n > a.list_cap) return;
  for (int i = t; i < n; i += kChunkThreads) a.list[(int64_t)b * a.list_cap + at + i] = list[i];
}

template <class IN>
__global__ void __launch_bounds__(kChunkThreads)
sample_chunk_kernel(SampleArgs a) {
  __shared__ uint64_t cells[kSampBins * kChunkCols];
  static_assert(kSampBins * kChunkCols >= kChunkList, "the list takes the cells' place");
  __shared__ SampleShared sh;
  const int b = blockIdx.y, c = blockIdx.x, t = threadIdx.x;
  const typename IN::T* row = static_cast<const typename IN::T*>(a.x) + (int64_t)b * a.ld;
  const SampleSettings set(a, b);
  if (set.greedy()) return;
  RowMaxima<kChunkThreads> maxima;
  const float top = maxima.load(a, b, sh);
  if (c == 0 && t == 0) a.top[b] = top;
  if (top == -INFINITY) return;
  const SampleRow r(top, set.T);
  int v0, v1;
  chunk_range(row_vectors<IN>(row, a.vocab), a.chunks, c, v0, v1);
  if (set.by_list()) {
    const float bound = list_bound<kChunkThreads>(set, r, sh, [&](auto f) {
#pragma unroll
      for (int i = 0; i < RowMaxima<kChunkThreads>::kMine; ++i) f(r.see(maxima.z[i]));
    });
    hand_over<IN>(a, b, row, v0, v1, r, cells, sh, [&](float v) { return v >= bound; });
    return;
  }
  for (int i = t; i < kSampBins * kChunkCols; i += kChunkThreads) cells[i] = 0;
  __syncthreads();
  uint64_t* own = cells + (t & (kChunkCols - 1));
  uint64_t above = 0, above_mass = 0;
  sweep<IN, 1>(row, a.vocab, v0 + t, v1, kChunkThreads, [&](const auto& z, int) {
    // two tokens' weights at a time, wanted or not: a weight alone is a chain of 20 dependent instructions
#pragma unroll
    for (int e = 0; e < IN::kVec; e += 2) {
      float place[2];
      double w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float v = r.see(z[e + i]);
        place[i] = r.place(v);
        w[i] = exp2_small(r.log2_weight(SampleRow::alive(place[i]) ? v : r.top));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (SampleRow::alive(place[i])) {
          if (set.m > 0.0 && w[i] >= set.m) {
            above += 1;
            above_mass += SampleRow::mass(w[i]);
          }
          add_to_cell(&own[(int)place[i] * kChunkCols], w[i]);
        }
    }
  });
  above = block_sum<kChunkThreads>(above, sh.red_u);   // and the barrier after the cells' additions
  above_mass = block_sum<kChunkThreads>(above_mass, sh.red_u);
  const int64_t at = (int64_t)b * a.chunks + c;
  {
    static_assert(kSampBins == kChunkThreads, "a thread sums up a bin");
    uint64_t mass = 0;
    uint32_t count = 0;
#pragma unroll
    for (int i = 0; i < kChunkCols; ++i) {   // every thread from a column of its own on: no bank conflicts
      const uint64_t w = cells[t * kChunkCols + ((i + t) & (kChunkCols - 1))];
      mass += w & (kSampCount - 1);
      count += (uint32_t)(w >> 51);
    }
    a.bin_mass[at * kSampBins + t] = mass;
    a.bin_count[at * kSampBins + t] = count;
  }
  if (t == 0) {
    a.above[at] = (uint32_t)above;
    a.above_mass[at] = above_mass;
  }
}

// The bins of a row from those of its chunks, by kSampBins threads or more.
__device__ __forceinline__ void row_bins(const SampleArgs& a, int b, SampleShared& sh, uint64_t& above, uint64_t& above_mass) {
  const int t = threadIdx.x;
  const int64_t at = (int64_t)b * a.chunks;
  if (t < kSampBins) {
    uint64_t mass = 0;
    uint32_t count = 0;
#pragma unroll 16
    for (int c = 0; c < a.chunks; ++c) {
      mass += a.bin_mass[(at + c) * kSampBins + t];
      count += a.bin_count[(at + c) * kSampBins + t];
    }
    sh.row.mass[t] = mass;
    sh.row.count[t] = count;
  }
  above = above_mass = 0;
#pragma unroll 8
  for (int c = 0; c < a.chunks; ++c) {
    above += a.above[at + c];
    above_mass += a.above_mass[at + c];
  }
  __syncthreads();
  before_bins(sh.row);
}

template <class IN>
__global__ void __launch_bounds__(kChunkThreads)
sample_gather_kernel(SampleArgs a) {
  __shared__ uint64_t list[kChunkList];
  __shared__ SampleShared sh;
  const int b = blockIdx.y, c = blockIdx.x;
  const SampleSettings set(a, b);
  if (set.greedy() || set.by_list()) return;
  const typename IN::T* row = static_cast<const typename IN::T*>(a.x) + (int64_t)b * a.ld;
  const float top = a.top[b];
  if (top == -INFINITY) return;
  const SampleRow r(top, set.T);
  uint64_t above, above_mass;
  row_bins(a, b, sh, above, above_mass);
  if (c == 0) {   // for the workgroup that finishes the row
    const int t = threadIdx.x;
    a.row_mass[(int64_t)b * (kSampBins + 2) + t] = sh.row.mass[t];
    a.row_count[(int64_t)b * kSampBins + t] = sh.row.count[t];
    if (t == 0) {
      a.row_mass[(int64_t)b * (kSampBins + 2) + kSampBins] = above_mass;
      a.row_mass[(int64_t)b * (kSampBins + 2) + kSampBins + 1] = above;
    }
  }
  const Needed needed(set, sh.row, above, above_mass);
  int v0, v1;
  chunk_range(row_vectors<IN>(row, a.vocab), a.chunks, c, v0, v1);
  hand_over<IN>(a, b, row, v0, v1, r, list, sh, [&](float v) { return needed.has(r.place(v)); });
}

template <class IN>
__global__ void __launch_bounds__(kSampThreads)
sample_finish_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint64_t cells[];
  __shared__ SampleShared sh;
  const int t = threadIdx.x, b = blockIdx.x;
  const typename IN::T* row = static_cast<const typename IN::T*>(a.x) + (int64_t)b * a.ld;
  const SampleSettings set(a, b);
  if (set.greedy()) {
    Best best{-INFINITY, 0x7fffffff};
    if (t < a.chunks) best = Best{a.maxima[(int64_t)b * a.chunks * a.per + t], a.best[(int64_t)b * a.chunks + t]};
    best = block_best<kSampThreads>(best, sh);
    if (t == 0) a.out[b] = best.i;
    return;
  }
  const float top = a.top[b];
  int token;
  if (top == -INFINITY) {
    token = argmax_row<IN, kSampThreads>(row, a.vocab, 0, row_vectors<IN>(row, a.vocab), sh).i;
  } else {
    const SampleRow r(top, set.T);
    const uint32_t listed = a.n_list[b];
    const int n = listed <= (uint32_t)a.list_cap ? (int)listed : -1;
    for (int i = t; i < n; i += kSampThreads) cells[i] = a.list[(int64_t)b * a.list_cap + i];
    __syncthreads();
    if (set.by_list() && n >= 0) {
      sort_list(cells, cells + kSampList, n);
      sum_list(cells, cells + kSampList, n, r, sh);
      token = draw_from_list(cells, cells + kSampList, n, set.k, set.p, set.m, set.u, ~0ull, r);
    } else {
      uint64_t above, above_mass;
      if (set.by_list()) {   // more than could be handed over
        fill_bins<IN>(row, a.vocab, r, set.m, cells, sh, above, above_mass);
      } else {
        const uint64_t* mass = a.row_mass + (int64_t)b * (kSampBins + 2);
        if (t < kSampBins) {
          sh.row.mass[t] = mass[t];
          sh.row.count[t] = a.row_count[(int64_t)b * kSampBins + t];
        }
        above_mass = mass[kSampBins];
        above = mass[kSampBins + 1];
        __syncthreads();
        before_bins(sh.row);
      }
      token = draw_from_bins<IN>(row, a.vocab, r, cells, sh, set, above, above_mass, n);
    }
  }
  if (t == 0) a.out[b] = token;
}

// How a call's rows are cut.  chunks 0: one workgroup takes a row whole.
struct SamplePlan {
  int chunks, per, list_cap;
  int64_t words;   // of 8 bytes, of the workspace
};
static SamplePlan sample_plan(int rows, int vocab) {
  if (vocab < 16384) return SamplePlan{0, 0, 0, 0};
  int c = 2048 / rows;
  c = c < 1 ? 1 : c > 16 ? 16 : c;
  const int most = vocab / 2048, least = (vocab + kChunkMost - 1) / kChunkMost;
  c = c > most ? most : c;
  c = c < least ? least : c;
  SamplePlan p{c, kChunkThreads, rows <= 512 ? kSampList : rows <= 4096 ? kSampList / 4 : kSampList / 16, 0};
  while (p.per * c > kMaxima && p.per > 8) p.per /= 2;
  p.words = (int64_t)rows * ((int64_t)c * (p.per / 2 + kSampBins + kSampBins / 2 + 2) + p.list_cap + 1 +
                              kSampBins + 2 + kSampBins / 2);
  return p;
}

template <class IN>
static int sample_launch(SampleArgs a, const SamplePlan& p, uint64_t* ws, hipStream_t s) {
  constexpr size_t lds = (size_t)kSampBins * kSampCols * sizeof(uint64_t);
  static_assert((size_t)kSampList * 16 == lds, "list and prefix take the bins' place");
  if (p.chunks == 0) {
    TQ_RETURN_IF_HIP_ERROR((allow_lds<sample_kernel<IN>>(lds)));
    hipLaunchKernelGGL(sample_kernel<IN>, dim3(a.rows), dim3(kSampThreads), lds, s, a);
    return (int)hipGetLastError();
  }
  const int64_t n = (int64_t)a.rows * p.chunks;
  a.chunks = p.chunks;
  a.per = p.per;
  a.list_cap = p.list_cap;
  a.bin_mass = ws;
  a.list = a.bin_mass + n * kSampBins;
  a.above_mass = a.list + (int64_t)a.rows * p.list_cap;
  a.row_mass = a.above_mass + n;
  a.maxima = reinterpret_cast<float*>(a.row_mass + (int64_t)a.rows * (kSampBins + 2));
  a.bin_count = reinterpret_cast<uint32_t*>(a.maxima + n * p.per);
  a.row_count = a.bin_count + n * kSampBins;
  a.above = a.row_count + (int64_t)a.rows * kSampBins;
  a.best = reinterpret_cast<int32_t*>(a.above + n);
  a.n_list = reinterpret_cast<uint32_t*>(a.best + n);
  a.top = reinterpret_cast<float*>(a.n_list + a.rows);
  TQ_RETURN_IF_HIP_ERROR((allow_lds<sample_finish_kernel<IN>>(lds)));
  const dim3 grid(p.chunks, a.rows), block(kChunkThreads);
  hipLaunchKernelGGL(sample_max_kernel<IN>, grid, block, 0, s, a);
  // what no row of the call has to do, where one number sets all rows
  const bool greedy = !a.temperature && !(a.temperature0 > 0.0f);
  const int k = a.top_k0 < a.vocab ? a.top_k0 : 0;
  const bool lists = !a.top_k && (k > 0 ? k <= kSampTopK : !a.top_p && !a.min_p && a.top_p0 >= 1.0f && a.min_p0 > 0.0f);
  if (!greedy) hipLaunchKernelGGL(sample_chunk_kernel<IN>, grid, block, 0, s, a);
  if (!greedy && !lists) hipLaunchKernelGGL(sample_gather_kernel<IN>, grid, block, 0, s, a);
  hipLaunchKernelGGL(sample_finish_kernel<IN>, dim3(a.rows), dim3(kSampThreads), lds, s, a);
  return (int)hipGetLastError();
}

}  // namespace tq

using namespace tq;

extern "C" int64_t tq_sample_workspace_elems(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > kSampMaxVocab) return 0;
  return sample_plan(rows, vocab).words;
}

extern "C" int tq_sample_tokens(const void* logits, int64_t logits_stride, int dtype, int rows, int vocab,
                                const float* uniform, const float* temperature, float temperature_all,
                                const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all,
                                const float* min_p, float min_p_all, int64_t* tokens, int64_t* workspace,
                                int64_t workspace_elems, void* stream) {
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_FP16 && dtype != TQ_DTYPE_FP32) return TQ_ERR_DTYPE;
  if (rows < 0 || rows > 65535 || vocab <= 0 || vocab > kSampMaxVocab || (rows > 1 && logits_stride < vocab))
    return TQ_ERR_ARG;
  if (rows == 0) return TQ_OK;
  if (!logits || !uniform || !tokens) return TQ_ERR_ARG;
  const size_t size = dtype == TQ_DTYPE_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return TQ_ERR_ALIGN;
  SampleArgs a{};
  a.x = logits; a.ld = logits_stride; a.u = uniform;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.temperature0 = temperature_all; a.top_k0 = top_k_all; a.top_p0 = top_p_all; a.min_p0 = min_p_all;
  a.out = tokens; a.rows = rows; a.vocab = vocab;
  const SamplePlan p = sample_plan(rows, vocab);
  if (p.chunks && (!workspace || workspace_elems < p.words)) return TQ_ERR_WORKSPACE;
  uint64_t* ws = reinterpret_cast<uint64_t*>(workspace);
  if (reinterpret_cast<uintptr_t>(ws) & 7u) return TQ_ERR_ALIGN;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == TQ_DTYPE_BF16) return sample_launch<H16In<Bf16>>(a, p, ws, s);
  if (dtype == TQ_DTYPE_FP16) return sample_launch<H16In<Fp16>>(a, p, ws, s);
  return sample_launch<F32In>(a, p, ws, s);
}

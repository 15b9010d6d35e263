// tq_paged.hip -- block tables of a paged KV cache, and its INT8 codes: quantized append and read-back, gfx950.
//
// The cache (tq_kv8_cache): pages of `block` tokens, each cut into units of 16 tokens.  Per page, kv head and unit:
//   k_codes [16 tokens][D], v_codes [D][16 tokens] (int8), one fp32 scale each.
// A unit of one head is 16 D contiguous bytes either way.  The values are stored transposed because the attention's
// P V product takes them as a matrix operand whose lanes each hold consecutive tokens of one dimension.
#include "tq_common.h"

namespace tq {

// ---- block tables -----------------------------------------------------------
//
// One step over all rows (requests), in row order:
//   a finished row pushes its ceil(length / block) pages on the free stack; its length becomes 0;
//   row b then asks for n = max(new_tokens[b], 0) tokens and need = ceil((length + n) / block) - ceil(length / block)
//   pages, and is granted them iff they fit the table's width, the inclusive sum of the needs does not pass the free
//   pages (a row that needs none is not held up by this), and the inclusive sum of the tokens does not pass max_tokens.
//   Granted rows pop their pages in row order and get the next places of the slot list.
// The sums are exclusive / inclusive prefix sums over the rows, so one workgroup does them (a chunk of one row per
// thread at a time, carries in registers); pages and tokens are then dealt to the threads flat, each finding its row by
// a binary search in the chunk's prefix sums in LDS.  What it moves is little (8 bytes a token); the bound is the chain
// of waits of one workgroup: 64 rows with a token each 4 us, about an empty launch; 256 rows that all end and take 115
// thousand tokens (12 thousand pages, every page's and token's row searched for) 19 us with the slots' launch.
constexpr int kTabThreads = 1024;

struct TablesArgs {
  const int32_t* new_tokens;
  const uint8_t* finished;
  int32_t* table;
  int64_t ld;
  int32_t* lengths;
  int32_t* free_list;
  int free_cap;
  int32_t* free_count;
  int32_t* slots;
  int32_t* positions;
  int32_t* query_start;
  uint8_t* granted;
  int rows, width, block, max_tokens;
};

// Inclusive sums over the workgroup of two 64-bit values per thread (64 bits: the sums of what rows ask for may pass 32).
struct Pair64 {
  int64_t a, b;
};
template <int NT>
__device__ inline Pair64 scan_inclusive(Pair64 x, Pair64* wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int64_t a = __shfl_up(x.a, off), b = __shfl_up(x.b, off);
    if (lane >= off) {
      x.a += a;
      x.b += b;
    }
  }
  if constexpr (NT > kWave) {
    if (lane == kWave - 1) wave_sums[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      x.a += wave_sums[w].a;
      x.b += wave_sums[w].b;
    }
    __syncthreads();   // the next scan writes wave_sums again
  }
  return x;
}

// Per item: the last index r in [0, N) with start[r] <= x (start ascending, start[0] <= x; N a power of two).  The
// items' searches run side by side: one alone waits for LDS log2(N) times.
constexpr int kFlat = 4;
template <int N>
__device__ __forceinline__ void last_at_most(const int64_t* start, const int64_t (&x)[kFlat], int (&r)[kFlat]) {
#pragma unroll
  for (int j = 0; j < kFlat; ++j) r[j] = 0;
#pragma unroll
  for (int step = N / 2; step > 0; step >>= 1)
#pragma unroll
    for (int j = 0; j < kFlat; ++j) r[j] = start[r[j] + step] <= x[j] ? r[j] + step : r[j];
}

// A page that is not one of the cache's (a damaged list) gives a slot that the cache's kernels skip, or another page's.
__device__ inline int32_t slot_of(int32_t page, int block, int at) { return (int32_t)((uint32_t)page * block + at); }

template <int NT, bool TOKENS>
__global__ void __launch_bounds__(NT)
tables_step_kernel(TablesArgs a) {
  __shared__ Pair64 wave_sums[NT / kWave];
  __shared__ int64_t start_pages[NT], start_tokens[NT];
  __shared__ int32_t row_len[NT], row_have[NT];
  __shared__ Pair64 carry, total;   // of the last thread
  const int t = threadIdx.x;
  const int64_t count0 = min(max(a.free_count[0], 0), a.free_cap);

  // ---- finished rows give their pages back
  int64_t pushed = 0;
  if (a.finished != nullptr) {
    for (int r0 = 0; r0 < a.rows; r0 += NT) {
      const int b = r0 + t;
      int held = 0;
      if (b < a.rows && a.finished[b])
        held = min((int)(((uint32_t)max(a.lengths[b], 0) + a.block - 1) / (uint32_t)a.block), a.width);
      const Pair64 inc = scan_inclusive<NT>(Pair64{held, 0}, wave_sums);
      start_pages[t] = inc.a - held;
      if (t == NT - 1) total = inc;
      __syncthreads();
      const int64_t n = total.a;
      for (int64_t i0 = t; i0 < n; i0 += kFlat * NT) {
        int64_t i[kFlat];
        int r[kFlat], page[kFlat];
        int32_t* entry[kFlat];
#pragma unroll
        for (int j = 0; j < kFlat; ++j) i[j] = i0 + j * NT;
        last_at_most<NT>(start_pages, i, r);
#pragma unroll
        for (int j = 0; j < kFlat; ++j) {
          entry[j] = a.table + (int64_t)(r0 + r[j]) * a.ld + (i[j] - start_pages[r[j]]);
          if (i[j] < n) page[j] = *entry[j];
        }
#pragma unroll
        for (int j = 0; j < kFlat; ++j) {
          const int64_t at = count0 + pushed + i[j];
          if (i[j] < n && at < a.free_cap) a.free_list[at] = page[j];
          if (i[j] < n) *entry[j] = -1;
        }
      }
      pushed += n;
      __syncthreads();   // the next chunk writes the sums; the pops below read the list
    }
  }
  const int64_t count = min(count0 + pushed, (int64_t)a.free_cap);

  // ---- rows take pages and places
  Pair64 asked{0, 0}, taken{0, 0};   // (pages, tokens) of the chunks before
  for (int r0 = 0; r0 < a.rows; r0 += NT) {
    const int b = r0 + t;
    const bool live = b < a.rows;
    int64_t len = 0, n = 0, have = 0, need = 0;
    bool fits = false;
    if (live) {
      len = (a.finished != nullptr && a.finished[b]) ? 0 : max(a.lengths[b], 0);
      n = max(a.new_tokens[b], 0);
      fits = len + n <= (int64_t)a.width * a.block;
      // 32 bits hold these: len < 2^31, and len + n <= width * block < 2^31 where it fits
      have = ((uint32_t)len + a.block - 1) / (uint32_t)a.block;
      need = fits ? ((uint32_t)(len + n) + a.block - 1) / (uint32_t)a.block - have : 0;
    }
    const Pair64 inc = scan_inclusive<NT>(Pair64{need, fits ? n : 0}, wave_sums);
    const bool ok = live && fits && (need == 0 || asked.a + inc.a <= count) && asked.b + inc.b <= a.max_tokens;
    if (!ok) need = n = 0;
    const Pair64 got = scan_inclusive<NT>(Pair64{need, n}, wave_sums);
    start_pages[t] = got.a - need;
    start_tokens[t] = got.b - n;
    row_len[t] = (int32_t)len;
    row_have[t] = (int32_t)min(have, (int64_t)a.width);
    if (t == NT - 1) {
      carry = inc;
      total = got;
    }
    if (live) {
      a.granted[b] = ok ? 1 : 0;
      a.lengths[b] = (int32_t)(len + n);
      a.query_start[b] = (int32_t)(taken.b + got.b - n);
    }
    __syncthreads();
    const Pair64 chunk = total;
    for (int64_t i0 = t; i0 < chunk.a; i0 += kFlat * NT) {
      int64_t i[kFlat];
      int r[kFlat], page[kFlat];
#pragma unroll
      for (int j = 0; j < kFlat; ++j) {
        i[j] = i0 + j * NT;
        if (i[j] < chunk.a) page[j] = a.free_list[count - 1 - taken.a - i[j]];
      }
      last_at_most<NT>(start_pages, i, r);
#pragma unroll
      for (int j = 0; j < kFlat; ++j)
        if (i[j] < chunk.a) a.table[(int64_t)(r0 + r[j]) * a.ld + row_have[r[j]] + (i[j] - start_pages[r[j]])] = page[j];
    }
    if constexpr (TOKENS) {
      for (int64_t i0 = t; i0 < chunk.b; i0 += kFlat * NT) {
        int64_t i[kFlat];
        int r[kFlat], page[kFlat];
        uint32_t pos[kFlat], page_at[kFlat];
#pragma unroll
        for (int j = 0; j < kFlat; ++j) i[j] = i0 + j * NT;
        last_at_most<NT>(start_tokens, i, r);
#pragma unroll
        for (int j = 0; j < kFlat; ++j) {
          pos[j] = (uint32_t)(row_len[r[j]] + (i[j] - start_tokens[r[j]]));
          page_at[j] = pos[j] / (uint32_t)a.block;
          const int64_t fresh = (int64_t)page_at[j] - row_have[r[j]];   // < 0: a page that the row had
          const int32_t* from = fresh < 0 ? a.table + (int64_t)(r0 + r[j]) * a.ld + page_at[j]
                                          : a.free_list + (count - 1 - taken.a - (start_pages[r[j]] + fresh));
          if (i[j] < chunk.b) page[j] = *from;
        }
#pragma unroll
        for (int j = 0; j < kFlat; ++j) {
          if (i[j] >= chunk.b) continue;
          a.slots[taken.b + i[j]] = page[j] < 0 ? -1 : slot_of(page[j], a.block, (int)(pos[j] - page_at[j] * a.block));
          a.positions[taken.b + i[j]] = (int32_t)pos[j];
        }
      }
    }
    asked.a += carry.a;
    asked.b += carry.b;
    taken.a += chunk.a;
    taken.b += chunk.b;
    __syncthreads();   // the next chunk writes the sums
  }
  if (t == 0) {
    a.query_start[a.rows] = (int32_t)taken.b;
    a.free_count[0] = (int32_t)(count - taken.a);
  }
  if constexpr (TOKENS) {
    for (int64_t i = taken.b + t; i < a.max_tokens; i += NT) {
      a.slots[i] = -1;
      a.positions[i] = 0;
    }
  }
}

// The slot list of many tokens, a launch of its own: the table, the lengths and the rows' places are there.
constexpr int kSlotThreads = 256;
__global__ void __launch_bounds__(kSlotThreads)
tables_slots_kernel(TablesArgs a) {
  const int i = blockIdx.x * kSlotThreads + threadIdx.x;
  if (i >= a.max_tokens) return;
  int32_t slot = -1, pos = 0;
  if (i < a.query_start[a.rows]) {
    int lo = 0, hi = a.rows;   // last row with query_start <= i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.query_start[mid] <= i) lo = mid;
      else hi = mid;
    }
    const int first = a.query_start[lo], n = a.query_start[lo + 1] - first;
    pos = a.lengths[lo] - n + (i - first);
    const int32_t page = a.table[(int64_t)lo * a.ld + pos / a.block];
    slot = page < 0 ? -1 : slot_of(page, a.block, pos % a.block);
  }
  a.slots[i] = slot;
  a.positions[i] = pos;
}

// ---- append -------------------------------------------------------------------
//
// Per unit and head, over the new tokens x of the unit (a: their absmax; below 2^-100 it counts as 0):
//   s = max(s_old, a / 127),  s_old = 0 when no older token is in the unit;  new codes rint(x (1 / s));
//   older codes c become rint(c (s_old / s)) when the scale grew.  All fp32, divisions correctly rounded.
// One wave takes the units whose first new token is among its `window` tokens of the list, for one head of K or V; it
// sees which those are from the slots themselves, so no list of units is made.  A window of 16 tokens holds the start
// of about one unit of a prompt; a window of 1 keeps a decoding step's units, one token each, on a wave each.
// The bound is memory: 16-bit rows in, codes out.  4 prompts of 2048 tokens, 8 kv heads of 128: 50 MB in 14.5 us,
// 3.5 TB/s where a large copy reaches 4.9 (one wave a token, clamps and roundings in fp32, loads behind branches: 38).
struct AppendArgs {
  const uint16_t* x[2];
  int64_t x_st[2], x_sh[2];
  const int32_t* slots;
  int8_t* codes[2];
  float* scales[2];
  int tokens, window, kv_heads, units;   // units per page
  int unit_shift;                // log2(units)
  int64_t n_slots;
};

constexpr float kTinyAbsmax = 7.888609052210118e-31f;   // 2^-100

// Two 16-bit values in a word, as bits: |x| orders like the integers.
template <class XT>
constexpr uint32_t kInfBits = std::is_same<XT, Bf16>::value ? 0x7f80u : 0x7c00u;

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max_abs2(uint32_t m, uint32_t w) {   // both halves
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                                __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
// NaN -> 0, infinities -> the largest finite value
template <class XT>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  uint32_t r = 0;
#pragma unroll
  for (int sh = 0; sh < 32; sh += 16) {
    const uint32_t x = (w >> sh) & 0xffffu, m = x & 0x7fffu;
    r |= (m < kInfBits<XT> ? x : m == kInfBits<XT> ? x - 1 : 0u) << sh;
  }
  return r;
}

// The absmax of the unit whose values the wave's lanes hold; values that are not finite are replaced in place.
template <class XT, int N>
__device__ __forceinline__ float unit_absmax(uint32_t (&v)[N]) {
  for (;;) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max_abs2(m, v[i]);
    m = max(m & 0xffffu, m >> 16);
    m = __float_as_uint(wave_max_nonneg(__uint_as_float(m)));   // an integer maximum over the lanes
    if (m < kInfBits<XT>) return XT::to_f32((uint16_t)m);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = finite2<XT>(v[i]);
  }
}

// rint(x r) in the low byte: |x r| <= 127 (1 + 2^-22), and adding 1.5 * 2^23 rounds to an integer, ties to even
__device__ __forceinline__ uint32_t code_of(float x, float r) { return __float_as_uint(x * r + 12582912.0f); }
__device__ __forceinline__ uint32_t bytes4(uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {   // the low bytes
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b3, b2, 0x0c0c0400u), __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u),
                               0x05040100u);
}
template <class XT>
__device__ __forceinline__ float half_of(uint32_t w, int i) { return XT::to_f32((uint16_t)(w >> (16 * i))); }
__device__ inline float byte_code(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }

struct UnitScale {
  float s, inv, shrink;
  bool grew;
  __device__ UnitScale(float absmax, float old) {
    const float a = absmax < kTinyAbsmax ? 0.0f : absmax;
    s = fmaxf(old, a / 127.0f);
    inv = s > 0.0f ? 1.0f / s : 0.0f;
    grew = s > old;
    shrink = s > 0.0f ? old / s : 0.0f;
  }
};

// One unit of one head: `src` names each offset's new token (-1: none), `first` is one of them.
template <class XT, int D>
__device__ __forceinline__ void append_unit(const AppendArgs& a, int h, int kv, int64_t unit, const int (&src)[16],
                                            int first) {
  const int lane = threadIdx.x & 63;
  int begun = 16;   // the unit held tokens 0 .. begun - 1 before
  bool whole = true;
#pragma unroll
  for (int o = 15; o >= 0; --o) {
    if (src[o] >= 0) begun = o;
    else whole = false;
  }
  const int64_t cell = ((unit >> a.unit_shift) * a.kv_heads + h) * a.units + (unit & (a.units - 1));
  float* scale_at = a.scales[kv] + cell;
  int8_t* codes = a.codes[kv] + cell * (16 * D);
  const float old = begun > 0 ? *scale_at : 0.0f;
  const uint16_t* x = a.x[kv] + (int64_t)h * a.x_sh[kv];

  // All loads are issued before the first is used: an offset without a new token reads `first` and drops it.
  if (kv == 0) {
    // lane: 8 dimensions of every kRows-th token
    constexpr int kLanes = D / 8, kRows = kWave / kLanes, kSteps = 16 / kRows;
    const int ch = lane % kLanes, rg = lane / kLanes;
    uint32_t v[kSteps * 4];
    u32x2 oc[kSteps];
    int sr[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      sr[i] = src[kRows * i];
#pragma unroll
      for (int r = 1; r < kRows; ++r) sr[i] = rg == r ? src[kRows * i + r] : sr[i];
      const int row = sr[i] >= 0 ? sr[i] : first;
      const u32x4 w = *reinterpret_cast<const u32x4*>(x + (int64_t)row * a.x_st[0] + ch * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * i + e] = w[e];
    }
    if (begun > 0) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) oc[i] = *reinterpret_cast<const u32x2*>(codes + (rg + kRows * i) * D + ch * 8);
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * i + e] = sr[i] >= 0 ? v[4 * i + e] : 0u;
    const UnitScale u(unit_absmax<XT>(v), old);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      u32x2 w;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint32_t lo = v[4 * i + 2 * p], hi = v[4 * i + 2 * p + 1];
        w[p] = bytes4(code_of(half_of<XT>(lo, 0), u.inv), code_of(half_of<XT>(lo, 1), u.inv),
                      code_of(half_of<XT>(hi, 0), u.inv), code_of(half_of<XT>(hi, 1), u.inv));
      }
      if (sr[i] >= 0) *reinterpret_cast<u32x2*>(codes + (rg + kRows * i) * D + ch * 8) = w;
    }
    if (begun > 0 && u.grew) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        u32x2 w;
#pragma unroll
        for (int p = 0; p < 2; ++p)
          w[p] = bytes4(code_of(byte_code(oc[i][p], 0), u.shrink), code_of(byte_code(oc[i][p], 1), u.shrink),
                        code_of(byte_code(oc[i][p], 2), u.shrink), code_of(byte_code(oc[i][p], 3), u.shrink));
        if (rg + kRows * i < begun) *reinterpret_cast<u32x2*>(codes + (rg + kRows * i) * D + ch * 8) = w;
      }
    }
    if (lane == 0) *scale_at = u.s;
  } else {
    // lane: all 16 tokens of kDims dimensions (a unit's row of 16 bytes each)
    constexpr int kDims = D / kWave;
    uint32_t v[16];
    u32x4 oc[kDims];
#pragma unroll
    for (int o = 0; o < 16; ++o) {
      const uint16_t* p = x + (int64_t)(src[o] >= 0 ? src[o] : first) * a.x_st[1] + lane * kDims;
      if constexpr (kDims == 2) v[o] = *reinterpret_cast<const uint32_t*>(p);
      else v[o] = *p;
    }
    if (!whole) {
#pragma unroll
      for (int d = 0; d < kDims; ++d) oc[d] = *reinterpret_cast<const u32x4*>(codes + (lane * kDims + d) * 16);
    }
#pragma unroll
    for (int o = 0; o < 16; ++o) v[o] = src[o] >= 0 ? v[o] : 0u;
    const UnitScale u(unit_absmax<XT>(v), old);
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      u32x4 w;
#pragma unroll
      for (int p = 0; p < 4; ++p)
        w[p] = bytes4(code_of(half_of<XT>(v[4 * p], d), u.inv), code_of(half_of<XT>(v[4 * p + 1], d), u.inv),
                      code_of(half_of<XT>(v[4 * p + 2], d), u.inv), code_of(half_of<XT>(v[4 * p + 3], d), u.inv));
      if (!whole) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          uint32_t now = 0, c = oc[d][p];
          if (begun > 0 && u.grew)
            c = bytes4(code_of(byte_code(c, 0), u.shrink), code_of(byte_code(c, 1), u.shrink),
                       code_of(byte_code(c, 2), u.shrink), code_of(byte_code(c, 3), u.shrink));
#pragma unroll
          for (int e = 0; e < 4; ++e) now |= src[4 * p + e] >= 0 ? 0xffu << (8 * e) : 0u;
          uint32_t kept = 0;   // offsets at and above `begun` without a new token stay as they were
#pragma unroll
          for (int e = 0; e < 4; ++e) kept |= 4 * p + e >= begun ? 0xffu << (8 * e) : 0u;
          w[p] = (w[p] & now) | (((c & ~kept) | (oc[d][p] & kept)) & ~now);
        }
      }
      *reinterpret_cast<u32x4*>(codes + (lane * kDims + d) * 16) = w;
    }
    if (lane == 0) *scale_at = u.s;
  }
}

template <class XT, int D>
__global__ void __launch_bounds__(256)
kv8_append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + wave) * a.window;
  const int h = blockIdx.y, kv = blockIdx.z;
  if (t0 >= a.tokens) return;
  // the unit of each lane's token (-1: none), and of the token before it
  const auto load_slot = [&](int64_t t) {
    const int32_t s = t < a.tokens ? a.slots[t] : -1;
    return s < a.n_slots ? s : -1;
  };
  const int slot = load_slot(t0 + lane), unit = slot < 0 ? -1 : slot >> 4;
  int before = __shfl_up(unit, 1);
  if (lane == 0) before = t0 > 0 ? load_slot(t0 - 1) : -1, before = before < 0 ? -1 : before >> 4;
  uint32_t todo = (uint32_t)__ballot(lane < a.window && unit >= 0 && unit != before);   // window <= 16
  for (; todo; todo &= todo - 1) {
    const int i = __builtin_ctz(todo);
    const int mine = __builtin_amdgcn_readlane(unit, i);
    // the run of tokens of this unit; each offset's source is the last token that names it
    int src[16];
#pragma unroll
    for (int o = 0; o < 16; ++o) src[o] = -1;
    int64_t base = t0;
    int at = slot, at_unit = unit;
    uint64_t skip = (1ull << i) - 1;   // lanes before the run
    for (;;) {
      const uint64_t out = ~(__ballot(at_unit == mine) | skip);
      const uint64_t run = (out ? (out & (0 - out)) - 1 : ~0ull) & ~skip;
#pragma unroll
      for (int o = 0; o < 16; ++o) {
        const uint64_t named = __ballot((at & 15) == o) & run;
        if (named) src[o] = (int)(base + 63 - __builtin_clzll(named));
      }
      if (out) break;
      base += kWave;
      if (base >= a.tokens) break;
      at = load_slot(base + lane);
      at_unit = at < 0 ? -1 : at >> 4;
      skip = 0;
    }
    append_unit<XT, D>(a, h, kv, mine, src, (int)t0 + i);
  }
}

// ---- read ----------------------------------------------------------------------
//
// code * scale, rounded once, of the listed slots (slots outside the cache: zeros).  One wave per 16 list entries,
// head and K or V.  Keys are copied row by row; values, stored transposed, unit by unit: the wave takes the unit of its
// first entry not yet written, and with it every entry of that unit (a list in token order has one or two units).
// The bound is memory: 8192 tokens, 8 kv heads of 128: 50 MB in 10 us, as fast as a large copy.
struct ReadArgs {
  const int32_t* slots;
  const int8_t* codes[2];
  const float* scales[2];
  uint16_t* out[2];
  int64_t o_st[2], o_sh[2];
  int n, kv_heads, units, unit_shift;
  int64_t n_slots;
};

template <class XT, int D>
__global__ void __launch_bounds__(256)
kv8_read_kernel(ReadArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = (blockIdx.x * 4 + wave) * 16;
  const int h = blockIdx.y, kv = blockIdx.z;
  if (n0 >= a.n) return;
  const int entry = n0 + (lane & 15);
  int64_t slot = entry < a.n ? (int64_t)a.slots[entry] : -1;
  if (slot >= a.n_slots) slot = -1;
  const int my_slot = (int)slot;   // n_slots < 2^31
  uint16_t* out = a.out[kv] + (int64_t)h * a.o_sh[kv];
  if (kv == 0) {
    constexpr int kLanes = D / 8, kRows = kWave / kLanes, kSteps = 16 / kRows;
    const int ch = lane % kLanes, rg = lane / kLanes;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int e = rg + kRows * i;
      const int64_t s = __shfl(my_slot, e);
      if (n0 + e >= a.n) continue;
      u32x4 w{0, 0, 0, 0};
      if (s >= 0) {
        const int64_t unit = s >> 4;
        const int64_t cell = ((unit >> a.unit_shift) * a.kv_heads + h) * a.units + (unit & (a.units - 1));
        const u32x2 c = *reinterpret_cast<const u32x2*>(a.codes[0] + cell * (16 * D) + (s & 15) * D + ch * 8);
        const float sc = a.scales[0][cell];
#pragma unroll
        for (int p = 0; p < 4; ++p)
          w[p] = XT::pack2(byte_code(c[p >> 1], 2 * (p & 1)) * sc, byte_code(c[p >> 1], 2 * (p & 1) + 1) * sc);
      }
      *reinterpret_cast<u32x4*>(out + (int64_t)(n0 + e) * a.o_st[0] + ch * 8) = w;
    }
  } else {
    constexpr int kDims = D / kWave;
    uint32_t left = (1u << min(16, a.n - n0)) - 1;   // entries not yet written (wave-uniform)
    const auto put = [&](int e, const float (&y)[kDims]) {
      uint16_t* p = out + (int64_t)(n0 + e) * a.o_st[1] + lane * kDims;
      if constexpr (kDims == 2) *reinterpret_cast<uint32_t*>(p) = XT::pack2(y[0], y[1]);
      else *p = XT::from_f32(y[0]);
    };
    while (left) {
      const int e0 = __builtin_ctz(left);
      const int s0 = __builtin_amdgcn_readlane(my_slot, e0);
      if (s0 < 0) {
        const float zero[kDims] = {};
        put(e0, zero);
        left &= left - 1;
        continue;
      }
      const int64_t unit = s0 >> 4;
      const uint32_t same = (uint32_t)__ballot(my_slot >= 0 && (my_slot >> 4) == (s0 >> 4)) & left;
      left &= ~same;
      const int64_t cell = ((unit >> a.unit_shift) * a.kv_heads + h) * a.units + (unit & (a.units - 1));
      u32x4 c[kDims];
#pragma unroll
      for (int d = 0; d < kDims; ++d)
        c[d] = *reinterpret_cast<const u32x4*>(a.codes[1] + cell * (16 * D) + (lane * kDims + d) * 16);
      const float sc = a.scales[1][cell];
      for (uint32_t todo = same; todo; todo &= todo - 1) {
        const int e = __builtin_ctz(todo);
        const int o = __builtin_amdgcn_readlane(my_slot, e) & 15;
        float y[kDims];
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const uint32_t lo = (o & 4) ? c[d][1] : c[d][0], hi = (o & 4) ? c[d][3] : c[d][2];
          y[d] = (float)(int8_t)(((o & 8) ? hi : lo) >> (8 * (o & 3))) * sc;
        }
        put(e, y);
      }
    }
  }
}

static int check_cache(const tq_kv8_cache* c) {
  if (c == nullptr || c->pages < 0 || c->kv_heads <= 0) return TQ_ERR_ARG;
  if (c->head_dim != 64 && c->head_dim != 128) return TQ_ERR_ARG;
  if (c->block < 16 || c->block > 1024 || (c->block & (c->block - 1)) != 0) return TQ_ERR_ARG;
  if ((int64_t)c->pages * c->block >= (1LL << 31)) return TQ_ERR_ARG;   // slots are 32-bit
  if (c->pages == 0) return TQ_OK;
  if (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales) return TQ_ERR_ARG;
  if (!aligned16(c->k_codes) || !aligned16(c->v_codes)) return TQ_ERR_ALIGN;
  return TQ_OK;
}

// Waves of window 1 end at once unless their token begins a unit, 15 of 16 in a prompt; wide windows make a wave of a
// decoding step append unit after unit, 2 us each.  So: 2048 to 4096 waves, as far as a window of 16 goes.  Measured in
// us at 8 kv heads of 128, windows 1 / 2 / 4 / 8 / 16:
//   64 requests of one token     4.2   6.1  10.0  17.9  33.1   (rule: 1)
//   512 requests of one token   11.7  11.2  12.8  18.8  34.2   (2)
//   a prompt of 512              6.8   4.7   5.3   5.4   5.3   (2)
//   512 requests of 4 tokens    27.8  20.9  20.3  20.6  24.1   (8)
//   4 prompts of 2048           60.0  33.4  22.0  17.4  14.2   (16)
static int append_window(int tokens, int kv_heads) {
  const int64_t rows = (int64_t)tokens * kv_heads;
  int window = 1;
  while (window < 16 && rows > 2048 * (int64_t)window) window *= 2;
  return window;
}

static int log2_exact(int x) { return 31 - __builtin_clz((unsigned)x); }

}  // namespace tq

using namespace tq;

extern "C" int tq_block_tables_step(const int32_t* new_tokens, const uint8_t* finished, int32_t* table,
                                    int64_t table_stride, int32_t* lengths, int32_t* free_list, int free_capacity,
                                    int32_t* free_count, int32_t* slots, int32_t* positions, int32_t* query_start,
                                    uint8_t* granted, int rows, int width, int block, int max_tokens, void* stream) {
  if (rows < 0 || width < 0 || block <= 0 || max_tokens < 0 || free_capacity < 0) return TQ_ERR_ARG;
  if ((int64_t)width * block >= (1LL << 31) || (int64_t)free_capacity * block >= (1LL << 31)) return TQ_ERR_ARG;
  if (rows > 0 && (!new_tokens || !lengths || !granted || table_stride < width || (width > 0 && !table)))
    return TQ_ERR_ARG;
  if (!free_count || !query_start || (free_capacity > 0 && !free_list)) return TQ_ERR_ARG;
  if (max_tokens > 0 && (!slots || !positions)) return TQ_ERR_ARG;
  const TablesArgs a{new_tokens, finished, table, table_stride, lengths, free_list, free_capacity, free_count,
                     slots, positions, query_start, granted, rows, width, block, max_tokens};
  hipStream_t s = static_cast<hipStream_t>(stream);
  // up to 4096 tokens one workgroup writes the slots too; above, a launch over all CUs does
  const bool one = max_tokens <= 4096;
  if (one && rows <= 64 && max_tokens <= 64)
    hipLaunchKernelGGL((tables_step_kernel<64, true>), dim3(1), dim3(64), 0, s, a);
  else if (one)
    hipLaunchKernelGGL((tables_step_kernel<kTabThreads, true>), dim3(1), dim3(kTabThreads), 0, s, a);
  else {
    hipLaunchKernelGGL((tables_step_kernel<kTabThreads, false>), dim3(1), dim3(kTabThreads), 0, s, a);
    hipLaunchKernelGGL(tables_slots_kernel, dim3((max_tokens + kSlotThreads - 1) / kSlotThreads), dim3(kSlotThreads),
                       0, s, a);
  }
  return (int)hipGetLastError();
}

extern "C" int tq_kv8_append(const tq_kv8_cache* cache, const void* k, int64_t k_stride_t, int64_t k_stride_h,
                             const void* v, int64_t v_stride_t, int64_t v_stride_h, int dtype, const int32_t* slots,
                             int tokens, void* stream) {
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_FP16) return TQ_ERR_DTYPE;
  const int rc = check_cache(cache);
  if (rc != TQ_OK) return rc;
  if (tokens < 0) return TQ_ERR_ARG;
  if (tokens == 0 || cache->pages == 0) return TQ_OK;
  if (!k || !v || !slots) return TQ_ERR_ARG;
  if (!aligned16(k) || !aligned16(v) || (k_stride_t % 8) || (k_stride_h % 8) || (v_stride_t % 8) || (v_stride_h % 8))
    return TQ_ERR_ALIGN;
  if (cache->kv_heads > 65535) return TQ_ERR_ARG;
  const int units = cache->block / 16;
  const int window = append_window(tokens, cache->kv_heads);
  const AppendArgs a{{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v)},
                     {k_stride_t, v_stride_t}, {k_stride_h, v_stride_h}, slots,
                     {cache->k_codes, cache->v_codes}, {cache->k_scales, cache->v_scales},
                     tokens, window, cache->kv_heads, units, log2_exact(units), (int64_t)cache->pages * cache->block};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 g((tokens + 4 * window - 1) / (4 * window), cache->kv_heads, 2);
  const bool bf = dtype == TQ_DTYPE_BF16;
  if (cache->head_dim == 128) {
    if (bf) hipLaunchKernelGGL((kv8_append_kernel<Bf16, 128>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv8_append_kernel<Fp16, 128>), g, dim3(256), 0, s, a);
  } else {
    if (bf) hipLaunchKernelGGL((kv8_append_kernel<Bf16, 64>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv8_append_kernel<Fp16, 64>), g, dim3(256), 0, s, a);
  }
  return (int)hipGetLastError();
}

extern "C" int tq_kv8_read(const tq_kv8_cache* cache, const int32_t* slots, int n, int dtype, void* k_out,
                           int64_t k_stride_n, int64_t k_stride_h, void* v_out, int64_t v_stride_n,
                           int64_t v_stride_h, void* stream) {
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_FP16) return TQ_ERR_DTYPE;
  const int rc = check_cache(cache);
  if (rc != TQ_OK) return rc;
  if (n < 0 || cache->kv_heads > 65535) return TQ_ERR_ARG;
  if (n == 0) return TQ_OK;
  if (!slots || !k_out || !v_out) return TQ_ERR_ARG;
  if (!aligned16(k_out) || !aligned16(v_out) || (k_stride_n % 8) || (k_stride_h % 8) || (v_stride_n % 8) ||
      (v_stride_h % 8))
    return TQ_ERR_ALIGN;
  const int units = cache->block / 16;
  const ReadArgs a{slots, {cache->k_codes, cache->v_codes}, {cache->k_scales, cache->v_scales},
                   {static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out)}, {k_stride_n, v_stride_n},
                   {k_stride_h, v_stride_h}, n, cache->kv_heads, units, log2_exact(units),
                   (int64_t)cache->pages * cache->block};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 g((n + 63) / 64, cache->kv_heads, 2);
  const bool bf = dtype == TQ_DTYPE_BF16;
  if (cache->head_dim == 128) {
    if (bf) hipLaunchKernelGGL((kv8_read_kernel<Bf16, 128>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv8_read_kernel<Fp16, 128>), g, dim3(256), 0, s, a);
  } else {
    if (bf) hipLaunchKernelGGL((kv8_read_kernel<Bf16, 64>), g, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv8_read_kernel<Fp16, 64>), g, dim3(256), 0, s, a);
  }
  return (int)hipGetLastError();
}

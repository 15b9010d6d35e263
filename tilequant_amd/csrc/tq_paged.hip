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
// a binary search in the chunk's prefix sums in LDS.
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

// Last index i in [0, n) with start[i] <= x (start ascending, start[0] <= x).
__device__ inline int last_at_most(const int64_t* start, int n, int64_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
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
        held = min((int)(((int64_t)max(a.lengths[b], 0) + a.block - 1) / a.block), a.width);
      const Pair64 inc = scan_inclusive<NT>(Pair64{held, 0}, wave_sums);
      start_pages[t] = inc.a - held;
      if (t == NT - 1) total = inc;
      __syncthreads();
      const int64_t n = total.a;
      for (int64_t i = t; i < n; i += NT) {
        const int r = last_at_most(start_pages, NT, i);
        int32_t* entry = a.table + (int64_t)(r0 + r) * a.ld + (i - start_pages[r]);
        const int64_t at = count0 + pushed + i;
        if (at < a.free_cap) a.free_list[at] = *entry;
        *entry = -1;
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
      have = (len + a.block - 1) / a.block;
      need = fits ? (len + n + a.block - 1) / a.block - have : 0;
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
    for (int64_t i = t; i < chunk.a; i += NT) {
      const int r = last_at_most(start_pages, NT, i);
      a.table[(int64_t)(r0 + r) * a.ld + row_have[r] + (i - start_pages[r])] = a.free_list[count - 1 - taken.a - i];
    }
    if constexpr (TOKENS) {
      for (int64_t i = t; i < chunk.b; i += NT) {
        const int r = last_at_most(start_tokens, NT, i);
        const int64_t pos = row_len[r] + (i - start_tokens[r]);
        const int page_at = (int)(pos / a.block);
        const int32_t page = page_at < row_have[r]
                                 ? a.table[(int64_t)(r0 + r) * a.ld + page_at]
                                 : a.free_list[count - 1 - taken.a - (start_pages[r] + page_at - row_have[r])];
        a.slots[taken.b + i] = page < 0 ? -1 : slot_of(page, a.block, (int)(pos - (int64_t)page_at * a.block));
        a.positions[taken.b + i] = (int32_t)pos;
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
// One wave per (token, head, K or V); the wave of a unit's first new token takes the whole unit, the others end at once
// (they cost less than a list of units would).  The bound is memory: 16-bit rows in, codes out.
struct AppendArgs {
  const uint16_t* x[2];
  int64_t x_st[2], x_sh[2];
  const int32_t* slots;
  int8_t* codes[2];
  float* scales[2];
  int tokens, kv_heads, units;   // units per page
  int unit_shift;                // log2(units)
  int64_t n_slots;
};

constexpr float kTinyAbsmax = 7.888609052210118e-31f;   // 2^-100

// NaN -> 0, infinities -> the largest finite value
template <class XT>
__device__ inline float finite(float x) {
  constexpr float top = std::is_same<XT, Bf16>::value ? 3.3895313892515355e38f : 65504.0f;
  return x != x ? 0.0f : fminf(fmaxf(x, -top), top);
}

__device__ inline uint32_t code_byte(float v) {   // rint and clamp to a signed byte
  return (uint32_t)(int)__builtin_amdgcn_fmed3f(__builtin_rintf(v), -127.0f, 127.0f) & 0xffu;
}
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

template <class XT, int D>
__global__ void __launch_bounds__(256)
kv8_append_kernel(AppendArgs a) {
  __shared__ int src_all[4][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x * 4 + wave;
  const int h = blockIdx.y, kv = blockIdx.z;
  if (t >= a.tokens) return;
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.n_slots) return;
  const int64_t unit = slot >> 4;   // over all pages
  if (t > 0) {
    const int64_t prev = a.slots[t - 1];
    if (prev >= 0 && (prev >> 4) == unit) return;   // not the unit's first new token
  }
  // the run of tokens of this unit: each offset's source is the last token that names it
  int* src_of = src_all[wave];
  if (lane < 16) src_of[lane] = -1;
  __builtin_amdgcn_wave_barrier();
  for (int t0 = t; t0 < a.tokens; t0 += kWave) {
    const int tt = t0 + lane;
    const int64_t sl = tt < a.tokens ? (int64_t)a.slots[tt] : -1;
    const uint64_t in = __ballot(sl >= 0 && (sl >> 4) == unit);
    const int n = in == ~0ull ? kWave : __builtin_ctzll(~in);
    if (lane < n) atomicMax(&src_of[sl & 15], tt);
    if (n < kWave) break;
  }
  __builtin_amdgcn_s_waitcnt(0xC07F);   // LDS operations of this wave
  asm volatile("" ::: "memory");
  int src[16];
  int begun = 16;   // the unit held tokens 0 .. begun - 1 before
#pragma unroll
  for (int o = 15; o >= 0; --o) {
    src[o] = __builtin_amdgcn_readfirstlane(src_of[o]);
    if (src[o] >= 0) begun = o;
  }
  const int64_t page = unit >> a.unit_shift;
  const int64_t cell = (page * a.kv_heads + h) * a.units + (unit & (a.units - 1));   // (page, head, unit)
  float* scale_at = a.scales[kv] + cell;
  int8_t* codes = a.codes[kv] + cell * (16 * D);
  const float old = begun > 0 ? *scale_at : 0.0f;
  const uint16_t* x = a.x[kv] + (int64_t)h * a.x_sh[kv];

  if (kv == 0) {
    // lane: 8 dimensions of every kRows-th token
    constexpr int kLanes = D / 8, kRows = kWave / kLanes, kSteps = 16 / kRows;
    const int ch = lane % kLanes, rg = lane / kLanes;
    u32x4 v[kSteps];
    u32x2 oc[kSteps];
    int sr[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int o = rg + kRows * i;
      sr[i] = src_of[o];
      v[i] = u32x4{0, 0, 0, 0};
      oc[i] = u32x2{0, 0};
      if (sr[i] >= 0) v[i] = *reinterpret_cast<const u32x4*>(x + (int64_t)sr[i] * a.x_st[0] + ch * 8);
      else if (o < begun) oc[i] = *reinterpret_cast<const u32x2*>(codes + o * D + ch * 8);
    }
    float f[kSteps][8], m = 0.0f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[i][e] = finite<XT>(XT::to_f32((uint16_t)(v[i][e >> 1] >> (16 * (e & 1)))));
        m = fmaxf(m, fabsf(f[i][e]));
      }
    const UnitScale u(wave_max_nonneg(m), old);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int o = rg + kRows * i;
      u32x2 w{0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[e >> 2] |= code_byte(sr[i] >= 0 ? f[i][e] * u.inv : byte_code(oc[i][e >> 2], e & 3) * u.shrink) << (8 * (e & 3));
      if (sr[i] >= 0 || (o < begun && u.grew)) *reinterpret_cast<u32x2*>(codes + o * D + ch * 8) = w;
    }
    if (lane == 0) *scale_at = u.s;
  } else {
    // lane: all 16 tokens of kDims dimensions (a unit's row of 16 bytes each)
    constexpr int kDims = D / kWave;
    u32x4 oc[kDims];
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      oc[d] = u32x4{0, 0, 0, 0};
      if (begun > 0 || src[15] < 0) oc[d] = *reinterpret_cast<const u32x4*>(codes + (lane * kDims + d) * 16);
    }
    uint32_t v[16];
#pragma unroll
    for (int o = 0; o < 16; ++o) {
      v[o] = 0;
      if (src[o] >= 0) {
        const uint16_t* p = x + (int64_t)src[o] * a.x_st[1] + lane * kDims;
        if constexpr (kDims == 2) v[o] = *reinterpret_cast<const uint32_t*>(p);
        else v[o] = *p;
      }
    }
    float f[16][kDims], m = 0.0f;
#pragma unroll
    for (int o = 0; o < 16; ++o)
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        f[o][d] = finite<XT>(XT::to_f32((uint16_t)(v[o] >> (16 * d))));
        m = fmaxf(m, fabsf(f[o][d]));
      }
    const UnitScale u(wave_max_nonneg(m), old);
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      u32x4 w = oc[d];
#pragma unroll
      for (int o = 0; o < 16; ++o) {
        const int sh = 8 * (o & 3);
        const bool now = src[o] >= 0;
        if (now || (o < begun && u.grew)) {
          const uint32_t c = code_byte(now ? f[o][d] * u.inv : byte_code(oc[d][o >> 2], o & 3) * u.shrink);
          w[o >> 2] = (w[o >> 2] & ~(0xffu << sh)) | (c << sh);
        }
      }
      *reinterpret_cast<u32x4*>(codes + (lane * kDims + d) * 16) = w;
    }
    if (lane == 0) *scale_at = u.s;
  }
}

// ---- read ----------------------------------------------------------------------
//
// code * scale, rounded once, of the listed slots (slots outside the cache: zeros).  One wave per 16 list entries,
// head and K or V.  Keys are copied row by row; values, stored transposed, unit by unit: the wave takes the unit of its
// first entry not yet written, and with it every entry of that unit (a list in token order has one or two units).
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
  const AppendArgs a{{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v)},
                     {k_stride_t, v_stride_t}, {k_stride_h, v_stride_h}, slots,
                     {cache->k_codes, cache->v_codes}, {cache->k_scales, cache->v_scales},
                     tokens, cache->kv_heads, units, log2_exact(units), (int64_t)cache->pages * cache->block};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 g((tokens + 3) / 4, cache->kv_heads, 2);
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

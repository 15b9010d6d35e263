// tq_paged_attention.hip -- attention over the paged INT8 KV cache (tq_kv8_cache), gfx950.
//
// Sequence b holds len = lengths[b] tokens in the pages of table row b; its n queries are its last n tokens (query i
// sits at position len - n + i and sees the keys up to there).  With G = q_heads / kv_heads, s_u / t_u the fp32 scales
// of a 16-token unit's keys / values and c, d their codes:
//   out[i, h] = sum_j p_j t_u(j) d_j / sum_j p_j,   p_j = exp(scale s_u(j) q . c_j - max),   j <= len - n + i.
//
// Both products run on v_mfma_f32_16x16x32_f16 with codes widened to fp16, which holds them exactly:
//   K: a code byte + 128 zero-extended to 16 bits IS the fp16 subnormal (code + 128) 2^-24, and the matrix core takes
//      subnormals as they are: one v_perm for two codes.  The 128 sum(q) it adds goes in as the accumulator's initial
//      value; it is of the size of the result itself, so the fp32 sums lose nothing to it.
//   V: 0x6400 | byte is 1024 + byte; a packed fp16 subtraction of 1152 gives the code.  (The bias is not folded here:
//      summed over a long sequence it would outgrow the result.)
//   q: each row is divided by the power of two of its absmax (exact), so that bf16's range fits fp16; elements under
//      2^-25 of the row's largest are rounded to that step.
//   P: p_j t_u(j) / 2^M with M the running maximum over log2(p_j t_u(j)), so it is in [0, 1] whatever the values' scale:
//      rounding it to fp16 (2^-12 relative) is the one rounding between the inputs and the fp32 result.  The softmax sum
//      adds the unrounded numbers over t_u.  A unit whose values are all zero (t_u = 0) enters the sum with
//      t_u = 2^-8 in its place, which its codes of 0 do not feel.
// Operand layout: S^T = K Q^T with keys as A rows, so that a lane holds the scores of one query row (column lane % 16)
// for all 16 keys of one unit (lane / 16): one key scale, one value scale per lane, and the scores are P's operand of
// O^T = V^T P^T as they stand.  For that, row r = 4 u + v of the A block m holds key 16 u + 4 m + v of the 64-key tile.
#include "tq_common.h"

#include <float.h>

namespace tq {

constexpr float kLog2e8 = 1.4426950408889634f;
constexpr int kKv8Tile = 64;    // keys per tile: four units
constexpr int kKv8Rows = 16;    // query rows (token, head of the group) of a decode workgroup

struct Kv8Args {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const int8_t* k;
  const int8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* table;
  int64_t ld;
  const int32_t* lengths;
  const int32_t* query_start;   // nullptr: one query per sequence
  uint16_t* out;
  int64_t o_st, o_sh;
  float* part;                  // [tokens * q_heads][n_splits][D + 2]: o, M, l
  int tokens, batch, q_heads, kv_heads, G, max_query;
  int pages, unit_shift, units;
  int len_cap;                  // the most tokens a sequence counts as having: the table's width, the caller's bound
  int n_splits, chunk;          // keys per split, a multiple of 64
  int zero_rest;                // rows of no answered query are written 0
  int64_t head_bytes;           // bytes of one (page, head): units * 16 * D
  float scale_log2, scale_sign; // |scale| log2(e), its sign
};

// The rows of one sequence, clamped into the query array whatever the device arrays say.
struct Kv8Seq {
  int len, n, first;   // cached tokens, queries to answer, index of the first query
  int before;          // tokens before the first query: query i sees keys 0 .. before + i
};
__device__ inline Kv8Seq kv8_seq(const Kv8Args& a, int b) {
  Kv8Seq s;
  s.len = min(max(a.lengths[b], 0), a.len_cap);
  s.first = b;
  int n = 1;
  if (a.query_start != nullptr) {
    s.first = min(max(a.query_start[b], 0), a.tokens);
    n = min(max(a.query_start[b + 1], s.first), a.tokens) - s.first;
  }
  s.before = s.len - n;
  s.n = min(n, a.max_query);
  return s;
}

// The rows of one kv head that no answered query of sequence b takes (past max_query of it), and a share of those before
// the first and behind the last sequence, written 0 by part `part` of `parts` of this sequence's workgroups.  (Filling
// the whole output before took 7 of 138 us for 4 prompts of up to 2048 tokens, and a launch.)
template <int D>
__device__ inline void kv8_zero_rest(const Kv8Args& a, int b, int h, const Kv8Seq& sq, int part, int parts) {
  const auto zero = [&](int64_t t0, int t1, int64_t step) {
    for (int64_t t = t0; t < t1; t += step)
      for (int i = threadIdx.x; i < a.G * (D / 8); i += blockDim.x)
        *reinterpret_cast<u32x4*>(a.out + t * a.o_st + (int64_t)(h * a.G + i / (D / 8)) * a.o_sh + i % (D / 8) * 8) =
            u32x4{0, 0, 0, 0};
  };
  const int first = min(max(a.query_start[0], 0), a.tokens), last = min(max(a.query_start[a.batch], 0), a.tokens);
  const int next = min(max(a.query_start[b + 1], sq.first), a.tokens);
  const int64_t share = (int64_t)b * parts + part, shares = (int64_t)a.batch * parts;
  zero((int64_t)sq.first + sq.n + part, next, parts);
  zero(share, first, shares);
  zero(last + share, a.tokens, shares);
}

__device__ inline float g4_sum(float x) {   // over lanes l, l ^ 16, l ^ 32, l ^ 48; the same association in every lane
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  unsigned b = __float_as_uint(x);
  u2 r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  b = __float_as_uint(x);
  r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ inline float g4_max(float x) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  unsigned b = __float_as_uint(x);
  u2 r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  b = __float_as_uint(x);
  r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 8 codes (two dwords) -> an fp16 operand of subnormals (code + 128) 2^-24
__device__ inline v4i widen_k(uint32_t lo, uint32_t hi) {
  lo ^= 0x80808080u;
  hi ^= 0x80808080u;
  v4i r;
  r[0] = (int)__builtin_amdgcn_perm(0u, lo, 0x0c010c00u);
  r[1] = (int)__builtin_amdgcn_perm(0u, lo, 0x0c030c02u);
  r[2] = (int)__builtin_amdgcn_perm(0u, hi, 0x0c010c00u);
  r[3] = (int)__builtin_amdgcn_perm(0u, hi, 0x0c030c02u);
  return r;
}
// 8 codes -> their values in fp16
__device__ inline v4i widen_v(uint32_t lo, uint32_t hi) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  lo ^= 0x80808080u;
  hi ^= 0x80808080u;
  const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
  v4i r;
  r[0] = __builtin_bit_cast(int, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) - off);
  r[1] = __builtin_bit_cast(int, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) - off);
  r[2] = __builtin_bit_cast(int, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) - off);
  r[3] = __builtin_bit_cast(int, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) - off);
  return r;
}

__device__ inline uint32_t pack_h2(float a, float b) {   // round to nearest even
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), h2));
}

// One query row as B operands: lane (column c, group g) holds dimensions 64 hf + 16 g .. + 15 of its row (operand 2 hf:
// the first 8 of them, 2 hf + 1: the others; a K operand of the same index holds the same dimensions).  `factor`
// turns a product with key codes into a log2 score before the key scale; `bias` cancels the codes' 128.
template <class XT, int D>
struct QueryRow {
  v4i op[D / 32];
  float factor, bias;
  __device__ void load(const uint16_t* row, bool live, const Kv8Args& a, int g) {
    u32x4 w[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      w[i] = u32x4{0, 0, 0, 0};
      if (live) w[i] = *reinterpret_cast<const u32x4*>(row + 64 * (i >> 1) + 16 * g + 8 * (i & 1));
    }
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) m = max8<XT>(w[i], m);
    m = g4_max(m);
    const int e = min(max((int)((__float_as_uint(m) >> 23) & 255u) - 127, -126), 126);   // 2^e <= m < 2^(e + 1)
    const float down = __uint_as_float((uint32_t)(127 - e) << 23) * a.scale_sign;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t h = pack_h2(XT::to_f32((uint16_t)(w[i][p] & 0xffffu)) * down,
                                   XT::to_f32((uint16_t)(w[i][p] >> 16)) * down);
        op[i][p] = (int)h;
        sum += Fp16::to_f32((uint16_t)(h & 0xffffu)) + Fp16::to_f32((uint16_t)(h >> 16));
      }
    bias = g4_sum(sum) * (-128.0f * 5.9604644775390625e-08f);   // -128 * 2^-24
    factor = __uint_as_float((uint32_t)(127 + e) << 23) * 16777216.0f * a.scale_log2;
  }
};

// The table's entry for a unit below the key limit (-1 beyond), and whether it is a page of the cache; page 0 stands in.
__device__ inline int32_t kv8_entry(const Kv8Args& a, const int32_t* row, int unit, int limit) {
  return unit * 16 < limit ? row[unit >> a.unit_shift] : -1;
}
__device__ inline int64_t kv8_page(const Kv8Args& a, int32_t entry, bool* ok) {
  *ok = (uint32_t)entry < (uint32_t)a.pages;
  return *ok ? entry : 0;
}

// Running softmax of one query row per lane column: M, the sum (of this lane's units), and what each tile does to them.
struct Softmax {
  float M, l;
};

// A value scale as the softmax takes it: log2 and reciprocal of what P is multiplied with.
struct ValueScale {
  float log, inv;
  __device__ inline explicit ValueScale(float vs) {
    const float t = vs > 0.0f ? vs : 0.00390625f;
    log = __builtin_amdgcn_logf(t);
    inv = __builtin_amdgcn_rcpf(t);
  }
};

// The tile's probabilities as the P operands, from the raw products; returns the factor of what was summed before.
// live: the lane's unit counts; MASK: of its 16 keys (the lane's key index is 4 m + v) the row sees the first nv.
template <bool MASK>
__device__ __forceinline__ float softmax_tile(v4f (&s)[4], bool live, int nv, float f, const ValueScale& vs, Softmax& sm,
                                              v4i (&p)[2]) {
  if constexpr (MASK) {
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int v = 0; v < 4; ++v) s[m][v] = 4 * m + v < nv ? s[m][v] : -3.0e38f;
    live = live && nv > 0;
  }
  // three at a time: 8 instructions, where a tree of pairs makes 20, each of whose leaves is first made canonical
  float top = s[0][0];
#pragma unroll
  for (int j = 1; j < 15; j += 2) top = fmaxf(fmaxf(top, s[j >> 2][j & 3]), s[(j + 1) >> 2][(j + 1) & 3]);
  top = fmaxf(fmaxf(top, s[3][3]), -FLT_MAX);
  const float mine = live ? fmaf(top, f, vs.log) : -INFINITY;
  const float M = fmaxf(sm.M, g4_max(mine));
  const float ref = M == -INFINITY ? 0.0f : M;
  const float c = live ? vs.log - ref : -INFINITY;   // f is 0 where the unit does not count: the exponentials are 0
  float sum = 0.0f;
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    float e[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      e[v] = __builtin_amdgcn_exp2f(fmaf(s[m][v], f, c));
      if constexpr (MASK) e[v] = 4 * m + v < nv ? e[v] : 0.0f;
      sum += e[v];
    }
    p[m >> 1][2 * (m & 1)] = (int)pack_h2(e[0], e[1]);
    p[m >> 1][2 * (m & 1) + 1] = (int)pack_h2(e[2], e[3]);
  }
  const float alpha = __builtin_amdgcn_exp2f(sm.M - ref);
  sm.M = M;
  sm.l = fmaf(sm.l, alpha, sum * vs.inv);
  return alpha;
}

// ---- few query rows: split over the keys ------------------------------------------
//
// Workgroup (split, sequence x kv head, row tile): NW waves take the split's 64-key tiles in turn, each with a running
// softmax of its own over 16 query rows; a tile's codes go straight from memory to the wave that multiplies them (K: 8,
// V: 8 16-byte loads per lane at D = 128).  The waves' results are joined through LDS in wave order.
// The bound is memory: 4 sequences of 131072 tokens, 8 kv heads of 128, 1.08 GB: 188 us, 5.7 TB/s.
template <class XT, int D, int NW>
__global__ void __launch_bounds__(NW * kWave)
kv8_split_kernel(Kv8Args a) {
  constexpr int HF = D / 64;    // 64-dimension halves of a key row
  constexpr int DB = D / 16;    // 16-dimension blocks of the output
  __shared__ __align__(16) float wo[NW][kKv8Rows][D + 4];
  __shared__ float wm[NW][kKv8Rows], wl[NW][kKv8Rows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int split = blockIdx.x;
  const int b = blockIdx.y / a.kv_heads, h = blockIdx.y - b * a.kv_heads;
  const Kv8Seq sq = kv8_seq(a, b);
  const int rows = sq.n * a.G, r0 = blockIdx.z * kKv8Rows;
  if (a.zero_rest && split == 0) kv8_zero_rest<D>(a, b, h, sq, blockIdx.z, gridDim.z);
  if (r0 >= rows) return;
  const int last_i = min(sq.n - 1, (r0 + kKv8Rows - 1) / a.G);
  const int hi = sq.before + last_i + 1;   // keys seen by the tile's last row (may be <= 0)
  const int key0 = split * a.chunk, key1 = min(key0 + a.chunk, hi);
  if (split > 0 && key0 >= hi) return;   // the merge does not read this record
  const int r = r0 + c;
  const bool live = r < rows;
  const int qi = live ? r / a.G : 0, qh = live ? h * a.G + (r - qi * a.G) : 0;
  const int seen = live ? sq.before + qi + 1 : key1;   // keys this lane's row sees (rows past the last: any)

  QueryRow<XT, D> qr;
  qr.load(a.q + (int64_t)(sq.first + qi) * a.q_st + (int64_t)qh * a.q_sh, live, a, g);

  const int32_t* row = a.table + (int64_t)b * a.ld;
  v4f o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = v4f{0.f, 0.f, 0.f, 0.f};
  Softmax sm{-INFINITY, 0.0f};

  // a tile's table entries are loaded a tile ahead: the codes' loads wait for nothing else
  int base = key0 + wave * kKv8Tile;
  int32_t ek = kv8_entry(a, row, (base >> 4) + (c >> 2), key1), ev = kv8_entry(a, row, (base >> 4) + g, key1);
  for (; base < key1; base += NW * kKv8Tile) {
    // units: of the key this lane loads as an A row, and of the keys whose scores it holds (and whose values it loads)
    const int uk = (base >> 4) + (c >> 2), uv = (base >> 4) + g;
    bool okk, okv;
    const int64_t pk = kv8_page(a, ek, &okk), pv = kv8_page(a, ev, &okv);
    const int8_t* kp = a.k + (pk * a.kv_heads + h) * a.head_bytes + (uk & (a.units - 1)) * (16 * D) + (c & 3) * D + g * 16;
    const int8_t* vp = a.v + (pv * a.kv_heads + h) * a.head_bytes + (uv & (a.units - 1)) * (16 * D) + c * 16;
    u32x4 kw[4][HF], vw[DB];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int f = 0; f < HF; ++f) kw[m][f] = *reinterpret_cast<const u32x4*>(kp + 4 * m * D + 64 * f);
    const int64_t cell = (pv * a.kv_heads + h) * a.units + (uv & (a.units - 1));
    float ks = a.ks[cell], vs = a.vs[cell];
#pragma unroll
    for (int d = 0; d < DB; ++d) vw[d] = *reinterpret_cast<const u32x4*>(vp + d * 256);
    ek = kv8_entry(a, row, uk + NW * (kKv8Tile / 16), key1);
    ev = kv8_entry(a, row, uv + NW * (kKv8Tile / 16), key1);
    const int nv = okv ? min(max(min(seen, key1) - uv * 16, 0), 16) : 0;
    if (nv == 0) ks = 0.0f, vs = 1.0f;   // whatever the scales of a page that is not there are
    const bool whole = __all(nv == 16 || nv == 0);

    v4f s[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      s[m] = v4f{qr.bias, qr.bias, qr.bias, qr.bias};
#pragma unroll
      for (int f = 0; f < HF; ++f) {
        s[m] = mfma16<Fp16>(widen_k(kw[m][f][0], kw[m][f][1]), qr.op[2 * f], s[m]);
        s[m] = mfma16<Fp16>(widen_k(kw[m][f][2], kw[m][f][3]), qr.op[2 * f + 1], s[m]);
      }
    }
    v4i p[2];
    const float before = sm.M;
    const ValueScale vsc(vs);
    const float alpha = whole ? softmax_tile<false>(s, nv > 0, nv, qr.factor * ks, vsc, sm, p)
                              : softmax_tile<true>(s, nv > 0, nv, qr.factor * ks, vsc, sm, p);
    if (__any(sm.M != before)) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 4; ++v) o[d][v] *= alpha;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      o[d] = mfma16<Fp16>(widen_v(vw[d][0], vw[d][1]), p[0], o[d]);
      o[d] = mfma16<Fp16>(widen_v(vw[d][2], vw[d][3]), p[1], o[d]);
    }
  }

  // ---- join the waves
  const float l = g4_sum(sm.l);
  if (g == 0) {
    wm[wave][c] = sm.M;
    wl[wave][c] = l;
  }
#pragma unroll
  for (int d = 0; d < DB; ++d) *reinterpret_cast<v4f*>(&wo[wave][c][16 * d + 4 * g]) = o[d];
  __syncthreads();
  for (int e = threadIdx.x; e < kKv8Rows * D; e += NW * kWave) {
    const int rr = e / D, d = e - rr * D;
    if (r0 + rr >= rows) break;
    float M = wm[0][rr];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, wm[w][rr]);
    const float ref = M == -INFINITY ? 0.0f : M;
    float O = 0.0f, L = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {   // weight 0 for a wave without a key; the NaN of a row that has one stays
      const float f = __builtin_amdgcn_exp2f(wm[w][rr] - ref);
      O = fmaf(f, wo[w][rr][d], O);
      L = fmaf(f, wl[w][rr], L);
    }
    const int i = (r0 + rr) / a.G, hh = h * a.G + (r0 + rr - i * a.G);
    const int64_t tok = sq.first + i;
    if (a.n_splits == 1) {
      a.out[tok * a.o_st + (int64_t)hh * a.o_sh + d] = XT::from_f32(L != 0.0f ? O / L : 0.0f);
    } else {
      float* rec = a.part + ((tok * a.q_heads + hh) * a.n_splits + split) * (D + 2);
      rec[d] = O;
      if (d == 0) {
        rec[D] = M;
        rec[D + 1] = L;
      }
    }
  }
}

// ---- many query rows: tiles of 128 rows ---------------------------------------------
//
// Workgroup (sequence x kv head, row tile, split): four waves of 32 query rows each over 64-key tiles.  The four waves
// widen a tile's codes once, a quarter each, into LDS in operand order (1 KiB per operand, lane after lane: no bank
// conflicts either way), two tiles deep, and every wave multiplies its rows with all of them.
// The bound is instruction issue, two waves a SIMD: matrix instructions take 30% of the SIMDs' cycles, the vector
// instructions (per tile and wave 170 of softmax, 32 of them exponentials, and 85 of widening) 52%.  4 prompts of 1500 to
// 2048 tokens, 24 / 8 heads of 128: 131 us, 0.64 PFLOP/s of what the mask leaves; 512 tokens over 16384: 0.75; a large
// fp16 product reaches 1.19.  48 rows a wave, or the next tile's scores beside this tile's softmax, spill (203 us and more);
// 32 x 32 x 16 products, half as many, took 146.
constexpr int kKv8Block = 128;   // rows per workgroup
constexpr int kKv8Waves = 4;

template <class XT, int D>
__global__ void __launch_bounds__(kKv8Waves * kWave, 2)
kv8_block_kernel(Kv8Args a) {
  constexpr int HF = D / 64, DB = D / 16, KS = D / 32;
  constexpr int KO = 4 * KS;       // K operands of a tile
  constexpr int VO = 2 * DB;       // V operands
  extern __shared__ __align__(16) int8_t smem[];
  v4i* kl = reinterpret_cast<v4i*>(smem);               // [2][KO][64]
  v4i* vl = kl + 2 * KO * kWave;                        // [2][VO][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int b = blockIdx.x / a.kv_heads, h = blockIdx.x - b * a.kv_heads;
  const int split = blockIdx.z;
  const Kv8Seq sq = kv8_seq(a, b);
  const int rows = sq.n * a.G;
  if (a.zero_rest && split == 0) kv8_zero_rest<D>(a, b, h, sq, blockIdx.y, gridDim.y);
  // The last row tiles have the most keys: they go first, over all sequences and heads (4 prompts of up to 2048
  // tokens, 8 kv heads: 143 us when this was tried, 173 with all tiles of a head before the next head's).
  const int tiles = (rows + kKv8Block - 1) / kKv8Block;
  const int tile = tiles - 1 - (int)blockIdx.y;
  if (tile < 0) return;
  const int r0 = tile * kKv8Block;
  const int last_i = min(sq.n - 1, (r0 + kKv8Block - 1) / a.G);
  const int hi = sq.before + last_i + 1;
  const int key0 = split * a.chunk, key1 = min(key0 + a.chunk, hi);
  if (split > 0 && key0 >= hi) return;

  QueryRow<XT, D> qr[2];
  int seen[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = r0 + wave * 32 + 16 * x + c;
    const bool live = r < rows;
    const int qi = live ? r / a.G : 0, qh = live ? h * a.G + (r - qi * a.G) : 0;
    seen[x] = live ? min(sq.before + qi + 1, key1) : key1;   // rows past the last: any
    qr[x].load(a.q + (int64_t)(sq.first + qi) * a.q_st + (int64_t)qh * a.q_sh, live, a, g);
  }
  const int32_t* row = a.table + (int64_t)b * a.ld;
  v4f o[2][DB];
  Softmax sm[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    sm[x] = Softmax{-INFINITY, 0.0f};
#pragma unroll
    for (int d = 0; d < DB; ++d) o[x][d] = v4f{0.f, 0.f, 0.f, 0.f};
  }

  // this wave's quarter of a tile: key block m = wave, and DB / 4 blocks of the values; table entries a tile ahead
  constexpr int VD = DB / 4;
  u32x4 kw[HF], vw[VD];
  float ks, vs;
  bool there;   // the lane's unit lies in a page of the cache
  int32_t ek = kv8_entry(a, row, (key0 >> 4) + (c >> 2), key1), ev = kv8_entry(a, row, (key0 >> 4) + g, key1);
  const auto fetch = [&](int base) {
    const int uk = (base >> 4) + (c >> 2), uv = (base >> 4) + g;
    bool okk;
    const int64_t pk = kv8_page(a, ek, &okk), pv = kv8_page(a, ev, &there);
    const int8_t* kp = a.k + (pk * a.kv_heads + h) * a.head_bytes + (uk & (a.units - 1)) * (16 * D) +
                       (4 * wave + (c & 3)) * D + g * 16;
    const int8_t* vp = a.v + (pv * a.kv_heads + h) * a.head_bytes + (uv & (a.units - 1)) * (16 * D) +
                       (16 * VD * wave + c) * 16;
#pragma unroll
    for (int f = 0; f < HF; ++f) kw[f] = *reinterpret_cast<const u32x4*>(kp + 64 * f);
#pragma unroll
    for (int d = 0; d < VD; ++d) vw[d] = *reinterpret_cast<const u32x4*>(vp + d * 256);
    const int64_t cell = (pv * a.kv_heads + h) * a.units + (uv & (a.units - 1));
    ks = a.ks[cell];
    vs = a.vs[cell];
    ek = kv8_entry(a, row, uk + kKv8Tile / 16, key1);
    ev = kv8_entry(a, row, uv + kKv8Tile / 16, key1);
  };
  const auto stage = [&](int buf) {
#pragma unroll
    for (int f = 0; f < HF; ++f) {
      kl[(buf * KO + wave * KS + 2 * f) * kWave + lane] = widen_k(kw[f][0], kw[f][1]);
      kl[(buf * KO + wave * KS + 2 * f + 1) * kWave + lane] = widen_k(kw[f][2], kw[f][3]);
    }
#pragma unroll
    for (int d = 0; d < VD; ++d) {
      vl[(buf * VO + (VD * wave + d) * 2) * kWave + lane] = widen_v(vw[d][0], vw[d][1]);
      vl[(buf * VO + (VD * wave + d) * 2 + 1) * kWave + lane] = widen_v(vw[d][2], vw[d][3]);
    }
  };

  if (key0 < key1) {
    fetch(key0);
    stage(0);
    int buf = 0;
    // keys that every row of this wave sees
    const int all = min(key1, sq.before + min((r0 + wave * 32) / a.G, sq.n - 1) + 1);
    for (int base = key0; base < key1; base += kKv8Tile) {
      const int ub = base + 16 * g;
      const bool live = there && ub < key1;
      const float ksc = live ? ks : 0.0f;   // whatever the scales of a unit that is not there are
      const ValueScale vsc(live ? vs : 1.0f);
      __syncthreads();   // the tile is staged; nobody reads the other buffer any more
      const bool more = base + kKv8Tile < key1;
      if (more) fetch(base + kKv8Tile);
      // Operands are read once for both row blocks, a group ahead of the products that take them: the scheduling
      // barriers keep the compiler from moving the reads down to their use, where each product waits for LDS (512 tokens
      // over 16384, 24 / 8 heads: 137 us against 141).
      v4f s[2][4];
      v4i kk[2][KS];
#pragma unroll
      for (int i = 0; i < KS; ++i) kk[0][i] = kl[(buf * KO + i) * kWave + lane];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (m < 3) {
#pragma unroll
          for (int i = 0; i < KS; ++i) kk[(m + 1) & 1][i] = kl[(buf * KO + (m + 1) * KS + i) * kWave + lane];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 2; ++x) s[x][m] = v4f{qr[x].bias, qr[x].bias, qr[x].bias, qr[x].bias};
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) s[x][m] = mfma16<Fp16>(kk[m & 1][i], qr[x].op[i], s[x][m]);
      }
      v4i vv[2][4];   // of two dimension blocks; the first are read under the softmax
#pragma unroll
      for (int i = 0; i < 4; ++i) vv[0][i] = vl[(buf * VO + i) * kWave + lane];
      __builtin_amdgcn_sched_barrier(0);
      v4i p[2][2];
      float alpha[2];
      bool moved = false;
      const bool whole = base + kKv8Tile <= all;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float before = sm[x].M;
        if (whole)
          alpha[x] = softmax_tile<false>(s[x], live, 16, qr[x].factor * ksc, vsc, sm[x], p[x]);
        else
          alpha[x] = softmax_tile<true>(s[x], live, min(max(seen[x] - ub, 0), 16), qr[x].factor * ksc, vsc, sm[x], p[x]);
        moved |= sm[x].M != before;
      }
      if (__any(moved)) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int v = 0; v < 4; ++v) o[x][d][v] *= alpha[x];
      }
#pragma unroll
      for (int d = 0; d < DB; d += 2) {
        if (d + 2 < DB) {
#pragma unroll
          for (int i = 0; i < 4; ++i) vv[(d / 2 + 1) & 1][i] = vl[(buf * VO + 2 * (d + 2) + i) * kWave + lane];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 0; x < 2; ++x) o[x][d + e] = mfma16<Fp16>(vv[(d / 2) & 1][2 * e + k], p[x][k], o[x][d + e]);
      }
      buf ^= 1;
      if (more) stage(buf);
    }
  }

  // lane (c, g): dimensions 16 d + 4 g + v of its row
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float l = g4_sum(sm[x].l);
    const int r = r0 + wave * 32 + 16 * x + c;
    if (r >= rows) continue;
    const int i = r / a.G, hh = h * a.G + (r - i * a.G);
    const int64_t tok = sq.first + i;
    if (a.n_splits == 1) {
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      uint16_t* out = a.out + tok * a.o_st + (int64_t)hh * a.o_sh;
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        u32x2 w;
        w[0] = XT::pack2(o[x][d][0] * inv, o[x][d][1] * inv);
        w[1] = XT::pack2(o[x][d][2] * inv, o[x][d][3] * inv);
        *reinterpret_cast<u32x2*>(out + 16 * d + 4 * g) = w;
      }
    } else {
      float* rec = a.part + ((tok * a.q_heads + hh) * a.n_splits + split) * (D + 2);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        float2* at = reinterpret_cast<float2*>(rec + 16 * d + 4 * g);   // records are 8-byte aligned
        at[0] = float2{o[x][d][0], o[x][d][1]};
        at[1] = float2{o[x][d][2], o[x][d][3]};
      }
      if (g == 0) {
        rec[D] = sm[x].M;
        rec[D + 1] = l;
      }
    }
  }
}

// ---- joining the splits ----------------------------------------------------------
//
// One wave per (token, query head), splits in order, eight at a time so that their loads go out together: 4 us for 32
// tokens of 28 heads in up to 17 splits, about an empty launch.
template <class XT, int D>
__global__ void __launch_bounds__(256)
kv8_merge_kernel(Kv8Args a) {
  constexpr int PD = D / kWave;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= (int64_t)a.tokens * a.q_heads) return;
  const int tok = (int)(row / a.q_heads), h = (int)(row - (int64_t)tok * a.q_heads);
  int b = tok;
  if (a.query_start != nullptr) {   // the last sequence that starts at or before tok
    int lo = 0, hi = a.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.query_start[mid] <= tok) lo = mid;
      else hi = mid;
    }
    b = lo;
  }
  const Kv8Seq sq = kv8_seq(a, b);
  if (tok < sq.first || tok >= sq.first + sq.n) return;   // rows of no sequence are left as they are
  const int keys = sq.before + (tok - sq.first) + 1;
  const int n = keys > 0 ? min((keys + a.chunk - 1) / a.chunk, a.n_splits) : 0;
  const float* rec = a.part + row * a.n_splits * (D + 2);
  float M = -INFINITY, L = 0.0f, O[PD] = {};
  for (int s0 = 0; s0 < n; s0 += 8) {
    float m[8], l[8], o[8][PD];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float* at = rec + (int64_t)min(s0 + j, n - 1) * (D + 2);
      m[j] = s0 + j < n ? at[D] : -INFINITY;
      l[j] = at[D + 1];
#pragma unroll
      for (int d = 0; d < PD; ++d) o[j][d] = at[lane * PD + d];
    }
    float Mb = M;
#pragma unroll
    for (int j = 0; j < 8; ++j) Mb = fmaxf(Mb, m[j]);
    const float ref = Mb == -INFINITY ? 0.0f : Mb;
    const float r = __builtin_amdgcn_exp2f(M - ref);
    L *= r;
#pragma unroll
    for (int d = 0; d < PD; ++d) O[d] *= r;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float w = __builtin_amdgcn_exp2f(m[j] - ref);   // 0 for a record of no keys
      L = fmaf(w, l[j], L);
#pragma unroll
      for (int d = 0; d < PD; ++d) O[d] = fmaf(w, o[j][d], O[d]);
    }
    M = Mb;
  }
  const float inv = L != 0.0f ? 1.0f / L : 0.0f;
  uint16_t* out = a.out + (int64_t)tok * a.o_st + (int64_t)h * a.o_sh + lane * PD;
  if constexpr (PD == 2) *reinterpret_cast<uint32_t*>(out) = XT::pack2(O[0] * inv, O[1] * inv);
  else *out = XT::from_f32(O[0] * inv);
}

// ---- host ----------------------------------------------------------------------
struct Kv8Plan {
  bool block;       // the 128-row kernel
  int waves;        // of a split workgroup
  int row_tiles, n_splits, chunk;
};

// Split kernel: a workgroup's waves take 64 keys each in turn.  Up to kKv8Alone keys one workgroup of 8 waves takes a
// sequence's kv head whole, which needs no join (one sequence of 613 tokens, 8 kv heads: 8.3 us, against 6.2 + 2.7 us and
// a launch more in splits of 256).  Else 4 waves: one tile a wave while that makes at most kKv8Fine workgroups (32 ragged
// sequences of up to 4099 tokens, 4 kv heads: 13.6 us, in chunks of 768 keys 16.4: the longest one's chain of tiles is
// what is waited for); beyond, chunks that make kKv8Resident workgroups, three a compute unit, so that all run at once
// (4 x 131072 tokens, 8 kv heads, in 4096 workgroups 200 us, in 1024 187, in 768 188).
// 128-row kernel: split only where the row tiles do not fill the chip, in chunks of 512 keys or more.
constexpr int kKv8Alone = 1024;
constexpr int kKv8Resident = 768;
constexpr int kKv8Fine = 3 * kKv8Resident;

static Kv8Plan kv8_plan(int batch, int q_heads, int kv_heads, int max_query, int max_len) {
  Kv8Plan p;
  const int64_t rows = (int64_t)max_query * (q_heads / kv_heads);
  p.block = rows > 2 * kKv8Rows;
  const int per = p.block ? kKv8Block : kKv8Rows;
  p.row_tiles = (int)((rows + per - 1) / per);
  const int64_t groups = (int64_t)batch * kv_heads * p.row_tiles;
  p.waves = 4;
  int64_t chunk;
  if (p.block) {
    const int64_t most = (max_len + 511) / 512;
    int64_t splits = 512 / groups;
    splits = splits < 1 ? 1 : splits > most ? most : splits;
    chunk = splits > 1 ? ((max_len + splits - 1) / splits + kKv8Tile - 1) / kKv8Tile * kKv8Tile : max_len;
  } else if (max_len <= kKv8Alone) {
    p.waves = 8;
    chunk = max_len;
  } else {
    const int64_t step = 4 * kKv8Tile;
    const int64_t fine = groups * ((max_len + step - 1) / step);
    chunk = fine <= kKv8Fine ? step : step * ((fine + kKv8Resident - 1) / kKv8Resident);
  }
  if (chunk < kKv8Tile) chunk = kKv8Tile;
  if (chunk > (1 << 30)) chunk = 1 << 30;
  p.chunk = (int)chunk;
  p.n_splits = (int)((max_len + chunk - 1) / chunk);
  if (p.n_splits < 1) p.n_splits = 1;
  return p;
}

template <class XT, int D>
static int kv8_launch(const Kv8Args& a, const Kv8Plan& p, hipStream_t s) {
  if (p.block) {
    constexpr size_t lds = (size_t)2 * (4 * (D / 32) + 2 * (D / 16)) * 1024;
    TQ_RETURN_IF_HIP_ERROR((allow_lds<kv8_block_kernel<XT, D>>(lds)));
    hipLaunchKernelGGL((kv8_block_kernel<XT, D>), dim3(a.batch * a.kv_heads, p.row_tiles, p.n_splits),
                       dim3(kKv8Waves * kWave), lds, s, a);
  } else {
    const dim3 grid(p.n_splits, a.batch * a.kv_heads, p.row_tiles);
    if (p.waves == 8)
      hipLaunchKernelGGL((kv8_split_kernel<XT, D, 8>), grid, dim3(8 * kWave), 0, s, a);
    else
      hipLaunchKernelGGL((kv8_split_kernel<XT, D, 4>), grid, dim3(4 * kWave), 0, s, a);
  }
  if (p.n_splits > 1)
    hipLaunchKernelGGL((kv8_merge_kernel<XT, D>), dim3((unsigned)(((int64_t)a.tokens * a.q_heads + 3) / 4)), dim3(256),
                       0, s, a);
  return (int)hipGetLastError();
}

}  // namespace tq

using namespace tq;

extern "C" int64_t tq_kv8_attention_workspace_elems(int tokens, int batch, int q_heads, int kv_heads, int head_dim,
                                                    int max_query, int max_len) {
  if (tokens <= 0 || batch <= 0 || q_heads <= 0 || kv_heads <= 0 || max_query <= 0 || max_len <= 0 ||
      q_heads % kv_heads != 0)
    return 0;
  const Kv8Plan p = kv8_plan(batch, q_heads, kv_heads, max_query, max_len);
  return p.n_splits > 1 ? (int64_t)tokens * q_heads * p.n_splits * (head_dim + 2) : 0;
}

extern "C" int tq_kv8_attention(const tq_kv8_cache* cache, const void* q, int64_t q_stride_t, int64_t q_stride_h,
                                int dtype, const int32_t* table, int64_t table_stride, int width,
                                const int32_t* lengths, const int32_t* query_start, int tokens, int batch,
                                int q_heads, int max_query, int max_len, float scale, void* out,
                                int64_t out_stride_t, int64_t out_stride_h, int zero_rest, float* workspace,
                                int64_t workspace_elems, void* stream) {
  if (dtype != TQ_DTYPE_BF16 && dtype != TQ_DTYPE_FP16) return TQ_ERR_DTYPE;
  if (cache == nullptr || cache->pages <= 0 || cache->kv_heads <= 0) return TQ_ERR_ARG;
  if (cache->head_dim != 64 && cache->head_dim != 128) return TQ_ERR_ARG;
  if (cache->block < 16 || cache->block > 1024 || (cache->block & (cache->block - 1)) != 0) return TQ_ERR_ARG;
  if (tokens < 0 || batch < 0 || q_heads <= 0 || q_heads % cache->kv_heads != 0 || width < 0 || max_len < 0 ||
      max_query < 0)
    return TQ_ERR_ARG;
  const int G = q_heads / cache->kv_heads;
  if (G > 128 || !(scale == scale) || scale - scale != 0.0f) return TQ_ERR_ARG;
  if (query_start == nullptr && (tokens != batch || max_query != 1)) return TQ_ERR_ARG;
  if ((int64_t)width * cache->block >= (1LL << 31) || (int64_t)batch * cache->kv_heads > 65535) return TQ_ERR_ARG;
  if ((int64_t)max_query * G >= (1LL << 31) || (int64_t)tokens * q_heads >= (1LL << 33)) return TQ_ERR_ARG;
  if (tokens == 0 || batch == 0 || max_query == 0) return TQ_OK;
  if (!q || !out || !lengths || table_stride < width || (width > 0 && !table)) return TQ_ERR_ARG;
  if (!cache->k_codes || !cache->v_codes || !cache->k_scales || !cache->v_scales) return TQ_ERR_ARG;
  if (!aligned16(q) || !aligned16(out) || !aligned16(cache->k_codes) || !aligned16(cache->v_codes) ||
      (q_stride_t % 8) || (q_stride_h % 8) || (out_stride_t % 8) || (out_stride_h % 8))
    return TQ_ERR_ALIGN;
  const int64_t room = (int64_t)width * cache->block;
  const Kv8Plan p = kv8_plan(batch, q_heads, cache->kv_heads, max_query, max_len);
  if (p.n_splits > 65535 || p.row_tiles > 65535) return TQ_ERR_ARG;
  if (p.n_splits > 1 && (!workspace || workspace_elems < (int64_t)tokens * q_heads * p.n_splits * (cache->head_dim + 2)))
    return TQ_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 7u) return TQ_ERR_ALIGN;
  Kv8Args a{};
  a.q = static_cast<const uint16_t*>(q); a.q_st = q_stride_t; a.q_sh = q_stride_h;
  a.k = cache->k_codes; a.v = cache->v_codes; a.ks = cache->k_scales; a.vs = cache->v_scales;
  a.table = table; a.ld = table_stride; a.lengths = lengths; a.query_start = query_start;
  a.out = static_cast<uint16_t*>(out); a.o_st = out_stride_t; a.o_sh = out_stride_h;
  a.part = workspace;
  a.tokens = tokens; a.batch = batch; a.q_heads = q_heads; a.kv_heads = cache->kv_heads; a.G = G;
  a.max_query = max_query;
  a.pages = cache->pages; a.len_cap = (int)(max_len < room ? max_len : room); a.units = cache->block / 16;
  a.unit_shift = 31 - __builtin_clz((unsigned)a.units);
  a.n_splits = p.n_splits; a.chunk = p.chunk; a.zero_rest = zero_rest && query_start != nullptr;
  a.head_bytes = (int64_t)cache->block * cache->head_dim;
  a.scale_log2 = (scale < 0 ? -scale : scale) * kLog2e8;
  a.scale_sign = scale < 0 ? -1.0f : 1.0f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->head_dim == 128)
    return dtype == TQ_DTYPE_BF16 ? kv8_launch<Bf16, 128>(a, p, s) : kv8_launch<Fp16, 128>(a, p, s);
  return dtype == TQ_DTYPE_BF16 ? kv8_launch<Bf16, 64>(a, p, s) : kv8_launch<Fp16, 64>(a, p, s);
}

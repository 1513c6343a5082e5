// Grouped-query attention of new tokens over a paged cache held in 4 bits (paged_int4.h), causal, in full or over a
// sliding window whose first positions stay visible. Ranges, tiles of 16 rows and the join are
// paged_attention.hip's (paged_attention.h).
//
// With k = z + (c - 8) step and v likewise, per group g of dims:
//   q.k_j = sum_g step_jg sum_d q_d (c_jd - 8) + z_jg U_g,   U_g = sum of q_d over the group,
//   out_d = [sum_j (w_j step_jg) (c_jd - 8) + sum_j w_j z_jg] / sum_j w_j,   w_j = exp(scale q.k_j - max).
// The matrix cores take c - 8, a whole number that fp16 holds exactly; what depends on the position, its step and
// offset, is applied outside in fp32, one fused multiply per score and group. So nothing of K is rounded, and of V
// only the weight w_j step_jg, to fp16, for bf16 too: its 11 bits are the closer, and the units below keep its range.
//
// Units. A row of bf16 q is scaled by the power of two that brings its largest element below 2^14: fp16 keeps its bits down
// to 2^-30 of the largest, and elements below 2^-38 are lost. Weights are held times 2^8 over a power of two, 2^ve, that
// follows the row's largest step so far (kept like the maximum): fp16 keeps weights down to 2^-32 of it. Sums in these
// units, of weights (up to 2^(14 - ve)) and of weights times offsets, have to stay inside fp32 where steps are 0 too (a
// group of one value): 2^ve begins at fp16's least step, whose offsets are below 2^16; with bf16, where it begins at
// 2^-80, it follows 2^-40 of the largest offset too, which is below any step of the same group but 0. So 2^25
// positions sum to at most 2^119.
#include "paged_attention.h"
#include "paged_int4.h"

namespace {

using namespace ldk;

// A power of two from its exponent, -126 .. 127.
__device__ __forceinline__ float pow2i(int e) { return u2f((uint32_t)(e + 127) << 23); }

// 8 params of the type as fp32.
template <typename E>
__device__ __forceinline__ void params8(const u32x4& v, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2_t a = unpack2<E>(v[i]);
    f[2 * i] = a[0], f[2 * i + 1] = a[1];
  }
}
// The largest of 8 params that are not negative, whose bits order as they do.
template <typename E>
__device__ __forceinline__ float largest8(const u32x4& v) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  auto h = [](uint32_t w) { return __builtin_bit_cast(u16x2, w); };  // (by value: a cast of v[i] itself is of v[0])
  const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(h(v[0]), h(v[1])), __builtin_elementwise_max(h(v[2]), h(v[3])));
  const uint16_t t = __builtin_elementwise_max(m[0], m[1]);
  return (float)__builtin_bit_cast(typename E::T, t);
}
// The largest of three, NaN aside (the compiler's own would first make a number of what it does not know to be one).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Two words of codes less 8 as fp16, the low four bits' (the even step's or block's) and the high four bits' operands.
// 1024 + c and 1024 + 16 c have the code in fp16's last bits. The masks are in registers, so that each is one
// instruction with its or.
struct Codes {
  u32x4 low, high;
};
struct Unpack {
  uint32_t low, high, magic;
  __device__ __forceinline__ Unpack() : low(sgpr_const<kLow4>()), high(sgpr_const<kHigh4>()), magic(vgpr_const<0x64006400u>()) {}
  __device__ __forceinline__ Codes operator()(uint32_t a, uint32_t b) const {
    const half2_t less = {(half_t)-1032.0f, (half_t)-1032.0f}, by = {(half_t)0.0625f, (half_t)0.0625f}, less72 = {(half_t)-72.0f, (half_t)-72.0f};
    const uint32_t w[4] = {a, a >> 8, b, b >> 8};
    Codes r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.low[i] = h22u(u2h2((w[i] & low) | magic) + less);
      r.high[i] = h22u(__builtin_elementwise_fma(u2h2((w[i] & high) | magic), by, less72));
    }
    return r;
  }
};

constexpr float kLag4 = 6.0f;  // powers of two that a row's maximum may lag (3: prompts of 8755 tokens 246 us instead of 231)
constexpr int kUnit4 = 8;      // weights times 2^kUnit4: 2^(kLag4 + kUnit4 + 1) is inside fp16
template <typename E>
constexpr bool kWide4 = E::kOnes == BF16::kOnes;  // of fp32's range: q is scaled, and the unit follows offsets
template <typename E>
constexpr int kLeast4 = kWide4<E> ? -80 : -24;  // of the weights' unit
// What the unit of the weights follows, of steps up to sm and 8 offsets (NaN aside: what it weights is NaN).
template <typename E>
__device__ __forceinline__ float follow8(float sm, const float* z) {
  if constexpr (kWide4<E>) {
    float m;
    asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(m) : "v"(z[0]), "v"(z[1]), "v"(z[2]));
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(m) : "v"(m), "v"(z[3]), "v"(z[4]));
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(m) : "v"(m), "v"(z[5]), "v"(z[6]));
    sm = fmaxf(sm, fmaxf(m, __builtin_fabsf(z[7])) * 0x1p-40f);
  }
  return sm;
}
// In words of two bf16 steps, whose offsets are the word four lanes on, puts 2^-40 of an offset in the place of a step that is
// smaller, which is 0 (times a code less 8, that is at most 2^-37 of the offset beside it); words of offsets stay. As
// numbers of 16 bits: infinities and NaN, 0x7F80 on, wrap to negative ones, and 40 less in the exponent.
struct Follow {
  uint32_t mask, wrap, less;  // in registers of each lane: scalar ones are short
  __device__ __forceinline__ Follow(bool offsets)
      : mask(offsets ? 0u : 0x7FFF7FFFu), wrap(offsets ? 0x80008000u : 0x00800080u), less(vgpr_const<0x14801480u>()) {
    asm volatile("" : "+v"(mask), "+v"(wrap));
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t word) const {
    typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
    auto two = [](uint32_t v) { return __builtin_bit_cast(i16x2, v); };
    const i16x2 z = two(__builtin_amdgcn_update_dpp(0, word, 0x104, 0xf, 0xf, true) & mask) + two(wrap);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(two(word), __builtin_elementwise_sub_sat(z, two(less))));
  }
};

// A row of q as the matrix cores' operands, 2^qs q in fp16: lane c16 + 16 kb has row c16's dims 8kb + 32s .. + 7, raw in
// qb; us: the row's sums over the groups in the same units (of the elements as they came: what fp16 loses of the
// smallest is below a sum's own rounding). Returns qs; fp16 q stays as it is.
template <typename E, int NS, int NG>
__device__ __forceinline__ int scale_q(u32x4* qb, float* us) {
  int qs = 0;
  if constexpr (kWide4<E>) {
    float amax = 0.0f;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2_t f = unpack2<E>(qb[s][i]);
        amax = max3(amax, __builtin_fabsf(f[0]), __builtin_fabsf(f[1]));
      }
    amax = max_xor32(max_xor16(amax));
    qs = 13 - max(-100, min(127, (int)(f2u(amax) >> 23) - 127));  // amax < 2^(14 - qs)
  }
  const float by = pow2i(qs);
#pragma unroll
  for (int g = 0; g < NG; ++g) us[g] = 0.0f;
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2_t f = unpack2<E>(qb[s][i]);
      us[s * NG / NS] += f[0] + f[1];
      if constexpr (kWide4<E>) qb[s][i] = pack2<F16>(f[0] * by, f[1] * by);
    }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    us[g] = add_xor32(add_xor16(us[g])) * by;
    if (!(__builtin_fabsf(us[g]) < __builtin_inff())) us[g] = __builtin_nanf("");  // a row with an infinity: no score
  }
  return qs;
}
// The exponents' factor of scores formed as 2^qs q.k: finite and, as -inf 0 is NaN, not 0.
__device__ __forceinline__ float score_factor(float scale, int qs) {
  return fmaxf(0x1p-126f, fminf(scale * 1.44269504088896341f * pow2i(-qs), 0x1p126f));
}

// ---- few rows
//
// A workgroup takes up to 16 rows of one kv head over a range of chunks. Both products have the row as the matrix
// cores' column, so that a lane's scores, weights, sums and outputs are one row's. Of a tile of R = 16 / C rows (a token's few
// query heads) the 16 columns take C chunks at once: q stands in the columns of one chunk (zeros in the others) when
// that chunk's K is the operand, so that the scores of all of them fill one accumulator, and the weights of one chunk's
// columns when its V is. What is done per score is then done once for C chunks on full lanes, and each column
// is a partial result over positions of its own; they meet at the end. A wave's loads are a group of chunks ahead.
//
// Long contexts are bound by what a CU has in flight: 64 tokens of 28/4 heads (95 MB) 27 us and 4.9 for the merge, 3.4 TB/s where
// a 2 GiB copy reaches 4.9; the CUs are busy for 20 us of it, the rest is the last ranges' unequal ends. Next to it stands the vector
// unit, 59% of the busy cycles (9 instructions per word of 8 codes, some 110 per group of columns), the matrix cores 11%.
// 40 tokens of 20/20 heads of 64 in groups of 32 (131 MB) 38 us. Short contexts are bound by the latency of finding the range,
// the page, its codes and of two launches: one token behind a window of 1024, 9.9 us.
// Waves of a SIMD that the registers are to leave room for: as many as need no spilling (two groups of dims of 128 with 2, 3
// waves: two contexts of 100000 positions 20.1, 21.7 us; four groups: 64 sequences 46, 118 us).
template <int HD, int NG>
constexpr int kSplitOcc = HD == 64 || NG == 1 ? 3 : 2;
constexpr int kPad = 4;  // floats after a row of outputs in LDS: 16 rows' float4 in different banks
constexpr int kWaves = 4;
// Chunks of a range, at least: two for each wave (with 4, 8, 12: one token of 28/4 heads after 4000 positions 10.7, 10.2, 11.3 us,
// after 16000 16.3, 12.1, 12.8).
constexpr int kMinRange4 = 8;
// Ranges of a sequence, at most (64, 128, 256: two contexts of 100000 positions 26.4, 21.9, 24.6 us, with the merge).
constexpr int kMaxRanges4 = 128;

// Over the 64 lanes.
template <int N>
__device__ __forceinline__ int row_ror_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, 0x120 + N, 0xf, 0xf, false);
}
__device__ __forceinline__ int wave_sum(int v) {
  v += row_ror_i<1>(v), v += row_ror_i<2>(v), v += row_ror_i<4>(v), v += row_ror_i<8>(v);
  auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = p[0] + p[1];
  p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return p[0] + p[1];
}
__device__ __forceinline__ int wave_max(int v) {
  v = max(v, row_ror_i<1>(v)), v = max(v, row_ror_i<2>(v)), v = max(v, row_ror_i<4>(v)), v = max(v, row_ror_i<8>(v));
  auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max((int)p[0], (int)p[1]);
  p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((int)p[0], (int)p[1]);
}
// Chunks of a range, of `sum` chunks (of up to 64 sequences: below 2^26) in sequences of at most `most`.
__device__ __forceinline__ int range_chunks4(const PagedArgs& a, int sum, int most) {
  const int per = min((sum + a.spare - 1) / a.spare, most);
  return max(per, max(kMinRange4, (most + kMaxRanges4 - 1) / kMaxRanges4));
}
// The sequence and range of workgroup `slot` of up to 64 sequences, one per lane. Whole ranges come first and each
// sequence's last, shorter one after them, so that the short ones fill what the whole ones leave of the CUs.
__device__ __forceinline__ Slot find_slot4(const PagedArgs& a, int slot, int lane) {
  if (a.map) {
    const int b = a.map[1 + slot];
    if (b < 0) return Slot{-1, 0, 1, 0, 0};
    const int first = a.plan[2 * b];
    return Slot{b, slot - first, a.plan[2 * b + 1], first, a.map[0]};
  }
  const int n = lane < a.B ? seq_span(a, lane).n : 0;
  const int per = range_chunks4(a, wave_sum(n), wave_max(n));
  const int whole = n / per, rest = lane < a.B && (n % per || !n) ? 1 : 0;  // whole < 2^9: both in one word
  int end = whole << 16 | rest;  // inclusive scan over the lanes
  for (int off = 1; off < a.B; off *= 2) {
    const int v = __shfl_up(end, off);
    if (lane >= off) end += v;
  }
  const int wholes = __builtin_amdgcn_readlane(end, a.B - 1) >> 16;
  const int w1 = end >> 16, r1 = end & 0xffff;
  const bool mine = slot < wholes ? slot >= w1 - whole && slot < w1 : rest && slot - wholes == r1 - 1;
  const uint64_t has = __ballot(mine);
  if (!has) return Slot{-1, 0, 1, 0, per};
  const int src = __builtin_ctzll(has);
  return Slot{src, slot < wholes ? slot - __builtin_amdgcn_readlane(w1 - whole, src) : __builtin_amdgcn_readlane(whole, src),
              __builtin_amdgcn_readlane(whole + rest, src), __builtin_amdgcn_readlane(w1 - whole + r1 - rest, src), per};
}

// LDS: q's operands and 16 bytes of zeros, the row's sums and scale; then the waves' results.
constexpr int q4_bytes(int hd, int ng) { return 32 * hd + 64 + 16 * 4 * (ng + 3) + 64; }
constexpr int split4_lds(int hd, int ng, int nw) { return q4_bytes(hd, ng) + nw * kRows * (2 + hd + kPad) * 4; }

template <typename E, int HD, int NG, int NW, int C>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(kSplitOcc<HD, NG>))) void paged_split4_kernel(PagedArgs a) {
  typedef typename E::T T;
  typedef T T4 __attribute__((ext_vector_type(4)));
  typedef Int4Block<HD, NG> L;
  constexpr int NS = HD / 32, NB = HD / 16, NP = HD / 64;  // K dim steps, V dim blocks, pairs of steps
  constexpr int NL = HD / 64;                              // 16-byte loads per lane of K's codes, and of V's
  __shared__ __align__(16) unsigned char lds[split4_lds(HD, NG, NW)];
  unsigned char* const q_at = lds;                         // [NS][64 lanes] 16 bytes, then zeros
  float(*const us_at)[kRows] = reinterpret_cast<float(*)[kRows]>(lds + 32 * HD + 64);  // [NG + 1]: sums; then qs
  float(*const ml)[kRows] = us_at + NG + 1;                // [2]: the rows' maxima and sums
  int* const found = reinterpret_cast<int*>(ml + 2);
  float(*const mw)[kRows] = reinterpret_cast<float(*)[kRows]>(lds + q4_bytes(HD, NG));
  float(*const lw)[kRows] = mw + NW;
  float(*const ow)[kRows][HD + kPad] = reinterpret_cast<float(*)[kRows][HD + kPad]>(lds + q4_bytes(HD, NG) + NW * kRows * 8);
  const int tid = threadIdx.x, lane = tid & 63, wg = (int)blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, kb = lane >> 4;
  const int xy = a.nkv * a.nt, bxy = wg % xy;
  const int kvh = bxy % a.nkv, tile = bxy / a.nkv;
  constexpr int R = 16 / C;
  const int r16 = c16 % R, col = c16 / R;  // this lane's row and chunk of a group

  // ---- one wave finds the range for all
  Slot sl{wg / xy, 0, 1, wg / xy, kAll};  // without a plan every sequence is one range
  if (a.plan) {
    if (wave == 0) {
      sl = find_slot4(a, wg / xy, lane);
      if (lane == 0) found[0] = sl.b, found[1] = sl.split, found[2] = sl.ranges, found[3] = sl.first, found[4] = sl.per;
    }
    lds_barrier();
    auto uniform = [&](int i) { return __builtin_amdgcn_readfirstlane(found[i]); };
    sl = Slot{uniform(0), uniform(1), uniform(2), uniform(3), uniform(4)};
  }
  if (sl.b < 0) return;
  Span sp = seq_span(a, sl.b);  // one sequence's for the whole workgroup: scalars, and with them what is formed of them
  sp.s.row0 = __builtin_amdgcn_readfirstlane(sp.s.row0);
  sp.s.n = __builtin_amdgcn_readfirstlane(sp.s.n);
  sp.s.pos0 = __builtin_amdgcn_readfirstlane(sp.s.pos0);
  sp.cs = __builtin_amdgcn_readfirstlane(sp.cs);
  sp.lo = __builtin_amdgcn_readfirstlane(sp.lo);
  sp.n = __builtin_amdgcn_readfirstlane(sp.n);
  if (a.plan && !a.map && kvh == 0 && tile == 0 && sl.split == 0 && tid == 0) {
    a.plan[2 * sl.b] = sl.first;
    a.plan[2 * sl.b + 1] = sl.ranges;
  }
  const int rows = min(kRows, sp.s.n * a.gq - tile * kRows);  // this tile's
  if (rows <= 0) return;
  // this lane's row and the positions that it sees: lo..hi and below sinks
  const int p = sp.s.pos0 + (tile * kRows + r16) / a.gq;
  const int hi = r16 < rows ? min(p, a.cap - 1) : -1;
  const int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
  // of the tile's rows: the last position and the first that one of them sees past the sinks, and that all see
  const int pt0 = sp.s.pos0 + tile * kRows / a.gq, pt1 = sp.s.pos0 + (tile * kRows + rows - 1) / a.gq;
  const int thi = min(pt1, a.cap - 1), tlo = a.window > 0 ? max(0, pt0 - a.window + 1) : 0;
  const int alo = a.window > 0 ? max(0, pt1 - a.window + 1) : 0;

  // The maximum that is subtracted may lag the largest score by kLag4; it and the unit of the weights move where a lane
  // finds more, and with them what is summed so far. Scores start from -m (0 while m is -inf), so that differences
  // are formed before they are scaled: what m f1 rounds away would rescale a row at every chunk.
  float m_run = -__builtin_inff(), less = 0.0f, limit = -__builtin_inff(), l = 0.0f;
  int ve = kLeast4<E>;           // 2^ve: the column's largest step's power of two
  float ms[NG];                  // sum of w z
  float4_t o[NB];                // O^T[dim 16b + 4kb + r][column c16]; l, ms and o in units of 2^(kUnit4 - ve)
#pragma unroll
  for (int g = 0; g < NG; ++g) ms[g] = 0.0f;
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const Unpack unpacked;
  const int32_t* const trow = a.table + (int64_t)sl.b * a.ldt;
  const char* const pool = (const char*)a.k + (int64_t)kvh * a.cpp.n * L::kBytes;
  const uint32_t pstride = (uint32_t)a.kps * 2;  // bytes: below 2^32
  const int jbegin = (int)min(sl.split * (int64_t)sl.per, (int64_t)sp.n), jend = (int)min((sl.split + (int64_t)1) * sl.per, (int64_t)sp.n);
  const int group = min(C, max(1, (jend - jbegin + NW - 1) / NW));  // chunks that a wave takes at once
  // The chunk j of the range and, where its page is in the pool and a row of the tile sees some of it, its block; else null
  auto chunk_at = [&](int j) __attribute__((always_inline)) { return j < sp.cs ? j : j - sp.cs + sp.lo; };
  auto block_of = [&](int j, int c, int page_id, int sub) __attribute__((always_inline)) {
    const int cb = c * kChunkPos;
    const bool live = j < jend && cb <= thi && (cb + kChunkPos > tlo || cb < a.sinks) && (uint32_t)page_id < (uint32_t)a.pages;
    return live ? pool + (uint64_t)(uint32_t)page_id * pstride + (uint32_t)sub * (uint32_t)L::kBytes : nullptr;
  };
  // Of the group from chunk j0 on: each lane's chunk c, its page id, and then its block and the block's steps and offsets (of
  // no block: any, they are masked)
  auto page_of = [&](int j0, int& c, int& sub) __attribute__((always_inline)) {
    c = chunk_at(min(j0 + col, jend - 1));
    int at;
    chunk_page(a.cpp, c, at, sub);
    return trow[at];
  };
  struct Loaded {
    u32x4 w[NL];
  };
  // codes of chunk i of a group, its block from a lane that has it; zeros where there is none
  auto load = [&](const char* mine, int i, int from) __attribute__((always_inline)) {
    const uint64_t m = (uint64_t)mine;
    const uint64_t u = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)m, i * R) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(m >> 32), i * R) << 32;
    const auto rs = buffer_rsrc(u ? (const char*)u + from : pool, u ? 16 * HD : 0);
    Loaded r;
#pragma unroll
    for (int t = 0; t < NL; ++t) r.w[t] = buffer_load16(rs, (uint32_t)(t * 1024 + lane * 16));
    return r;
  };
  u32x4 kp[NG][2], vp[NG][2];
  auto params = [&](const char* mine) __attribute__((always_inline)) {
    const char* const at = (mine ? mine : pool) + kb * 32;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kp[g][i] = *reinterpret_cast<const u32x4*>(at + L::kParams + g * 128 + i * 16);
        vp[g][i] = *reinterpret_cast<const u32x4*>(at + L::kVParams + g * 128 + i * 16);
      }
  };
  const int step = NW * group;
  int j0 = jbegin + wave * group, c, cn, subn;
  const char *mine = nullptr, *next = nullptr;
  Loaded x[C], y[C];
  if (j0 < jend) {
    int sub;
    const int id = page_of(j0, c, sub), idn = page_of(j0 + step, cn, subn);
    mine = block_of(col < group ? j0 + col : kAll, c, id, sub);
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = load(mine, i, 0);
    params(mine);
#pragma unroll
    for (int i = 0; i < C; ++i) y[i] = load(mine, i, L::kV);
    next = block_of(col < group ? j0 + step + col : kAll, cn, idn, subn);
  }
  // ---- with the first codes on their way, one wave prepares q for all
  if (wave == 0) {
    const int row = tile * kRows + r16;
    const T* qrow = (const T*)a.q + (int64_t)(sp.s.row0 + row / a.gq) * a.ldq + (int64_t)(kvh * a.gq + row % a.gq) * HD;
    u32x4 qb[NS];
    float us[NG];
#pragma unroll
    for (int t = 0; t < NS; ++t)
      qb[t] = r16 < rows ? *reinterpret_cast<const u32x4*>(qrow + 32 * t + 8 * kb) : u32x4{0, 0, 0, 0};
    const int qs = scale_q<E, NS, NG>(qb, us);
#pragma unroll
    for (int t = 0; t < NS; ++t) *reinterpret_cast<u32x4*>(q_at + (t * 64 + lane) * 16) = qb[t];
    if (lane < 4) reinterpret_cast<uint32_t*>(q_at + 32 * HD)[lane] = 0;
    if (kb == 0) {
#pragma unroll
      for (int g = 0; g < NG; ++g) us_at[g][c16] = us[g];
      us_at[NG][c16] = __builtin_bit_cast(float, qs);
    }
  }
  lds_barrier();
  float us[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) us[g] = us_at[g][c16];
  const int qs = __builtin_bit_cast(int, us_at[NG][c16]);
  const float f1 = score_factor(a.scale, qs);
  for (; j0 < jend; j0 += step) {
    int c2, sub2;
    const int id2 = page_of(j0 + 2 * step, c2, sub2);
    // ---- scores of positions 8kb + e of this lane's chunk
    float4_t acc[2][NG];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < NG; ++g) acc[h][g] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < C; ++i) {
      // q in this chunk's columns; elsewhere zeros
      int at_q = lane * 16;
      asm volatile("" : "+v"(at_q));  // read each time: registers do not hold C copies of q beside the rest
      const unsigned char* const src = q_at + (C == 1 || col == i ? at_q : 32 * HD);
      const int stride = C == 1 || col == i ? 1024 : 0;
      u32x4 qb[NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) qb[s] = *reinterpret_cast<const u32x4*>(src + s * stride);
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Codes k = HD == 128 ? unpacked(x[i].w[h % NL][2 * n], x[i].w[h % NL][2 * n + 1]) : unpacked(x[i].w[0][2 * h], x[i].w[0][2 * h + 1]);
          acc[h][2 * n * NG / NS] = F16::mfma(k.low, qb[2 * n], acc[h][2 * n * NG / NS]);
          acc[h][(2 * n + 1) * NG / NS] = F16::mfma(k.high, qb[2 * n + 1], acc[h][(2 * n + 1) * NG / NS]);
        }
      x[i] = load(next, i, 0);
    }
    float sv[8];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float st[8], z[8];
      params8<E>(kp[g][0], st);
      params8<E>(kp[g][1], z);
#pragma unroll
      for (int e = 0; e < 8; ++e) sv[e] = __builtin_fmaf(st[e], acc[e >> 2][g][e & 3], __builtin_fmaf(z[e], us[g], g ? sv[e] : less));
    }
    // chunks that not every row sees whole, or that are not there: what a row does not see has no score, and steps and
    // offsets of 0 (they may be anything, and 0 x NaN is NaN)
    const int cb = c * kChunkPos;
    if (__any(!mine || cb + kChunkPos - 1 > pt0 || (cb < alo && cb + kChunkPos > a.sinks))) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p0 = cb + 8 * kb + 2 * i;
        const bool on0 = mine && p0 <= hi && (p0 >= lo || p0 < a.sinks), on1 = mine && p0 + 1 <= hi && (p0 + 1 >= lo || p0 + 1 < a.sinks);
        sv[2 * i] = on0 ? sv[2 * i] : -__builtin_inff();
        sv[2 * i + 1] = on1 ? sv[2 * i + 1] : -__builtin_inff();
        const uint32_t mk = (on0 ? 0x0000FFFFu : 0u) | (on1 ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int g = 0; g < NG; ++g) vp[g][0][i] &= mk, vp[g][1][i] &= mk;
      }
    }
    float sm = largest8<E>(vp[0][0]);
#pragma unroll
    for (int g = 1; g < NG; ++g) sm = fmaxf(sm, largest8<E>(vp[g][0]));
    if constexpr (kWide4<E>) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float z[8];
        params8<E>(vp[g][1], z);
        sm = follow8<E>(sm, z);
      }
    }
    float mc = max3(max3(max3(sv[0], sv[1], sv[2]), sv[3], sv[4]), max3(sv[5], sv[6], sv[7]), sv[7]);
    if (__any(mc > limit || sm >= pow2i(ve + 1))) {
      mc = max_xor32(max_xor16(mc));
      sm = max_xor32(max_xor16(sm));
      const float old = less, m_new = fmaxf(m_run, mc - old);
      const float now = m_new == -__builtin_inff() ? 0.0f : -m_new, more = old - now;
      const int vn = min(126, max(ve, (int)(f2u(sm) >> 23) - 127));
      const float was = m_run == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(-more * f1), al = __builtin_ldexpf(was, ve - vn);
      l = __builtin_ldexpf(l * was, ve - vn);
#pragma unroll
      for (int g = 0; g < NG; ++g) ms[g] = __builtin_ldexpf(ms[g] * was, ve - vn);
#pragma unroll
      for (int b = 0; b < NB; ++b) o[b] *= al;
#pragma unroll
      for (int e = 0; e < 8; ++e) sv[e] -= more;
      m_run = m_new;
      less = now;
      limit = m_new == -__builtin_inff() ? m_new : kLag4 / f1;
      ve = vn;
    }
    const float unit = (float)(kUnit4 - ve);
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e], f1, unit));
#pragma unroll
    for (int e = 0; e < 8; ++e) l += w[e];
    u32x4 pw[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float st[8], z[8];
      params8<E>(vp[g][0], st);
      params8<E>(vp[g][1], z);
#pragma unroll
      for (int e = 0; e < 8; ++e) ms[g] = __builtin_fmaf(w[e], z[e], ms[g]);
#pragma unroll
      for (int e = 0; e < 4; ++e) pw[g][e] = pack2<F16>(w[2 * e] * st[2 * e], w[2 * e + 1] * st[2 * e + 1]);
    }
    params(next);
    // ---- the weights of each chunk's columns times its V
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const uint32_t mk = C == 1 || col == i ? 0xFFFFFFFFu : 0u;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const u32x4 pi = {pw[g][0] & mk, pw[g][1] & mk, pw[g][2] & mk, pw[g][3] & mk};
#pragma unroll
        for (int t = g * NB / 2 / NG; t < (g + 1) * NB / 2 / NG; ++t) {  // the group's pairs of blocks
          const Codes v = unpacked(y[i].w[t / 2][2 * (t % 2)], y[i].w[t / 2][2 * (t % 2) + 1]);
          o[2 * t] = F16::mfma(v.low, pi, o[2 * t]);
          o[2 * t + 1] = F16::mfma(v.high, pi, o[2 * t + 1]);
        }
      }
      y[i] = load(next, i, L::kV);
    }
    mine = next, c = cn, cn = c2;
    next = block_of(col < group ? j0 + 2 * step + col : kAll, c2, id2, sub2);
  }

  // ---- what the columns have, in q.k's and v's own units; then a row's columns and the waves meet
  const float one = pow2i(ve - kUnit4), sc = a.scale * 1.44269504088896341f;
  l = add_xor32(add_xor16(l)) * one;
#pragma unroll
  for (int g = 0; g < NG; ++g) ms[g] = add_xor32(add_xor16(ms[g])) * one;
  if (kb == 0) {
    mw[wave][c16] = m_run * pow2i(-qs);
    lw[wave][c16] = l;
  }
  if (r16 < rows) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float4_t v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = __builtin_fmaf(o[b][r], one, ms[b * NG / NB]);
      *reinterpret_cast<float4_t*>(&ow[wave][c16][16 * b + 4 * kb]) = v;
    }
  }
  lds_barrier();
  if (tid < rows) {  // a row's maximum and sum, and the columns' factors in the place of their maxima
    float mv[NW * C], M = -__builtin_inff(), ls = 0.0f;
#pragma unroll
    for (int i = 0; i < NW * C; ++i) {
      mv[i] = mw[i / C][i % C * R + tid];
      M = fmaxf(M, mv[i]);
    }
#pragma unroll
    for (int i = 0; i < NW * C; ++i) {
      const float f = mv[i] != -__builtin_inff() ? __builtin_amdgcn_exp2f((mv[i] - M) * sc) : 0.0f;
      ls = __builtin_fmaf(lw[i / C][i % C * R + tid], f, ls);
      mw[i / C][i % C * R + tid] = f;
    }
    ml[0][tid] = M, ml[1][tid] = ls;
  }
  lds_barrier();
  float* part = a.part + (part_at(a, sl.b, sp.s.row0, sl.first, sl.split, tile) * a.nkv + kvh) * part_floats(HD);
  for (int e = tid; e < rows * (HD / 4); e += NW * 64) {
    const int j = e / (HD / 4), d = e % (HD / 4) * 4;
    float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NW * C; ++i) {
      const float f = mw[i / C][i % C * R + j];
      const float4_t x = *reinterpret_cast<const float4_t*>(&ow[i / C][i % C * R + j][d]);
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = __builtin_fmaf(x[r], f, v[r]);
    }
    const float ls = ml[1][j], over = ls != 0.0f ? 1.0f / ls : 0.0f;
    if (sl.ranges == 1) {
      const int g = tile * kRows + j;
      T* dst = (T*)a.out + (int64_t)(sp.s.row0 + g / a.gq) * a.ldo + (int64_t)(kvh * a.gq + g % a.gq) * HD + d;
      T4 y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = (T)bounded<E>(v[r] * over);
      *reinterpret_cast<T4*>(dst) = y;
    } else {
      *reinterpret_cast<float4_t*>(part + 2 * kRows + j * HD + d) = v;
      if (d == 0) {
        part[2 * j] = ml[0][j];
        part[2 * j + 1] = ls;
      }
    }
  }
}

// ---- blocks of rows that share K and V through LDS
//
// As paged_attention.hip's: CG x KG waves take 32 CG rows of one kv head, wave (kg, cg) 32 rows (two column tiles) over the
// chunks kg, kg + KG, ... of the block's range. The waves of a K group unpack each chunk once for all of its
// rows, ahead of its use: each wave its part of the codes, into whole tiles of c - 8 in an LDS slot, and of the steps and
// offsets, as fp32. What a wave unpacks it has loaded a step before. One barrier per chunk. With one K group (128 rows)
// there are three slots and a chunk's scores are formed a step ahead: their products run beside the exponentials of
// the chunk before. (Not with four groups of dims, whose products 256 registers do not hold beside the rest.)
//
// The vector unit bounds it, 63% (heads of 64: 72%) of the cycles with two or three waves a SIMD, the matrix cores 25% (20%):
// per score 2 instructions to form it, 2 for its exponential, 4 for its sums and weight, and unpacking a quarter of 9 per 8
// codes. 8755 tokens of 32/8 heads behind a window of 1000 (bf16) 231 us, 540 TFLOP/s; 509 of 14/2 heads of 64 after
// 20000 96 us with the merge, 385 TFLOP/s; with groups of 64 and 32 dims the former take 257 (fp16) and 362 us (bf16). Of the
// bf16 figures 2% are the unit's following offsets (Follow; as maxima beside the steps' 4 to 6%), 1% its being each row's own. Tried to
// no gain: the products in the compiler's scheduling groups, V's tiles read ahead of their products, wave priorities.
template <int BT, int NG>
constexpr bool kAhead4 = kBlockKG<BT> == 1 && NG < 4;

// LDS bytes: of a slot its tiles, steps and offsets (as much as the K group's threads write); of a K group its slots; the
// K groups' m and l per column tile and lane.
constexpr int param4_words(int ng, int cg) { return (64 * ng + cg * 64 - 1) / (cg * 64); }  // per thread
constexpr int slot4_bytes(int hd, int ng, int cg) { return hd / 8 * 1024 + param4_words(ng, cg) * cg * 64 * 8; }
constexpr int block4_lds(int hd, int ng, int cg, int kg, int s) { return kg * s * slot4_bytes(hd, ng, cg) + (kg > 1 ? cg * kg * 4 * 64 * 4 : 0); }

template <typename E, int HD, int NG, int BT>
__global__ __launch_bounds__(kBlockThreads<BT>) __attribute__((amdgpu_waves_per_eu(2))) void paged_block4_kernel(PagedArgs a) {
  typedef typename E::T T;
  typedef T T4 __attribute__((ext_vector_type(4)));
  typedef Int4Block<HD, NG> L;
  constexpr int CG = BT / 32, KG = kBlockKG<BT>, NS = HD / 32, NB = HD / 16, NP = HD / 64;
  constexpr int NU = 4 / CG;                                  // of a chunk's four quarters of codes, a wave's
  constexpr int NT = 2 * NP;                                  // tiles of a quarter
  constexpr int PW = param4_words(NG, CG);                    // words of steps and offsets per thread
  constexpr bool AHEAD = kAhead4<BT, NG>;
  constexpr int S = AHEAD ? 3 : 2, kSlot = slot4_bytes(HD, NG, CG);
  static_assert(KG == 1 || KG * S * kSlot >= (KG - 1) * CG * 2 * NB * 64 * 16, "the K groups meet in the slots");
  __shared__ __align__(16) unsigned char lds[block4_lds(HD, NG, CG, KG, S)];
  const int tid = threadIdx.x, lane = tid & 63, wg = (int)blockIdx.x, split = (int)blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave / CG, cg = wave % CG;
  const int c16 = lane & 15, kb = lane >> 4;
  const int kvh = wg % a.nkv, tile = a.btiles - 1 - wg / a.nkv;  // longest blocks first
  const Block bk = find_block<0>(a, tile, BT);
  if (bk.rows <= 0) return;
  const int per = block_range(a, bk.n, KG);
  const int j0 = split * per;
  if (split && j0 >= bk.n) return;  // the first range runs with no chunk too: its rows are written
  const int nsteps = max(0, min(per, bk.n - j0));
  const int n = (nsteps + KG - 1) / KG;  // steps of a K group (the last ones may be dead)

  // this lane's two rows see the positions above hi - window up to hi, and those below sinks; rows past
  // the block's are not stored
  const int window = a.window > 0 ? a.window : kAll;
  auto row_of = [&](int ct, int ln, int& tok, int& head) __attribute__((always_inline)) {
    const int r = bk.r0 + min(32 * cg + 16 * ct + (ln & 15), bk.rows - 1);
    tok = r / a.gq;
    head = kvh * a.gq + r % a.gq;
  };
  int hi[2];
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    int t, h;
    row_of(ct, lane, t, h);
    hi[ct] = max(-1, bk.pos0 + t);
  }
  // of the block: positions that every row sees, all_lo .. first, and that one sees, any_lo .. last
  const int all_lo = a.window > 0 ? max(0, bk.last - a.window + 1) : 0;
  const int any_lo = a.window > 0 ? max(0, bk.first - a.window + 1) : 0;

  // the block's chunks in order: those that every row sees whole (fl .. fl + nf - 1), the sinks', the others
  const int fl = max(bk.lo, (all_lo + kChunkPos - 1) / kChunkPos);
  const int nf = max(0, min(bk.lo + bk.n - bk.cs, (min(bk.first, kAll - 1) + 1) / kChunkPos) - fl);
  auto chunk_of = [&](int j) __attribute__((always_inline)) {
    const int i = j0 + j * KG + kg;
    int d = i - nf - bk.cs + bk.lo < fl ? bk.lo - nf - bk.cs : bk.lo - bk.cs;
    d = i < nf + bk.cs ? -nf : d;
    return i + (i < nf ? fl : d);
  };
  // the page of a step that is to be loaded next. Its id comes as the codes do: read through the scalar cache, its way back
  // would be waited for with the next read of LDS
  const auto table = buffer_rsrc(a.table + (int64_t)bk.b * a.ldt, (uint32_t)kAll);
  int page, sub, c_page;
  auto next_page = [&](int j) __attribute__((always_inline)) {
    c_page = j * KG + kg < nsteps ? chunk_of(j) : 0;
    int at;
    chunk_page(a.cpp, c_page, at, sub);
    page = (int)__builtin_amdgcn_raw_buffer_load_b32(table, at * 4, 0, 0);
  };
  uint32_t have = 0;  // bit i: whether the step i before the last one loaded has a page
  int nfull = min(n, max(0, nf - j0 - kg + KG - 1) / KG);  // unmasked steps: to the first without a page
  struct Raw {
    u32x4 codes[NU];
    uint32_t params[PW];
    int c;
  };
  const int gt = cg * 64 + lane;  // of the K group's threads
  // A chunk's bytes that this thread unpacks; no page (an id outside the pool, a step past the range): zeros
  const char* const pool = (const char*)a.k + (int64_t)kvh * a.cpp.n * L::kBytes;
  const uint32_t pstride = (uint32_t)a.kps * 2;  // bytes: below 2^32
  auto load = [&](int j) __attribute__((always_inline)) {
    const uint32_t id = (uint32_t)__builtin_amdgcn_readfirstlane(page);
    const bool ok = (j * KG + kg < nsteps) & (id < (uint32_t)a.pages);
    const auto rs = buffer_rsrc(pool + (uint64_t)(ok ? id : 0u) * pstride + (uint32_t)sub * (uint32_t)L::kBytes, ok ? L::kBytes : 0);
    Raw r;
    r.c = c_page;
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = cg + CG * i;
      if constexpr (HD == 128) {
        r.codes[i] = buffer_load16(rs, (uint32_t)(u * 1024 + lane * 16));
      } else {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(rs, (uint32_t)((u >> 1) * 1024 + lane * 16 + (u & 1) * 8), 0, 0);
        r.codes[i] = u32x4{v[0], v[1], 0, 0};
      }
    }
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int w = gt + i * CG * 64;
      r.params[i] = __builtin_amdgcn_raw_buffer_load_b32(rs, (uint32_t)(w < 64 * NG ? L::kParams + w * 4 : L::kBytes), 0, 0);
    }
    have = __builtin_amdgcn_readfirstlane(have << 1 | (ok ? 1u : 0u));
    nfull = __builtin_amdgcn_readfirstlane(ok ? nfull : min(nfull, j));
    next_page(j + 1);
    return r;
  };
  unsigned char* const slots = lds + kg * S * kSlot;
  auto slot_of = [&](int j) __attribute__((always_inline)) { return slots + (S == 2 ? j & 1 : j % 3) * kSlot; };
  const Unpack unpacked;
  const Follow follow(gt & 4);
  auto unpack = [&](const Raw& r, int j) __attribute__((always_inline)) {
    unsigned char* const to = slot_of(j);
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int t = 0; t < NP; ++t) {
        const Codes c = unpacked(r.codes[i][2 * t], r.codes[i][2 * t + 1]);
        unsigned char* const at = to + ((cg + CG * i) * NT + 2 * t) * 1024 + lane * 16;
        *reinterpret_cast<u32x4*>(at) = c.low;
        *reinterpret_cast<u32x4*>(at + 1024) = c.high;
      }
    // word w of the params: of k or v, group, position / 8, step or offset, a pair of positions. What no row of the block
    // sees may be anything: zero
    float* const par = reinterpret_cast<float*>(to + HD / 8 * 1024);
    const int cb = r.c * kChunkPos;
    const bool edge = (cb + kChunkPos - 1 > bk.last) | ((cb < any_lo) & (cb + kChunkPos > a.sinks));  // for the whole workgroup
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      const int w = gt + i * CG * 64;
      const int pos = (w >> 3 & 3) * 8 + (w & 3) * 2, kind = (w >> 2 & 1) + (w >= 32 * NG ? 2 : 0), g = w / 32 % NG;
      float2_t f = unpack2<E>(kWide4<E> ? follow(r.params[i]) : r.params[i]);
      if (edge) {
        const int p0 = cb + pos;
        f[0] = (p0 <= bk.last) & ((p0 >= any_lo) | (p0 < a.sinks)) ? f[0] : 0.0f;
        f[1] = (p0 + 1 <= bk.last) & ((p0 + 1 >= any_lo) | (p0 + 1 < a.sinks)) ? f[1] : 0.0f;
      }
      // (threads past the last word write behind them)
      *reinterpret_cast<float2_t*>(par + (w < 64 * NG ? (kind * NG + g) * 32 + pos : 2 * w)) = f;
    }
  };
  constexpr int D = AHEAD ? 2 : 1;  // steps ahead that are unpacked
  next_page(0);
  {
    Raw r[D];
#pragma unroll
    for (int i = 0; i < D; ++i) r[i] = load(i);
#pragma unroll
    for (int i = 0; i < D; ++i) unpack(r[i], i);
  }
  Raw raw = load(D);  // (one step's: a copy of registers that a load is to fill would wait for it)

  // this wave's q operands
  u32x4 q[2][NS];
  float us[2][NG], f1[2];
  int qs[2];
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    int t, h;
    row_of(ct, lane, t, h);
    const T* src = (const T*)a.q + (int64_t)(bk.row0 + t) * a.ldq + (int64_t)h * HD + 8 * kb;
#pragma unroll
    for (int s = 0; s < NS; ++s) q[ct][s] = *reinterpret_cast<const u32x4*>(src + 32 * s);
    qs[ct] = scale_q<E, NS, NG>(q[ct], us[ct]);
    f1[ct] = score_factor(a.scale, qs[ct]);
  }
  float m_run[2], less[2], limit[2], l[2], ms[2][NG];
  float unit[2];      // kUnit4 - ve, 2^ve the row's largest step's power of two: the units of l, ms and o
  float top = pow2i(kLeast4<E> + 1);  // 2^(ve + 1) of the rows' smaller one
  float4_t o[2][NB];  // O^T[dim 16b + 4kb + r][row c16], unnormalised
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    m_run[ct] = limit[ct] = -__builtin_inff();
    less[ct] = l[ct] = 0.0f;
    unit[ct] = (float)(kUnit4 - kLeast4<E>);
#pragma unroll
    for (int g = 0; g < NG; ++g) ms[ct][g] = 0.0f;
#pragma unroll
    for (int b = 0; b < NB; ++b) o[ct][b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  auto unit_exponent = [](float u) { return kUnit4 - (int)u; };
  auto param = [&](const unsigned char* slot, int kind, int g, float* f) __attribute__((always_inline)) {
    const float* const par = reinterpret_cast<const float*>(slot + HD / 8 * 1024) + (kind * NG + g) * 32 + 8 * kb;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4_t v = *reinterpret_cast<const float4_t*>(par + 4 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[4 * i + e] = v[e];
    }
  };
  float4_t acc[AHEAD ? NG : 1][2][2];  // [half][column tile]: a chunk's products by group of dims
  float sv[2][8];                      // its scores less the row's maximum, then its weights
  auto products = [&](const unsigned char* from, int g, float4_t (&x)[2][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int s = g * NS / NG; s < (g + 1) * NS / NG; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 k = *reinterpret_cast<const u32x4*>(from + (h * NS + s) * 1024 + lane * 16);
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
          const float4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
          x[h][ct] = F16::mfma(k, q[ct][s], s % (NS / NG) ? x[h][ct] : zero);
        }
      }
  };
  auto fold = [&](const unsigned char* from, int g, const float4_t (&x)[2][2]) __attribute__((always_inline)) {
    float st[8], z[8];
    param(from, 0, g, st);
    param(from, 1, g, z);
#pragma unroll
    for (int ct = 0; ct < 2; ++ct)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        sv[ct][e] = __builtin_fmaf(st[e], x[e >> 2][ct][e & 3], __builtin_fmaf(z[e], us[ct][g], g ? sv[ct][e] : less[ct]));
  };
  auto products_ahead = [&](int j) __attribute__((always_inline)) {
    if constexpr (AHEAD)
#pragma unroll
      for (int g = 0; g < NG; ++g) products(slot_of(j), g, acc[g]);
  };
  auto fold_ahead = [&](int j) __attribute__((always_inline)) {
    if constexpr (AHEAD)
#pragma unroll
      for (int g = 0; g < NG; ++g) fold(slot_of(j), g, acc[g]);
  };
  auto step = [&](auto maskedc, int j) __attribute__((always_inline)) {
    constexpr bool kMasked = decltype(maskedc)::value;
    lds_barrier();
    const unsigned char* const from = slot_of(j);
    const int cb = kMasked ? chunk_of(j) * kChunkPos : 0;
    const bool there = !kMasked || (have >> D & 1);
    if constexpr (!AHEAD) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        products(from, g, acc[0]);
        fold(from, g, acc[0]);
        if constexpr (NG == 4) __builtin_amdgcn_sched_barrier(0);  // one group at a time: 256 registers hold no more
      }
    }
    bool seen[2][8];
    float mc[2], sm[2] = {0.0f, 0.0f};  // the largest score, and the largest step of what the row sees
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (kMasked) {
          const int p = cb + 8 * kb + e;
          seen[ct][e] = there && p <= hi[ct] && (p > hi[ct] - window || p < a.sinks);
          sv[ct][e] = seen[ct][e] ? sv[ct][e] : -__builtin_inff();
        }
      }
      mc[ct] = max3(max3(max3(sv[ct][0], sv[ct][1], sv[ct][2]), sv[ct][3], sv[ct][4]), max3(sv[ct][5], sv[ct][6], sv[ct][7]), sv[ct][7]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float st[8];
      param(from, 2, g, st);
      if constexpr (kMasked) {
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
          for (int e = 0; e < 8; ++e) sm[ct] = fmaxf(sm[ct], seen[ct][e] ? st[e] : 0.0f);
      } else {
        sm[0] = max3(max3(max3(sm[0], st[0], st[1]), st[2], st[3]), max3(st[4], st[5], st[6]), st[7]);
      }
    }
    if constexpr (!kMasked) sm[1] = sm[0];
    if (__any(mc[0] > limit[0] || mc[1] > limit[1] || sm[0] >= top || (kMasked && sm[1] >= top))) {
#pragma unroll
      for (int ct = 0; ct < 2; ++ct) {
        const int ve = unit_exponent(unit[ct]), vn = min(126, max(ve, (int)(f2u(max_xor32(max_xor16(sm[ct]))) >> 23) - 127)), by = ve - vn;
        unit[ct] = (float)(kUnit4 - vn);
        const float mx = max_xor32(max_xor16(mc[ct]));
        const float old = less[ct], m_new = fmaxf(m_run[ct], mx - old);
        const float now = m_new == -__builtin_inff() ? 0.0f : -m_new, more = old - now;
        const float was = m_run[ct] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(-more * f1[ct]), al = __builtin_ldexpf(was, by);
        l[ct] = __builtin_ldexpf(l[ct] * was, by);
#pragma unroll
        for (int g = 0; g < NG; ++g) ms[ct][g] = __builtin_ldexpf(ms[ct][g] * was, by);
#pragma unroll
        for (int b = 0; b < NB; ++b) o[ct][b] *= al;
#pragma unroll
        for (int e = 0; e < 8; ++e) sv[ct][e] -= more;
        m_run[ct] = m_new;
        less[ct] = now;
        limit[ct] = m_new == -__builtin_inff() ? m_new : kLag4 / f1[ct];
      }
      top = pow2i(unit_exponent(fmaxf(unit[0], unit[1])) + 1);
    }
    products_ahead(j + 1);
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sv[ct][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[ct][e], f1[ct], unit[ct]));
        l[ct] += sv[ct][e];
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float st[8], z[8];
      param(from, 2, g, st);
      param(from, 3, g, z);
      u32x4 pw[2];
#pragma unroll
      for (int ct = 0; ct < 2; ++ct) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // what this row does not see and another does may be NaN
          const bool on = !kMasked || seen[ct][e];
          ms[ct][g] = __builtin_fmaf(sv[ct][e], on ? z[e] : 0.0f, ms[ct][g]);
          x[e] = sv[ct][e] * (on ? st[e] : 0.0f);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) pw[ct][e] = pack2<F16>(x[2 * e], x[2 * e + 1]);
      }
#pragma unroll
      for (int b = g * NB / NG; b < (g + 1) * NB / NG; ++b) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(from + (2 * NS + b) * 1024 + lane * 16);
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) o[ct][b] = F16::mfma(v, pw[ct], o[ct][b]);
      }
      if constexpr (NG == 4) __builtin_amdgcn_sched_barrier(0);
    }
    unpack(raw, j + D);
    raw = load(j + D + 1);
    fold_ahead(j + 1);
  };
  if (AHEAD) {
    lds_barrier();
    products_ahead(0);
    fold_ahead(0);
  }
  int j = 0;
  for (; j < nfull; ++j) step(IntC<0>(), j);
  for (; j < n; ++j) step(IntC<1>(), j);

  // ---- what the rows have, in q.k's and v's own units; groups past the first leave it to the first, lane for lane
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    const float one = pow2i(-(int)unit[ct]);
    l[ct] = add_xor32(add_xor16(l[ct])) * one;
    m_run[ct] *= pow2i(-qs[ct]);
#pragma unroll
    for (int g = 0; g < NG; ++g) ms[ct][g] = add_xor32(add_xor16(ms[ct][g]));
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[ct][b][r] = (o[ct][b][r] + ms[ct][b * NG / NB]) * one;
  }
  float4_t* const red = reinterpret_cast<float4_t*>(lds);  // [wave - CG][2 NB][64]
  float(*const mls)[4][64] = reinterpret_cast<float(*)[4][64]>(lds + KG * S * kSlot);
  if constexpr (KG > 1) {
    lds_barrier();  // the slots have been read
    if (kg > 0) {
#pragma unroll
      for (int ct = 0; ct < 2; ++ct) {
        mls[wave][2 * ct][lane] = m_run[ct];
        mls[wave][2 * ct + 1][lane] = l[ct];
#pragma unroll
        for (int b = 0; b < NB; ++b) red[((wave - CG) * 2 * NB + NB * ct + b) * 64 + lane] = o[ct][b];
      }
    }
    lds_barrier();
    if (kg > 0) return;
  }
  const float sc = a.scale * 1.44269504088896341f;
  const bool direct = bk.n <= per;  // a lone range
  float* const part = a.bpart + (((int64_t)tile * a.nkv + kvh) * a.bsplits + split) * BT * (2 + HD);
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    float mv[KG], f[KG], M = m_run[ct], ls = 0.0f;
    mv[0] = m_run[ct];
#pragma unroll
    for (int g = 1; g < KG; ++g) {
      mv[g] = mls[cg + g * CG][2 * ct][lane];
      M = fmaxf(M, mv[g]);
    }
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      f[g] = mv[g] != -__builtin_inff() ? __builtin_amdgcn_exp2f((mv[g] - M) * sc) : 0.0f;
      ls = __builtin_fmaf(g ? mls[cg + g * CG][2 * ct + 1][lane] : l[ct], f[g], ls);
    }
    const float over = ls != 0.0f ? 1.0f / ls : 0.0f;
    const int col = 32 * cg + 16 * ct + c16;
    int t, h;
    row_of(ct, lane, t, h);
    T* dst = (T*)a.out + (int64_t)(bk.row0 + t) * a.ldo + (int64_t)h * HD + 4 * kb;
    float* pdst = part + 2 * BT + col * HD + 4 * kb;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float4_t v = o[ct][b] * f[0];
#pragma unroll
      for (int g = 1; g < KG; ++g) {
        const float4_t w = red[((cg + (g - 1) * CG) * 2 * NB + NB * ct + b) * 64 + lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = __builtin_fmaf(w[r], f[g], v[r]);
      }
      if (col < bk.rows) {
        if (direct) {
          T4 y;
#pragma unroll
          for (int r = 0; r < 4; ++r) y[r] = (T)bounded<E>(v[r] * over);
          *reinterpret_cast<T4*>(dst + 16 * b) = y;
        } else {
          *reinterpret_cast<float4_t*>(pdst + 16 * b) = v;
        }
      }
    }
    if (!direct && kb == 0 && col < bk.rows) {
      part[2 * col] = M;
      part[2 * col + 1] = ls;
    }
  }
}

// Chunks up to which a sequence is one range, without a merge (19 chunks 8.8 us, in ranges 9.9; 24 chunks 8.9 and 10.0; 34
// chunks 11.5 and 9.7).
constexpr int kSingle4 = 28;
// More sequences have their ranges found in a launch before (256 sequences of 20/20 heads of 64, to 1500 positions: 77 us; found
// by every workgroup, four sequences a lane, 104; 200 of 28/4 heads 36 and 38).
constexpr int kPlanSeqs4 = 64;

Plan make_plan4(int64_t T, int64_t B, int64_t max_q, int64_t max_len, int64_t window, int64_t sinks, int nq, int nkv, int hd) {
  Plan p;
  const int64_t gq = nq / nkv, rows = T * gq;
  if (max_q * gq > 2 * kRows) {  // blocks of rows
    // blocks of 128 rows where a sequence has 96 on average (from 48 on: 400 tokens of 32/8 heads beside 30 that decode 114 us, not 75)
    p.bt = rows >= 96 * B ? 128 : 64;
    p.btiles = rows / p.bt + B;
    // Blocks are cut along the positions while they do not fill the card: this many workgroups (two a CU with heads of 128,
    // three with 64), unless a half or a third of it is there uncut. us with half, this and twice as many: 300 tokens of 32/8
    // heads 43.8, 34.4, 33.4, 200 of 28/4 after 10000 87, 68, 76; blocks of 64 rows, 150 tokens of 28/4 beside 12 that decode 86, 57,
    // 65; heads of 64, 509 tokens of 14/2 after 20000 138, 98. Uncut from a half and from a third: 2000 tokens of 12/2 heads of
    // 128 65.7 and 73.7, 2 x 1500 of 14/2 of 64 73.4 and 48.9.
    const int64_t fill = p.bt == 64 ? 320 : hd == 128 ? 512 : 768, whole = nkv * p.btiles;
    const bool uncut = (hd == 128 ? 2 : 3) * whole >= fill;
    // Tiles of 16 rows that each unpack what they read are the faster up to some 20 a sequence, but against whole blocks of 128
    // rows. us in blocks and in tiles: 16 x 9 tokens of 28/4 heads after 4000 46.0, 34.3; 40 x 11 of 32/8 175, 104; 4 x 60 of 32/8
    // alone 16.2, 7.4; 50 of 12/2 after 8000 30.2, 22.7; 60 of 32/8 beside 200 that decode 127, 72; 32 x 1 to 40 108, 76.
    // They are even with 8 x 40 of 28/4 (46, 47) and 20 x 64 of 32/8 after 500 (41, 42), and slower with several prompts
    // beside tokens: 8 x 64 beside 32 that decode 60, 69. Where whole blocks are left alone: 40 x 30 of 32/8 after 3000 146, 166.
    // (And not where there would be a million of them, most of them of sequences of fewer rows.)
    if (max_q * gq > 20 * kRows || (p.bt == 128 && uncut) || B * nkv * (max_q * gq / kRows) > (1 << 20)) {
      p.bsplits = uncut ? 1 : std::max<int64_t>(1, std::min<int64_t>(32, fill / whole));
      if (p.bsplits > 1) p.bpart_bytes = p.btiles * nkv * p.bsplits * p.bt * (2 + hd) * 4;
      p.bytes = workspace_bytes(p, B);
      return p;
    }
    p.bt = p.btiles = 0;
  }
  p.nt = (max_q * gq + kRows - 1) / kRows;
  if (most_chunks(max_len, max_q, window, sinks) <= kSingle4) {
    p.slots = B;
    return p;
  }
  const int64_t w = nkv * p.nt, most = rows / kRows + B;  // the batch has most tiles or fewer
  // Whole ranges for two workgroups a CU, and more for the sequences' last, shorter ones, whose number is not known here:
  // us with 512 / w, this and 512 / w + B / 2: 64 sequences of 28/4 heads 33.8, 32.4, 35.7; 40 of 20/20 heads of 64 43.8,
  // 42.3, 42.9; half and twice the 512: 37 to 39 and 33 to 38.
  p.spare = std::max<int64_t>(1, 512 / w + std::min(most, B * p.nt) / (4 * p.nt));
  p.slots = B + p.spare;
  p.mapped = B > kPlanSeqs4;
  // (of nt tiles a sequence: one prompt of 80 tokens of 32/8 heads beside 1000 that decode, 1.7 GB and not 0.1)
  if (p.nt > 1) p.tiles = most;
  p.part_bytes = (p.nt > 1 ? p.tiles + p.spare * p.nt : p.slots) * nkv * part_floats(hd) * 4;
  p.bytes = workspace_bytes(p, B);
  return p;
}

template <typename E, int HD, int NG>
void launch_split(const PagedArgs& a, unsigned grid, hipStream_t s) {
  const int rows = a.max_q * a.gq;  // of a sequence, at most: its one tile's, or 16
  if constexpr (HD == 64) {
    if (rows <= 4) return paged_split4_kernel<E, HD, NG, kWaves, 4><<<grid, kWaves * 64, 0, s>>>(a);
  }
  if (rows <= 8)
    paged_split4_kernel<E, HD, NG, kWaves, 2><<<grid, kWaves * 64, 0, s>>>(a);
  else
    paged_split4_kernel<E, HD, NG, kWaves, 1><<<grid, kWaves * 64, 0, s>>>(a);
}

template <typename E, int HD, int NG>
int launch(const PagedArgs& a, const Plan& p, int dtype, hipStream_t s) {
  (void)hipGetLastError();
  int st;
  if (p.mapped && (st = ldk::paged_find_ranges(a, s))) return st;
  const dim3 blocks((unsigned)(p.btiles * a.nkv), (unsigned)p.bsplits);
  if (p.bt == 128)
    paged_block4_kernel<E, HD, NG, 128><<<blocks, kBlockThreads<128>, 0, s>>>(a);
  else if (p.bt)
    paged_block4_kernel<E, HD, NG, 64><<<blocks, kBlockThreads<64>, 0, s>>>(a);
  else
    launch_split<E, HD, NG>(a, (unsigned)(p.slots * a.nkv * p.nt), s);
  if ((st = ldk::check_launch("paged_attention_int4")) || !p.bytes) return st;
  return ldk::paged_join(a, dtype, HD, p.bt, s);
}
template <typename E>
int launch(const PagedArgs& a, const Plan& p, int dtype, int hd, int group, hipStream_t s) {
  if (hd == 64) return group == 32 ? launch<E, 64, 2>(a, p, dtype, s) : launch<E, 64, 1>(a, p, dtype, s);
  return group == 32 ? launch<E, 128, 4>(a, p, dtype, s) : group == 64 ? launch<E, 128, 2>(a, p, dtype, s) : launch<E, 128, 1>(a, p, dtype, s);
}

}  // namespace

extern "C" int64_t ldk_paged_attention_int4_workspace_bytes(int64_t T, int64_t B, int64_t max_q, int64_t max_len, int64_t window,
                                                            int64_t sinks, int nq, int nkv, int head_dim) {
  if (T <= 0 || T > (int64_t(1) << 24) || B <= 0 || B > 65535 || max_q <= 0 || max_q > (int64_t(1) << 24) || max_len <= 0 ||
      max_len > ldk::kMaxPositions || window < 0 || sinks < 0 || nq <= 0 || nkv <= 0 || nq % nkv || nq > 4096 ||
      (head_dim != 64 && head_dim != 128)) {
    return -ldk::fail(LDK_ERR_INVALID,
                      "paged_attention_int4_workspace_bytes: T=%lld B=%lld max_q=%lld max_len=%lld window=%lld sinks=%lld nq=%d "
                      "nkv=%d head_dim=%d",
                      (long long)T, (long long)B, (long long)max_q, (long long)max_len, (long long)window, (long long)sinks, nq,
                      nkv, head_dim);
  }
  return make_plan4(T, B, max_q, max_len, window, sinks, nq, nkv, head_dim).bytes;
}

extern "C" int ldk_paged_attention_int4(const void* q, int64_t ldq, int dtype, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                        const int32_t* block_table, int64_t ldt, int64_t max_pages, const void* kv_pages,
                                        int64_t page_stride, int64_t num_pages, int64_t page_size, void* out, int64_t ldo,
                                        int64_t T, int64_t B, int64_t max_q, int nq, int nkv, int head_dim, int group,
                                        int64_t window, int64_t sinks, float scale, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
  static const char* fn = "paged_attention_int4";
  if (!q || !kv_lens || !block_table || !kv_pages || !out) return ldk::fail(LDK_ERR_INVALID, "%s: null pointer", fn);
  int st = ldk::check_int4_pool(fn, dtype, nkv, head_dim, group, page_stride, num_pages, page_size, ldt, max_pages);
  if (st || (st = ldk::check_int4_batch(fn, T, B, 65535, cu_seqlens))) return st;
  if (nq <= 0 || nq % nkv || nq > 4096)
    return ldk::fail(LDK_ERR_INVALID, "%s: nq=%d must be a positive multiple of nkv=%d (at most 4096)", fn, nq, nkv);
  if (max_q <= 0 || max_q > T) return ldk::fail(LDK_ERR_INVALID, "%s: max_q=%lld outside 1..%lld", fn, (long long)max_q, (long long)T);
  if (window < 0 || sinks < 0) return ldk::fail(LDK_ERR_INVALID, "%s: window=%lld sinks=%lld", fn, (long long)window, (long long)sinks);
  if (!(scale > 1e-20f && scale < 1e20f)) return ldk::fail(LDK_ERR_INVALID, "%s: scale=%g must be positive", fn, (double)scale);
  if (ldq < (int64_t)nq * head_dim || ldo < (int64_t)nq * head_dim)
    return ldk::fail(LDK_ERR_INVALID, "%s: strides ldq=%lld ldo=%lld below what they step over", fn, (long long)ldq, (long long)ldo);
  if (!ldk::aligned(q, 16) || !ldk::aligned(out, 16) || !ldk::aligned(kv_pages, 16) || ldq % 8 || ldo % 8 || page_stride % 8 ||
      !ldk::aligned(kv_lens, 4) || !ldk::aligned(cu_seqlens, 4) || !ldk::aligned(block_table, 4) || !ldk::aligned(workspace, 16))
    return ldk::fail(LDK_ERR_ALIGN, "%s: q, out, workspace and the pages 16-byte aligned with strides of multiples of 8 elements", fn);
  const Plan p = make_plan4(cu_seqlens ? T : B, B, cu_seqlens ? max_q : 1, max_pages * page_size, window, sinks, nq, nkv, head_dim);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
    return ldk::fail(LDK_ERR_INVALID, "%s: workspace of %lld bytes, this call needs %lld", fn, (long long)workspace_bytes, (long long)p.bytes);
  if (!launchable(p, T, nq, nkv)) return ldk::fail(LDK_ERR_UNSUPPORTED, "%s: T=%lld rows of nq=%d heads are too many for a launch", fn, (long long)T, nq);
  const int big = 1 << 30;  // a window or sinks past every position
  PagedArgs a{};
  a.q = q, a.ldq = ldq, a.out = out, a.ldo = ldo;
  a.cu = cu_seqlens, a.kv_lens = kv_lens, a.table = block_table, a.ldt = ldt;
  a.k = kv_pages, a.kps = page_stride;
  lay_out(a, p, workspace, B);
  a.T = cu_seqlens ? (int)T : (int)B, a.B = (int)B, a.max_q = cu_seqlens ? (int)max_q : 1;
  a.nq = nq, a.nkv = nkv, a.gq = nq / nkv, a.nt = (int)p.nt;
  a.pages = (int)num_pages, a.cpp = page_div(page_size / kChunkPos), a.cap = (int)(max_pages * page_size);
  a.window = (int)std::min<int64_t>(window, big), a.sinks = (int)std::min<int64_t>(sinks, big);
  a.slots = (int)p.slots, a.spare = (int)p.spare;
  a.btiles = (int)p.btiles, a.bsplits = (int)p.bsplits, a.bdirect = 1;
  a.scale = scale;
  hipStream_t s = (hipStream_t)stream;
  return dtype == LDK_F16 ? launch<ldk::F16>(a, p, dtype, head_dim, group, s) : launch<ldk::BF16>(a, p, dtype, head_dim, group, s);
}

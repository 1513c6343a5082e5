// Grouped-query attention of new tokens over a paged cache (pages and sequences: paged.h): causal, in
// full or over a sliding window whose first positions stay visible, with the positions of a prefix that
// the whole batch shares looked up in one table.
//
// For a token at position p:  out = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q.k_j - max),  over the
// positions j <= p of its sequence with (window == 0 or j > p - window or j < sinks). A token that sees
// nothing (kv_lens 0, a position below 0, only absent pages) gives zeros.
//
// Rows. The query heads of a kv head and the tokens that share it are the rows of one product: row
// r = token * gq + head (gq = nq / nkv), so one token's whole group and, with more tokens, their
// groups, fill the matrix cores' 16-wide tiles, and each K and V byte is read once per tile.
//
// paged_split_kernel: a workgroup takes 16 rows of one kv head over a range of 32-position chunks,
// chunk w, w + NW, ... of it by wave w. Scores are S^T = K Q^T (a K tile is the A operand), whose
// lanes hold 8 consecutive positions of one row: the softmax numerators go straight into P V as its A
// operand, V^T tiles being the B operand, with an online maximum and sum in fp32 per wave; the waves
// meet in LDS. The numerators are rounded to the element type before they weight V (the matrix cores
// take nothing wider; fp16's are held times 2^7, which keeps weights down to 2^-32), and their sum is
// taken of what they were rounded to, so that a row that one position dominates gets that position's v
// whatever its numerator rounds to.
//
// paged_block_kernel: a workgroup takes 64 or 128 rows of one kv head, which share K and V through LDS.
// For prompts, and for the prefix that a whole batch shares, whose rows are all tokens of the batch.
//
// Ranges. The lengths are on the device, so the split is made there: every sequence has its visible
// chunks (those of the sinks, then those of the window) cut into ranges of `per` chunks, one `per` for
// the whole batch such that all ranges fit the launch's slots; a ragged batch gets ranges of equal
// work. Each wave finds its slot's sequence from the lengths alone, or, of more than 64 sequences, in what
// paged_plan_kernel found in a launch before. Sequences with more than one range leave {max, sum} and the
// unnormalised output in the workspace, and paged_merge_kernel, the next launch on the stream, joins them.
#include "lds_dma.h"
#include "paged_attention.h"

namespace {

using namespace ldk;

// find_slot for many sequences, once instead of by every wave: one workgroup. spare != 0.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedArgs a) {
  constexpr int NW = kPlanThreads / 64;
  __shared__ int64_t sums[NW];
  __shared__ int mosts[NW], totals[NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t sum = 0;
  int most = 0;
  for (int b = tid; b < a.B; b += kPlanThreads) {
    const int n = seq_span(a, b).n;
    sum += n;
    most = max(most, n);
  }
  sum = wave_sum64(sum);
  most = wave_max_i(most);
  if (lane == 0) sums[wave] = sum, mosts[wave] = most;
  __syncthreads();
  sum = 0, most = 0;
  for (int w = 0; w < NW; ++w) sum += sums[w], most = max(most, mosts[w]);
  const int per = range_chunks(a, sum, most);
  if (tid == 0) a.map[0] = per;
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + tid, n = b < a.B ? max(1, (seq_span(a, b).n + per - 1) / per) : 0;
    int end = n;  // inclusive scan over the lanes
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
      const int v = __shfl_up(end, off);
      if (lane >= off) end += v;
    }
    if (lane == 63) totals[wave] = end;
    __syncthreads();
    int first = base + end - n;
    for (int w = 0; w < NW; ++w) {
      first += w < wave ? totals[w] : 0;
      base += totals[w];
    }
    if (b < a.B) a.plan[2 * b] = first, a.plan[2 * b + 1] = n;
    for (int i = first; i < min(first + n, a.slots); ++i) a.map[1 + i] = b;
    __syncthreads();  // the totals have been read
  }
  for (int i = base + tid; i < a.slots; i += kPlanThreads) a.map[1 + i] = -1;
}

// LDS bytes of split_rows: per wave the 16 rows' m, l and outputs.
constexpr int split_lds(int hd, int nw) { return nw * kRows * (2 + hd) * 4; }

// Workgroup wg of the split: NW waves. Memory bounds it where the contexts are long: 64 tokens of 28/4
// heads over 364 MB 76 us, 4.8 TB/s, the rate of a 2 GiB copy; the latency of finding the ranges and of two
// launches where they are short (one token behind a window of 1024: 10.0 us with the merge).
template <typename E, int HD, int NW>
__device__ __forceinline__ void split_rows(const PagedArgs& a, int wg, unsigned char* lds) {
  typedef typename E::T T;
  constexpr int NS = HD / 32, NB = HD / 16;  // K dim steps, V dim blocks
  float(*const mw)[kRows] = reinterpret_cast<float(*)[kRows]>(lds);
  float(*const lw)[kRows] = mw + NW;
  float(*const ow)[kRows][HD] = reinterpret_cast<float(*)[kRows][HD]>(lds + NW * kRows * 8);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, kb = lane >> 4;
  const int xy = a.nkv * a.nt, bxy = wg % xy;
  const int kvh = bxy % a.nkv, tile = bxy / a.nkv;
  const Slot sl = find_slot(a, wg / xy, lane);
  if (sl.b < 0) return;
  const Span sp = seq_span(a, sl.b);
  if (a.plan && !a.map && kvh == 0 && tile == 0 && sl.split == 0 && tid == 0) {
    a.plan[2 * sl.b] = sl.first;
    a.plan[2 * sl.b + 1] = sl.ranges;
  }
  const int rows = min(kRows, sp.s.n * a.gq - tile * kRows);  // this tile's
  if (rows <= 0) return;
  // this lane's row (column of the score tiles) and the positions that it sees: lo..hi and below sinks
  const int row = tile * kRows + c16, tok = row / a.gq;
  const int p = sp.s.pos0 + tok;
  int hi = c16 < rows ? min(p, a.cap - 1) : -1;
  int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
  // of the tile: its last position and the first that any of its rows sees past the sinks
  const int pt0 = sp.s.pos0 + tile * kRows / a.gq, pt1 = sp.s.pos0 + (tile * kRows + rows - 1) / a.gq;
  const int thi = min(pt1, a.cap - 1), tlo = a.window > 0 ? max(0, pt0 - a.window + 1) : 0;
  // B operands: row c16's q at dims 8kb + 32s .. + 7
  const T* qrow = (const T*)a.q + (int64_t)(sp.s.row0 + tok) * a.ldq + (int64_t)(kvh * a.gq + row % a.gq) * HD;
  u32x4 qb[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s)
    qb[s] = c16 < rows ? *reinterpret_cast<const u32x4*>(qrow + 32 * s + 8 * kb) : u32x4{0, 0, 0, 0};

  const float sc = a.scale * 1.44269504088896341f;
  float m_run = -__builtin_inff();
  float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};  // of rows 4kb .. 4kb+3's numerators as rounded, by a column of ones
  const u32x4 ones = {E::kOnes, E::kOnes, E::kOnes, E::kOnes};
  float4_t o[NB];  // O[rows 4kb .. 4kb+3][dim 16b + c16], unnormalised
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const ScalarInts trow = (ScalarInts)(uintptr_t)(a.table + (int64_t)sl.b * a.ldt);
  const int jend = (int)min((sl.split + (int64_t)1) * sl.per, (int64_t)sp.n);
  const uint32_t lane_off = (uint32_t)(c16 * 64 + kb * 16);
  const uint32_t chunk_bytes = kChunkPos * HD * 2;
  for (int j = sl.split * sl.per + wave; j < jend; j += NW) {
    const int c = j < sp.cs ? j : j - sp.cs + sp.lo;
    const int cb = c * kChunkPos;
    if (cb > thi || (cb + kChunkPos <= tlo && cb >= a.sinks)) continue;
    int at, sub;
    chunk_page(a.cpp, c, at, sub);
    const int page = trow[at];
    if (page < 0 || page >= a.pages) continue;
    const int64_t in_page = ((int64_t)kvh * a.cpp.n + sub) * (kChunkPos * HD);
    const auto krs = buffer_rsrc((const T*)a.k + page * a.kps + in_page, chunk_bytes);
    const auto vrs = buffer_rsrc((const T*)a.vt + page * a.vps + in_page, chunk_bytes);
    u32x4 kr[2 * NS], vr[NB];
#pragma unroll
    for (int t = 0; t < 2 * NS; ++t) kr[t] = buffer_load16(krs, (uint32_t)(t * 1024) + lane_off);
#pragma unroll
    for (int t = 0; t < NB; ++t) vr[t] = buffer_load16(vrs, (uint32_t)(t * 1024) + lane_off);
    float4_t acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      acc[0] = E::mfma(kr[s], qb[s], acc[0]);
      acc[1] = E::mfma(kr[NS + s], qb[s], acc[1]);
    }
    float sv[8], mc = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int pj = cb + 8 * kb + e;
      sv[e] = pj <= hi && (pj >= lo || pj < a.sinks) ? acc[e >> 2][e & 3] : -__builtin_inff();
      mc = fmaxf(mc, sv[e]);
    }
    mc = max_xor32(max_xor16(mc));
    const float m_new = fmaxf(m_run, mc);
    // a row that has seen nothing so far keeps m = -inf; its exponents are taken against 0. Differences are
    // formed before they are scaled: what m sc rounds away would rescale a row at every chunk
    const float base = m_new == -__builtin_inff() ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f((m_run - base) * sc);
    m_run = m_new;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e] - base, sc, E::kShift));
    u32x4 pa;
#pragma unroll
    for (int e = 0; e < 4; ++e) pa[e] = pack2<E>(x[2 * e], x[2 * e + 1]);
    // V at positions that no row of the tile sees is not this call's data: zero, so that 0 x NaN is not
    if (cb + kChunkPos - 1 > thi || (cb < tlo && cb + kChunkPos > a.sinks)) {
      uint32_t mk[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int p0 = cb + 8 * kb + 2 * e;
        mk[e] = (p0 <= thi && (p0 >= tlo || p0 < a.sinks) ? 0x0000FFFFu : 0u) |
                (p0 + 1 <= thi && (p0 + 1 >= tlo || p0 + 1 < a.sinks) ? 0xFFFF0000u : 0u);
      }
#pragma unroll
      for (int t = 0; t < NB; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) vr[t][e] &= mk[e];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float al = __shfl(alpha, 4 * kb + r);
      sum[r] *= al;
#pragma unroll
      for (int b = 0; b < NB; ++b) o[b][r] *= al;
    }
    sum = E::mfma(pa, ones, sum);
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = E::mfma(pa, vr[b], o[b]);
  }

  // ---- the waves meet
  if (kb == 0) mw[wave][c16] = m_run;
  if (c16 == 0) *reinterpret_cast<float4_t*>(&lw[wave][4 * kb]) = sum;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (4 * kb + r < rows) {
#pragma unroll
      for (int b = 0; b < NB; ++b) ow[wave][4 * kb + r][16 * b + c16] = o[b][r];
    }
  lds_barrier();
  float* part = a.part + (int64_t)wg * part_floats(HD);
  for (int e = tid; e < rows * HD; e += NW * 64) {
    const int j = e / HD, d = e % HD;
    float mv[NW], lv[NW], ov[NW], M = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      mv[w] = mw[w][j];
      lv[w] = lw[w][j];
      ov[w] = ow[w][j][d];
    }
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, mv[w]);
    float l = 0.0f, v = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = mv[w] != -__builtin_inff() ? __builtin_amdgcn_exp2f((mv[w] - M) * sc) : 0.0f;
      l = __builtin_fmaf(lv[w], f, l);
      v = __builtin_fmaf(ov[w], f, v);
    }
    if (sl.ranges == 1 && !a.skip) {
      const int g = tile * kRows + j;
      T* dst = (T*)a.out + (int64_t)(sp.s.row0 + g / a.gq) * a.ldo + (int64_t)(kvh * a.gq + g % a.gq) * HD;
      dst[d] = (T)(l != 0.0f ? v / l : 0.0f);
    } else {
      part[2 * kRows + e] = v;
      if (d == 0) {
        part[2 * j] = M;
        part[2 * j + 1] = l;
      }
    }
  }
}

template <typename E, int HD, int NW>
__global__ __launch_bounds__(NW * 64) void paged_split_kernel(PagedArgs a) {
  __shared__ __align__(16) unsigned char lds[split_lds(HD, NW)];
  split_rows<E, HD, NW>(a, (int)blockIdx.x, lds);
}

// ---- blocks of rows that share K and V through LDS
//
// A workgroup of CG x KG waves takes 32 CG rows of one kv head: wave (kg, cg) has 32 rows (two MFMA
// column tiles) over the 32-position chunks kg, kg + KG, ... of the block's range. The waves of a K
// group share each chunk's K and V tiles through an S-slot LDS ring filled by 16-byte loads to LDS (a
// tile's lane l reads the 16 bytes lane l wrote: no bank conflicts), so a byte from L2 serves 32 CG
// rows and a byte from LDS 32. One barrier per chunk; a chunk's V, and with four slots the next
// chunk's K, leaves LDS before the MFMAs ahead of those that need it. P.V is O^T = V^T P with the row
// as the column, so a lane's scores, maximum, sum and outputs are the same rows' and the online softmax
// needs no shuffles beyond the maximum over a tile's positions. Chunks that every row sees whole run
// without masks. Page ids come through the scalar cache, one chunk ahead of their loads.
//
// Bound by the order of a wave's own work, scores, softmax and P.V of a chunk one after the other between two
// barriers: 5 windowed prompts of 32/8 heads (124 GFLOP) 169 us, 734 TFLOP/s, 61% of a large matrix product's
// rate, with the vector unit busy 48% and the matrix unit 35% of a CU's cycles. On those prompts, in us: 1420 with
// split_rows (16 rows read K and V from L2), 269 with two K groups of 128 rows that met at every
// barrier, 203 as four waves per workgroup and two workgroups per CU, 178 with the numerators' sum on the
// matrix unit and the lagging maximum, the rest from forming maxima only where a score passes the limit.
//
// MODE 0: the rows of one sequence's new tokens over its visible chunks. Sequence b's tiles begin at
// index cu[b] gq / rows + b (n gq rows need at most one tile more than floor((cu + n) gq / rows) -
// floor(cu gq / rows)); a workgroup finds its sequence with a binary search. MODE 1: the rows of all
// tokens over the shared prefix.
constexpr float kLag = 8.0f;

// LDS bytes of block_rows: the ring, and the K groups' m and l per column tile and lane.
constexpr int block_lds(int hd, int cg, int kg, int s) { return kg * s * 2 * kChunkPos * hd * 2 + cg * kg * 4 * 64 * 4; }

// Block wg of the launch's tiles x kv heads, range split of it.
template <typename E, int HD, int CG, int KG, int S, int MODE>
__device__ __forceinline__ void block_rows(const PagedArgs& a, int wg, int split, unsigned char* lds) {
  typedef typename E::T T;
  typedef T T4 __attribute__((ext_vector_type(4)));
  constexpr int BT = 32 * CG, NS = HD / 32, NB = HD / 16;
  constexpr int KB = kChunkPos * HD * 2;  // bytes of a chunk's K (and of its V): NB tiles
  constexpr int LI = NB / CG;             // K (and V) tiles each wave loads per chunk
  constexpr bool AHEAD = S >= 4;          // deep enough to read the next chunk's K a step early
  static_assert(CG * LI == NB && S >= 2 && (LI == 1 || LI % 2 == 0), "whole loads per wave, two slots");
  static_assert(KG * S * 2 * KB >= (KG - 1) * CG * 2 * NB * 64 * 16, "the K groups meet in the ring");
  unsigned char* const ring = lds;
  float(*const mls)[4][64] = reinterpret_cast<float(*)[4][64]>(lds + KG * S * 2 * KB);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave / CG, cg = wave % CG;
  const int c16 = lane & 15, kb = lane >> 4;
  const int kvh = wg % a.nkv, tile = a.btiles - 1 - wg / a.nkv;  // longest blocks first
  const Block bk = find_block<MODE>(a, tile, BT);
  if (bk.rows <= 0) return;
  const int per = block_range(a, bk.n, KG);
  const int j0 = split * per;
  if (split && j0 >= bk.n) return;  // the first range runs with no chunk too: its rows are written
  const int nsteps = max(0, min(per, bk.n - j0));
  const int n = (nsteps + KG - 1) / KG;  // steps of a K group (the last ones may be dead)

  // this lane's two rows see the positions above hi - window up to hi, and those below sinks; rows past
  // the block's are not stored. thi, tlo: last and first of the column tiles (what V is kept of); all_hi,
  // all_lo: of the block (which chunks every row sees whole)
  const int window = a.window > 0 ? a.window : kAll;
  auto row_of = [&](int ct, int ln, int& tok, int& head) __attribute__((always_inline)) {
    const int r = bk.r0 + min(32 * cg + 16 * ct + (ln & 15), bk.rows - 1);
    tok = r / a.gq;
    head = kvh * a.gq + r % a.gq;
  };
  int hi[2], thi[2], tlo[2], all_hi, all_lo = 0;
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    int t, h;
    row_of(ct, lane, t, h);
    const int p = max(-1, MODE == 1 ? row_position(a, t) : bk.pos0 + t);
    const int l = max(0, p - window + 1);
    hi[ct] = p;
    // over the 16 rows (all four lane groups hold the same 16)
    int mx = p, mn = l;
#pragma unroll
    for (int off = 1; off < 16; off *= 2) {
      mx = max(mx, __shfl_xor(mx, off));
      mn = min(mn, __shfl_xor(mn, off));
    }
    thi[ct] = __builtin_amdgcn_readfirstlane(mx);
    tlo[ct] = __builtin_amdgcn_readfirstlane(mn);
  }
  if constexpr (MODE == 1) {
    int mn = kAll;
    for (int i = lane; i < bk.rows; i += 64) {
      const int p = row_position(a, (bk.r0 + i) / a.gq);
      mn = p < 0 ? mn : min(mn, p);  // rows without a position: the merge takes nothing of them
    }
#pragma unroll
    for (int off = 1; off < 64; off *= 2) mn = min(mn, __shfl_xor(mn, off));
    all_hi = __builtin_amdgcn_readfirstlane(mn);
  } else {
    all_hi = bk.first;
    all_lo = a.window > 0 ? max(0, bk.last - a.window + 1) : 0;
  }
  const int whi = max(thi[0], thi[1]), wlo = min(tlo[0], tlo[1]);  // of the wave's rows

  // the block's chunks in order: those that every row sees whole (fl .. fl + nf - 1), the sinks', the others
  const int fl = max(bk.lo, (all_lo + kChunkPos - 1) / kChunkPos);
  const int nf = max(0, min(bk.lo + bk.n - bk.cs, (min(all_hi, kAll - 1) + 1) / kChunkPos) - fl);
  auto chunk_of = [&](int j) __attribute__((always_inline)) {
    const int i = j0 + j * KG + kg;
    int d = i - nf - bk.cs + bk.lo < fl ? bk.lo - nf - bk.cs : bk.lo - bk.cs;
    d = i < nf + bk.cs ? -nf : d;
    return i + (i < nf ? fl : d);
  };
  // Step j of this K group loads from: the chunk's page, its id read through the scalar cache, and its place
  // in the page. No page (an id outside the pool, a step past the range): zeros are loaded
  const ScalarInts table = (ScalarInts)(uintptr_t)(MODE == 1 ? a.ptable : a.table + (int64_t)bk.b * a.ldt);
  const ScalarInts ptable = (ScalarInts)(uintptr_t)a.ptable;
  int page, sub;
  auto next_page = [&](int j) __attribute__((always_inline)) {
    const bool in = j * KG + kg < nsteps;
    const int c = in ? chunk_of(j) : 0;
    int at;
    chunk_page(a.cpp, c, at, sub);
    page = (MODE == 0 && c < a.pchunks ? ptable : table)[at];  // first used a step later
  };
  const uint32_t dma_off = (uint32_t)(c16 * 64 + kb * 16 + cg * LI * 1024);
  unsigned char* const kring = ring + kg * S * 2 * KB;
  unsigned char* const vring = kring + KB;
  auto usable = [&](int j) __attribute__((always_inline)) { return j * KG + kg < nsteps && (uint32_t)page < (uint32_t)a.pages; };
  // K or V of the chunk into slot j % S
  const char* const kpool = (const char*)a.k + (int64_t)kvh * a.cpp.n * KB;
  const char* const vpool = (const char*)a.vt + (int64_t)kvh * a.cpp.n * KB;
  const uint32_t kstride = (uint32_t)a.kps * 2, vstride = (uint32_t)a.vps * 2;  // bytes: below 2^32
  auto load = [&](const char* pool, uint32_t stride, unsigned char* slots, int j) __attribute__((always_inline)) {
    const bool ok = usable(j);
    const char* at = pool + (uint64_t)(ok ? (uint32_t)page : 0u) * stride + (uint32_t)sub * (uint32_t)KB;
    const u32x4 rs = raw_rsrc_uniform(at, ok ? KB : 0);
    unsigned char* const to = slots + (j % S) * 2 * KB + cg * LI * 1024;
    if constexpr (LI % 2 == 0) {
#pragma unroll
      for (int i = 0; i < LI; i += 2) dma_buffer16x2(rs, dma_off + i * 1024, dma_off + (i + 1) * 1024, lds_addr(to + i * 1024));
    } else {
      dma_buffer16(rs, dma_off, 0u, lds_addr(to));
    }
  };
  uint32_t have = 0;  // bit i: whether the step i before the last one loaded has a page
  int nfull = min((nsteps + KG - 1) / KG, max(0, nf - j0 - kg + KG - 1) / KG);  // unmasked steps: to the first without one
  auto loaded = [&](int j) __attribute__((always_inline)) {
    const bool ok = usable(j);
    have = __builtin_amdgcn_readfirstlane(have << 1 | (ok ? 1u : 0u));
    nfull = __builtin_amdgcn_readfirstlane(ok ? nfull : min(nfull, j));
    next_page(j + 1);
  };
  next_page(0);
#pragma unroll
  for (int j = 0; j < S - 1; ++j) {
    load(kpool, kstride, kring, j);
    load(vpool, vstride, vring, j);
    loaded(j);
  }

  // this wave's q operands: waited for here, once, so that the compiler has no load of its own left to
  // wait for inside the loop (its count does not know the loads to LDS)
  u32x4 q[2][NS];
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    int t, h;
    row_of(ct, lane, t, h);
    const T* src = (const T*)a.q + (int64_t)(bk.row0 + t) * a.ldq + (int64_t)h * HD + 8 * kb;
#pragma unroll
    for (int s = 0; s < NS; ++s) q[ct][s] = *reinterpret_cast<const u32x4*>(src + 32 * s);
  }
#pragma unroll
  for (int ct = 0; ct < 2; ++ct)
#pragma unroll
    for (int s = 0; s < NS; ++s) asm volatile("" : "+v"(q[ct][s]));

  const float sc = a.scale * 1.44269504088896341f;
  float m_run[2] = {-__builtin_inff(), -__builtin_inff()};
  float4_t sum[2];     // of the numerators as rounded, by a row of ones in the place of V^T: every element is row c16's
  float4_t o[2][NB];   // O^T[dim 16b + 4kb + r][row c16], unnormalised
  float4_t acc[2][2];  // [row half hb][column tile]: scores of positions 8kb + 4hb + r, less the row's maximum so far
  u32x4 ph[2];         // numerators: the B operand of P.V
#pragma unroll
  for (int ct = 0; ct < 2; ++ct)
#pragma unroll
    for (int b = 0; b < NB; ++b) o[ct][b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll
  for (int ct = 0; ct < 2; ++ct) sum[ct] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const u32x4 ones = {E::kOnes, E::kOnes, E::kOnes, E::kOnes};
  u32x4 kt[NB], vv[NB];  // a chunk's K and V, read ahead of the MFMAs before the ones that use them
  auto tiles = [&](u32x4 (&t)[NB], const unsigned char* src) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NB; ++i) t[i] = *reinterpret_cast<const u32x4*>(src + i * 1024 + lane * 16);
    __builtin_amdgcn_sched_barrier(0);
  };
  // the products are added to -m_run (0 while m_run is -inf), so that a row's exponents need no difference
  float4_t less[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
  auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int hb = 0; hb < 2; ++hb)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) acc[hb][ct] = E::mfma(kt[NS * hb + s], q[ct][s], s ? acc[hb][ct] : less[ct]);
  };
  auto pv = [&](auto maskedc, int cb0) __attribute__((always_inline)) {
    uint32_t mk[2][4];
    if constexpr (decltype(maskedc)::value) {  // zero V that no row of the tile sees (0 x NaN)
#pragma unroll
      for (int ct = 0; ct < 2; ++ct)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int p0 = cb0 + 8 * kb + 2 * e;
          mk[ct][e] = (p0 <= thi[ct] && (p0 >= tlo[ct] || p0 < a.sinks) ? 0x0000FFFFu : 0u) |
                      (p0 + 1 <= thi[ct] && (p0 + 1 >= tlo[ct] || p0 + 1 < a.sinks) ? 0xFFFF0000u : 0u);
        }
    }
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) sum[ct] = E::mfma(ones, ph[ct], sum[ct]);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int ct = 0; ct < 2; ++ct) {
        u32x4 v = vv[b];
        if constexpr (decltype(maskedc)::value)
          v = u32x4{v[0] & mk[ct][0], v[1] & mk[ct][1], v[2] & mk[ct][2], v[3] & mk[ct][3]};
        o[ct][b] = E::mfma(v, ph[ct], o[ct][b]);
      }
    __builtin_amdgcn_sched_barrier(0);
  };
  // The maximum that is subtracted may lag the largest score by kLag (in powers of two): the numerators
  // then reach 2^(kLag + kShift), inside every type, and the outputs are rescaled once or twice a block instead of
  // at most of its chunks (16 rows rarely all keep their maximum over a chunk).
  const float lag = kLag / sc;
  float limit[2] = {-__builtin_inff(), -__builtin_inff()};  // lag, -inf while m_run is
  auto softmax = [&](auto maskedc, int cb0) __attribute__((always_inline)) {
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
      float mc = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (decltype(maskedc)::value) {
          const int p = cb0 + 8 * kb + e;
          if (p > hi[ct] || (p <= hi[ct] - window && p >= a.sinks)) acc[e >> 2][ct][e & 3] = -__builtin_inff();
        }
        mc = fmaxf(mc, acc[e >> 2][ct][e & 3]);
      }
      if (__any(mc > limit[ct])) {  // of any lane: the rows' maxima are only formed here
        mc = max_xor32(max_xor16(mc));
        // a row that has seen nothing so far keeps m = -inf; its scores are less 0. One that keeps its
        // maximum keeps its sums to the bit
        const float old = less[ct][0], m_new = fmaxf(m_run[ct], mc - old);
        const float now = m_new == -__builtin_inff() ? 0.0f : -m_new, more = old - now;
        const float alpha = m_run[ct] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(-more * sc);
        sum[ct] *= alpha;
#pragma unroll
        for (int b = 0; b < NB; ++b) o[ct][b] *= alpha;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e >> 2][ct][e & 3] -= more;
        m_run[ct] = m_new;
        less[ct] = float4_t{now, now, now, now};
        limit[ct] = m_new == -__builtin_inff() ? m_new : lag;
      }
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[e >> 2][ct][e & 3], sc, E::kShift));
#pragma unroll
      for (int e = 0; e < 4; ++e) ph[ct][e] = pack2<E>(x[2 * e], x[2 * e + 1]);
    }
  };
  auto step = [&](auto maskedc, int j) __attribute__((always_inline)) {
    // stage j (and with a deep ring j + 1) has landed, and every wave is done with step j - 1, whose
    // slot takes stage j + S - 1
    wait_vm<AHEAD ? (S - 3) * 2 * LI : (S - 2) * 2 * LI>();
    ring_barrier();
    const int cb0 = chunk_of(j) * kChunkPos;
    const bool live = !decltype(maskedc)::value || ((have >> (S - 2) & 1) && cb0 <= whi && (cb0 + kChunkPos > wlo || cb0 < a.sinks));
    if (!AHEAD && live) tiles(kt, kring + (j % S) * 2 * KB);
    if (live) scores();
    load(kpool, kstride, kring, j + S - 1);
    if (live) {
      tiles(vv, vring + (j % S) * 2 * KB);
      softmax(maskedc, cb0);
    }
    load(vpool, vstride, vring, j + S - 1);
    loaded(j + S - 1);
    if (AHEAD) tiles(kt, kring + ((j + 1) % S) * 2 * KB);
    if (live) pv(maskedc, cb0);
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));  // lgkmcnt(0): no LDS read is left pending
  };
  wait_vm<0>();  // the first stages, with q
  ring_barrier();
  if (AHEAD) tiles(kt, kring);
  int j = 0;
  for (; j < nfull; ++j) step(IntC<0>(), j);
  for (; j < n; ++j) step(IntC<1>(), j);
  wait_vm<0>();
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));
  ring_barrier();  // the ring is free: every wave's loads have landed and its reads are done

  // ---- the K groups meet: groups past the first leave m, l and O, lane for lane
  const float l_w[2] = {sum[0][0], sum[1][0]};
  float4_t* const red = reinterpret_cast<float4_t*>(ring);  // [wave - CG][2 NB][64]
  if (kg > 0) {
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
      mls[wave][2 * ct][lane] = m_run[ct];
      mls[wave][2 * ct + 1][lane] = l_w[ct];
#pragma unroll
      for (int b = 0; b < NB; ++b) red[((wave - CG) * 2 * NB + NB * ct + b) * 64 + lane] = o[ct][b];
    }
  }
  lds_barrier();
  if (kg > 0) return;
  const bool direct = a.bdirect && bk.n <= per;  // a lone range
  float* const part = a.bpart + (((int64_t)tile * a.nkv + kvh) * a.bsplits + split) * BT * (2 + HD);
#pragma unroll
  for (int ct = 0; ct < 2; ++ct) {
    float mv[KG], lv[KG], M = m_run[ct];
    mv[0] = m_run[ct];
    lv[0] = l_w[ct];
#pragma unroll
    for (int g = 1; g < KG; ++g) {
      mv[g] = mls[cg + g * CG][2 * ct][lane];
      lv[g] = mls[cg + g * CG][2 * ct + 1][lane];
      M = fmaxf(M, mv[g]);
    }
    float f[KG], l = 0.0f;
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      f[g] = mv[g] != -__builtin_inff() ? __builtin_amdgcn_exp2f((mv[g] - M) * sc) : 0.0f;
      l = __builtin_fmaf(lv[g], f[g], l);
    }
    const int col = 32 * cg + 16 * ct + c16;
    int t, h, ln = lane;
    asm volatile("" : "+v"(ln));  // formed again here rather than kept in registers over the loop
    row_of(ct, ln, t, h);
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
          for (int r = 0; r < 4; ++r) y[r] = (T)(l != 0.0f ? v[r] / l : 0.0f);
          *reinterpret_cast<T4*>(dst + 16 * b) = y;
        } else {
          *reinterpret_cast<float4_t*>(pdst + 16 * b) = v;
        }
      }
    }
    if (!direct && kb == 0 && col < bk.rows) {
      part[2 * col] = M;
      part[2 * col + 1] = l;
    }
  }
}

template <typename E, int HD, int BT>
__global__ __launch_bounds__(kBlockThreads<BT>) __attribute__((amdgpu_waves_per_eu(2))) void paged_block_kernel(PagedArgs a) {
  constexpr int CG = BT / 32, KG = kBlockKG<BT>, S = kBlockSlots<BT>;
  __shared__ __align__(16) unsigned char lds[block_lds(HD, CG, KG, S)];
  block_rows<E, HD, CG, KG, S, 0>(a, (int)blockIdx.x, (int)blockIdx.y, lds);
}

// Behind a shared prefix: its blocks, which the matrix cores bound, and the sequences' own positions, which
// the memory does, in one launch, so that a CU runs some of each. Groups of 8 workgroups (one per XCD)
// are of one kind, the kinds spread evenly over the launch. 128 sequences of up to 900 positions behind
// 16384, 32/8 heads (205 MB, 35 GFLOP): 120 us in two launches, 104 in one, 95 now
// with the merge.
template <typename E, int HD, int BT>
__global__ __launch_bounds__(kBlockThreads<BT>) __attribute__((amdgpu_waves_per_eu(2))) void paged_prefix_kernel(PagedArgs a) {
  constexpr int CG = BT / 32, KG = kBlockKG<BT>, S = kBlockSlots<BT>, NW = kBlockThreads<BT> / 64;
  constexpr int kBlockLds = block_lds(HD, CG, KG, S), kSplitLds = split_lds(HD, NW);
  __shared__ __align__(16) unsigned char lds[kBlockLds > kSplitLds ? kBlockLds : kSplitLds];
  const int tiles = a.btiles * a.nkv, nblock = tiles * a.bsplits;
  const int64_t gb = (nblock + 7) / 8, gs = (a.slots * a.nkv * a.nt + 7) / 8, g = blockIdx.x / 8;
  const int before = (int)(g * gb / (gb + gs));  // block groups before this one
  if ((g + 1) * gb / (gb + gs) > before) {
    const int wg = before * 8 + (int)(blockIdx.x % 8);
    if (wg < nblock) block_rows<E, HD, CG, KG, S, 1>(a, wg % tiles, wg / tiles, lds);
  } else {
    const int wg = (int)(g - before) * 8 + (int)(blockIdx.x % 8);
    if (wg < a.slots * a.nkv * a.nt) split_rows<E, HD, NW>(a, wg, lds);
  }
}

// ---- joining the ranges of one (token, query head)
//
// Rows come from paged_split_kernel's slots, from paged_block_kernel's splits, or (behind a shared
// prefix) from both; ones whose only range has written the output are left alone. A wave per row takes
// 2 or 4 ranges at once, lane d of a range's dims 4d on (one range at once, 509 tokens of 14/2 heads of 64
// in 13 ranges each: 77 us for attention and merge instead of 74; four heads of a token per wave: 128
// sequences behind 16384 positions 107 us instead of 97). Where rows are few, WR = 8 waves per row take
// ranges w, w + 8, ..., one at once, and meet in LDS (as above: 10.2 us instead of 10.0).
constexpr int kMergeWaves = 8;  // of a workgroup

template <typename E, int HD, int WR, int BT>
__global__ __launch_bounds__(kMergeWaves * 64) void paged_merge_kernel(PagedArgs a) {
  typedef typename E::T T;
  constexpr int VL = WR == 1 ? 4 : HD / 64, LR = HD / VL, G = 64 / LR;  // dims per lane, lanes per range, ranges at once
  typedef T out_t __attribute__((ext_vector_type(VL)));
  typedef float vec_t __attribute__((ext_vector_type(VL)));
  __shared__ float ms[kMergeWaves], ls[kMergeWaves];
  __shared__ __align__(16) vec_t os[kMergeWaves][LR];
  const int lane = threadIdx.x & 63, ld = lane % LR;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w = wave % WR;
  const int64_t item = (int64_t)blockIdx.x * (kMergeWaves / WR) + wave / WR;
  const int t = (int)(item / a.nq), h = (int)(item % a.nq);
  int b = t;
  bool run = t < a.T;
  if (run && a.cu) {
    b = -1;
    for (int lo = 0, hi = a.B; lo < hi;) {
      const int mid = (lo + hi) / 2;
      if (a.cu[mid] <= t)
        b = mid, lo = mid + 1;
      else
        hi = mid;
    }
    run = b >= 0;
  }
  SeqRows s{};
  if (run) s = seq_rows(a.cu, a.kv_lens, b, a.T);
  const int tok = t - s.row0;
  run = run && tok < min(s.n, a.max_q);
  const bool nothing = s.pos0 + tok < 0;  // zeros
  int first = 0, na = 0;
  if (run && a.slots) {
    first = a.plan[2 * b];
    na = nothing ? 0 : a.plan[2 * b + 1];
    run = a.skip || a.plan[2 * b + 1] > 1;
  }
  if (WR == 1 && !run) return;
  const float sc = a.scale * 1.44269504088896341f;
  const int kvh = h / a.gq, row = tok * a.gq + h % a.gq;
  // the two lists: {m, l} and outputs of range i at p + i * step (the tiles' first range at p0)
  const int64_t sa = (int64_t)a.nkv * a.nt * part_floats(HD);
  auto part = [&](int split) { return a.part + (part_at(a, b, s.row0, first, split, row / kRows) * a.nkv + kvh) * part_floats(HD); };
  const float *p0 = part(0), *pa = part(1) - sa;
  const float* pb = nullptr;
  int nb = 0, jb = 0;
  if (run && a.bsplits && !nothing) {
    int tile, n;
    if (a.bdirect) {
      tile = (int)(s.row0 * (int64_t)a.gq / BT) + b + row / BT;
      n = sequence_block(a, b, s, row / BT * BT, BT).n;
      jb = row % BT;
    } else {
      const int r = t * a.gq + h % a.gq;
      tile = r / BT;
      n = a.pchunks;
      jb = r % BT;
    }
    const int per = block_range(a, n, kBlockKG<BT>);
    nb = (n + per - 1) / per;
    run = !a.bdirect || nb > 1;
    pb = a.bpart + ((int64_t)tile * a.nkv + kvh) * a.bsplits * BT * (2 + HD);
  }
  if (WR == 1 && !run) return;
  float M = -__builtin_inff(), l = 0.0f;
  vec_t o = vec_t(0.0f);
  // the factor from maximum m to mn
  auto factor = [&](float m, float mn) __attribute__((always_inline)) {
    return m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * sc);
  };
  if (run) {
#pragma unroll 4
    for (int r = w * G + lane / LR; r < na + nb; r += WR * G) {
      const bool split = r < na;
      const float* p = split ? (r ? pa + r * sa : p0) : pb + (int64_t)(r - na) * BT * (2 + HD);
      const int j = split ? row % kRows : jb, rows = split ? kRows : BT;
      const float m = p[2 * j], lr = p[2 * j + 1];
      const vec_t v = *reinterpret_cast<const vec_t*>(p + 2 * rows + j * HD + VL * ld);
      const float mn = fmaxf(M, m), f0 = factor(M, mn), f1 = factor(m, mn);
      l = l * f0 + lr * f1;
#pragma unroll
      for (int i = 0; i < VL; ++i) o[i] = __builtin_fmaf(v[i], f1, o[i] * f0);
      M = mn;
    }
  }
  if constexpr (G > 1) {  // the wave's groups of lanes meet
    const float mn = max_xor32(G == 4 ? max_xor16(M) : M), f = factor(M, mn);
    l *= f, o *= f;
#pragma unroll
    for (int off = LR; off < 64; off *= 2) {
      l += __shfl_xor(l, off);
#pragma unroll
      for (int i = 0; i < VL; ++i) o[i] += __shfl_xor(o[i], off);
    }
  }
  if constexpr (WR > 1) {
    if (lane == 0) {
      ms[wave] = M;
      ls[wave] = l;
    }
    os[wave][ld] = o;
    __syncthreads();
    if (!run || w) return;
    float mn = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < WR; ++i) mn = fmaxf(mn, ms[wave + i]);
    l = 0.0f, o = vec_t(0.0f);
#pragma unroll
    for (int i = 0; i < WR; ++i) {
      const float fw = factor(ms[wave + i], mn);
      l = __builtin_fmaf(ls[wave + i], fw, l);
      const vec_t v = os[wave + i][ld];
#pragma unroll
      for (int d = 0; d < VL; ++d) o[d] = __builtin_fmaf(v[d], fw, o[d]);
    }
  }
  if (lane >= LR) return;
  out_t y;
#pragma unroll
  for (int i = 0; i < VL; ++i) y[i] = (T)bounded<E>(l != 0.0f ? o[i] / l : 0.0f);
  *reinterpret_cast<out_t*>((T*)a.out + (int64_t)t * a.ldo + (int64_t)h * HD + VL * ld) = y;
}

// Up to this many chunks a sequence is one range, with nothing to merge; and up to kSingleMany where the
// sequences alone are workgroups for half of the CUs (one streams about 70 GB/s). Graph-timed, one range /
// ranges and merge, us: 1 sequence of 12/2 heads at 300 positions 8.1 / 10.3, 600 9.7 / 10.4, 1100 13.6 / 10.5;
// 64 of 28/4 at 1050 29 / 40.
constexpr int kSingle = 20, kSingleMany = 36;
// More sequences than a wave's lanes have their ranges found by paged_plan_kernel, a launch before: every wave's
// own search grows with the batch. Graph-timed, own search / launch, us: 28/4 heads, 200 to 1000 positions, 96
// sequences 37 / 35, 256 72 / 60, 1024 437 / 244, 4096 4119 / 949; 100 to 4000 positions, 96 78 / 79, 512 404 / 370.
constexpr int kPlanSeqs = 64;

Plan make_plan(int64_t T, int64_t B, int64_t max_q, int64_t max_len, int64_t window, int64_t sinks, int64_t prefix_len,
               int nq, int nkv, int hd) {
  Plan p;
  const int64_t gq = nq / nkv, rows = T * gq;
  // a sequence's rows past two tiles share K and V in LDS; those that fill a block do so behind a prefix too, and
  // with them every other sequence's of the call (127 tokens and a chunk of 64 behind 16384, 32/8 heads: 828 us; 128
  // tokens 111)
  const bool block = max_q * gq > (prefix_len ? 128 : 2 * kRows);
  p.apart = prefix_len && !block;
  if (!block) {
    p.nt = (max_q * gq + kRows - 1) / kRows;
    if (!prefix_len && most_chunks(max_len, max_q, window, sinks) <= (B * nkv * p.nt >= 128 ? kSingleMany : kSingle)) {
      p.slots = B;
      return p;
    }
    // As many workgroups as run at once (a CU holds one of head_dim 128, two of 64) where that leaves half as
    // many ranges again as there are sequences. Else a range is at most two thirds of what a CU would
    // have to read (all of it behind a prefix, whose blocks keep the CUs busy too): with half of it / all, 64
    // sequences of up to 16000 positions 85 / 92 us against 80, 100 of up to 4000 30 / 26 against 25
    const int64_t w = nkv * p.nt, round = (hd == 128 ? 256 : 512) / w;
    p.spare = 2 * round >= 3 * B ? 0 : std::max<int64_t>(1, (prefix_len ? 256 : 384) / w);
    p.slots = p.spare ? B + p.spare : round;
    p.mapped = p.spare && B > kPlanSeqs;
    p.part_bytes = p.slots * w * part_floats(hd) * 4;
  }
  if (block || p.apart) {
    // 128 rows where the sequences have about as many, else 64; split for two workgroups of 128 rows a CU (three
    // of head_dim 64), or one of 64. With 384 / 512 / 640 workgroups of 128 rows, us: 200 tokens after 10000
    // positions, 28/4 heads, 56 / 51 / 60, 300 after 6000, 32/8, 65 / 54 / 62; with 512 / 768 / 896 of head_dim 64: 509
    // after 20000, 16/16, 75 / 71 / 84. With 192 / 320 / 448 of 64 rows: 4 times 10 after 5000, 32/8, 29 / 26 / 36, 50
    // after 8000, 16/16 of 64, 18 / 17 / 24. With 2 kv heads, where 32 ranges are the limit, all alike. Not split
    // where they are a third as many unsplit: the merge then costs more than fuller CUs save (2 prompts of
    // 1500, 14/2 heads of 64, in one range / two: 34 / 68 us)
    auto tiles = [&](int bt) { return p.apart ? (rows + bt - 1) / bt : rows / bt + B; };
    p.bt = rows >= 96 * (p.apart ? 1 : B) ? 128 : 64;
    p.btiles = tiles(p.bt);
    const int64_t fill = p.bt == 64 ? 320 : hd == 128 ? 512 : 768;
    const int64_t whole = nkv * p.btiles;
    p.bsplits = !p.apart && 3 * whole >= fill ? 1 : std::max<int64_t>(1, std::min<int64_t>(32, fill / whole));
    if (p.apart || p.bsplits > 1) p.bpart_bytes = p.btiles * nkv * p.bsplits * p.bt * (2 + hd) * 4;
  }
  p.bytes = workspace_bytes(p, B);
  return p;
}

template <typename E, int HD, int BT>
int launch_rows(const PagedArgs& a, const Plan& p, hipStream_t s) {
  if (a.skip) {
    const int64_t groups = (p.btiles * a.nkv * p.bsplits + 7) / 8 + (p.slots * a.nkv * p.nt + 7) / 8;
    paged_prefix_kernel<E, HD, BT><<<(unsigned)(8 * groups), kBlockThreads<BT>, 0, s>>>(a);
  } else {
    paged_block_kernel<E, HD, BT><<<dim3((unsigned)(p.btiles * a.nkv), (unsigned)p.bsplits), kBlockThreads<BT>, 0, s>>>(a);
  }
  return ldk::check_launch("paged_attention block");
}

template <typename E, int HD>
int launch(const PagedArgs& a, const Plan& p, int dtype, hipStream_t s) {
  (void)hipGetLastError();
  int st;
  if (p.mapped && (st = paged_find_ranges(a, s))) return st;
  if (p.bt) {
    st = p.bt == 128 ? launch_rows<E, HD, 128>(a, p, s) : launch_rows<E, HD, 64>(a, p, s);
  } else {
    paged_split_kernel<E, HD, 8><<<(unsigned)(p.slots * a.nkv * p.nt), 8 * 64, 0, s>>>(a);
    st = ldk::check_launch("paged_attention split");
  }
  if (st || !p.bytes) return st;  // no bytes: no sequence has more than one range
  return paged_join(a, dtype, HD, p.bt, s);
}

template <typename E, int HD>
int join(const PagedArgs& a, int64_t bt, hipStream_t s) {
  const bool few = (int64_t)a.T * a.nq < 512;
  const int64_t waves = (int64_t)a.T * a.nq * (few ? kMergeWaves : 1);
  const unsigned grid = (unsigned)((waves + kMergeWaves - 1) / kMergeWaves);
  if (bt == 128)
    few ? paged_merge_kernel<E, HD, kMergeWaves, 128><<<grid, kMergeWaves * 64, 0, s>>>(a)
        : paged_merge_kernel<E, HD, 1, 128><<<grid, kMergeWaves * 64, 0, s>>>(a);
  else
    few ? paged_merge_kernel<E, HD, kMergeWaves, 64><<<grid, kMergeWaves * 64, 0, s>>>(a)
        : paged_merge_kernel<E, HD, 1, 64><<<grid, kMergeWaves * 64, 0, s>>>(a);
  return ldk::check_launch("paged_attention merge");
}

int run(const char* fn, const void* q, int64_t ldq, int dtype, const int32_t* cu, const int32_t* kv_lens,
        const int32_t* table, int64_t ldt, int64_t max_pages, const int32_t* ptable, int64_t prefix_len, const void* k,
        int64_t kps, const void* vt, int64_t vps, int64_t num_pages, int64_t page_size, void* out, int64_t ldo, int64_t T,
        int64_t B, int64_t max_q, int nq, int nkv, int hd, int64_t window, int64_t sinks, float scale, void* ws,
        int64_t ws_bytes, void* stream) {
  if (!q || !kv_lens || !table || !k || !vt || !out || (prefix_len && !ptable)) return ldk::fail(LDK_ERR_INVALID, "%s: null pointer", fn);
  if (dtype != LDK_F16 && dtype != LDK_BF16) return ldk::fail(LDK_ERR_INVALID, "%s: dtype %d (fp16 or bf16)", fn, dtype);
  if (hd != 64 && hd != 128) return ldk::fail(LDK_ERR_UNSUPPORTED, "%s: head_dim=%d (64 or 128)", fn, hd);
  if (nq <= 0 || nkv <= 0 || nq % nkv || nq > 4096)
    return ldk::fail(LDK_ERR_INVALID, "%s: nq=%d must be a positive multiple of nkv=%d (at most 4096)", fn, nq, nkv);
  if (T <= 0 || T > (int64_t(1) << 24) || B <= 0 || B > 65535)
    return ldk::fail(LDK_ERR_INVALID, "%s: T=%lld tokens (1..2^24) of B=%lld sequences (1..65535)", fn, (long long)T, (long long)B);
  if (!cu && T < B) return ldk::fail(LDK_ERR_INVALID, "%s: T=%lld rows for B=%lld sequences of one token", fn, (long long)T, (long long)B);
  if (max_q <= 0 || max_q > T) return ldk::fail(LDK_ERR_INVALID, "%s: max_q=%lld outside 1..%lld", fn, (long long)max_q, (long long)T);
  if (page_size < 32 || page_size % 32 || page_size > 65536)
    return ldk::fail(LDK_ERR_UNSUPPORTED, "%s: page_size=%lld must be a multiple of 32 up to 65536", fn, (long long)page_size);
  if (num_pages <= 0 || num_pages > INT32_MAX || max_pages <= 0 || ldt < max_pages || max_pages > ldk::kMaxPositions / page_size)
    return ldk::fail(LDK_ERR_INVALID, "%s: num_pages=%lld max_pages=%lld ldt=%lld", fn, (long long)num_pages, (long long)max_pages, (long long)ldt);
  if (prefix_len < 0 || prefix_len % page_size || prefix_len > max_pages * page_size)
    return ldk::fail(LDK_ERR_INVALID, "%s: prefix_len=%lld must be whole pages of %lld, at most the tables' %lld", fn,
                     (long long)prefix_len, (long long)page_size, (long long)max_pages);
  if (window < 0 || sinks < 0) return ldk::fail(LDK_ERR_INVALID, "%s: window=%lld sinks=%lld", fn, (long long)window, (long long)sinks);
  if (!(scale > 1e-20f && scale < 1e20f)) return ldk::fail(LDK_ERR_INVALID, "%s: scale=%g must be positive", fn, (double)scale);
  const int64_t per = (int64_t)nkv * page_size * hd;
  if (kps > INT32_MAX || vps > INT32_MAX) return ldk::fail(LDK_ERR_UNSUPPORTED, "%s: page strides %lld %lld past 2^31", fn, (long long)kps, (long long)vps);
  if (kps < per || vps < per || ldq < (int64_t)nq * hd || ldo < (int64_t)nq * hd)
    return ldk::fail(LDK_ERR_INVALID, "%s: strides ldq=%lld ldo=%lld pages %lld %lld below what they step over", fn,
                     (long long)ldq, (long long)ldo, (long long)kps, (long long)vps);
  if (!ldk::aligned(q, 16) || !ldk::aligned(out, 16) || !ldk::aligned(k, 16) || !ldk::aligned(vt, 16) || ldq % 8 ||
      ldo % 8 || kps % 8 || vps % 8 || !ldk::aligned(kv_lens, 4) || !ldk::aligned(cu, 4) || !ldk::aligned(table, 4) ||
      !ldk::aligned(ptable, 4) || !ldk::aligned(ws, 16))
    return ldk::fail(LDK_ERR_ALIGN, "%s: q, out, workspace and the pages 16-byte aligned with strides of multiples of 8 elements", fn);
  const Plan p = make_plan(cu ? T : B, B, cu ? max_q : 1, max_pages * page_size, window, sinks, prefix_len, nq, nkv, hd);
  if (p.bytes > 0 && (!ws || ws_bytes < p.bytes))
    return ldk::fail(LDK_ERR_INVALID, "%s: workspace of %lld bytes, this call needs %lld", fn, (long long)ws_bytes, (long long)p.bytes);
  if (!launchable(p, T, nq, nkv)) return ldk::fail(LDK_ERR_UNSUPPORTED, "%s: T=%lld rows of nq=%d heads are too many for a launch", fn, (long long)T, nq);
  const int big = 1 << 30;  // a window or sinks past every position
  PagedArgs a{};
  a.q = q, a.ldq = ldq, a.out = out, a.ldo = ldo;
  a.cu = cu, a.kv_lens = kv_lens, a.table = table, a.ptable = ptable, a.ldt = ldt;
  a.k = k, a.vt = vt, a.kps = kps, a.vps = vps;
  lay_out(a, p, ws, B);
  a.T = cu ? (int)T : (int)B, a.B = (int)B, a.max_q = cu ? (int)max_q : 1;
  a.nq = nq, a.nkv = nkv, a.gq = nq / nkv, a.nt = (int)p.nt;
  a.pages = (int)num_pages, a.cpp = page_div(page_size / kChunkPos), a.cap = (int)(max_pages * page_size);
  a.pchunks = (int)(prefix_len / kChunkPos), a.skip = p.apart ? a.pchunks : 0;
  a.window = (int)std::min<int64_t>(window, big), a.sinks = (int)std::min<int64_t>(sinks, big);
  a.slots = (int)p.slots, a.spare = (int)p.spare;
  a.btiles = (int)p.btiles, a.bsplits = (int)p.bsplits, a.bdirect = !p.apart;
  a.scale = scale;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == LDK_F16) return hd == 128 ? launch<ldk::F16, 128>(a, p, dtype, s) : launch<ldk::F16, 64>(a, p, dtype, s);
  return hd == 128 ? launch<ldk::BF16, 128>(a, p, dtype, s) : launch<ldk::BF16, 64>(a, p, dtype, s);
}

}  // namespace

namespace ldk {

int paged_find_ranges(const PagedArgs& a, hipStream_t s) {
  paged_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
  return check_launch("paged_attention plan");
}

int paged_join(const PagedArgs& a, int dtype, int hd, int64_t bt, hipStream_t s) {
  if (dtype == LDK_F16) return hd == 128 ? join<F16, 128>(a, bt, s) : join<F16, 64>(a, bt, s);
  return hd == 128 ? join<BF16, 128>(a, bt, s) : join<BF16, 64>(a, bt, s);
}

}  // namespace ldk

extern "C" int64_t ldk_paged_attention_workspace_bytes(int64_t T, int64_t B, int64_t max_q, int64_t max_len, int64_t window,
                                                       int64_t sinks, int64_t prefix_len, int nq, int nkv, int head_dim) {
  if (T <= 0 || T > (int64_t(1) << 24) || B <= 0 || B > 65535 || max_q <= 0 || max_q > (int64_t(1) << 24) || max_len <= 0 ||
      max_len > ldk::kMaxPositions || window < 0 || sinks < 0 || prefix_len < 0 || nq <= 0 || nkv <= 0 || nq % nkv ||
      nq > 4096 || (head_dim != 64 && head_dim != 128)) {
    return -ldk::fail(LDK_ERR_INVALID,
                      "paged_attention_workspace_bytes: T=%lld B=%lld max_q=%lld max_len=%lld window=%lld sinks=%lld "
                      "prefix_len=%lld nq=%d nkv=%d head_dim=%d",
                      (long long)T, (long long)B, (long long)max_q, (long long)max_len, (long long)window, (long long)sinks,
                      (long long)prefix_len, nq, nkv, head_dim);
  }
  return make_plan(T, B, max_q, max_len, window, sinks, prefix_len, nq, nkv, head_dim).bytes;
}

extern "C" int ldk_paged_attention(const void* q, int64_t ldq, int dtype, const int32_t* cu_seqlens,
                                   const int32_t* kv_lens, const int32_t* block_table, int64_t ldt, int64_t max_pages,
                                   const void* k_pages, int64_t k_page_stride, const void* vt_pages,
                                   int64_t vt_page_stride, int64_t num_pages, int64_t page_size, void* out, int64_t ldo,
                                   int64_t T, int64_t B, int64_t max_q, int nq, int nkv, int head_dim, int64_t window,
                                   int64_t sinks, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  return run("paged_attention", q, ldq, dtype, cu_seqlens, kv_lens, block_table, ldt, max_pages, nullptr, 0, k_pages,
             k_page_stride, vt_pages, vt_page_stride, num_pages, page_size, out, ldo, T, B, max_q, nq, nkv, head_dim, window,
             sinks, scale, workspace, workspace_bytes, stream);
}

extern "C" int ldk_shared_prefix_attention(const void* q, int64_t ldq, int dtype, const int32_t* cu_seqlens,
                                           const int32_t* kv_lens, const int32_t* block_table, int64_t ldt,
                                           int64_t max_pages, const int32_t* prefix_table, int64_t prefix_len,
                                           const void* k_pages, int64_t k_page_stride, const void* vt_pages,
                                           int64_t vt_page_stride, int64_t num_pages, int64_t page_size, void* out,
                                           int64_t ldo, int64_t T, int64_t B, int64_t max_q, int nq, int nkv, int head_dim,
                                           float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  return run("shared_prefix_attention", q, ldq, dtype, cu_seqlens, kv_lens, block_table, ldt, max_pages, prefix_table,
             prefix_len, k_pages, k_page_stride, vt_pages, vt_page_stride, num_pages, page_size, out, ldo, T, B, max_q, nq,
             nkv, head_dim, 0, 0, scale, workspace, workspace_bytes, stream);
}

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
// take nothing wider), their sum is taken from the unrounded values.
//
// Ranges. The lengths are on the device, so the split is made there: every sequence has its visible
// chunks (those of the sinks, then those of the window) cut into ranges of `per` chunks, one `per` for
// the whole batch such that all ranges fit the launch's slots; a ragged batch gets ranges of equal
// work. Each wave finds its slot's sequence from the lengths alone. Sequences with more than one
// range leave {max, sum} and the unnormalised output in the workspace, and paged_merge_kernel, the
// next launch on the stream, joins them.
#include <algorithm>

#include "paged.h"

namespace {

using namespace ldk;

struct PagedArgs {
  const void* q;
  int64_t ldq;
  const int32_t *cu, *kv_lens, *table, *ptable;  // ptable: the shared prefix's pages
  int64_t ldt;
  const void *k, *vt;
  int64_t kps, vps;  // page strides, elements
  void* out;
  int64_t ldo;
  float* part;    // partials, per (slot, kv head, tile): [16 rows]{m, l} and [16 rows][hd]
  int32_t* plan;  // [B][2]: first slot and ranges of every sequence
  int T, B, max_q, nq, nkv, gq, nt;  // nt: 16-row tiles of a sequence
  int pages, cpp, cap;               // cpp: chunks per page; cap: positions a sequence can hold
  int pchunks;                       // chunks of the shared prefix
  int window, sinks, slots;
  float scale;
};

constexpr int kRows = 16;
constexpr int kMinRange = 4;     // chunks of a range, at least
constexpr int kMaxRanges = 128;  // ranges of a sequence

// The visible chunks of a sequence's new tokens: cs chunks from 0 (the sinks), then those from lo on.
struct Span {
  SeqRows s;
  int cs, lo, n;
};
__device__ __forceinline__ Span seq_span(const PagedArgs& a, int b) {
  Span x;
  x.s = seq_rows(a.cu, a.kv_lens, b, a.T);
  x.s.n = min(x.s.n, a.max_q);
  const int hi = min(x.s.pos0 + x.s.n - 1, a.cap - 1);  // the last position that a row sees
  const int hc = hi < 0 || x.s.n <= 0 ? 0 : hi / kChunkPos + 1;
  x.lo = a.window > 0 ? max(0, x.s.pos0 - a.window + 1) / kChunkPos : 0;
  x.lo = min(x.lo, hc);
  x.cs = min((min(a.sinks, a.cap) + kChunkPos - 1) / kChunkPos, x.lo);
  x.n = x.cs + hc - x.lo;
  return x;
}

__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor((long long)v, off);
  return v;
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off));
  return v;
}

// The sequence and range of a slot: every wave forms it from the lengths of the whole batch. Every
// sequence has at least one range (its rows have to be written); sum over b of max(1, ceil(n_b / per))
// <= B + total / per <= slots.
struct Slot {
  int b, split, ranges, first, per;  // b < 0: none
};
__device__ __forceinline__ Slot find_slot(const PagedArgs& a, int slot, int lane) {
  const int each = (a.B + 63) / 64, b0 = lane * each, b1 = min(b0 + each, a.B);
  int64_t sum = 0;
  int most = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = seq_span(a, b).n;
    sum += n;
    most = max(most, n);
  }
  sum = wave_sum64(sum);
  most = wave_max_i(most);
  const int spare = a.slots - a.B;
  int64_t per = (sum + spare - 1) / spare;
  per = max(per, (int64_t)max(kMinRange, (most + kMaxRanges - 1) / kMaxRanges));
  Slot r{-1, 0, 1, 0, (int)per};
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += max(1, (seq_span(a, b).n + r.per - 1) / r.per);
  int end = mine;  // inclusive scan over the lanes
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int v = __shfl_up(end, off);
    if (lane >= off) end += v;
  }
  int at = end - mine;
  const uint64_t has = __ballot(slot >= at && slot < end);
  if (!has) return r;
  for (int b = b0; b < b1; ++b) {
    const int n = max(1, (seq_span(a, b).n + r.per - 1) / r.per);
    if (slot >= at && slot < at + n) {
      r.b = b;
      r.split = slot - at;
      r.ranges = n;
      r.first = at;
    }
    at += n;
  }
  const int src = __builtin_ctzll(has);
  r.b = __builtin_amdgcn_readlane(r.b, src);
  r.split = __builtin_amdgcn_readlane(r.split, src);
  r.ranges = __builtin_amdgcn_readlane(r.ranges, src);
  r.first = __builtin_amdgcn_readlane(r.first, src);
  return r;
}

__device__ __forceinline__ float max_xor16(float v) {
  auto p = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(p[0]), u2f(p[1]));
}
__device__ __forceinline__ float max_xor32(float v) {
  auto p = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(p[0]), u2f(p[1]));
}

// Floats of one partial: 16 rows of {m, l} and of hd outputs.
constexpr int part_floats(int hd) { return kRows * (2 + hd); }

template <typename E, int HD, int NW>
__global__ __launch_bounds__(NW * 64) void paged_split_kernel(PagedArgs a) {
  typedef typename E::T T;
  constexpr int NS = HD / 32, NB = HD / 16;  // K dim steps, V dim blocks
  __shared__ float mw[NW][kRows], lw[NW][kRows];
  __shared__ __align__(16) float ow[NW][kRows][HD];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, kb = lane >> 4;
  const int xy = a.nkv * a.nt, bxy = (int)blockIdx.x % xy;
  const int kvh = bxy % a.nkv, tile = bxy / a.nkv;
  const Slot sl = find_slot(a, (int)blockIdx.x / xy, lane);
  if (sl.b < 0) return;
  const Span sp = seq_span(a, sl.b);
  if (kvh == 0 && tile == 0 && sl.split == 0 && tid == 0) {
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
  float m_run = -__builtin_inff(), l_lane = 0.0f;
  float4_t o[NB];  // O[rows 4kb .. 4kb+3][dim 16b + c16], unnormalised
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const int32_t* trow = a.table + (int64_t)sl.b * a.ldt;
  const int jend = min((sl.split + 1) * sl.per, sp.n);
  const uint32_t lane_off = (uint32_t)(c16 * 64 + kb * 16);
  const uint32_t chunk_bytes = kChunkPos * HD * 2;
  for (int j = sl.split * sl.per + wave; j < jend; j += NW) {
    const int c = j < sp.cs ? j : j - sp.cs + sp.lo;
    const int cb = c * kChunkPos;
    if (cb > thi || (cb + kChunkPos <= tlo && cb >= a.sinks)) continue;
    const int page = c < a.pchunks ? a.ptable[c / a.cpp] : trow[c / a.cpp];
    if (page < 0 || page >= a.pages) continue;
    const int64_t in_page = ((int64_t)kvh * a.cpp + c % a.cpp) * (kChunkPos * HD);
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
    // a row that has seen nothing so far keeps m = -inf; its exponents are taken against 0
    const float base = m_new == -__builtin_inff() ? 0.0f : m_new * sc;
    const float alpha = __builtin_amdgcn_exp2f(__builtin_fmaf(m_run, sc, -base));
    m_run = m_new;
    float ls = 0.0f, x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e], sc, -base));
      ls += x[e];
    }
    u32x4 pa;
#pragma unroll
    for (int e = 0; e < 4; ++e) pa[e] = pack2<E>(x[2 * e], x[2 * e + 1]);
    l_lane = __builtin_fmaf(l_lane, alpha, ls);
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
#pragma unroll
      for (int b = 0; b < NB; ++b) o[b][r] *= al;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = E::mfma(pa, vr[b], o[b]);
  }

  // ---- the waves meet
  const float l_w = add_xor32(add_xor16(l_lane));
  if (kb == 0) {
    mw[wave][c16] = m_run;
    lw[wave][c16] = l_w;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (4 * kb + r < rows) {
#pragma unroll
      for (int b = 0; b < NB; ++b) ow[wave][4 * kb + r][16 * b + c16] = o[b][r];
    }
  lds_barrier();
  float* part = a.part + (int64_t)blockIdx.x * part_floats(HD);
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
    if (sl.ranges == 1) {
      const int g = tile * kRows + j;
      T* dst = (T*)a.out + (int64_t)(sp.s.row0 + g / a.gq) * a.ldo + (int64_t)(kvh * a.gq + g % a.gq) * HD;
      dst[d] = (T)(l > 0.0f ? v / l : 0.0f);
    } else {
      part[2 * kRows + e] = v;
      if (d == 0) {
        part[2 * j] = M;
        part[2 * j + 1] = l;
      }
    }
  }
}

// Joins the ranges of one (token, query head): a workgroup per row, wave w the ranges w, w + NW, ...,
// lane d the dims d and d + 64.
constexpr int kMergeWaves = 8;

template <typename E, int HD>
__global__ __launch_bounds__(kMergeWaves * 64) void paged_merge_kernel(PagedArgs a) {
  typedef typename E::T T;
  constexpr int ND = HD / 64;
  __shared__ float ms[kMergeWaves], ls[kMergeWaves], os[kMergeWaves][HD];
  const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = a.plan[2 * b], n = a.plan[2 * b + 1];
  if (n <= 1) return;
  const SeqRows s = seq_rows(a.cu, a.kv_lens, b, a.T);
  const int tok = blockIdx.x;
  if (tok >= min(s.n, a.max_q)) return;
  const int kvh = h / a.gq, row = tok * a.gq + h % a.gq, tile = row / kRows, j = row % kRows;
  const float sc = a.scale * 1.44269504088896341f;
  const int64_t step = (int64_t)a.nkv * a.nt * part_floats(HD);
  const float* p0 = a.part + ((int64_t)first * a.nkv * a.nt + tile * a.nkv + kvh) * part_floats(HD);
  float M = -__builtin_inff(), l = 0.0f, o[ND] = {};
  for (int r = wave; r < n; r += kMergeWaves) {
    const float* p = p0 + r * step;
    const float m = p[2 * j], lr = p[2 * j + 1];
    const float mn = fmaxf(M, m);
    const float f0 = M == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((M - mn) * sc);
    const float f1 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * sc);
    l = l * f0 + lr * f1;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] = o[i] * f0 + p[2 * kRows + j * HD + lane + 64 * i] * f1;
    M = mn;
  }
  if (lane == 0) {
    ms[wave] = M;
    ls[wave] = l;
  }
#pragma unroll
  for (int i = 0; i < ND; ++i) os[wave][lane + 64 * i] = o[i];
  __syncthreads();
  for (int d = threadIdx.x; d < HD; d += kMergeWaves * 64) {
    float MM = -__builtin_inff(), L = 0.0f, v = 0.0f;
    for (int w = 0; w < kMergeWaves; ++w) MM = fmaxf(MM, ms[w]);
    for (int w = 0; w < kMergeWaves; ++w) {
      const float f = ms[w] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((ms[w] - MM) * sc);
      L += ls[w] * f;
      v += os[w][d] * f;
    }
    ((T*)a.out)[(int64_t)(s.row0 + tok) * a.ldo + (int64_t)h * HD + d] = (T)(L > 0.0f ? v / L : 0.0f);
  }
}

// What a call launches, from its sizes alone.
struct Plan {
  int nt, slots;
  int64_t part_bytes, bytes;  // the partials', and with the plan's after them
};
Plan make_plan(int64_t B, int64_t max_q, int nq, int nkv, int hd) {
  Plan p;
  p.nt = (int)((max_q * (nq / nkv) + kRows - 1) / kRows);
  // about two workgroups per CU beyond one for each sequence
  const int64_t spare = std::max<int64_t>(1, 512 / ((int64_t)nkv * p.nt));
  p.slots = (int)(B + spare);
  p.part_bytes = (int64_t)p.slots * nkv * p.nt * part_floats(hd) * 4;
  p.bytes = p.part_bytes + B * 8;
  return p;
}

template <typename E, int HD>
int launch(const PagedArgs& a, hipStream_t s) {
  (void)hipGetLastError();
  paged_split_kernel<E, HD, 8><<<(unsigned)a.slots * a.nkv * a.nt, 8 * 64, 0, s>>>(a);
  const int st = ldk::check_launch("paged_attention");
  if (st) return st;
  paged_merge_kernel<E, HD><<<dim3((unsigned)a.max_q, (unsigned)a.nq, (unsigned)a.B), kMergeWaves * 64, 0, s>>>(a);
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
  if (kps < per || vps < per || ldq < (int64_t)nq * hd || ldo < (int64_t)nq * hd)
    return ldk::fail(LDK_ERR_INVALID, "%s: strides ldq=%lld ldo=%lld pages %lld %lld below what they step over", fn,
                     (long long)ldq, (long long)ldo, (long long)kps, (long long)vps);
  if (!ldk::aligned(q, 16) || !ldk::aligned(out, 16) || !ldk::aligned(k, 16) || !ldk::aligned(vt, 16) || ldq % 8 ||
      ldo % 8 || kps % 8 || vps % 8 || !ldk::aligned(kv_lens, 4) || !ldk::aligned(cu, 4) || !ldk::aligned(table, 4) ||
      !ldk::aligned(ptable, 4) || !ldk::aligned(ws, 16))
    return ldk::fail(LDK_ERR_ALIGN, "%s: q, out, workspace and the pages 16-byte aligned with strides of multiples of 8 elements", fn);
  const Plan p = make_plan(B, cu ? max_q : 1, nq, nkv, hd);
  if (!ws || ws_bytes < p.bytes)
    return ldk::fail(LDK_ERR_INVALID, "%s: workspace of %lld bytes, this call needs %lld", fn, (long long)ws_bytes, (long long)p.bytes);
  if ((int64_t)p.slots * nkv * p.nt > INT32_MAX) return ldk::fail(LDK_ERR_UNSUPPORTED, "%s: too many workgroups", fn);
  const int big = 1 << 30;  // a window or sinks past every position
  PagedArgs a{q, ldq, cu, kv_lens, table, ptable, ldt, k, vt, kps, vps, out, ldo, (float*)ws,
              (int32_t*)((char*)ws + p.part_bytes), cu ? (int)T : (int)B, (int)B, cu ? (int)max_q : 1, nq, nkv, nq / nkv, p.nt,
              (int)num_pages, (int)(page_size / 32), (int)(max_pages * page_size), (int)(prefix_len / 32),
              (int)std::min<int64_t>(window, big), (int)std::min<int64_t>(sinks, big), p.slots, scale};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == LDK_F16) return hd == 128 ? launch<ldk::F16, 128>(a, s) : launch<ldk::F16, 64>(a, s);
  return hd == 128 ? launch<ldk::BF16, 128>(a, s) : launch<ldk::BF16, 64>(a, s);
}

}  // namespace

extern "C" int64_t ldk_paged_attention_workspace_bytes(int64_t T, int64_t B, int64_t max_q, int64_t prefix_len, int nq,
                                                       int nkv, int head_dim) {
  if (T <= 0 || T > (int64_t(1) << 24) || B <= 0 || B > 65535 || max_q <= 0 || max_q > (int64_t(1) << 24) || prefix_len < 0 || nq <= 0 || nkv <= 0 ||
      nq % nkv || nq > 4096 || (head_dim != 64 && head_dim != 128)) {
    return -ldk::fail(LDK_ERR_INVALID, "paged_attention_workspace_bytes: T=%lld B=%lld max_q=%lld prefix_len=%lld nq=%d nkv=%d head_dim=%d",
                      (long long)T, (long long)B, (long long)max_q, (long long)prefix_len, nq, nkv, head_dim);
  }
  return make_plan(B, max_q, nq, nkv, head_dim).bytes;
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

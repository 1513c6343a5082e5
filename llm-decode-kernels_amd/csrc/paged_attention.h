// What the kernels of attention over a paged cache share, whatever their pages hold: the call's arguments, the
// visible chunks of a sequence and their split into ranges, blocks of rows, and the host's plan of launches
// (paged_attention.hip, paged_attention_int4.hip). Not part of the C ABI.
#pragma once

#include <algorithm>

#include "paged.h"

namespace ldk {

struct PagedArgs {
  const void* q;
  int64_t ldq;
  const int32_t *cu, *kv_lens, *table, *ptable;  // ptable: the shared prefix's pages
  int64_t ldt;
  const void *k, *vt;
  int64_t kps, vps;  // page strides, elements
  void* out;
  int64_t ldo;
  float* part;    // paged_split_kernel's partials, per (slot, tile, kv head): [16 rows]{m, l} and [16 rows][hd] (part_at)
  float* bpart;   // paged_block_kernel's, per (tile, kv head, split): [rows]{m, l} and [rows][hd]
  int32_t* plan;  // [B][2]: first slot and ranges of every sequence
  int32_t* map;   // of many sequences: [0] chunks of a range, [1 + slot] its sequence; else null
  int T, B, max_q, nq, nkv, gq, nt;  // nt: 16-row tiles of a sequence
  int tiles;                         // partials of a sequence's own tiles alone: the call's tiles; else 0
  int pages, cap;                    // cap: positions a sequence can hold
  PageDiv cpp;                       // chunks per page
  int pchunks, skip;                 // chunks of the shared prefix; of them, those that its own blocks take
  int window, sinks, slots, spare;
  int btiles, bsplits, bdirect;      // the block kernel's tiles and splits; a lone range writes the output
  float scale;
};

typedef const __attribute__((address_space(4))) int32_t* ScalarInts;  // read through the scalar cache

constexpr int kRows = 16;
template <int N>
struct IntC {
  static constexpr int value = N;
};
// Of paged_block_kernel, by a block's rows: the waves that split its chunks between them, and LDS slots.
template <int BT>
constexpr int kBlockKG = BT == 128 ? 1 : 4;
template <int BT>
constexpr int kBlockSlots = BT == 128 ? 4 : 2;
template <int BT>
constexpr int kBlockThreads = BT / 32 * kBlockKG<BT> * 64;
constexpr int kAll = 0x7fffffff;
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
  if (a.skip) x.cs = 0, x.lo = min(a.skip, hc);  // the shared prefix is another kernel's
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
// sequence has at least one range (its rows have to be written), so sum over b of max(1, ceil(n_b / per))
// <= B + total / per: with per = total / spare it fits B + spare slots. Where the launch is to be one round
// of workgroups (spare 0), per is the least for which the sum fits the slots, found by bisection.
struct Slot {
  int b, split, ranges, first, per;  // b < 0: none
};
// Chunks of a range, of `sum` chunks in sequences of at most `most`.
__device__ __forceinline__ int range_chunks(const PagedArgs& a, int64_t sum, int most) {
  const int ways = a.spare ? a.spare : a.slots;
  const int per = (int)min((sum + ways - 1) / ways, (int64_t)most);
  return max(per, max(kMinRange, (most + kMaxRanges - 1) / kMaxRanges));
}
__device__ __forceinline__ Slot find_slot(const PagedArgs& a, int slot, int lane) {
  if (!a.plan) return Slot{slot, 0, 1, slot, kAll};  // every sequence in one range
  if (a.map) {                                       // paged_plan_kernel has found it
    const int b = a.map[1 + slot];
    if (b < 0) return Slot{-1, 0, 1, 0, 0};
    const int first = a.plan[2 * b];
    return Slot{b, slot - first, a.plan[2 * b + 1], first, a.map[0]};
  }
  const int each = (a.B + 63) / 64, b0 = lane * each, b1 = min(b0 + each, a.B);
  int64_t sum = 0;
  int most = 0, n0 = 0;
  for (int b = b0; b < b1; ++b) {
    const int n = seq_span(a, b).n;
    sum += n;
    most = max(most, n);
    n0 = n;
  }
  sum = wave_sum64(sum);
  most = wave_max_i(most);
  int per = range_chunks(a, sum, most);
  if (!a.spare && a.B > 1) {
    int hi = max(per, (int)min((int64_t)most, (sum + a.slots - a.B - 1) / (a.slots - a.B)));
    while (per < hi) {
      const int mid = (per + hi) / 2;
      float c = 0.0f;  // exact: below 2^24
      if (each == 1) {
        if (b0 < b1) c = (float)max(1, (n0 + mid - 1) / mid);
      } else {
        for (int b = b0; b < b1; ++b) c += (float)max(1, (seq_span(a, b).n + mid - 1) / mid);
      }
      if (__builtin_amdgcn_readfirstlane((int)sum_lanes_strided<1>(c)) <= a.slots)
        hi = mid;
      else
        per = mid + 1;
    }
  }
  Slot r{-1, 0, 1, 0, per};
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

// Place among the partials, in kv heads, of the range `split` of the 16 rows `tile` of sequence b, whose first row is row0
// and first slot `first`. Slot by slot, nt tiles each; or, where the call's tiles are counted, first the tiles of every
// sequence's first range as the call's rows have them (sequence b's from row0 gq / 16 + b on, rounded down: its
// ceil(n gq / 16) end before the next one's begin), then nt for each of the ranges past the first, of which there are
// `spare` at most, first - b of them before b's.
__device__ __forceinline__ int64_t part_at(const PagedArgs& a, int b, int row0, int first, int split, int tile) {
  if (!a.tiles) return (int64_t)(first + split) * a.nt + tile;
  return split ? a.tiles + (int64_t)(first - b + split - 1) * a.nt + tile : row0 * (int64_t)a.gq / kRows + b + tile;
}

// ---- blocks of rows (the kernels' own words on them stand there)

struct Block {
  int b, row0, pos0;     // MODE 0: the sequence, its first row and position
  int r0, rows;          // the block's first row (of the sequence's, or of the call's) and its number
  int first, last;       // positions of the first and last row (MODE 0)
  int cs, lo, n;         // visible chunks
};
// The block of sequence b's rows from r0 on. rows == 0: none.
__device__ __forceinline__ Block sequence_block(const PagedArgs& a, int b, const SeqRows& s, int r0, int BT) {
  Block k{};
  k.b = b;
  k.row0 = s.row0;
  k.pos0 = s.pos0;
  k.r0 = r0;
  k.rows = r0 < 0 ? 0 : max(0, min(BT, min(s.n, a.max_q) * a.gq - r0));
  if (k.rows <= 0) return k;
  k.first = k.pos0 + k.r0 / a.gq;
  k.last = k.pos0 + (k.r0 + k.rows - 1) / a.gq;
  const int hi = min(k.last, a.cap - 1), hc = hi < 0 ? 0 : hi / kChunkPos + 1;
  k.lo = min(a.window > 0 ? max(0, k.first - a.window + 1) / kChunkPos : 0, hc);
  k.cs = min((min(a.sinks, a.cap) + kChunkPos - 1) / kChunkPos, k.lo);
  k.n = k.cs + hc - k.lo;
  return k;
}
// The block of tile x (uniform).
template <int MODE>
__device__ __forceinline__ Block find_block(const PagedArgs& a, int x, int BT) {
  Block k{};
  if constexpr (MODE == 1) {
    k.r0 = x * BT;
    k.rows = min(BT, a.T * a.gq - k.r0);
    k.last = kAll;
    k.n = a.pchunks;
    return k;
  }
  int b = 0;
  for (int lo = 0, hi = a.B; lo < hi;) {
    const int mid = (lo + hi) / 2;
    if ((int64_t)(a.cu ? max(a.cu[mid], 0) : mid) * a.gq / BT + mid <= x)
      b = mid, lo = mid + 1;
    else
      hi = mid;
  }
  const SeqRows s = seq_rows(a.cu, a.kv_lens, b, a.T);
  return sequence_block(a, b, s, (x - (int)(s.row0 * (int64_t)a.gq / BT) - b) * BT, BT);
}
// Chunks of a block's range, a multiple of kg.
__device__ __forceinline__ int block_range(const PagedArgs& a, int n, int kg) {
  const int per = (n + a.bsplits - 1) / a.bsplits;
  return max(2 * kg, (per + kg - 1) / kg * kg);
}
// The position of row t of the call's (-1: no sequence's), by its sequence.
__device__ __forceinline__ int row_position(const PagedArgs& a, int t) {
  int b = t;
  if (a.cu) {
    b = -1;
    for (int lo = 0, hi = a.B; lo < hi;) {  // the last b with cu[b] <= t
      const int mid = (lo + hi) / 2;
      if (a.cu[mid] <= t)
        b = mid, lo = mid + 1;
      else
        hi = mid;
    }
    if (b < 0) return -1;
  }
  const SeqRows s = seq_rows(a.cu, a.kv_lens, b, a.T);
  return t - s.row0 < min(s.n, a.max_q) ? s.pos0 + t - s.row0 : -1;
}

// ---- the host's side

// What a call launches, from its sizes alone.
struct Plan {
  bool apart = false;                               // the shared prefix in blocks of its own
  int64_t nt = 0, slots = 0, spare = 0, tiles = 0;  // paged_split_kernel, slots == 0: not launched
  int64_t bt = 0, btiles = 0, bsplits = 0;          // paged_block_kernel, bt == 0: not launched
  bool mapped = false;                              // paged_plan_kernel
  int64_t part_bytes = 0, bpart_bytes = 0, bytes = 0;
};
// Chunks that a token sees at most, from the positions a table holds and the window.
inline int64_t most_chunks(int64_t max_len, int64_t max_q, int64_t window, int64_t sinks) {
  const int64_t all = (max_len + kChunkPos - 1) / kChunkPos;
  if (!window) return all;
  return std::min(all, (window + max_q + kChunkPos - 2) / kChunkPos + 1 + (sinks + kChunkPos - 1) / kChunkPos);
}
// The workspace: both kernels' partials, [B] first slots and ranges, the slots' sequences.
inline int64_t workspace_bytes(const Plan& p, int64_t B) {
  return p.part_bytes + p.bpart_bytes + (p.part_bytes ? B * 8 : 0) + (p.mapped ? (p.slots + 1) * 4 : 0);
}
inline void lay_out(PagedArgs& a, const Plan& p, void* ws, int64_t B) {
  a.part = (float*)ws;
  a.tiles = (int)p.tiles;
  a.bpart = (float*)((char*)ws + p.part_bytes);
  a.plan = p.part_bytes ? (int32_t*)((char*)ws + p.part_bytes + p.bpart_bytes) : nullptr;
  a.map = p.mapped ? a.plan + 2 * B : nullptr;
}
// A launch holds fewer than 2^32 threads.
inline bool launchable(const Plan& p, int64_t T, int nq, int nkv) {
  const int64_t most = (int64_t(1) << 32) / 512 - 8;
  return p.slots * nkv * p.nt + p.btiles * nkv * std::max<int64_t>(1, p.bsplits) < most && T * nq < most * 8;
}

// The launches around the ranges' own, on stream s: the sequences' ranges where p.mapped (before), and the ranges' join
// where p.bytes (after). E and HD of the partials by dtype and head_dim; a.plan, a.map and the partials as p lays them out.
int paged_find_ranges(const PagedArgs& a, hipStream_t s);
int paged_join(const PagedArgs& a, int dtype, int hd, int64_t bt, hipStream_t s);

}  // namespace ldk

// Appending new tokens to a paged cache: RoPE on q and k, k and v written into the pages at each
// token's position, q returned in rows of its own. Pages and sequences: paged.h.
//
// Rotation of a head x of hd dims, h = hd / 2, by the angles a_j = r * inv_freq[j] of the token's
// position r (its cache position, or rope_pos):
//   (x_j, x_{j+h}) -> (x_j cos a_j - x_{j+h} sin a_j, x_{j+h} cos a_j + x_j sin a_j).
// r * inv_freq in fp32 is off by r 2^-24 (0.01 radians at position 150000), so the product is formed
// in 64 bits and reduced there to a fraction of a turn; its cosine and sine, and the rotation, are
// fp32 and the results are rounded once to the element type. v is copied.
//
// Bound by the bytes: each of the T (nq + 2 nkv) hd elements is read and written once. Two forms:
//  - append_token_kernel, one new token per sequence: a workgroup per token; the angles are formed
//    once per token through LDS while the rows' loads are in flight.
//  - append_chunk_kernel, ragged prompts: a workgroup takes the new tokens of one 32-position chunk of
//    one sequence, so that K and V^T leave as whole 1 KB tiles (v turned in LDS).
#include <algorithm>

#include "paged_rope.h"

namespace {

using namespace ldk;

struct AppendArgs {
  const void* qkv;
  int64_t ldqkv;
  const int32_t *cu, *kv_lens, *table;
  int64_t ldt;
  const int64_t* rope_pos;  // or null: the cache positions
  const float* inv_freq;    // [hd/2], or null: no rotation
  void *k, *vt, *q;
  int64_t kps, vps, ldq;    // page strides and q's row stride, elements
  int T, B, nq, nkv, pages, cpp, cap;  // cpp: chunks per page; cap: positions a table row holds
};

// Element offsets inside a page's kv head of K at (chunk c, position r of it, dim d) and of V^T.
template <int HD>
__device__ __forceinline__ int k_at(int c, int r, int d) {
  return ((c * 2 + ((r >> 2) & 1)) * (HD / 32) + (d >> 5)) * kTileElems + (4 * (r >> 3) + (r & 3)) * 32 + (d & 31);
}
template <int HD>
__device__ __forceinline__ int vt_at(int c, int r, int d) {
  return (c * (HD / 16) + (d >> 4)) * kTileElems + (d & 15) * 32 + r;
}

constexpr int kTokThreads = 256;

// Thread i of a token's workgroups (y) takes 8 dims of a q or k head and their partners, or 8 of a v head; its
// loads go out before the angles, whose length and page loads and trigonometry they then cover. Latency
// bounds it: graph-timed 3.2 us for one token of 12/2 heads, 4.5 for 96 of 32/8 (2.4 MB).
template <typename E, int HD>
__global__ __launch_bounds__(kTokThreads) void append_token_kernel(AppendArgs a) {
  typedef typename E::T T;
  constexpr int LH = HD / 16;  // lanes per q or k head
  constexpr int LV = HD / 8;   // lanes per v head
  __shared__ __align__(16) float cs[2][HD / 2];
  const int t = blockIdx.x, tid = threadIdx.x, i = tid + (int)blockIdx.y * kTokThreads;
  const int pairs = (a.nq + a.nkv) * LH, j = i - pairs;
  const bool rot = i < pairs, val = !rot && j < a.nkv * LV;
  const int h = rot ? i / LH : j / LV, d = (rot ? i % LH : j % LV) * 8;
  const T* row = (const T*)a.qkv + (int64_t)t * a.ldqkv;
  u32x4 x0{}, x1{};
  if (rot) {
    x0 = *reinterpret_cast<const u32x4*>(row + (int64_t)h * HD + d);
    x1 = *reinterpret_cast<const u32x4*>(row + (int64_t)h * HD + HD / 2 + d);
  } else if (val) {
    x0 = *reinterpret_cast<const u32x4*>(row + (int64_t)(a.nq + a.nkv + h) * HD + d);
  }
  const int p = seq_rows(nullptr, a.kv_lens, t, a.T).pos0;
  int64_t page = -1;
  if (p >= 0 && p < a.cap) page = a.table[(int64_t)t * a.ldt + p / (kChunkPos * a.cpp)];
  if (a.inv_freq) {  // uniform
    if (tid < HD / 2) angle(a.rope_pos ? a.rope_pos[t] : (int64_t)p, a.inv_freq[tid], &cs[0][tid], &cs[1][tid]);
    __syncthreads();
  }
  const bool wr = page >= 0 && page < a.pages;
  const int c = p >= 0 ? p / kChunkPos % a.cpp : 0, r = p & 31;
  if (rot) {
    if (a.inv_freq) rotate8<E>(x0, x1, &cs[0][d], &cs[1][d]);
    if (h < a.nq) {
      T* q = (T*)a.q + (int64_t)t * a.ldq + (int64_t)h * HD;
      *reinterpret_cast<u32x4*>(q + d) = x0;
      *reinterpret_cast<u32x4*>(q + HD / 2 + d) = x1;
    } else if (wr) {
      T* k = (T*)a.k + page * a.kps + (int64_t)(h - a.nq) * a.cpp * kChunkPos * HD;
      *reinterpret_cast<u32x4*>(k + k_at<HD>(c, r, d)) = x0;
      *reinterpret_cast<u32x4*>(k + k_at<HD>(c, r, HD / 2 + d)) = x1;
    }
  } else if (val && wr) {
    uint16_t* v = (uint16_t*)a.vt + page * a.vps + (int64_t)h * a.cpp * kChunkPos * HD;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[vt_at<HD>(c, r, d + e)] = (uint16_t)(x0[e >> 1] >> (16 * (e & 1)));
  }
}

constexpr int kChunkThreads = 256;

// Workgroup x: of the sequences' chunks, sequence b's begin at index cu[b] / 32 + 2b (at most
// (n + 62) / 32 chunks hold its n new tokens, which is at most floor((cu + n) / 32) - floor(cu / 32)
// + 2). Each workgroup finds its sequence with a binary search. Memory bounds it: 21.3 us for 97 MB (7
// prompts, 28/4 heads), 4.6 TB/s, 94% of the rate of a 2 GiB copy.
template <typename E, int HD>
__global__ __launch_bounds__(kChunkThreads) void append_chunk_kernel(AppendArgs a) {
  typedef typename E::T T;
  constexpr int LH = HD / 16, NS = HD / 32;
  __shared__ __align__(16) float cs[2][kChunkPos][HD / 2 + 4];
  __shared__ __align__(16) uint16_t vs[kChunkPos][HD + 2];
  const int tid = threadIdx.x, x = blockIdx.x;
  int b = 0;
  for (int lo = 0, hi = a.B; lo < hi;) {  // the last b whose first index is not past x
    const int mid = (lo + hi) / 2;
    if (max(a.cu[mid], 0) / kChunkPos + 2 * mid <= x)
      b = mid, lo = mid + 1;
    else
      hi = mid;
  }
  const SeqRows sr = seq_rows(a.cu, a.kv_lens, b, a.T);
  if (sr.n <= 0) return;
  // the chunk's new tokens: rows t0 .. t0 + nt - 1 at its positions r0 ..; chunks are counted from the
  // one that holds pos0 (rounded down, for positions below 0 too)
  const int ci = x - (sr.row0 / kChunkPos + 2 * b);
  const int c0 = (sr.pos0 >= 0 ? sr.pos0 : sr.pos0 - (kChunkPos - 1)) / kChunkPos + ci;
  const int64_t base = (int64_t)c0 * kChunkPos;
  const int first = max(0, (int)(sr.pos0 - base));                      // in the chunk
  const int last = (int)min((int64_t)kChunkPos, sr.pos0 + (int64_t)sr.n - base);  // one past
  if (first >= last) return;
  const int t0 = sr.row0 + (int)(base + first - sr.pos0) - first;  // row of the chunk's position 0
  int64_t page = -1;
  if (c0 >= 0 && base < a.cap) page = a.table[(int64_t)b * a.ldt + c0 / a.cpp];
  const bool wr = page >= 0 && page < a.pages;
  const int c = c0 >= 0 ? c0 % a.cpp : 0;
  if (a.inv_freq) {
    for (int i = tid; i < kChunkPos * (HD / 2); i += kChunkThreads) {
      const int r = i / (HD / 2), j = i % (HD / 2);
      if (r >= first && r < last)
        angle(a.rope_pos ? a.rope_pos[t0 + r] : base + r, a.inv_freq[j], &cs[0][r][j], &cs[1][r][j]);
    }
  }
  __syncthreads();
  const T* rows = (const T*)a.qkv;
  for (int h = (int)blockIdx.y; h < a.nq + 2 * a.nkv; h += (int)gridDim.y) {
    if (h < a.nq) {
      for (int i = tid; i < kChunkPos * LH; i += kChunkThreads) {
        const int r = i / LH, d = i % LH * 8;
        if (r < first || r >= last) continue;
        const T* src = rows + (int64_t)(t0 + r) * a.ldqkv + (int64_t)h * HD;
        u32x4 x0 = *reinterpret_cast<const u32x4*>(src + d), x1 = *reinterpret_cast<const u32x4*>(src + HD / 2 + d);
        if (a.inv_freq) rotate8<E>(x0, x1, &cs[0][r][d], &cs[1][r][d]);
        T* q = (T*)a.q + (int64_t)(t0 + r) * a.ldq + (int64_t)h * HD;
        *reinterpret_cast<u32x4*>(q + d) = x0;
        *reinterpret_cast<u32x4*>(q + HD / 2 + d) = x1;
      }
    } else if (h < a.nq + a.nkv) {
      if (!wr) continue;
      // item i: 8 dims of row i / 4 % 16 of the tile (row half, dim step s) and of (row half, s + NS / 2)
      T* k = (T*)a.k + page * a.kps + (int64_t)(h - a.nq) * a.cpp * kChunkPos * HD;
      for (int i = tid; i < kChunkPos * LH; i += kChunkThreads) {
        const int e = i & 3, row = (i >> 2) & 15, s = (i >> 6) % (NS / 2), hb = (i >> 6) / (NS / 2);
        const int r = 8 * (row >> 2) + 4 * hb + (row & 3), d = 32 * s + 8 * e;
        if (r < first || r >= last) continue;
        const T* src = rows + (int64_t)(t0 + r) * a.ldqkv + (int64_t)h * HD;
        u32x4 x0 = *reinterpret_cast<const u32x4*>(src + d), x1 = *reinterpret_cast<const u32x4*>(src + HD / 2 + d);
        if (a.inv_freq) rotate8<E>(x0, x1, &cs[0][r][d], &cs[1][r][d]);
        *reinterpret_cast<u32x4*>(k + k_at<HD>(c, r, d)) = x0;
        *reinterpret_cast<u32x4*>(k + k_at<HD>(c, r, HD / 2 + d)) = x1;
      }
    } else {
      if (!wr) continue;
      __syncthreads();  // the v head before has been read
      for (int i = tid; i < kChunkPos * (HD / 8); i += kChunkThreads) {
        const int r = i / (HD / 8), d = i % (HD / 8) * 8;
        if (r < first || r >= last) continue;
        const u32x4 v = *reinterpret_cast<const u32x4*>(rows + (int64_t)(t0 + r) * a.ldqkv + (int64_t)h * HD + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(&vs[r][d + 2 * j]) = v[j];
      }
      __syncthreads();
      uint16_t* v = (uint16_t*)a.vt + page * a.vps + (int64_t)(h - a.nq - a.nkv) * a.cpp * kChunkPos * HD;
      // item i: dim i / 4, positions 8 (i % 4) .. + 7
      for (int i = tid; i < HD * 4; i += kChunkThreads) {
        const int d = i >> 2, r = 8 * (i & 3);
        if (r >= first && r + 8 <= last) {
          u32x4 y;
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = (uint32_t)vs[r + 2 * j][d] | ((uint32_t)vs[r + 2 * j + 1][d] << 16);
          *reinterpret_cast<u32x4*>(v + vt_at<HD>(c, r, d)) = y;
        } else {
          for (int j = max(r, first); j < min(r + 8, last); ++j) v[vt_at<HD>(c, j, d)] = vs[j][d];
        }
      }
    }
  }
}

template <typename E, int HD>
int launch(const AppendArgs& a, hipStream_t s) {
  (void)hipGetLastError();
  if (!a.cu) {
    const int items = (a.nq + a.nkv) * (HD / 16) + a.nkv * (HD / 8);
    append_token_kernel<E, HD><<<dim3((unsigned)a.T, (unsigned)((items + kTokThreads - 1) / kTokThreads)), kTokThreads, 0, s>>>(a);
  } else {
    const unsigned gx = (unsigned)(a.T / kChunkPos + 2 * a.B);
    const int hb = std::min(a.nq + 2 * a.nkv, std::max(1, 1024 / (int)(a.T / kChunkPos + a.B)));
    append_chunk_kernel<E, HD><<<dim3(gx, (unsigned)hb), kChunkThreads, 0, s>>>(a);
  }
  return ldk::check_launch("paged_append");
}

}  // namespace

extern "C" int ldk_paged_append(const void* qkv, int64_t ldqkv, int dtype, const int32_t* cu_seqlens,
                                const int32_t* kv_lens, const int32_t* block_table, int64_t ldt, int64_t max_pages,
                                const int64_t* rope_pos, const float* inv_freq, void* k_pages, int64_t k_page_stride,
                                void* vt_pages, int64_t vt_page_stride, int64_t num_pages, int64_t page_size,
                                void* q_out, int64_t ldq, int64_t T, int64_t B, int nq, int nkv, int head_dim,
                                void* stream) {
  static const char* fn = "paged_append";
  if (!qkv || !kv_lens || !block_table || !k_pages || !vt_pages || !q_out) return ldk::fail(LDK_ERR_INVALID, "%s: null pointer", fn);
  if (dtype != LDK_F16 && dtype != LDK_BF16) return ldk::fail(LDK_ERR_INVALID, "%s: dtype %d (fp16 or bf16)", fn, dtype);
  if (head_dim != 64 && head_dim != 128) return ldk::fail(LDK_ERR_UNSUPPORTED, "%s: head_dim=%d (64 or 128)", fn, head_dim);
  if (nq <= 0 || nkv <= 0 || nq % nkv || nq > 4096)
    return ldk::fail(LDK_ERR_INVALID, "%s: nq=%d must be a positive multiple of nkv=%d (at most 4096)", fn, nq, nkv);
  if (T <= 0 || T > (int64_t(1) << 24) || B <= 0 || B > (int64_t(1) << 20))
    return ldk::fail(LDK_ERR_INVALID, "%s: T=%lld tokens (1..2^24) of B=%lld sequences (1..2^20)", fn, (long long)T, (long long)B);
  if (!cu_seqlens && T < B) return ldk::fail(LDK_ERR_INVALID, "%s: T=%lld rows for B=%lld sequences of one token", fn, (long long)T, (long long)B);
  if (page_size < 32 || page_size % 32 || page_size > 65536)
    return ldk::fail(LDK_ERR_UNSUPPORTED, "%s: page_size=%lld must be a multiple of 32 up to 65536", fn, (long long)page_size);
  if (num_pages <= 0 || num_pages > INT32_MAX || max_pages <= 0 || ldt < max_pages || max_pages > ldk::kMaxPositions / page_size)
    return ldk::fail(LDK_ERR_INVALID, "%s: num_pages=%lld max_pages=%lld ldt=%lld", fn, (long long)num_pages, (long long)max_pages, (long long)ldt);
  const int64_t per = (int64_t)nkv * page_size * head_dim;
  if (k_page_stride > INT32_MAX || vt_page_stride > INT32_MAX)
    return ldk::fail(LDK_ERR_UNSUPPORTED, "%s: page strides %lld %lld past 2^31", fn, (long long)k_page_stride, (long long)vt_page_stride);
  if (k_page_stride < per || vt_page_stride < per || ldqkv < (int64_t)(nq + 2 * nkv) * head_dim || ldq < (int64_t)nq * head_dim)
    return ldk::fail(LDK_ERR_INVALID, "%s: strides ldqkv=%lld ldq=%lld pages %lld %lld below what they step over", fn,
                     (long long)ldqkv, (long long)ldq, (long long)k_page_stride, (long long)vt_page_stride);
  if (!ldk::aligned(qkv, 16) || !ldk::aligned(q_out, 16) || !ldk::aligned(k_pages, 16) || !ldk::aligned(vt_pages, 16) ||
      ldqkv % 8 || ldq % 8 || k_page_stride % 8 || vt_page_stride % 8 || !ldk::aligned(kv_lens, 4) ||
      !ldk::aligned(cu_seqlens, 4) || !ldk::aligned(block_table, 4) || !ldk::aligned(rope_pos, 8) || !ldk::aligned(inv_freq, 4))
    return ldk::fail(LDK_ERR_ALIGN, "%s: qkv, q_out and the pages 16-byte aligned with strides of multiples of 8 elements", fn);
  const AppendArgs a{qkv, ldqkv, cu_seqlens, kv_lens, block_table, ldt, rope_pos, inv_freq, k_pages, vt_pages, q_out,
                     k_page_stride, vt_page_stride, ldq, cu_seqlens ? (int)T : (int)B, (int)B, nq, nkv, (int)num_pages,
                     (int)(page_size / 32), (int)(max_pages * page_size)};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == LDK_F16) return head_dim == 128 ? launch<ldk::F16, 128>(a, s) : launch<ldk::F16, 64>(a, s);
  return head_dim == 128 ? launch<ldk::BF16, 128>(a, s) : launch<ldk::BF16, 64>(a, s);
}

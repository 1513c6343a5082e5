// Reading the values of a paged cache held in 4 bits (paged_int4.h) back as rows [token, kv head, hd] of the cache's type:
// z + (code - 8) step in fp32 (the product is exact), rounded once, at most the type's largest number.
//
// A workgroup takes the rows of one 32-position chunk of one sequence and some of its kv heads. k's codes are rows
// already (a lane's 16 bytes are 8 dims of each step of one position); v's, whose bytes run along the positions, are turned
// in LDS.
//
// The stores bound it: 39439 positions of 8 heads of 128 in groups of 32, 50 MB of codes to 162 MB of values, 48 us, 4.4 TB/s (a
// 2 GiB copy: 4.9). 700 positions of 2 heads 4.6 us, the latency of the length, the page's id, the codes and the stores.
#include <algorithm>

#include "paged_int4.h"

namespace {

using namespace ldk;

struct Read4Args {
  const int32_t *cu, *kv_lens, *table;
  int64_t ldt;
  const void* pool;
  int64_t stride;
  void *k, *v;
  int64_t ldk, ldv;  // row strides, elements
  int T, B, nkv, pages, cpp, cap;
};

// The outermost codes of a group near the type's largest number may stand for a value past it, by the step's and the offset's
// rounding: it is read as the largest. most4: that number, or NaN for a group that is (as med3 of three NaN is).
template <typename E>
__device__ __forceinline__ float most4(float z) {
  return __builtin_fmaf(z, 0.0f, E::kMost);
}
template <typename E>
__device__ __forceinline__ float value4(uint32_t code, float step, float z, float most) {
  return __builtin_amdgcn_fmed3f(__builtin_fmaf((float)(int)code - 8.0f, step, z), -most, most);
}

constexpr int kThreads = 256;

template <typename E, int HD, int NG>
__global__ __launch_bounds__(kThreads) void read4_kernel(Read4Args a) {
  typedef typename E::T T;
  typedef Int4Block<HD, NG> L;
  constexpr int NB = HD / 16, NP = HD / 64;  // v's dim blocks; pairs of k's steps
  __shared__ __align__(16) T vs[kChunkPos][HD + 8];
  const int tid = threadIdx.x, x = blockIdx.x;
  int b = x;  // without cu: one row per sequence
  if (a.cu) {
    b = 0;
    for (int lo = 0, hi = a.B; lo < hi;) {  // the last b whose first index is not past x (as the append's chunks)
      const int mid = (lo + hi) / 2;
      if (max(a.cu[mid], 0) / kChunkPos + 2 * mid <= x)
        b = mid, lo = mid + 1;
      else
        hi = mid;
    }
  }
  const SeqRows sr = seq_rows(a.cu, a.kv_lens, b, a.T);
  if (sr.n <= 0) return;
  const int ci = a.cu ? x - (sr.row0 / kChunkPos + 2 * b) : 0;
  const int c0 = (sr.pos0 >= 0 ? sr.pos0 : sr.pos0 - (kChunkPos - 1)) / kChunkPos + ci;
  const int64_t base = (int64_t)c0 * kChunkPos;
  const int first = max(0, (int)(sr.pos0 - base));
  const int last = (int)min((int64_t)kChunkPos, sr.pos0 + (int64_t)sr.n - base);
  if (first >= last) return;
  const int t0 = sr.row0 + (int)(base + first - sr.pos0) - first;  // row of the chunk's position 0
  int64_t page = -1;
  if (c0 >= 0 && base < a.cap) page = a.table[(int64_t)b * a.ldt + c0 / a.cpp];
  const bool held = page >= 0 && page < a.pages;
  const int c = c0 >= 0 ? c0 % a.cpp : 0;
  for (int h = (int)blockIdx.y; h < a.nkv; h += (int)gridDim.y) {
    const unsigned char* blk = (const unsigned char*)a.pool + (held ? page * a.stride + ((int64_t)h * a.cpp + c) * L::kWords : 0) * 2;
    // ---- k: item i is lane i % 64 of the block's rows, of half i / 64: position r, dims 8kb .. of every step
    if (tid < 128) {
      const int i = tid & 15, kb = (tid >> 4) & 3, half = tid >> 6;
      const int r = 8 * (i >> 2) + 4 * half + (i & 3);
      if (r >= first && r < last) {
        T* dst = (T*)a.k + (int64_t)(t0 + r) * a.ldk + (int64_t)h * HD + 8 * kb;
        uint32_t w[2 * NP] = {};
        float step[NG] = {}, z[NG] = {}, most[NG] = {};
        if (held) {
#pragma unroll
          for (int n = 0; n < NP; ++n) {
            const u32x2 v = *reinterpret_cast<const u32x2*>(blk + int4_k_at<HD>(r, kb) + 8 * n);
            w[2 * n] = v[0], w[2 * n + 1] = v[1];
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const T* p = reinterpret_cast<const T*>(blk + L::kParams + int4_param_at(g, r));
            step[g] = (float)p[0], z[g] = (float)p[8], most[g] = most4<E>(z[g]);
          }
        }
#pragma unroll
        for (int s = 0; s < 2 * NP; ++s) {
          const int g = s * NG / (2 * NP);
          u32x4 y;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float f[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const int el = 2 * e + n;
              const uint32_t code = (w[2 * (s / 2) + (el >> 2)] >> (8 * int4_byte(el & 3) + 4 * (s & 1))) & 15u;
              f[n] = value4<E>(code, step[g], z[g], most[g]);
            }
            y[e] = pack2<E>(f[0], f[1]);
          }
          *reinterpret_cast<u32x4*>(dst + 32 * s) = y;
        }
      }
    }
    // ---- v: item u is 16 bytes, 8 positions of a column of 4 blocks
    __syncthreads();  // the head before has been stored
    for (int u = tid; u < HD; u += kThreads) {
      const int col = u & 15, kb = (u >> 4) & 3, quad = u >> 6;
      if (8 * kb + 8 <= first || 8 * kb >= last) continue;
      u32x4 w{};
      u32x4 st[2] = {}, zz[2] = {};  // of the quad's two pairs of blocks
      if (held) {
        w = *reinterpret_cast<const u32x4*>(blk + L::kV + u * 16);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const unsigned char* p = blk + L::kVParams + (2 * quad + t) * 2 * NG / NB * 128 + kb * 32;
          st[t] = *reinterpret_cast<const u32x4*>(p);
          zz[t] = *reinterpret_cast<const u32x4*>(p + 16);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // positions 2e, 2e + 1
          const float2_t s2 = unpack2<E>(st[t][e]), z2 = unpack2<E>(zz[t][e]);
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int el = 2 * e + n;
            const uint32_t byte = w[2 * t + (el >> 2)] >> (8 * int4_byte(el & 3));
            const float most = most4<E>(z2[n]);
            T* dst = &vs[8 * kb + el][(2 * quad + t) * 32 + col];
            dst[0] = (T)value4<E>(byte & 15u, s2[n], z2[n], most);
            dst[16] = (T)value4<E>(byte >> 4 & 15u, s2[n], z2[n], most);
          }
        }
    }
    __syncthreads();
    for (int i = tid; i < kChunkPos * (HD / 8); i += kThreads) {
      const int r = i / (HD / 8), d = i % (HD / 8) * 8;
      if (r < first || r >= last) continue;
      *reinterpret_cast<u32x4*>((T*)a.v + (int64_t)(t0 + r) * a.ldv + (int64_t)h * HD + d) = *reinterpret_cast<const u32x4*>(&vs[r][d]);
    }
  }
}

template <typename E, int HD, int NG>
int launch(const Read4Args& a, hipStream_t s) {
  (void)hipGetLastError();
  const unsigned gx = a.cu ? (unsigned)(a.T / kChunkPos + 2 * a.B) : (unsigned)a.B;
  const int hb = std::min(a.nkv, std::max(1, 2048 / (int)(a.T / kChunkPos + a.B)));
  read4_kernel<E, HD, NG><<<dim3(gx, (unsigned)hb), kThreads, 0, s>>>(a);
  return ldk::check_launch("paged_read_int4");
}
template <typename E>
int launch(const Read4Args& a, int hd, int group, hipStream_t s) {
  if (hd == 64) return group == 32 ? launch<E, 64, 2>(a, s) : launch<E, 64, 1>(a, s);
  return group == 32 ? launch<E, 128, 4>(a, s) : group == 64 ? launch<E, 128, 2>(a, s) : launch<E, 128, 1>(a, s);
}

}  // namespace

extern "C" int ldk_paged_read_int4(int dtype, const int32_t* cu_seqlens, const int32_t* kv_lens, const int32_t* block_table,
                                   int64_t ldt, int64_t max_pages, const void* kv_pages, int64_t page_stride,
                                   int64_t num_pages, int64_t page_size, void* k_out, int64_t ld_k, void* v_out, int64_t ld_v,
                                   int64_t T, int64_t B, int nkv, int head_dim, int group, void* stream) {
  static const char* fn = "paged_read_int4";
  if (!kv_lens || !block_table || !kv_pages || !k_out || !v_out) return ldk::fail(LDK_ERR_INVALID, "%s: null pointer", fn);
  int st = ldk::check_int4_pool(fn, dtype, nkv, head_dim, group, page_stride, num_pages, page_size, ldt, max_pages);
  if (st || (st = ldk::check_int4_batch(fn, T, B, int64_t(1) << 20, cu_seqlens))) return st;
  if (ld_k < (int64_t)nkv * head_dim || ld_v < (int64_t)nkv * head_dim)
    return ldk::fail(LDK_ERR_INVALID, "%s: strides %lld and %lld below what they step over", fn, (long long)ld_k, (long long)ld_v);
  if (!ldk::aligned(kv_pages, 16) || !ldk::aligned(k_out, 16) || !ldk::aligned(v_out, 16) || ld_k % 8 || ld_v % 8 ||
      page_stride % 8 || !ldk::aligned(kv_lens, 4) || !ldk::aligned(cu_seqlens, 4) || !ldk::aligned(block_table, 4))
    return ldk::fail(LDK_ERR_ALIGN, "%s: k_out, v_out and the pages 16-byte aligned with strides of multiples of 8 elements", fn);
  const Read4Args a{cu_seqlens, kv_lens, block_table, ldt, kv_pages, page_stride, k_out, v_out, ld_k, ld_v, cu_seqlens ? (int)T : (int)B,
                    (int)B, nkv, (int)num_pages, (int)(page_size / 32), (int)(max_pages * page_size)};
  hipStream_t s = (hipStream_t)stream;
  return dtype == LDK_F16 ? launch<ldk::F16>(a, head_dim, group, s) : launch<ldk::BF16>(a, head_dim, group, s);
}

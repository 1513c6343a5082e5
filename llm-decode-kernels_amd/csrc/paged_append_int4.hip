// Appending new tokens to a paged cache held in 4 bits (paged_int4.h): RoPE on q and k, k and v quantised into the
// pages at each token's position, q returned in rows of its own.
//
// The rotation is paged_append.hip's, of q in fp32. A code hangs on k at its borders, so k is rotated in 64 bits,
// angles included, and rounded to fp32 and then to the type: what is quantised is the same number however it is
// computed. The quantiser's fp32 steps are single IEEE operations, in the order that paged_int4.h writes.
//
// Two forms, as paged_append.hip has them: a workgroup per token of a decode step, and one per 32-position chunk of a
// ragged prompt.
#include <algorithm>

#include "paged_int4.h"
#include "paged_rope.h"

namespace {

using namespace ldk;

struct Append4Args {
  const void* qkv;
  int64_t ldqkv;
  const int32_t *cu, *kv_lens, *table;
  int64_t ldt;
  const int64_t* rope_pos;  // or null: the cache positions
  const float* inv_freq;    // [hd/2], or null: no rotation
  void *pool, *q;
  int64_t stride, ldq;      // page stride and q's row stride, elements
  int T, B, nq, nkv, pages, cpp, cap;  // cpp: chunks per page; cap: positions a table row holds
};

// cos and sin of pos * freq in 64 bits.
__device__ __forceinline__ void angle64(int64_t pos, float freq, double* c, double* s) {
  const double t = (double)pos * (double)freq * 0.15915494309189533577;  // turns
  sincospi(2.0 * (t - __builtin_rint(t)), s, c);
}
// The 8 pairs (x0[e], x1[e]) turned by the angles whose cos and sin are c[0..7], s[0..7], as values of the type.
template <typename E>
__device__ __forceinline__ void turn8(const u32x4& x0, const u32x4& x1, const double* c, const double* s, float* y0, float* y1) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2_t a = unpack2<E>(x0[i]), b = unpack2<E>(x1[i]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const double cj = c[2 * i + j], sj = s[2 * i + j];
      float f0 = (float)((double)a[j] * cj - (double)b[j] * sj), f1 = (float)((double)b[j] * cj + (double)a[j] * sj);
      asm volatile("" : "+v"(f0), "+v"(f1));  // fp32 numbers: the compiler would round the 64 bits to the type at once
      y0[2 * i + j] = (float)(typename E::T)f0;
      y1[2 * i + j] = (float)(typename E::T)f1;
    }
  }
}
template <typename E>
__device__ __forceinline__ void values8(const u32x4& x, float* y) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2_t a = unpack2<E>(x[i]);
    y[2 * i] = a[0], y[2 * i + 1] = a[1];
  }
}

// Minimum, maximum and whether all is finite of N values of each of LANES neighbouring lanes.
struct Spread {
  float lo, hi;
};
template <int N>
__device__ __forceinline__ Spread spread(const float* x) {
  Spread r{x[0], x[0]};
  bool fine = true;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    r.lo = fminf(r.lo, x[e]);
    r.hi = fmaxf(r.hi, x[e]);
    fine = fine && __builtin_fabsf(x[e]) < __builtin_inff();
  }
  if (!fine) r.hi = __builtin_inff();
  return r;
}
__device__ __forceinline__ Spread join(Spread a, Spread b) { return {fminf(a.lo, b.lo), fmaxf(a.hi, b.hi)}; }
template <int LANES>
__device__ __forceinline__ Spread over_lanes(Spread r) {
#pragma unroll
  for (int off = 1; off < LANES; off *= 2) r = join(r, {__shfl_xor(r.lo, off), __shfl_xor(r.hi, off)});
  return r;
}
// A group's step and offset, of the type.
struct Scale4 {
  float step, z;
};
template <typename E>
__device__ __forceinline__ Scale4 scale_of(Spread r) {
  typedef typename E::T T;
  if (r.hi == __builtin_inff()) return {0.0f, __builtin_nanf("")};
  const float step = (float)(T)((r.hi * 0.5f - r.lo * 0.5f) / 7.5f);
  return {step, (float)(T)((r.lo * 0.5f + r.hi * 0.5f) + step * 0.5f)};
}
// The codes of 8 values in the low halves of two words' bytes: the quotient, rounded to fp32, rounded to a whole number.
// Below 9 in size (beyond, the code is 0 or 15), x times the reciprocal is within 9 (2^-23 + 2^-24) of the quotient and that
// within 9 2^-24 of its rounding, 2^-18.8 in all: away from the halves by 2^-18 both round alike. Where one of a
// wave's 512 values is closer (of scattered ones: in 1 of 256 calls), or none of this holds (a step below 2^-126,
// infinities), the division decides. 5279 new tokens of 28/4 heads: 20.5 us, with the division alone 21.7.
__device__ __forceinline__ u32x2 codes8(const float* x, Scale4 s) {
  const float by = __builtin_amdgcn_rcpf(s.step);
  float t[8];
  bool sure = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = (x[e] - s.z) * by;
    t[e] = __builtin_rintf(y);
    sure = sure && __builtin_fabsf(y - t[e]) < 0.5f - 0x1p-18f;
  }
  if (__any(!sure)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = s.step > 0.0f ? __builtin_rintf((x[e] - s.z) / s.step) : 0.0f;
  }
  u32x2 w = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e >> 2] |= (uint32_t)fminf(fmaxf(t[e] + 8.0f, 0.0f), 15.0f) << (8 * int4_byte(e & 3));
  return w;
}
template <typename E>
__device__ __forceinline__ void put_scale(unsigned char* at, Scale4 s) {
  *reinterpret_cast<typename E::T*>(at) = (typename E::T)s.step;
  *reinterpret_cast<typename E::T*>(at + 16) = (typename E::T)s.z;
}

// Quantises position r of a block's k: lane j of the HD/16 of a head has dims 8j .. 8j+7 (y0) and HD/2 + 8j .. (y1).
template <typename E, int HD, int NG>
__device__ __forceinline__ void store_k(unsigned char* block, int r, int j, const float* y0, const float* y1) {
  typedef Int4Block<HD, NG> L;
  constexpr int LH = HD / 16;
  Spread s0 = spread<8>(y0), s1 = spread<8>(y1);
  if constexpr (NG == 1) {
    s0 = s1 = over_lanes<LH>(join(s0, s1));
  } else {
    s0 = over_lanes<NG == 4 ? 4 : LH>(s0);
    s1 = over_lanes<NG == 4 ? 4 : LH>(s1);
  }
  const Scale4 a = scale_of<E>(s0), b = scale_of<E>(s1);
  const u32x2 c0 = codes8(y0, a), c1 = codes8(y1, b);
  if constexpr (HD == 128) {  // dims of an even step of 32 meet those of the odd one, four lanes on
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = c0[i] | (__shfl_xor(c0[i], 4) << 4);
      w[2 + i] = c1[i] | (__shfl_xor(c1[i], 4) << 4);
    }
    if (j < 4) *reinterpret_cast<u32x4*>(block + int4_k_at<HD>(r, j)) = w;
  } else {
    *reinterpret_cast<u32x2*>(block + int4_k_at<HD>(r, j)) = u32x2{c0[0] | (c1[0] << 4), c0[1] | (c1[1] << 4)};
  }
  unsigned char* const p = block + L::kParams;
  if constexpr (NG == 1) {
    if (j == 0) put_scale<E>(p + int4_param_at(0, r), a);
  } else if constexpr (NG == 2) {
    if (j == 0) put_scale<E>(p + int4_param_at(0, r), a), put_scale<E>(p + int4_param_at(1, r), b);
  } else if (j % 4 == 0) {
    put_scale<E>(p + int4_param_at(j / 4, r), a);
    put_scale<E>(p + int4_param_at(2 + j / 4, r), b);
  }
}

// Quantises position r of a block's v: lane j of the HD/8 of a head has dims 8j .. 8j+7 (y). `bytes` gets the codes' bytes
// (the block's v, or a copy of it in LDS), `block` the steps and offsets.
template <typename E, int HD, int NG>
__device__ __forceinline__ void store_v(unsigned char* bytes, unsigned char* block, int r, int j, const float* y) {
  constexpr int LG = HD / NG / 8;  // lanes of a group
  const Scale4 s = scale_of<E>(over_lanes<LG>(spread<8>(y)));
  const u32x2 c = codes8(y, s);
  // an even block of 16 dims meets the odd one, two lanes on: each of the two lanes stores four of the eight bytes
  const bool odd = j & 2;
  const uint32_t other = __shfl_xor(odd ? c[0] : c[1], 2);
  const uint32_t w = odd ? other | (c[1] << 4) : c[0] | (other << 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) bytes[int4_v_at(r, (j & 1) * 8 + (odd ? 4 : 0) + e, j >> 2)] = (unsigned char)(w >> (8 * int4_byte(e)));
  if (j % LG == 0) put_scale<E>(block + Int4Block<HD, NG>::kVParams + int4_param_at(j / LG, r), s);
}

constexpr int kTokThreads = 256;

// Latency bounds it: the length, the page's id, the angles, one after the other. One token of 12/2 heads 3.8 us, 96 of 32/8
// 5.1.
// Thread i of a token's workgroups (y) takes 8 dims of a q or k head and their partners, or (from a wave's first lane
// on, so that a head's lanes stay in one wave) 8 of a v head; its loads go out before the angles.
template <typename E, int HD, int NG>
__global__ __launch_bounds__(kTokThreads) void append4_token_kernel(Append4Args a) {
  typedef typename E::T T;
  typedef Int4Block<HD, NG> L;
  constexpr int LH = HD / 16;  // lanes per q or k head
  constexpr int LV = HD / 8;   // lanes per v head
  __shared__ __align__(16) double cs[2][HD / 2];  // k's
  __shared__ __align__(16) float cq[2][HD / 2];   // q's, by another wave at the same time
  const int t = blockIdx.x, tid = threadIdx.x, i = tid + (int)blockIdx.y * kTokThreads;
  const int pairs = (a.nq + a.nkv) * LH, j = i - (pairs + 63) / 64 * 64;
  const bool rot = i < pairs, val = j >= 0 && j < a.nkv * LV;
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
    const int64_t at = a.rope_pos ? a.rope_pos[t] : (int64_t)p;
    if (tid < HD / 2)
      angle64(at, a.inv_freq[tid], &cs[0][tid], &cs[1][tid]);
    else if (tid >= 64 && tid < 64 + HD / 2)
      angle(at, a.inv_freq[tid - 64], &cq[0][tid - 64], &cq[1][tid - 64]);
    __syncthreads();
  }
  const bool wr = page >= 0 && page < a.pages;
  const int c = p >= 0 ? p / kChunkPos % a.cpp : 0, r = p & 31;
  // block of kv head g: where wr
  auto block = [&](int g) { return (unsigned char*)a.pool + (page * a.stride + ((int64_t)g * a.cpp + c) * L::kWords) * 2; };
  if (rot && h < a.nq) {
    if (a.inv_freq) rotate8<E>(x0, x1, &cq[0][d], &cq[1][d]);
    T* q = (T*)a.q + (int64_t)t * a.ldq + (int64_t)h * HD;
    *reinterpret_cast<u32x4*>(q + d) = x0;
    *reinterpret_cast<u32x4*>(q + HD / 2 + d) = x1;
  } else if (rot && wr) {
    float y0[8], y1[8];
    if (a.inv_freq)
      turn8<E>(x0, x1, &cs[0][d], &cs[1][d], y0, y1);
    else
      values8<E>(x0, y0), values8<E>(x1, y1);
    store_k<E, HD, NG>(block(h - a.nq), r, d / 8, y0, y1);
  } else if (val && wr) {
    float y[8];
    values8<E>(x0, y);
    store_v<E, HD, NG>(block(h) + L::kV, block(h), r, d / 8, y);
  }
}

constexpr int kChunkThreads = 256;

// Workgroup x: of the sequences' chunks, sequence b's begin at index cu[b] / 32 + 2b (at most
// (n + 62) / 32 chunks hold its n new tokens, which is at most floor((cu + n) / 32) - floor(cu / 32)
// + 2). Each workgroup finds its sequence with a binary search. The workgroups y of a chunk share the heads, k's first and q's
// last: what takes longest starts first. A thread has one position and 8 dims of every q and k head that
// it meets, so its 8 angles stay in registers; the next head's values come in while one is quantised. (With the
// angles in LDS for every head, which holds a CU to 4 workgroups: 26.7 us where this takes 20.4.)
//
// 5279 new tokens of 28/4 heads, 90 MB: 19 to 20 us, 4.5 TB/s. The vector unit is next to memory (67% of the busy cycles):
// its part for k, angles and rotation in 64 bits, is 4 to 6 us, v's 4, q's 4.
template <typename E, int HD, int NG>
__global__ __launch_bounds__(kChunkThreads) void append4_chunk_kernel(Append4Args a) {
  typedef typename E::T T;
  typedef Int4Block<HD, NG> L;
  constexpr int LH = HD / 16, LV = HD / 8;
  constexpr int HP = kChunkThreads / (kChunkPos * LH);  // q or k heads at once
  __shared__ __align__(16) unsigned char vs[16 * HD];  // a head's codes of v
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
  // the chunk's new tokens: rows t0 + first .. t0 + last - 1 at its positions first .. last - 1; chunks are counted from
  // the one that holds pos0 (rounded down, for positions below 0 too)
  const int ci = x - (sr.row0 / kChunkPos + 2 * b);
  const int c0 = (sr.pos0 >= 0 ? sr.pos0 : sr.pos0 - (kChunkPos - 1)) / kChunkPos + ci;
  const int64_t base = (int64_t)c0 * kChunkPos;
  const int first = max(0, (int)(sr.pos0 - base));                                // in the chunk
  const int last = (int)min((int64_t)kChunkPos, sr.pos0 + (int64_t)sr.n - base);  // one past
  if (first >= last) return;
  const int t0 = sr.row0 + (int)(base + first - sr.pos0) - first;  // row of the chunk's position 0
  int64_t page = -1;
  if (c0 >= 0 && base < a.cap) page = a.table[(int64_t)b * a.ldt + c0 / a.cpp];
  const bool wr = page >= 0 && page < a.pages;
  const int c = c0 >= 0 ? c0 % a.cpp : 0;
  const T* rows = (const T*)a.qkv;
  auto block = [&](int g) { return (unsigned char*)a.pool + (page * a.stride + ((int64_t)g * a.cpp + c) * L::kWords) * 2; };
  const int heads = a.nq + 2 * a.nkv, y = blockIdx.y;
  const int h0 = y * heads / (int)gridDim.y, h1 = (y + 1) * heads / (int)gridDim.y;  // of k's, then v's, then q's heads
  // ---- k and q: this thread's position, dims and first head
  const int d = tid % LH * 8, r = tid / LH % kChunkPos, hp = tid / (kChunkPos * LH);
  const bool mine = r >= first && r < last;
  const int64_t row = mine ? t0 + r : 0, at = !mine ? 0 : a.rope_pos ? a.rope_pos[row] : base + r;
  const int ke = wr ? min(h1, a.nkv) : 0;
  if (h0 + hp < ke && mine) {
    const T* src = rows + row * a.ldqkv + (int64_t)(a.nq + h0 + hp) * HD + d;
    u32x4 x0 = *reinterpret_cast<const u32x4*>(src), x1 = *reinterpret_cast<const u32x4*>(src + HD / 2);
    double ck[8], sk[8];
    if (a.inv_freq) {
#pragma unroll
      for (int e = 0; e < 8; ++e) angle64(at, a.inv_freq[d + e], &ck[e], &sk[e]);
    }
    for (int h = h0 + hp; h < ke; h += HP) {
      float y0[8], y1[8];
      if (a.inv_freq)
        turn8<E>(x0, x1, ck, sk, y0, y1);
      else
        values8<E>(x0, y0), values8<E>(x1, y1);
      if (h + HP < ke) {  // the next head's are on their way meanwhile
        src += HP * HD;
        x0 = *reinterpret_cast<const u32x4*>(src), x1 = *reinterpret_cast<const u32x4*>(src + HD / 2);
      }
      store_k<E, HD, NG>(block(h), r, d / 8, y0, y1);
    }
  }
  // ---- v
  constexpr int VI = kChunkPos * LV / kChunkThreads;  // items of a thread
  auto load_v = [&](int h, u32x4* xv) {
#pragma unroll
    for (int n = 0; n < VI; ++n) {
      const int r = (tid + n * kChunkThreads) / LV, d = tid % LV * 8;
      if (r >= first && r < last)
        xv[n] = *reinterpret_cast<const u32x4*>(rows + (int64_t)(t0 + r) * a.ldqkv + (int64_t)(a.nq + a.nkv + h) * HD + d);
    }
  };
  const int v0 = max(h0 - a.nkv, 0), ve = wr ? min(h1 - a.nkv, a.nkv) : 0;
  u32x4 xv[VI];
  if (v0 < ve) load_v(v0, xv);
  for (int h = v0; h < ve; ++h) {
    unsigned char* const blk = block(h);
    float y[VI][8];
#pragma unroll
    for (int n = 0; n < VI; ++n) values8<E>(xv[n], y[n]);
    if (h + 1 < ve) load_v(h + 1, xv);
    __syncthreads();  // the v head before has been copied
#pragma unroll
    for (int n = 0; n < VI; ++n) {
      const int r = (tid + n * kChunkThreads) / LV;
      if (r >= first && r < last) store_v<E, HD, NG>(vs, blk, r, tid % LV, y[n]);
    }
    __syncthreads();
    // item u: the 16 bytes of positions 8 (u / 16 % 4) .. + 7
    for (int u = tid; u < HD; u += kChunkThreads) {
      const int r0 = 8 * (u / 16 % 4);
      if (r0 >= first && r0 + 8 <= last) {
        *reinterpret_cast<u32x4*>(blk + L::kV + u * 16) = *reinterpret_cast<const u32x4*>(vs + u * 16);
      } else {
        for (int r = max(r0, first); r < min(r0 + 8, last); ++r) {
          const int at = u * 16 + ((r >> 2) & 1) * 4 + int4_byte(r & 3);
          blk[L::kV + at] = vs[at];
          blk[L::kV + at + 8] = vs[at + 8];
        }
      }
    }
  }
  // ---- q
  const int hq = max(h0 - 2 * a.nkv, 0) + hp, qe = h1 - 2 * a.nkv;
  if (hq - hp < qe && mine) {
    float cq[8], sq[8];
    if (a.inv_freq) {
#pragma unroll
      for (int e = 0; e < 8; ++e) angle(at, a.inv_freq[d + e], &cq[e], &sq[e]);
    }
#pragma unroll 2
    for (int h = hq; h < qe; h += HP) {
      const T* src = rows + row * a.ldqkv + (int64_t)h * HD + d;
      u32x4 x0 = *reinterpret_cast<const u32x4*>(src), x1 = *reinterpret_cast<const u32x4*>(src + HD / 2);
      if (a.inv_freq) rotate8<E>(x0, x1, cq, sq);
      T* q = (T*)a.q + row * a.ldq + (int64_t)h * HD + d;
      *reinterpret_cast<u32x4*>(q) = x0;
      *reinterpret_cast<u32x4*>(q + HD / 2) = x1;
    }
  }
}

template <typename E, int HD, int NG>
int launch(const Append4Args& a, hipStream_t s) {
  (void)hipGetLastError();
  if (!a.cu) {
    const int items = ((a.nq + a.nkv) * (HD / 16) + 63) / 64 * 64 + a.nkv * (HD / 8);
    append4_token_kernel<E, HD, NG><<<dim3((unsigned)a.T, (unsigned)((items + kTokThreads - 1) / kTokThreads)), kTokThreads, 0, s>>>(a);
  } else {
    const unsigned gx = (unsigned)(a.T / kChunkPos + 2 * a.B);
    // workgroups y: with 1024, 1280 and 2048 workgroups in all, us with the reading back of 5279 new tokens of 28/4 heads 31.5,
    // 29.7, 32.7; of 5622 of 32/8 46.7, 44.8, 44.1; of 3630 of 20/20 of 64 30.5, 29.0, 30.6
    const int hb = std::min(a.nq + 2 * a.nkv, std::max(1, 1280 / (int)(a.T / kChunkPos + a.B)));
    append4_chunk_kernel<E, HD, NG><<<dim3(gx, (unsigned)hb), kChunkThreads, 0, s>>>(a);
  }
  return ldk::check_launch("paged_append_int4");
}
template <typename E>
int launch(const Append4Args& a, int hd, int group, hipStream_t s) {
  if (hd == 64) return group == 32 ? launch<E, 64, 2>(a, s) : launch<E, 64, 1>(a, s);
  return group == 32 ? launch<E, 128, 4>(a, s) : group == 64 ? launch<E, 128, 2>(a, s) : launch<E, 128, 1>(a, s);
}

}  // namespace

extern "C" int ldk_paged_append_int4(const void* qkv, int64_t ldqkv, int dtype, const int32_t* cu_seqlens,
                                     const int32_t* kv_lens, const int32_t* block_table, int64_t ldt, int64_t max_pages,
                                     const int64_t* rope_pos, const float* inv_freq, void* kv_pages, int64_t page_stride,
                                     int64_t num_pages, int64_t page_size, void* q_out, int64_t ldq, int64_t T, int64_t B,
                                     int nq, int nkv, int head_dim, int group, void* stream) {
  static const char* fn = "paged_append_int4";
  if (!qkv || !kv_lens || !block_table || !kv_pages || !q_out) return ldk::fail(LDK_ERR_INVALID, "%s: null pointer", fn);
  int st = ldk::check_int4_pool(fn, dtype, nkv, head_dim, group, page_stride, num_pages, page_size, ldt, max_pages);
  if (st || (st = ldk::check_int4_batch(fn, T, B, int64_t(1) << 20, cu_seqlens))) return st;
  if (nq <= 0 || nq % nkv || nq > 4096)
    return ldk::fail(LDK_ERR_INVALID, "%s: nq=%d must be a positive multiple of nkv=%d (at most 4096)", fn, nq, nkv);
  if (ldqkv < (int64_t)(nq + 2 * nkv) * head_dim || ldq < (int64_t)nq * head_dim)
    return ldk::fail(LDK_ERR_INVALID, "%s: strides ldqkv=%lld ldq=%lld below what they step over", fn, (long long)ldqkv, (long long)ldq);
  if (!ldk::aligned(qkv, 16) || !ldk::aligned(q_out, 16) || !ldk::aligned(kv_pages, 16) || ldqkv % 8 || ldq % 8 ||
      page_stride % 8 || !ldk::aligned(kv_lens, 4) || !ldk::aligned(cu_seqlens, 4) || !ldk::aligned(block_table, 4) ||
      !ldk::aligned(rope_pos, 8) || !ldk::aligned(inv_freq, 4))
    return ldk::fail(LDK_ERR_ALIGN, "%s: qkv, q_out and the pages 16-byte aligned with strides of multiples of 8 elements", fn);
  const Append4Args a{qkv, ldqkv, cu_seqlens, kv_lens, block_table, ldt, rope_pos, inv_freq, kv_pages, q_out, page_stride, ldq,
                      cu_seqlens ? (int)T : (int)B, (int)B, nq, nkv, (int)num_pages, (int)(page_size / 32),
                      (int)(max_pages * page_size)};
  hipStream_t s = (hipStream_t)stream;
  return dtype == LDK_F16 ? launch<ldk::F16>(a, head_dim, group, s) : launch<ldk::BF16>(a, head_dim, group, s);
}

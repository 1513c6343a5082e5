// Element types, cache pages and ragged sequences of the paged operators (paged_append.hip,
// paged_attention.hip). Not part of the C ABI.
//
// The cache is a pool of pages of `page` positions (a multiple of 32). A page holds, per kv head, the
// tiles of the static cache (attention.hip), each one 16-byte load per lane of a wave:
//  - K:   [page/32 chunks][2 row halves hb][hd/32 dim steps s][16 rows i][32 dims]; row i of half hb of
//         a chunk holds its position 8(i/4) + 4hb + i%4, dims 32s .. 32s + 31;
//  - V^T: [page/32 chunks][hd/16 dim blocks][16 dims][32 positions].
// Position p of sequence b is row p % page of page table[b][p / page]. A page id outside [0, pages) is
// no page: an append writes nothing there and the attention does not see its positions.
//
// Sequence b of a ragged batch has the rows cu[b] .. cu[b+1] - 1 of the call's new tokens (row b alone
// where cu is null) and kv_lens[b] positions in the cache, the new tokens the last of them: its i-th
// new token is at position kv_lens[b] - (cu[b+1] - cu[b]) + i.
#pragma once

#include "ldk_common.h"

namespace ldk {

struct F16 {
  typedef half_t T;
  static constexpr uint32_t kOnes = 0x3C003C00u;  // (1, 1)
  static constexpr float kMost = 65504.0f;        // the largest finite number
  // softmax numerators are held times 2^kShift: a weight of 2^-25 of the largest, where fp16 alone ends,
  // would be lost, and with it a long context's many small ones beside a large one
  static constexpr float kShift = 7.0f;
  typedef half_t T2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ float4_t mfma(u32x4 a, u32x4 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  }
};
struct BF16 {
  typedef __bf16 T;
  static constexpr uint32_t kOnes = 0x3F803F80u;
  static constexpr float kMost = 0x1.FEp127f;
  static constexpr float kShift = 0.0f;
  typedef __bf16 T2 __attribute__((ext_vector_type(2)));
  typedef __bf16 T8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float4_t mfma(u32x4 a, u32x4 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b), c, 0, 0, 0);
  }
};

// Two floats rounded to nearest even, as one 32-bit word; and back.
template <typename E>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_t){a, b}, typename E::T2));
}
template <typename E>
__device__ __forceinline__ float2_t unpack2(uint32_t u) {
  return __builtin_convertvector(__builtin_bit_cast(typename E::T2, u), float2_t);
}
// x, or the type's largest number in the place of a finite one that would round to an infinity.
template <typename E>
__device__ __forceinline__ float bounded(float x) {
  return __builtin_fabsf(x) < __builtin_inff() ? __builtin_amdgcn_fmed3f(x, -E::kMost, E::kMost) : x;
}

constexpr int kChunkPos = 32;          // positions of a chunk
constexpr int kTileElems = 512;        // elements of a 1 KB tile
constexpr int64_t kMaxPositions = int64_t(1) << 25;  // of one sequence

// c / n and c % n of a chunk c < 2^20 by the chunks of a page, 1 <= n <= 2^11: with m = ceil(2^31 / n) =
// (2^31 + e) / n, e < n, 2 c m / 2^32 = c / n + c e / (n 2^31), and c e < 2^31 keeps its floor.
struct PageDiv {
  uint32_t n, m;
};
inline PageDiv page_div(int64_t n) { return {(uint32_t)n, (uint32_t)(((int64_t(1) << 31) + n - 1) / n)}; }
__device__ __forceinline__ void chunk_page(const PageDiv& d, int c, int& page, int& sub) {
  page = (int)__umulhi(2u * (uint32_t)c, d.m);
  sub = c - page * (int)d.n;
}

// The new rows and positions of sequence b.
struct SeqRows {
  int row0, n;   // rows row0 .. row0 + n - 1
  int pos0;      // position of row0 (negative where kv_lens is below the new tokens' count)
};
__device__ __forceinline__ SeqRows seq_rows(const int32_t* cu, const int32_t* kv_lens, int b, int T) {
  SeqRows s;
  s.row0 = cu ? cu[b] : b;
  const int end = cu ? cu[b + 1] : b + 1;
  s.n = end - s.row0;
  s.pos0 = max(kv_lens[b], -(1 << 30)) - s.n;
  if (s.row0 < 0 || end > T || s.row0 > end) s.n = 0;  // not rows of this call
  return s;
}

}  // namespace ldk

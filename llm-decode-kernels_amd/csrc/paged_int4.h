// A paged cache held in 4 bits (paged_append_int4.hip, paged_read_int4.hip, paged_attention_int4.hip); pages, tables
// and ragged sequences as in paged.h. Not part of the C ABI.
//
// A position's k (v) of a kv head is held in groups of 32, 64 or 128 dims, each with a step and an offset z of the
// cache's type, as codes 0..15:  value = z + (code - 8) step. Of a group's values x, which have the type (k after
// its rotation is rounded to it):
//   step = rnd((max/2 - min/2) / 7.5)   z = rnd((min/2 + max/2) + step/2)   code = clamp(rint((x - z) / step) + 8)
// in fp32, rnd to the type, so that codes 0 and 15 lie at the minimum and the maximum but for the roundings of step and z: with
// u half a step of the type at 1 (2^-11, bf16 2^-8) a value is off by at most step/2 + u (|z| + 7.5 step), which the
// offset rules where a group lies far from 0 (bf16 900 .. 904: z 904, and 900 is held as 901.9). step = 0: code 8. A group with
// a NaN or an infinity gets step 0 and z NaN; a value that the roundings put past the type's largest number is read as that.
// One pair per position (not per channel): a token is quantised as it
// comes, whatever its neighbours are, and a group's range is that of one head's dims; the finer groups keep a
// dim that is far larger than the others (as some of k's are) from coarsening all of them.
//
// A page holds [kv head][page/32 chunks][block of a chunk], a block the bytes
//   [0, 16 hd)      codes of k. Row i of half h holds position 8(i/4) + 4h + i%4 (paged.h's tiles). Lane kb 16 + i of
//                   a wave finds dims 8kb .. 8kb+7 of every step of 32 dims in 16 bytes (hd 128; of half h at 1024 h + 16
//                   lane) or in 8 (hd 64; at 16 lane + 8 h): 8 bytes per pair of steps, in them two words of 4 dims, in
//                   a word's byte 0, 2, 1, 3 dims 0, 1, 2, 3, the even step's in the low four bits;
//   [16 hd, 32 hd)  codes of v. Lane kb 16 + c finds positions 8kb .. 8kb+7 of dim c of every block of 16 dims in
//                   16 bytes per 4 blocks (at 1024 (b/4) + 16 lane): 8 bytes per pair of blocks, two words of 4 positions,
//                   bytes as above, the even block's in the low four bits;
//   then 128 bytes per group of k, and per group of v: [position / 8]{8 steps, 8 offsets}.
// A byte is one position's alone, so an append writes whole bytes and no two tokens meet in one. word & 0x000F000F are the
// codes of elements 0 and 1 in the low bits of two halves, (word >> 8) & 0x000F000F of 2 and 3, and with 0x00F000F0 the
// odd step's or block's: an or makes fp16 numbers of them.
#pragma once

#include "paged.h"

namespace ldk {

template <int HD, int NG>  // NG groups of HD / NG dims
struct Int4Block {
  static constexpr int kV = 16 * HD;                  // byte offsets: v's codes,
  static constexpr int kParams = 32 * HD;             // k's steps and offsets,
  static constexpr int kVParams = kParams + 128 * NG; // v's
  static constexpr int kBytes = kVParams + 128 * NG;
  static constexpr int kWords = kBytes / 2;           // elements of the pool's type
};

constexpr uint32_t kLow4 = 0x000F000Fu, kHigh4 = 0x00F000F0u;

// Byte of a word that holds element e of 4.
__host__ __device__ constexpr int int4_byte(int e) { return (e & 1) * 2 + (e >> 1); }

// Byte offset of the 8 bytes (hd 64) or 16 (hd 128: both pairs of steps) of position r's dims 8kb .. of a block's k.
template <int HD>
__device__ __forceinline__ int int4_k_at(int r, int kb) {
  const int half = (r >> 2) & 1, unit = kb * 16 + 4 * (r >> 3) + (r & 3);
  return HD == 128 ? half * 1024 + unit * 16 : unit * 16 + half * 8;
}
// Byte offset, from v's codes on, of position r's byte for column c of the pair t of 16-dim blocks.
__device__ __forceinline__ int int4_v_at(int r, int c, int t) {
  return (t >> 1) * 1024 + ((r >> 3) * 16 + c) * 16 + (t & 1) * 8 + ((r >> 2) & 1) * 4 + int4_byte(r & 3);
}
// Byte offset of a group's step for position r, from its params on; the offset z is 16 further.
__device__ __forceinline__ int int4_param_at(int g, int r) { return g * 128 + (r >> 3) * 32 + (r & 7) * 2; }

// The arguments that the entries share, checked; LDK_OK or a status with its message set.
inline int check_int4_pool(const char* fn, int dtype, int nkv, int hd, int group, int64_t page_stride, int64_t num_pages,
                           int64_t page_size, int64_t ldt, int64_t max_pages) {
  if (dtype != LDK_F16 && dtype != LDK_BF16) return fail(LDK_ERR_INVALID, "%s: dtype %d (fp16 or bf16)", fn, dtype);
  if (hd != 64 && hd != 128) return fail(LDK_ERR_UNSUPPORTED, "%s: head_dim=%d (64 or 128)", fn, hd);
  if ((group != 32 && group != 64 && group != 128) || group > hd)
    return fail(LDK_ERR_UNSUPPORTED, "%s: group=%d (32, 64 or 128, at most head_dim=%d)", fn, group, hd);
  if (nkv <= 0 || nkv > 4096) return fail(LDK_ERR_INVALID, "%s: nkv=%d (1..4096)", fn, nkv);
  if (page_size < 32 || page_size % 32 || page_size > 65536)
    return fail(LDK_ERR_UNSUPPORTED, "%s: page_size=%lld must be a multiple of 32 up to 65536", fn, (long long)page_size);
  if (num_pages <= 0 || num_pages > INT32_MAX || max_pages <= 0 || ldt < max_pages || max_pages > kMaxPositions / page_size)
    return fail(LDK_ERR_INVALID, "%s: num_pages=%lld max_pages=%lld ldt=%lld", fn, (long long)num_pages, (long long)max_pages, (long long)ldt);
  if (page_stride > INT32_MAX) return fail(LDK_ERR_UNSUPPORTED, "%s: page stride %lld past 2^31", fn, (long long)page_stride);
  if (page_stride < nkv * (page_size / 32) * (16 * hd + 128 * (hd / group)))
    return fail(LDK_ERR_INVALID, "%s: page stride %lld below a page", fn, (long long)page_stride);
  return LDK_OK;
}
inline int check_int4_batch(const char* fn, int64_t T, int64_t B, int64_t most_b, bool ragged) {
  if (T <= 0 || T > (int64_t(1) << 24) || B <= 0 || B > most_b)
    return fail(LDK_ERR_INVALID, "%s: T=%lld tokens (1..2^24) of B=%lld sequences (1..%lld)", fn, (long long)T, (long long)B, (long long)most_b);
  if (!ragged && T < B) return fail(LDK_ERR_INVALID, "%s: T=%lld rows for B=%lld sequences of one token", fn, (long long)T, (long long)B);
  return LDK_OK;
}

}  // namespace ldk

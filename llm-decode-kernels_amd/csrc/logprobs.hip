// Log probabilities of given tokens: per row of logits x[V], with m = max x and s = sum exp(x - m),
//   logprob = (x[token] - m) - ln s,   entropy = ln s - sum exp(x - m) (x - m) / s,
// and the `top` largest logits (NaN largest, the lowest index first on ties, as torch.argmax orders
// them) with their log probabilities. Every logit is read once.
//
// A row is cut into `splits` slices, one workgroup each; a wave takes tiles of 1024 consecutive logits
// of its slice (16 per lane, the next tile's loads in flight), tiles w, w + 4, ... by wave w.
//  - Sums: each lane keeps a maximum of its own and rescales its two sums once per tile, so a logit
//    costs one fma, one exp2, one add and one fma; y = x log2 e - base is in powers of two.
//    exp(-inf) * -inf would be NaN: a tile whose second sum is NaN is summed again with y clamped.
//  - The largest: each wave keeps candidates (64-bit keys, value then lower index) in its own LDS list
//    and a threshold below which nothing can be among them: the top-th largest of its 64 lanes'
//    running maxima (found bit by bit with ballots), which lets through about the logits that are
//    the largest so far. Tiles come in rising index order, so a later logit equal to the threshold
//    loses its tie. A list that fills up is cut back to its `top` largest. The lists' entries are
//    ranked by counting.
// Rows of several slices leave {base, s, sum, keys} per slice in the workspace, which the next launch
// joins with one wave per row. What bounds it: the bytes for 32-bit logits; for 16-bit ones the
// vector instructions come close (one exp2 is four instructions' time).
#include <algorithm>

#include "ldk_common.h"

namespace {

constexpr int kWaves = 4;
constexpr int kPer = 16;             // logits of a lane per tile
constexpr int kTileLogits = 64 * kPer;
constexpr int kTopMax = 64;          // a wave's lanes: the threshold is a lane's maximum
constexpr int kKeep = 128;           // candidates past which a list is cut back
constexpr int kCap = kKeep + kTileLogits;
constexpr int kMergeKeys = 1024;     // keys of a row's slices that the joining wave takes
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

struct LogprobArgs {
  const void* x;
  int64_t ld;
  const int64_t* tokens;
  float *logprob, *entropy, *top_lp;
  int64_t* top_ids;
  float* part;     // [rows][splits][4]: base, s, sum
  uint64_t* keys;  // [rows][splits][top], descending
  int64_t rows;
  int V, top, splits, slice;  // slice: tiles of a slice
};

// Unsigned order of the floats: NaN above +inf, -0 and +0 one value.
__device__ __forceinline__ uint32_t order(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
  if (v != v) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t o) {
  return __builtin_bit_cast(float, o == 0xffffffffu ? 0x7fc00000u : o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// The n-th largest (n in 1..64) of the 64 lanes' values: the largest t with at least n values >= t.
__device__ __forceinline__ uint32_t nth_largest(uint32_t v, int n) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    if (__popcll(__ballot(v >= c)) >= n) t = c;
  }
  return t;
}

// Cuts a wave's list of n keys to its `top` largest, in descending order at out[0 ..); absent ones are
// 0. Keys of one list differ (their indexes do) but for absent zeros, which the position tells apart.
__device__ __forceinline__ void rank_keys(const uint64_t* list, int n, int top, uint64_t* out, int lane) {
  for (int i = lane; i < n; i += 64) {
    const uint64_t key = list[i];
    int r = 0;
    for (int j = 0; j < n; ++j) {
      const uint64_t other = list[j];
      r += other > key || (other == key && j < i);
    }
    if (r < top) out[r] = key;
  }
  for (int i = n + lane; i < top; i += 64) out[i] = 0;
}

// What a row's sums become: the combination of two {base, s, sum} triples over one logits row.
struct Sums {
  float m, base, s, y;  // maximum, its power-of-two base, sum of 2^(x log2e - base) and of that times its exponent
};
__device__ __forceinline__ float base_of(float m) { return m == -__builtin_inff() ? 0.0f : m * kLog2e; }
// a's sums taken against another maximum m (not below a's).
__device__ __forceinline__ void rebase(Sums& a, float m) {
  const float base = base_of(m), d = a.base - base;
  const float f = a.m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(d);
  // nothing summed yet, or too far below to matter: 0, and not 0 x inf
  a.y = f == 0.0f ? a.s * 0.0f : f * __builtin_fmaf(d, a.s, a.y);
  a.s *= f;
  a.m = m;
  a.base = base;
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  const float m = fmaxf(a.m, b.m);
  rebase(a, m);
  rebase(b, m);
  a.s += b.s;
  a.y += b.y;
  return a;
}
__device__ __forceinline__ Sums wave_join(Sums a) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    a = join(a, Sums{__shfl_xor(a.m, off), __shfl_xor(a.base, off), __shfl_xor(a.s, off), __shfl_xor(a.y, off)});
  return a;
}

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<half_t>(half_t v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<uint16_t>(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }

// The answers of one row, from its sums and its sorted keys (lanes 0 .. top - 1 hold one each).
template <typename T>
__device__ __forceinline__ void finish(const LogprobArgs& a, int64_t row, const Sums& t, uint64_t key, int lane) {
  const float log_s = __builtin_amdgcn_logf(t.s);  // powers of two
  if (lane == 0) {
    const int64_t tok = a.tokens[row];
    float lp = __builtin_nanf("");
    if (tok >= 0 && tok < a.V) lp = (__builtin_fmaf(to_f<T>(((const T*)a.x)[row * a.ld + tok]), kLog2e, -t.base) - log_s) * kLn2;
    a.logprob[row] = lp;
    a.entropy[row] = (log_s - t.y / t.s) * kLn2;
  }
  if (lane < a.top) {
    a.top_lp[row * a.top + lane] = (__builtin_fmaf(from_order((uint32_t)(key >> 32)), kLog2e, -t.base) - log_s) * kLn2;
    a.top_ids[row * a.top + lane] = (int64_t)(uint32_t)~(uint32_t)key;
  }
}

template <typename T, bool TOP>
__global__ __launch_bounds__(kWaves * 64) void logprobs_kernel(LogprobArgs a) {
  constexpr int VEC = 16 / sizeof(T), NV = kPer / VEC;
  typedef T vec_t __attribute__((ext_vector_type(VEC)));
  __shared__ uint64_t lists[TOP ? kWaves : 1][TOP ? kCap : 1];
  __shared__ uint64_t best[TOP ? kWaves : 1][kTopMax], sorted[kTopMax];
  __shared__ Sums sums[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * 65535;
  if (row >= a.rows) return;
  const T* x = (const T*)a.x + row * a.ld;
  // 16-byte vectors from the address below the row's start on: logit i of vector v is v * VEC + i - head
  const int head = (int)((uintptr_t)x & 15) / (int)sizeof(T);
  const int first = (int)blockIdx.x * a.slice, tiles = min(a.slice, (a.V + head + kTileLogits - 1) / kTileLogits - first);

  // the 16 logits of this lane in tile t: vectors lane + 64 u of it, whole ones as 16-byte loads; -inf past
  // the row's ends (exp 0 and never among the largest unless the row has fewer numbers)
  auto load = [&](int t, vec_t (&v)[NV]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = ((first + t) * NV + u) * 64 * VEC + lane * VEC - head;
      if (i >= 0 && i + VEC <= a.V) {
        v[u] = *reinterpret_cast<const vec_t*>(x + i);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          T none;
          if constexpr (sizeof(T) == 4)
            none = -__builtin_inff();
          else
            none = __builtin_bit_cast(T, (uint16_t)(__is_same(T, half_t) ? 0xfc00 : 0xff80));
          v[u][e] = i + e >= 0 && i + e < a.V ? x[i + e] : none;
        }
      }
    }
  };

  Sums s{-__builtin_inff(), 0.0f, 0.0f, 0.0f};
  uint32_t thr = 0, lmax = 0;  // candidates are above thr; this lane's largest so far
  int n = 0, next_thr = 0, seen = 0;
  vec_t cur[NV], nxt[NV];
  if (wave < tiles) load(wave, cur);
  for (int t = wave; t < tiles; t += kWaves) {
    if (t + kWaves < tiles) load(t + kWaves, nxt);
    float v[kPer];
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[u * VEC + e] = to_f<T>(cur[u][e]);
    float tm = v[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) tm = fmaxf(tm, v[e]);
    rebase(s, fmaxf(s.m, tm));
    float ts = 0.0f, ty = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float y = __builtin_fmaf(v[e], kLog2e, -s.base), p = __builtin_amdgcn_exp2f(y);
      ts += p;
      ty = __builtin_fmaf(p, y, ty);
    }
    const bool odd = ty != ty;  // an infinity or a NaN among them
    if (__any(odd)) {
      ty = 0.0f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const float y = __builtin_fmaf(v[e], kLog2e, -s.base), p = __builtin_amdgcn_exp2f(y);
        ty = __builtin_fmaf(p, fmaxf(y, -1e30f), ty);
      }
    }
    s.s += ts;
    s.y += ty;
    if constexpr (TOP) {
      uint32_t tk = order(tm);
      if (ts != ts) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) tk = max(tk, order(v[e]));
      }
      lmax = max(lmax, tk);
      uint64_t hit = __ballot(tk > thr);
      if (hit) {
        uint32_t floor = thr;  // of this tile's candidates: above floor
        // a new threshold at tiles 0, 1, 3, 7, ... of the wave, and where many lanes hit
        if (seen >= next_thr || __popcll(hit) > a.top) {
          const uint32_t nth = nth_largest(lmax, a.top);
          if (nth > thr) {
            floor = nth - 1;  // this tile's equals are among the ones that made it
            thr = nth;
          }
          next_thr = 2 * seen + 1;
        }
        if (tk > floor) {
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const uint32_t o = order(v[e]);
            const int i = ((first + t) * NV + e / VEC) * 64 * VEC + lane * VEC + e % VEC - head;
            const bool take = o > floor && i >= 0 && i < a.V;
            const uint64_t mask = __ballot(take);
            if (take) lists[wave][n + __popcll(mask & ((uint64_t(1) << lane) - 1))] = ((uint64_t)o << 32) | (uint32_t)~i;
            n += __popcll(mask);
          }
        }
        // n is the same in every lane that took part: the others take the first hit's
        n = __builtin_amdgcn_readlane(n, __builtin_ctzll(__ballot(tk > floor) | (uint64_t(1) << 63)));
        if (n > kKeep) {
          ldk::wave_lds_sync();
          rank_keys(lists[wave], n, a.top, best[wave], lane);
          ldk::wave_lds_sync();
          if (lane < a.top) lists[wave][lane] = best[wave][lane];
          n = a.top;
          ldk::wave_lds_sync();
          thr = max(thr, (uint32_t)(lists[wave][a.top - 1] >> 32));
        }
      }
      ++seen;
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) cur[u] = nxt[u];
  }

  s = wave_join(s);
  if (lane == 0) sums[wave] = s;
  if constexpr (TOP) {
    ldk::wave_lds_sync();
    rank_keys(lists[wave], n, a.top, best[wave], lane);
  }
  __syncthreads();
  if constexpr (TOP) {
    if (lane < a.top) {
      const uint64_t key = best[wave][lane];
      int r = 0;
      for (int w = 0; w < kWaves; ++w)
        for (int j = 0; j < a.top; ++j) {
          const uint64_t other = best[w][j];
          r += other > key || (other == key && w * kTopMax + j < wave * kTopMax + lane);
        }
      if (r < a.top) sorted[r] = key;
    }
    __syncthreads();
  }
  if (wave) return;
  Sums all = sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) all = join(all, sums[w]);
  const uint64_t key = TOP && lane < a.top ? sorted[lane] : 0;
  if (a.splits == 1) {
    finish<T>(a, row, all, key, lane);
  } else {
    const int64_t at = row * a.splits + blockIdx.x;
    if (lane == 0) {
      float* p = a.part + at * 4;
      p[0] = all.m;
      p[1] = all.s;
      p[2] = all.y;
    }
    if (TOP && lane < a.top) a.keys[at * a.top + lane] = key;
  }
}

// Joins a row's slices: one wave per row.
template <typename T>
__global__ __launch_bounds__(64) void logprobs_join_kernel(LogprobArgs a) {
  __shared__ uint64_t list[kMergeKeys], sorted[kTopMax];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  Sums s{-__builtin_inff(), 0.0f, 0.0f, 0.0f};
  for (int i = lane; i < a.splits; i += 64) {
    const float* p = a.part + (row * a.splits + i) * 4;
    s = join(s, Sums{p[0], base_of(p[0]), p[1], p[2]});
  }
  s = wave_join(s);
  uint64_t key = 0;
  if (a.top) {
    const int total = a.splits * a.top;
    constexpr int PER = kMergeKeys / 64;
    uint64_t k[PER];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      k[i] = lane + 64 * i < total ? a.keys[row * total + lane + 64 * i] : 0;
      most = max(most, (uint32_t)(k[i] >> 32));
    }
    const uint32_t nth = nth_largest(most, a.top);
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool take = k[i] && (uint32_t)(k[i] >> 32) >= nth;
      const uint64_t mask = __ballot(take);
      if (take) list[n + __popcll(mask & ((uint64_t(1) << lane) - 1))] = k[i];
      n += __popcll(mask);
    }
    ldk::wave_lds_sync();
    rank_keys(list, n, a.top, sorted, lane);
    ldk::wave_lds_sync();
    if (lane < a.top) key = sorted[lane];
  }
  finish<T>(a, row, s, key, lane);
}

// Slices of a row: enough workgroups for the CUs, whole tiles for every wave, keys for one joining wave.
int plan_splits(int64_t rows, int64_t V, int top) {
  const int64_t most = std::max<int64_t>(1, V / (kWaves * kTileLogits));
  int64_t s = std::min<int64_t>(most, std::max<int64_t>(1, 1024 / rows));
  if (top) s = std::min<int64_t>(s, kMergeKeys / top);
  return (int)std::min<int64_t>(s, 512);
}
int64_t workspace_bytes(int64_t rows, int64_t V, int top) {
  const int64_t s = plan_splits(rows, V, top);
  return s == 1 ? 0 : rows * s * (16 + 8 * (int64_t)top);
}

template <typename T>
int launch(LogprobArgs& a, hipStream_t s) {
  (void)hipGetLastError();
  const dim3 grid((unsigned)a.splits, (unsigned)std::min<int64_t>(a.rows, 65535), (unsigned)((a.rows + 65534) / 65535));
  if (a.top)
    logprobs_kernel<T, true><<<grid, kWaves * 64, 0, s>>>(a);
  else
    logprobs_kernel<T, false><<<grid, kWaves * 64, 0, s>>>(a);
  const int st = ldk::check_launch("token_logprobs");
  if (st || a.splits == 1) return st;
  logprobs_join_kernel<T><<<(unsigned)a.rows, 64, 0, s>>>(a);
  return ldk::check_launch("token_logprobs join");
}

bool in_range(int64_t rows, int64_t V, int64_t top) {
  return rows > 0 && rows <= (int64_t(1) << 24) && V > 0 && V <= (int64_t(1) << 30) && top >= 0 && top <= kTopMax && top <= V;
}

}  // namespace

extern "C" int64_t ldk_token_logprobs_workspace_bytes(int64_t rows, int64_t V, int top) {
  if (!in_range(rows, V, top))
    return -ldk::fail(LDK_ERR_INVALID, "token_logprobs: rows=%lld (1..2^24) V=%lld (1..2^30) top=%d (0..%d, at most V)",
                      (long long)rows, (long long)V, top, kTopMax);
  return workspace_bytes(rows, V, top);
}

extern "C" int ldk_token_logprobs(const void* logits, int64_t ld, int dtype, const int64_t* tokens, int64_t rows, int64_t V,
                                  int top, float* logprob, float* entropy, float* top_logprobs, int64_t* top_ids,
                                  void* workspace, int64_t workspace_bytes_, void* stream) {
  static const char* fn = "token_logprobs";
  if (!logits || !tokens || !logprob || !entropy || (top && (!top_logprobs || !top_ids)))
    return ldk::fail(LDK_ERR_INVALID, "%s: null pointer", fn);
  if (!in_range(rows, V, top))
    return ldk::fail(LDK_ERR_INVALID, "%s: rows=%lld (1..2^24) V=%lld (1..2^30) top=%d (0..%d, at most V)", fn, (long long)rows,
                     (long long)V, top, kTopMax);
  if (ld < V && rows > 1) return ldk::fail(LDK_ERR_INVALID, "%s: ld=%lld below V=%lld", fn, (long long)ld, (long long)V);
  if (dtype != LDK_F16 && dtype != LDK_BF16 && dtype != LDK_F32) return ldk::fail(LDK_ERR_INVALID, "%s: unknown dtype %d", fn, dtype);
  if (!ldk::aligned(logits, dtype == LDK_F32 ? 4 : 2) || !ldk::aligned(tokens, 8) || !ldk::aligned(logprob, 4) ||
      !ldk::aligned(entropy, 4) || !ldk::aligned(top_logprobs, 4) || !ldk::aligned(top_ids, 8) || !ldk::aligned(workspace, 16))
    return ldk::fail(LDK_ERR_ALIGN, "%s: every array aligned to its elements, the workspace to 16 bytes", fn);
  const int64_t need = workspace_bytes(rows, V, top);
  if (need && (!workspace || workspace_bytes_ < need))
    return ldk::fail(LDK_ERR_INVALID, "%s: workspace of %lld bytes, this call needs %lld", fn, (long long)workspace_bytes_, (long long)need);
  LogprobArgs a{logits, ld, tokens, logprob, entropy, top_logprobs, top_ids, (float*)workspace, nullptr, rows, (int)V, top,
                plan_splits(rows, V, top), 0};
  a.keys = reinterpret_cast<uint64_t*>(a.part + 4 * rows * a.splits);
  // every row has at most 15 / 2 logits' room before its first vector
  const int tiles = (int)((V + 7 + kTileLogits - 1) / kTileLogits);
  a.slice = (tiles + a.splits - 1) / a.splits;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LDK_F16: return launch<half_t>(a, s);
    case LDK_BF16: return launch<uint16_t>(a, s);
    default: return launch<float>(a, s);
  }
}

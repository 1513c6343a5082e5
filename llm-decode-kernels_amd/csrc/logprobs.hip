// Log probabilities of given tokens: per row of logits x[V], with m = max x and s = sum exp(x - m),
//   logprob = (x[token] - m) - ln s,   entropy = ln s - sum exp(x - m) (x - m) / s,
// and the `top` largest logits (NaN largest, the lowest index first on ties, as torch.argmax orders
// them) with their log probabilities. Every logit is read once.
//
// A row is cut into `splits` slices, one workgroup each; a wave takes tiles of 1024 consecutive logits
// of its slice (16 per lane, the next tile's loads in flight), tiles w, w + 4, ... by wave w.
//  - Sums: the wave keeps one maximum m, and each lane two sums of 2^y and 2^y y with y = x log2 e -
//    m log2 e: a logit costs half a maximum, one fma, one exp2, one add and one fma. Only a tile that
//    raises the maximum rescales them. The maximum's own term is left out of the sums until another
//    replaces it, so that ln s = log1p(rest) keeps its digits where one token has nearly all the
//    probability. 2^-inf * -inf would be NaN: a tile whose second sum is NaN is summed again, clamped.
//    Of a maximum past 2^24 (words masked with a large finite number) m log2 e as rounded is off by whole
//    powers of two, or infinite. Such a wave sums nothing: next to a slice's larger maximum its logits have no
//    weight, and a slice whose maximum is far is read again, for y = (x - m) log2 e. (That as a branch of
//    every tile took 5 to 13% of the time of rows without such logits.)
//  - The largest: each wave keeps candidates (64-bit keys, value then lower index) in its own LDS list
//    and a floor that none of the `top` largest can be below. Its first is the top-th largest of its 64
//    lanes' maxima (found by ballots), which lets through about the logits that are the largest so
//    far; then the waves share theirs: where each has top/4 lanes at or above what it gives, the least
//    of the four has `top`. A list that fills up is cut back to its `top` largest. At the end the four
//    lists' survivors of the highest floor meet, and one wave ranks them by counting.
// Rows of several slices leave {m, sums, keys} per slice in the workspace, which the next launch
// joins with one wave per row.
//
// Bound by the vector instructions, close behind by memory: 1900 rows of 151936 bf16 (577 MB) with 20
// alternatives 150 us, 3.8 TB/s, the vector unit busy 69%; without alternatives 113 us, 5.1 TB/s.
// 77 rows of 50257 fp32 (15.5 MB, 20 alternatives) 23.6 us and one row of 151936 fp16 14.0: two launches, each a
// load's latency, the ballots of the first floor, and the ranking of the keys. Per lane maxima and a
// threshold per wave instead of the shared floors took 275 us on the first.
#include <algorithm>

#include "ldk_common.h"

namespace {

constexpr int kWaves = 4;
constexpr int kPer = 16;             // logits of a lane per tile
constexpr int kTileLogits = 64 * kPer;
constexpr int kTopMax = 64;          // a wave's lanes: the threshold is a lane's maximum
constexpr int kKeep = 128;           // candidates past which a list is cut back
constexpr int kCap = kKeep + 64;     // one more logit of every lane
constexpr int kCapPer = kCap / 64;
constexpr int kMergeKeys = 1024;     // keys of a row's slices that the joining wave takes
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

struct LogprobArgs {
  const void* x;
  int64_t ld;
  const int64_t* tokens;
  float *logprob, *entropy, *top_lp;
  int64_t* top_ids;
  float* part;     // [rows][splits][4]: m, s, y
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

// The float that exactly the numbers of keys above o are larger than (0x7fffffff would be -0: no key).
__device__ __forceinline__ float float_at(uint32_t o) { return from_order(o == 0x7fffffffu ? 0x7ffffffeu : o); }

// Maximum over the 64 lanes, in every lane (NaN does not count).
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, ldk::row_ror<1>(v));
  v = fmaxf(v, ldk::row_ror<2>(v));
  v = fmaxf(v, ldk::row_ror<4>(v));
  v = fmaxf(v, ldk::row_ror<8>(v));
  auto p = __builtin_amdgcn_permlane16_swap(ldk::f2u(v), ldk::f2u(v), false, false);
  v = fmaxf(ldk::u2f(p[0]), ldk::u2f(p[1]));
  p = __builtin_amdgcn_permlane32_swap(ldk::f2u(v), ldk::f2u(v), false, false);
  return fmaxf(ldk::u2f(p[0]), ldk::u2f(p[1]));
}

// The n-th largest of the wave's values, PER of each lane: the largest t with at least n values >= t, two
// bits a step from the top; with BITS < 32 only its upper bits, the others 0 (a bound below it).
template <int PER, int BITS>
__device__ __forceinline__ uint32_t nth_largest(const uint32_t (&v)[PER], int n) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 30; bit >= 32 - BITS; bit -= 2) {
    int c[3] = {0, 0, 0};
#pragma unroll
    for (int q = 0; q < 3; ++q)
#pragma unroll
      for (int i = 0; i < PER; ++i) c[q] += __popcll(__ballot(v[i] >= (t | (uint32_t)(q + 1) << bit)));
    t |= (c[2] >= n ? 3u : c[1] >= n ? 2u : c[0] >= n ? 1u : 0u) << bit;
  }
  return t;
}

// Rank of this lane's key among n keys in LDS (n a multiple of 8, 16-byte aligned): how many are larger,
// or equal and before position i. Real keys differ (their indexes do); absent ones are 0.
__device__ __forceinline__ int rank_key(const uint64_t* list, int n, uint64_t key, int i) {
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  int r = 0;
#pragma unroll 1
  for (int j = 0; j < n; j += 8) {
    u64x2 a[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = *reinterpret_cast<const u64x2*>(list + j + 2 * q);
#pragma unroll
    for (int q = 0; q < 8; ++q) r += a[q / 2][q % 2] > key || (a[q / 2][q % 2] == key && j + q < i);
  }
  return r;
}

// Position among the lanes whose bit of mask is set.
__device__ __forceinline__ int lane_rank(uint64_t mask, int lane) { return __popcll(mask & ((uint64_t(1) << lane) - 1)); }

// Writes the wave's keys, one of each lane that takes part, to list[n ..) and returns the new n.
__device__ __forceinline__ int append_keys(bool take, uint64_t key, uint64_t* list, int n, int lane) {
  const uint64_t mask = __ballot(take);
  if (take) list[n + lane_rank(mask, lane)] = key;
  return n + __popcll(mask);
}

// Cuts a wave's list of n <= kCap keys, n > top, to its largest: `top` of them, or up to kKeep / 2 where the
// last one's value is another's too. Returns their number; *value gets the top-th largest's.
__device__ __forceinline__ int cut_list(uint64_t* list, int n, int top, uint32_t* value, int lane) {
  ldk::wave_lds_sync();
  uint64_t k[kCapPer];
  uint32_t hi[kCapPer], lo[kCapPer];
#pragma unroll
  for (int i = 0; i < kCapPer; ++i) {
    k[i] = lane + 64 * i < n ? list[lane + 64 * i] : 0;
    hi[i] = (uint32_t)(k[i] >> 32);
  }
  const uint32_t nth = nth_largest<kCapPer, 32>(hi, top);
  int above = 0, equal = 0;
#pragma unroll
  for (int i = 0; i < kCapPer; ++i) {
    above += __popcll(__ballot(hi[i] > nth));
    equal += __popcll(__ballot(hi[i] == nth));
    lo[i] = hi[i] == nth ? (uint32_t)k[i] : 0u;
  }
  uint64_t least = (uint64_t)nth << 32;
  if (above + equal > kKeep / 2) least |= nth_largest<kCapPer, 32>(lo, top - above);  // the lowest indexes of them
  ldk::wave_lds_sync();
  n = 0;
#pragma unroll
  for (int i = 0; i < kCapPer; ++i) n = append_keys(k[i] >= least, k[i], list, n, lane);
  ldk::wave_lds_sync();
  *value = nth;
  return n;
}

// The `top` largest of `total` keys (absent ones 0) in descending order: lane r gets the r-th. The loops
// run as often as there are keys, mostly once or twice: code that runs once waits for its own fetch.
// list: LDS for total + 8 keys (may be where keys are), sorted: for kTopMax.
__device__ __forceinline__ uint64_t rank_keys(const uint64_t* keys, int total, int top, uint64_t* list, uint64_t* sorted,
                                              int lane) {
  uint32_t most[1] = {0};
#pragma unroll 1
  for (int i = lane; i < total; i += 64) most[0] = max(most[0], (uint32_t)(keys[i] >> 32));
  const uint32_t nth = nth_largest<1, 32>(most, top);
  int n = 0;
#pragma unroll 1
  for (int i = 0; i < total; i += 64) {  // in place: what is written lies before what is read next
    const uint64_t key = i + lane < total ? keys[i + lane] : 0;
    ldk::wave_lds_sync();
    n = append_keys(key != 0 && (uint32_t)(key >> 32) >= nth, key, list, n, lane);
  }
  if (lane < 8) list[n + lane] = 0;
  sorted[lane] = 0;
  ldk::wave_lds_sync();
#pragma unroll 1
  for (int i = lane; i < n; i += 64) {
    const uint64_t key = list[i];
    const int r = rank_key(list, (n + 7) & ~7, key, i);
    if (r < top) sorted[r] = key;
  }
  ldk::wave_lds_sync();
  return lane < top ? sorted[lane] : 0;
}

// A part of a row: its maximum m, and over its other logits the sums of 2^y and 2^y y, y = x log2 e -
// m log2 e (as rounded: base_of). m == -inf: nothing but -inf. Of a far m: y = (x - m) log2 e.
struct Sums {
  float m, s, y;
};
constexpr float kFar = 16777216.0f;    // 2^24, where what base_of rounds away reaches 1
constexpr float kNoSum = 2.0f * kFar;  // past it a wave sums nothing: between the two it may meet a near maximum
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) >= kFar && m != -__builtin_inff(); }
__device__ __forceinline__ float base_of(float m) { return m == -__builtin_inff() ? 0.0f : m * kLog2e; }
__device__ __forceinline__ float rounded_away(float m) { return __builtin_fmaf(m, kLog2e, -base_of(m)); }
// The maximum's own exponent: what base_of rounded away, 0 of a far one; no number of an infinity.
template <bool FAR>
__device__ __forceinline__ float residue(float m) {
  return FAR && is_far(m) ? m - m : rounded_away(m);
}
// From exponents against m to those against top >= m; finite, so that 0 times it is 0.
template <bool FAR>
__device__ __forceinline__ float step_to(float m, float top) {
  if (!FAR || !(is_far(m) || is_far(top))) return base_of(m) - base_of(top);
  return fmaxf((m - top) * kLog2e - residue<FAR>(m) + residue<FAR>(top), -1e9f);
}
// a's sums with its own maximum's term, taken against the maximum m >= a.m.
template <bool FAR>
__device__ __forceinline__ void rebase(Sums& a, float m) {
  const float d = step_to<FAR>(a.m, m), f = a.m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(d);
  if (a.m > -__builtin_inff()) {
    const float r = residue<FAR>(a.m), p = __builtin_amdgcn_exp2f(r);
    a.s += p;
    a.y = __builtin_fmaf(p, r, a.y);
  }
  a.y = f * __builtin_fmaf(d, a.s, a.y);
  a.s *= f;
  a.m = m;
}
template <bool FAR>
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  if (b.m > a.m) {
    const Sums t = a;
    a = b;
    b = t;
  }
  rebase<FAR>(b, a.m);
  a.s += b.s;
  a.y += b.y;
  return a;
}
// a's sums against its base as those against its maximum itself.
__device__ __forceinline__ void rebase_to_maximum(Sums& a) {
  const float r = rounded_away(a.m), f = __builtin_amdgcn_exp2f(-r);
  a.y = f * __builtin_fmaf(-r, a.s, a.y);
  a.s *= f;
}
// Over the lanes: the first that has the largest maximum keeps its term out.
template <bool FAR>
__device__ __forceinline__ Sums wave_join(Sums a, int lane) {
  const float m = wave_max(a.m);
  if (lane != __builtin_ctzll(__ballot(a.m == m) | (uint64_t(1) << 63))) rebase<FAR>(a, m);
  return Sums{m, ldk::sum_lanes_strided<1>(a.s), ldk::sum_lanes_strided<1>(a.y)};
}

template <typename T>
constexpr bool kCanBeFar = true;
template <>
constexpr bool kCanBeFar<half_t> = false;  // 65504 at most

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<half_t>(half_t v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<uint16_t>(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }

// The logit of the row's given token (NaN: outside the vocabulary). Read ahead of the row: two dependent loads.
template <typename T>
__device__ __forceinline__ float given_logit(const LogprobArgs& a, int64_t row) {
  const int64_t tok = a.tokens[row];
  return tok >= 0 && tok < a.V ? to_f<T>(((const T*)a.x)[row * a.ld + tok]) : __builtin_nanf("");
}

// The answers of one row, from its sums and its sorted keys (lanes 0 .. top - 1 hold one each).
template <typename T>
__device__ __forceinline__ void finish(const LogprobArgs& a, int64_t row, const Sums& t, float given, uint64_t key, int lane) {
  // against the maximum itself: without what its base rounded away
  const float r = residue<kCanBeFar<T>>(t.m), f = __builtin_amdgcn_exp2f(-r);
  const float rest = t.s * f, y = f * __builtin_fmaf(-r, t.s, t.y);
  const float log_s = log1pf(rest);
  if (lane == 0) {
    a.logprob[row] = (given - t.m) - log_s;
    a.entropy[row] = log_s - kLn2 * y / (1.0f + rest);
  }
  if (lane < a.top) {
    a.top_lp[row * a.top + lane] = (from_order((uint32_t)(key >> 32)) - t.m) - log_s;
    a.top_ids[row * a.top + lane] = (int64_t)(uint32_t)~(uint32_t)key;
  }
}

// Without alternatives 8 waves a SIMD hide the loads best, the most there are: the compiler then keeps to the
// scalar registers that they leave (1900 rows of 151936 bf16 126 us at 7 waves, 112 at 8).
template <typename T, bool TOP>
__global__ __launch_bounds__(kWaves * 64, sizeof(T) == 4 ? 5 : TOP ? 6 : 8) void logprobs_kernel(LogprobArgs a) {
  constexpr int VEC = 16 / sizeof(T), NV = kPer / VEC;
  typedef T vec_t __attribute__((ext_vector_type(VEC)));
  typedef vec_t unaligned_t __attribute__((aligned(sizeof(T))));
  __shared__ __align__(16) uint64_t lists[TOP ? kWaves : 1][TOP ? kCap : 1], pool[TOP ? kWaves * kCap + 8 : 1];
  __shared__ uint64_t sorted[kTopMax];
  __shared__ uint32_t shared_floor[kWaves];  // what each wave gives: top / 4 of its logits are at or above it
  __shared__ uint32_t floors[kWaves];
  __shared__ int pooled;
  __shared__ Sums sums[kWaves];
  __shared__ Sums far[kWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * 65535;
  if (row >= a.rows) return;
  const T* x = (const T*)a.x + row * a.ld;
  // whole vectors from the row's start on (rows of any alignment: the loads take any), then the numbers
  // that make up none, one per lane, as a tile of their own
  const int rest = a.V % VEC, whole = a.V - rest, vtiles = (whole + kTileLogits - 1) / kTileLogits;
  const int first = (int)blockIdx.x * a.slice, tiles = min(a.slice, vtiles + (rest ? 1 : 0) - first);

  // the row's index of element e of this lane in tile t (of the slice), V or more for none
  auto place = [&](int t, int e) __attribute__((always_inline)) {
    if (first + t >= vtiles) return whole + (e ? VEC : lane);
    return ((first + t) * NV + e / VEC) * 64 * VEC + lane * VEC + e % VEC;
  };
  // the vectors of this lane in tile t, a valid one in the place of none: loads under no condition, so that
  // the wait for a tile's can leave the next tile's in flight
  auto load = [&](int t, vec_t (&v)[NV]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NV; ++u) v[u] = *reinterpret_cast<const unaligned_t*>(x + min(place(t, u * VEC), whole - VEC));
  };

  // of a far maximum m: how many logits of the wave equal it, and the others' sums
  auto far_sums = [&](float m) __attribute__((always_inline)) {
    float equal = 0.0f, s = 0.0f, y = 0.0f;
    const int begin = min(first * kTileLogits, whole);
    const int end = first + tiles > vtiles ? a.V : min(whole, (first + tiles) * kTileLogits);
#pragma unroll 1
    for (int i = begin + tid; i < end; i += kWaves * 64) {
      const float v = to_f<T>(x[i]), e = (v - m) * kLog2e, p = v == m ? 0.0f : __builtin_amdgcn_exp2f(e);
      equal += v == m ? 1.0f : 0.0f;
      s += p;
      y = __builtin_fmaf(p, fmaxf(e, -1e30f), y);
    }
    return Sums{ldk::sum_lanes_strided<1>(equal), ldk::sum_lanes_strided<1>(s), ldk::sum_lanes_strided<1>(y)};
  };

  Sums s{-__builtin_inff(), 0.0f, 0.0f};  // m: of the wave
  float nb = 0.0f, lmax = -__builtin_inff();  // -base_of(m), or -inf for no sums; this lane's largest so far
  // Candidates' keys are above floor; `none` is below the key of every number. own: the last value of the
  // wave's own top so far: later logits that equal it come after it
  const uint32_t none = order(-__builtin_inff()) - 1;
  uint32_t own = none;
  int n = 0, next = 0, seen = 0;
  uint32_t lodd = 0;  // the largest of tiles whose sum was not a number
  const int quarter = (a.top + kWaves - 1) / kWaves;
  if constexpr (TOP) {
    if (tid < kWaves) shared_floor[tid] = none;
    if (tid == 0) pooled = 0;
    __syncthreads();
  }
  const float given = a.splits == 1 && wave == 0 ? given_logit<T>(a, row) : 0.0f;
  vec_t cur[NV], nxt[NV];
  if (whole) load(min(wave, vtiles - 1 - first), cur);
  for (int t = wave; t < tiles; t += kWaves) {
    if (whole) load(t + kWaves, nxt);
    float v[kPer];
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[u * VEC + e] = to_f<T>(cur[u][e]);
    if (first + t >= vtiles - 1) {  // the last tiles: -inf for none (exp 0, and not among the largest by its place)
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[e] = first + t < vtiles && place(t, e) < whole ? v[e] : -__builtin_inff();
      if (first + t == vtiles && lane < rest) v[0] = to_f<T>(x[whole + lane]);
    }
    float tm = v[0];
#pragma unroll
    for (int e = 1; e < kPer; ++e) tm = fmaxf(tm, v[e]);
    float ts = 0.0f, ty = 0.0f;
    if (__any(tm > s.m)) {  // a new maximum: its first lane leaves one logit that equals it out
      const float m = wave_max(tm);
      const bool holds = lane == __builtin_ctzll(__ballot(tm == m));
      // finite, so that 0 times it is 0 (infinite where a product overflows; past 0 only from -inf)
      const float d = fminf(fmaxf(base_of(s.m) - base_of(m), -1e9f), 0.0f);
      const float f = s.m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(d);
      if (lane == 0 && fabsf(s.m) <= kNoSum) {  // the old maximum's term joins lane 0's sums
        const float r = rounded_away(s.m), p = __builtin_amdgcn_exp2f(r);
        s.s += p;
        s.y = __builtin_fmaf(p, r, s.y);
      }
      s.y = f * __builtin_fmaf(d, s.s, s.y);
      s.s *= f;
      s.m = m;
      nb = fabsf(m) <= kNoSum ? -base_of(m) : -__builtin_inff();
      bool left = !holds;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const float y = __builtin_fmaf(v[e], kLog2e, nb);
        const bool out = !left && v[e] == m;
        const float p = out ? 0.0f : __builtin_amdgcn_exp2f(y);
        left |= out;
        ts += p;
        ty = __builtin_fmaf(p, fmaxf(y, -1e30f), ty);
      }
      asm volatile("" : "+v"(ts));  // the sum is formed here (left to where the branches join, its terms live on)
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const float y = __builtin_fmaf(v[e], kLog2e, nb), p = __builtin_amdgcn_exp2f(y);
        ts += p;
        ty = __builtin_fmaf(p, y, ty);
      }
      asm volatile("" : "+v"(ts));
      if (__any(ty != ty)) {  // an infinity or a NaN among them
        ty = 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const float y = __builtin_fmaf(v[e], kLog2e, nb), p = __builtin_amdgcn_exp2f(y);
          ty = __builtin_fmaf(p, fmaxf(y, -1e30f), ty);
        }
      }
    }
    s.s += ts;
    s.y += ty;
    if constexpr (TOP) {
      lmax = fmaxf(lmax, tm);
      const bool strange = __any(ts != ts);  // a NaN among them, or infinities
      if (strange && ts != ts) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) lodd = max(lodd, order(v[e]));
      }
      uint32_t floor = own;
      if (seen == next) {  // tiles 0, 1, 3, 7, ... of the wave
        const uint32_t mine[1] = {max(order(lmax), lodd)};
        if (seen == 0) {  // this tile's equals are among the ones that made it
          own = max(own, nth_largest<1, 20>(mine, a.top));
          floor = max(floor, own - 1);
        }
        const uint32_t give = nth_largest<1, 20>(mine, quarter);
        if (lane == 0 && give > none) __hip_atomic_store(&shared_floor[wave], give, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        next = 2 * seen + 1;
      }
      uint32_t least = 0xffffffffu;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) least = min(least, __hip_atomic_load(&shared_floor[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
      floor = max(floor, (uint32_t)__builtin_amdgcn_readfirstlane(least) - 1);
      floor = max(floor, none);
      const float floor_f = float_at(floor);
      const uint64_t hit = __ballot(tm > floor_f || ts != ts);
      if (hit || floor == none) {
        // by floats where they order as the keys do: no NaN, above -inf
        int from = 0;  // the elements from here on go the long way
        if (!strange && floor > none) {
          from = kPer;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const uint64_t mask = __ballot(v[e] > floor_f);
            if (mask && from == kPer) {
              if (n > kKeep) {
                from = e;
              } else {
                if (v[e] > floor_f) lists[wave][n + lane_rank(mask, lane)] = ((uint64_t)order(v[e]) << 32) | (uint32_t)~place(t, e);
                n += __popcll(mask);
              }
            }
          }
        }
        // the long way: what is left, read again, and the list cut back where it is full
        if (from < kPer || n > kKeep) {
          uint32_t value = 0;
#pragma unroll 1
          for (int e = from;; ++e) {
            if (n > kKeep) n = cut_list(lists[wave], n, a.top, &value, lane);
            if (e >= kPer) break;
            const int i = place(t, e);
            const uint32_t o = i < (first + t < vtiles ? whole : a.V) ? order(to_f<T>(x[i])) : 0u;
            n = append_keys(o > floor, ((uint64_t)o << 32) | (uint32_t)~i, lists[wave], n, lane);
          }
          own = max(own, value);
        }
      }
      ++seen;
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) cur[u] = nxt[u];
  }

  s.s = ldk::sum_lanes_strided<1>(s.s);
  s.y = ldk::sum_lanes_strided<1>(s.y);
  if (kCanBeFar<T> && is_far(s.m) && fabsf(s.m) <= kNoSum) rebase_to_maximum(s);
  if (lane == 0) sums[wave] = s;
  uint64_t key = 0;
  if constexpr (TOP) {
    if (seen > 1) {
      const uint32_t mine[1] = {max(order(lmax), lodd)};
      own = max(own, nth_largest<1, 20>(mine, a.top));
    }
    if (lane == 0) floors[wave] = own;
  }
  __syncthreads();
  if constexpr (kCanBeFar<T>) {
    float m = sums[0].m;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, sums[w].m);
    if (is_far(m) && m != __builtin_inff()) {  // of the slice (uniform): its logits are read again
      const Sums mine = far_sums(m);
      __syncthreads();  // every wave has read the maxima
      if (lane == 0) far[wave] = mine;
      __syncthreads();
      if (tid == 0) {
        Sums t{m, -1.0f, 0.0f};
        for (int w = 0; w < kWaves; ++w) t.s += far[w].m;  // how many equal the maximum
        for (int w = 0; w < kWaves; ++w) t.s += far[w].s, t.y += far[w].y;
        sums[0] = t;
      }
      if (tid > 0 && tid < kWaves) sums[tid] = Sums{-__builtin_inff(), 0.0f, 0.0f};
      __syncthreads();
    }
  }
  if constexpr (TOP) {  // what is at or above every floor, of all four lists
    uint32_t floor = none, least = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      floor = max(floor, floors[w]);
      least = min(least, shared_floor[w]);
    }
    floor = max(floor, least);
#pragma unroll 1
    for (int i = 0; i < n; i += 64) {
      const uint64_t k1 = i + lane < n ? lists[wave][i + lane] : 0;
      const bool take = k1 && (uint32_t)(k1 >> 32) >= floor;
      const int count = __popcll(__ballot(take));
      int at = 0;
      if (lane == 0) at = atomicAdd(&pooled, count);
      append_keys(take, k1, pool, __builtin_amdgcn_readfirstlane(at), lane);
    }
    __syncthreads();
    if (wave == 0) key = rank_keys(pool, pooled, a.top, pool, sorted, lane);
  }
  if (wave) return;
  Sums all = sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) all = join<kCanBeFar<T>>(all, sums[w]);
  if (a.splits == 1) {
    finish<T>(a, row, all, given, key, lane);
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
  __shared__ __align__(16) uint64_t list[kMergeKeys + 8];
  __shared__ uint64_t sorted[kTopMax];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const float given = given_logit<T>(a, row);
  Sums s{-__builtin_inff(), 0.0f, 0.0f};
  for (int i = lane; i < a.splits; i += 64) {
    const float* p = a.part + (row * a.splits + i) * 4;
    s = join<kCanBeFar<T>>(s, Sums{p[0], p[1], p[2]});
  }
  s = wave_join<kCanBeFar<T>>(s, lane);
  uint64_t key = 0;
  if (a.top) {
    const int total = a.splits * a.top;
    key = rank_keys(a.keys + row * total, total, a.top, list, sorted, lane);
  }
  finish<T>(a, row, s, given, key, lane);
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
  const int vec = dtype == LDK_F32 ? 4 : 8;
  const int tiles = (int)((V / vec * vec + kTileLogits - 1) / kTileLogits + (V % vec ? 1 : 0));
  a.slice = (tiles + a.splits - 1) / a.splits;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case LDK_F16: return launch<half_t>(a, s);
    case LDK_BF16: return launch<uint16_t>(a, s);
    default: return launch<float>(a, s);
  }
}

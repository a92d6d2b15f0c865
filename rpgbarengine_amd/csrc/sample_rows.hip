// One draw per row of logits (rpg_hip_sample_rows, include/rpg_hip.h). With
// w_i = exp((x_i - max) / T), the tokens ranked by (x descending, index
// ascending):
//   kept: rank < top_k; weight of the better tokens < top_p x weight of the
//         top_k ones; w_i >= min_p
//   token = the first index i with sum of the kept w up to i > u x their sum.
// All three limits keep a head of the ranking, so what is kept is everything
// up to one cut (a value and an index).
//
// Weights are summed as integers of 2^-44 (44 bits below the largest weight,
// at most 2^18 of them in 64 bits): sums are the same in any order, so atomics
// and slices cannot change a draw, and each is within half a unit of the exact
// weight. A weight itself is computed in double (a table of 2^(-j/32) and a
// polynomial of degree 5, 3e-15 relative).
//
// Four launches over (row, slice of the vocabulary), three where neither top_k nor
// top_p are given, without a sort:
//   Max    largest value (and its first index) and least finite one per slice,
//          the largest of every group of four threads' tokens
//   Count  histogram of 2048 equal steps of x below the row's maximum: count
//          and weight, slices added by atomics; the row's last slice looks up
//          the step that holds the cut. For a small top_k the list below at once,
//          down to the step of the k-th largest group
//   Split  a list of the tokens down to the cut's step; where those are more than
//          kList, the list of its own tokens and the weight above it per 4096 tokens
//   Draw   one workgroup a row: the list sorted and cut, then the draw, among
//          the list's tokens by index or in the unit that it falls into
// A step of more than kList tokens (thousands of equal values) and a cut whose
// step the histogram cannot tell (a large top_k whose last step decides
// top_p's) are found by Draw over the whole row, digit by digit.
//
// Bound: the logits' bytes, read once from HBM (later launches find them in
// the memory-side cache); for few rows what a row takes whatever its length: the
// launches, a histogram's 2048 steps, sorting a list. Measured, vocabulary of
// 151936: 192 bf16 rows, 58 MB (12 us for a large copy), greedy 24 us, top_k 40 50,
// min_p 48, temperature alone 75, top_p 95 (a weight in double and an LDS atomic
// for nearly every token), all mixed 84-92; 8 f32 rows with min_p 19 where the
// launches are four, 17 where they are three. One f32 row, in a captured graph:
// greedy 8.5 us (all that the four launches and one look at the logits take), no
// limits 16, top_k 40 22, top_p 27 (peaked) to 36 (flat), of which 31 with 4096 tokens.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "lanes.h"
#include "paged_dev.h"
#include "sample_rows.h"

namespace rpg {
namespace rows {
namespace {

using paged::BF16;
using paged::F16;
using paged::F32;
using paged::U4;
using paged::Unpack2;

constexpr int kThreads = 256;
constexpr int kBins = 2048;
constexpr int kDrawThreads = 1024;
constexpr int kList = 1024;      // tokens of the cut's step that Draw ranks in LDS
constexpr int kUnit = 4096;      // Draw looks for the token in a run of this many; slices are multiples of it
constexpr int kMaxUnits = 64;    // of a row: 262144 tokens
constexpr float kNone = -__builtin_inff();

struct Bin {
  uint64_t weight;
  uint32_t count, pad;
};
struct Cut;
struct SliceMax {
  float max, min;
  int32_t index, pad;
};

struct Layout {
  int slices, length;  // tokens per slice
  int groups;          // of a slice's tokens, whose maxima are kept: a thread's, or four threads'
  int64_t max_at, bins_at, weights_at, lists_at, counts_at, cuts_at, groups_at, bytes;
};

__host__ __device__ inline Layout LayoutOf(int64_t rows, int64_t vocab) {
  Layout l;
  // About 1500 workgroups where there are many rows, as many as the card holds at a
  // time, slices of 4096 tokens where there are few. 192 rows, us with half as
  // many / these / twice as many: mixed parameters 136 / 104 / 100, top_p 0.9 119 /
  // 132 / 160 (each slice adds its histogram to the row's).
  const int64_t most = (vocab + kUnit - 1) / kUnit;
  int64_t want = rows < 1 ? 1 : (1536 + rows - 1) / rows;
  want = want < 1 ? 1 : want > most ? most : want;
  want = want > kMaxUnits ? kMaxUnits : want;
  l.length = static_cast<int>(((vocab + want - 1) / want + kUnit - 1) / kUnit * kUnit);
  l.slices = static_cast<int>((vocab + l.length - 1) / l.length);
  l.groups = l.slices <= 8 ? kThreads : kThreads / 4;
  l.bins_at = 0;
  l.max_at = l.bins_at + rows * kBins * static_cast<int64_t>(sizeof(Bin));
  l.weights_at = l.max_at + rows * l.slices * static_cast<int64_t>(sizeof(SliceMax));
  l.lists_at = l.weights_at + rows * kMaxUnits * 8;
  l.counts_at = l.lists_at + rows * kList * 8;
  l.cuts_at = (l.counts_at + rows * 8 + 63) / 64 * 64;
  l.groups_at = l.cuts_at + rows * 64;
  l.bytes = l.groups_at + rows * l.slices * l.groups * 4;
  return l;
}

// One row's view of the work buffer.
struct Work {
  Bin* bins;
  SliceMax* max;
  uint64_t* weights;  // per unit
  uint64_t* list;  // rank keys
  uint32_t* count;  // tokens listed; slices counted
  Cut* cut;
  float* groups;
  __device__ Work(const SampleArgs& a, const Layout& l, int row)
      : bins(reinterpret_cast<Bin*>(a.work + l.bins_at) + static_cast<int64_t>(row) * kBins),
        max(reinterpret_cast<SliceMax*>(a.work + l.max_at) + static_cast<int64_t>(row) * l.slices),
        weights(reinterpret_cast<uint64_t*>(a.work + l.weights_at) + static_cast<int64_t>(row) * kMaxUnits),
        list(reinterpret_cast<uint64_t*>(a.work + l.lists_at) + static_cast<int64_t>(row) * kList),
        count(reinterpret_cast<uint32_t*>(a.work + l.counts_at) + 2 * row),
        cut(reinterpret_cast<Cut*>(a.work + l.cuts_at + static_cast<int64_t>(row) * 64)),
        groups(reinterpret_cast<float*>(a.work + l.groups_at) + static_cast<int64_t>(row) * l.slices * l.groups) {}
};

template <typename T>
constexpr int kPer = 16 / paged::kBytes<T>;  // values of a 16-byte load

// NaN is never chosen: it counts as -inf. Zeros are alike.
__device__ __forceinline__ float Clean(float x) { return x == x ? x + 0.0f : kNone; }

template <typename T>
__device__ __forceinline__ float One(const char* row, int i) {
  if constexpr (paged::kBytes<T> == 4) {
    return Clean(reinterpret_cast<const float*>(row)[i]);
  } else {
    float x, unused;
    Unpack2<T>(reinterpret_cast<const uint16_t*>(row)[i], &x, &unused);
    return Clean(x);
  }
}

// Two neighbouring values of a run: those of its first dword (16-bit types) or
// dwords (f32). Next moves on to the two behind them.
template <typename T>
__device__ __forceinline__ void RawTwo(U4 v, float* a, float* b) {
  if constexpr (paged::kBytes<T> == 4)
    *a = __uint_as_float(v[0]), *b = __uint_as_float(v[1]);
  else
    Unpack2<T>(v[0], a, b);
}
template <typename T>
__device__ __forceinline__ void Two(U4 v, float* a, float* b) {
  RawTwo<T>(v, a, b);
  *a = Clean(*a);
  *b = Clean(*b);
}
template <typename T>
__device__ __forceinline__ U4 Next(U4 v) {
  if constexpr (paged::kBytes<T> == 4) return U4{v[2], v[3], 0u, 0u};
  return U4{v[1], v[2], v[3], 0u};
}
template <typename T>
constexpr uint32_t kNoneBits = paged::kBytes<T> == 4 ? 0xFF800000u : __is_same(T, BF16) ? 0xFF80FF80u : 0xFC00FC00u;

// 2^(-j / 32)
__device__ const double kPow2[32] = {
    0x1.0000000000000p+0, 0x1.f50765b6e4540p-1, 0x1.ea4afa2a490dap-1, 0x1.dfc97337b9b5fp-1,
    0x1.d5818dcfba487p-1, 0x1.cb720dcef9069p-1, 0x1.c199bdd85529cp-1, 0x1.b7f76f2fb5e47p-1,
    0x1.ae89f995ad3adp-1, 0x1.a5503b23e255dp-1, 0x1.9c49182a3f090p-1, 0x1.93737b0cdc5e5p-1,
    0x1.8ace5422aa0dbp-1, 0x1.82589994cce13p-1, 0x1.7a11473eb0187p-1, 0x1.71f75e8ec5f74p-1,
    0x1.6a09e667f3bcdp-1, 0x1.6247eb03a5585p-1, 0x1.5ab07dd485429p-1, 0x1.5342b569d4f82p-1,
    0x1.4bfdad5362a27p-1, 0x1.44e086061892dp-1, 0x1.3dea64c123422p-1, 0x1.371a7373aa9cbp-1,
    0x1.306fe0a31b715p-1, 0x1.29e9df51fdee1p-1, 0x1.2387a6e756238p-1, 0x1.1d4873168b9aap-1,
    0x1.172b83c7d517bp-1, 0x1.11301d0125b51p-1, 0x1.0b5586cf9890fp-1, 0x1.059b0d3158574p-1};

constexpr double kOne = 17592186044416.0;  // 2^44: the largest weight

__device__ __forceinline__ uint64_t Mask(bool x) { return x ? ~uint64_t{0} : 0; }

// A row's parameters, from its slices' maxima.
struct Row {
  float max;     // -inf: nothing to draw from
  int32_t best;  // its first index
  float scale;   // histogram steps per unit of x
  double c32;    // 32 log2(e) / T
  bool greedy;
  int32_t k;      // 0: no limit
  double p, floor;  // 0: no limit; min_p in weight units
  float reach;      // how far below max a weight can reach the floor
  bool weightless_end;  // the histogram's last step holds only what has no weight

  // top_k so small that the tokens up to the k-th are listed whole: only their
  // number is needed of the histogram
  __device__ __forceinline__ bool Lean() const { return k > 0 && k <= kList / 2; }

  // top_k so small against the groups whose maxima are kept that the k-th largest
  // of those, which is no more than the k-th token, has few tokens above it: they
  // are listed without a histogram (192 rows of 151936, top_k 40: 37 us in
  // CountKernel with one, 18 without). Where at most a quarter of the groups hold one,
  // 1.15 k tokens spread over them do, and k more that crowd in a few: within kList.
  __device__ __forceinline__ bool Direct(const Layout& l) const {
    return k > 0 && k <= min(kList * 7 / 16, l.slices * l.groups / 4);
  }

  // The most tokens that a step of weight q may hold. Without top_k only that is
  // needed, and only to see whether the cut's list is short: a count would be a
  // second LDS atomic for every token (192 rows, top_p 0.9: 132 us with it, 106
  // without). A step spans a 65th of its weight; the margin is for the
  // rounding of Bin.
  __device__ __forceinline__ uint32_t Most(int bin, uint64_t q) const {
    const float low = __builtin_amdgcn_exp2f(44.0f - static_cast<float>(c32) * 0.03125f * (static_cast<float>(bin + 1) / scale)) * 0.98f;
    return q == 0 ? 0u : low >= 64.0f ? static_cast<uint32_t>(fminf(static_cast<float>(q) / low, 1e6f)) + 1u : 1u << 20;
  }

  // w 2^44, at most half a unit off when rounded (below half a unit: somewhere
  // there). 2^-y = 2^-(n / 32) 2^-(y - n / 32) with n the integer next to 32 y, found
  // by adding what leaves no bits for a fraction.
  __device__ __forceinline__ double Weight(float x, const double* pow2) const {
    const double d = x == max ? 0.0 : static_cast<double>(max) - static_cast<double>(x);
    const double y = fmin(d * c32, 46.0 * 32.0);  // (no branch: a run's weights are computed side by side)
    const double t = y + 0x1.8p52, z = ((t - 0x1.8p52) - y) * (0.69314718055994530942 / 32.0);  // ln 2 / 64 at most
    const int n = static_cast<int>(__builtin_bit_cast(uint64_t, t));
    double e = __builtin_fma(z, 1.0 / 120.0, 1.0 / 24.0);
    e = __builtin_fma(z, e, 1.0 / 6.0);
    e = __builtin_fma(z, e, 0.5);
    e = __builtin_fma(z, e, 1.0);
    e = __builtin_fma(z, e, 1.0);
    const uint64_t p = __builtin_bit_cast(uint64_t, pow2[n & 31]) + (static_cast<uint64_t>(44 - (n >> 5)) << 52);
    return e * __builtin_bit_cast(double, p);
  }
  // rounded to an integer (weights are below 2^52)
  static __device__ __forceinline__ uint64_t Units(double w) {
    return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
  }
  // Tokens without weight are not counted where that is plain: those of -inf, and
  // the last step of a histogram that ends where weights do (which may be most
  // of a row, on one counter). Where fewer than k are counted, top_k sets no limit.
  __device__ __forceinline__ bool Counted(float x, int bin) const {
    return x > kNone && !(weightless_end && bin == kBins - 1);
  }
  // false only where the weight is below the floor (the margin covers the
  // rounding of the difference and of reach)
  __device__ __forceinline__ bool MayReach(float x) const { return max - x <= reach || x == max; }
  // monotone: never less for a smaller x
  __device__ __forceinline__ int Bin(float x) const {
    return static_cast<int>(fminf((x == max ? 0.0f : max - x) * scale, static_cast<float>(kBins - 1)));
  }
};

// Row parameters; every thread of a wave gets them. The least weight that is
// not 0 lies 45.5 bits (31.54 nats) below the largest: the histogram spans
// that, or the row's values where those span less.
__device__ __forceinline__ Row RowOf(const SampleArgs& a, const Layout& l, const Work& w, int row) {
  const int lane = threadIdx.x & 63;
  SliceMax m = lane < l.slices ? w.max[lane] : SliceMax{kNone, -kNone, INT32_MAX, 0};
  const float max = lanes::WaveMaxF(m.max), min = -lanes::WaveMaxF(-m.min);
  const uint64_t at = __ballot(m.max == max);
  Row r;
  r.max = max;
  r.best = __shfl(m.index, __ffsll(static_cast<unsigned long long>(at)) - 1, 64);  // (slices in order)
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  r.greedy = !(t > 0.0f);
  r.c32 = 32.0 * 1.4426950408889634074 / static_cast<double>(t);
  const float weighty = 31.6f * t, span = fminf(weighty, max - min);
  // (both infinite: values further apart than a float reaches have weight too)
  r.weightless_end = weighty <= max - min && weighty < -kNone;
  // (finite: the maximum's own step is 0 x scale. Below a span of 6e-36, a temperature
  // of 1.9e-37, the steps are wider than they could be)
  r.scale = span > 0.0f ? fminf(static_cast<float>(kBins) / span, __FLT_MAX__) : 0.0f;
  const int32_t k = a.top_k != nullptr ? a.top_k[row] : 0;
  r.k = k > 0 && k < a.vocab ? k : 0;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  r.p = p > 0.0f && p < 1.0f ? static_cast<double>(p) : 0.0;
  const float f = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  r.floor = f > 0.0f ? static_cast<double>(fminf(f, 1.0f)) * kOne : 0.0;
  r.reach = t * (f > 0.0f ? -__logf(fminf(f, 1.0f)) * 1.0001f + 1e-3f : 31.6f);
  return r;
}

// f(run, i, lo) for the runs of 16 bytes of `length` tokens from `start` on, a
// run to a lane, kAhead of a lane's runs in flight. Tokens i .. i + kPer - 1 lie
// in the run; it stands for those from lo on (the row's last run reaches back
// into the one before it, and a lane behind the row has none: lo past its
// tokens). The length is a multiple of a workgroup's runs; whole waves go round
// together, so f may use their lanes. The loads take any alignment, depend on no
// branch (a join would wait for them) and never reach past the row. One copy of
// f: a launch starts on a cold instruction cache.
constexpr int kAhead = 4;
typedef U4 U4Any __attribute__((aligned(2)));
template <typename T, typename F>
__device__ __forceinline__ void ForRuns(const SampleArgs& a, const char* row, int start, int length, F&& f) {
  const int end = min(a.vocab, start + length), step = kThreads * kPer<T>;
  if (a.vocab < kPer<T>) {  // less than a run
    if (start > 0 || threadIdx.x >= 64) return;
    U4 v = {kNoneBits<T>, kNoneBits<T>, kNoneBits<T>, kNoneBits<T>};
    for (int e = 0; e < a.vocab; ++e) {
      const float x = One<T>(row, e);
      const uint32_t u = paged::kBytes<T> == 4 ? __float_as_uint(x) : reinterpret_cast<const uint16_t*>(row)[e];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (paged::kBytes<T> == 4 && k == e) v[k] = u;
        if (paged::kBytes<T> == 2 && k == e / 2) v[k] = e % 2 ? (v[k] & 0xFFFFu) | u << 16 : (v[k] & 0xFFFF0000u) | u;
      }
    }
    // (values past the row are -inf; the lane past kPer - vocab has none to stand for)
    f(v, 0, threadIdx.x == 0 ? 0 : kPer<T>);
    return;
  }
  const int wave_first = start + static_cast<int>(threadIdx.x / 64) * 64 * kPer<T>;
  const int n = wave_first < end ? (end - wave_first - 1) / step + 1 : 0;
  const int mine = start + threadIdx.x * kPer<T>, last = a.vocab - kPer<T>;
  auto load = [&](int r) {
    return *(const __attribute__((address_space(1))) U4Any*)(row + static_cast<int64_t>(min(mine + r * step, last)) * paged::kBytes<T>);
  };
  U4 ring[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) ring[k] = load(k);
#pragma unroll 1
  for (int r = 0; r < n; ++r) {
    const U4 run = ring[0];
#pragma unroll
    for (int k = 0; k + 1 < kAhead; ++k) ring[k] = ring[k + 1];
    ring[kAhead - 1] = load(r + kAhead);
    const int at = mine + r * step;
    f(run, min(at, last), at);
  }
}

// f(x, y, i) for neighbouring values of a run.
template <typename T, typename F>
__device__ __forceinline__ void ForTwo(U4 run, int i, F&& f) {
#pragma unroll 1
  for (int e = 0; e < kPer<T>; e += 2) {
    float x, y;
    Two<T>(run, &x, &y);
    f(x, y, i + e);
    run = Next<T>(run);
  }
}
// The largest value of a run, and the smallest (fmax and fmin pass NaN over).
template <typename T>
__device__ __forceinline__ float Top(U4 run) {
  float top = kNone;
#pragma unroll
  for (int e = 0; e < kPer<T>; e += 2) {
    float x, y;
    RawTwo<T>(run, &x, &y);
    top = fmaxf(top, fmaxf(x, y));
    run = Next<T>(run);
  }
  return top;
}
template <typename T>
__device__ __forceinline__ float Bottom(U4 run) {
  float low = -kNone;
#pragma unroll
  for (int e = 0; e < kPer<T>; e += 2) {
    float x, y;
    RawTwo<T>(run, &x, &y);
    low = fminf(low, fminf(x, y));
    run = Next<T>(run);
  }
  return low;
}

// grid (slice, row)
template <typename T>
__global__ __launch_bounds__(kThreads) void MaxKernel(SampleArgs a, Layout l) {
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const Work w(a, l, row);
  const char* x = a.logits + row * a.row_bytes;
  for (int i = slice * kThreads + tid; i < kBins; i += l.slices * kThreads) w.bins[i] = Bin{0, 0, 0};
  if (slice == 0 && tid == 0) w.count[0] = w.count[1] = 0;
  float most = kNone, least = -kNone;
  int at = INT32_MAX;  // the first run that holds `most`
  ForRuns<T>(a, x, slice * l.length, l.length, [&](U4 run, int i, int lo) {
    float top = Top<T>(run);
    if (__any(i != lo)) {  // the row's end: a token counts in one group only
      top = kNone;
      ForTwo<T>(run, i, [&](float y, float z, int t) {
        top = fmaxf(top, fmaxf(t >= lo ? y : kNone, t + 1 >= lo ? z : kNone));
      });
    }
    if (top > most) most = top, at = i;
    least = fminf(least, Bottom<T>(run));
  });
  if (__syncthreads_or(least == kNone)) {  // the least above -inf: a row with tokens ruled out
    least = -kNone;
    ForRuns<T>(a, x, slice * l.length, l.length, [&](U4 run, int i, int) {
      ForTwo<T>(run, i, [&](float y, float z, int) {
        least = fminf(least, fminf(y > kNone ? y : -kNone, z > kNone ? z : -kNone));
      });
    });
  }
  float quad = fmaxf(most, lanes::DppF<lanes::kQuadXor1>(most));
  quad = fmaxf(quad, lanes::DppF<lanes::kQuadXor2>(quad));
  if (l.groups == kThreads)
    w.groups[slice * kThreads + tid] = most;
  else if (tid % 4 == 0)
    w.groups[slice * l.groups + tid / 4] = quad;
  __shared__ SliceMax s[kThreads / 64];
  const float top = lanes::WaveMaxF(most);
  const float low = -lanes::WaveMaxF(-least);
  int first = most == top ? at : INT32_MAX;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
  if ((tid & 63) == 0) s[tid >> 6] = SliceMax{top, low, first, 0};
  __syncthreads();
  if (tid >= 64) return;
  SliceMax m = s[0];
#pragma unroll
  for (int i = 1; i < kThreads / 64; ++i) {
    if (s[i].max > m.max || (s[i].max == m.max && s[i].index < m.index)) m.max = s[i].max, m.index = s[i].index;
    m.min = fminf(m.min, s[i].min);
  }
  // the token in its run
  const bool here = m.max > kNone && tid < kPer<T> && m.index + tid < a.vocab && One<T>(x, m.index + tid) == m.max;
  m.index += __ffsll(static_cast<unsigned long long>(__ballot(here))) - 1;
  if (tid == 0) w.max[slice] = m;
}

__device__ __forceinline__ void LoadPow2(double* pow2) {
  if (threadIdx.x < 32) pow2[threadIdx.x] = kPow2[threadIdx.x];
}

// Order of the ranking: x descending, index ascending. The key of x grows with it.
__device__ __forceinline__ uint32_t KeyOf(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t RankKey(float x, int index) {
  return static_cast<uint64_t>(KeyOf(x)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ float ValueOf(uint64_t rank_key) {
  const uint32_t k = static_cast<uint32_t>(rank_key >> 32);
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ int IndexOf(uint64_t rank_key) {
  return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(rank_key));
}

// Sums over the threads before this one, in a workgroup of kN (every thread
// calls it), of weights and of counts.
template <int kN>
__device__ __forceinline__ uint64_t Before(uint64_t q, uint64_t* total, uint32_t n = 0, uint32_t* before_n = nullptr) {
  constexpr int kParts = kN / 64;
  __shared__ unsigned long long part[kParts];
  __shared__ uint32_t part_n[kParts];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned long long x = lanes::WaveInclusiveAdd(static_cast<unsigned long long>(q));
  const uint32_t c = before_n != nullptr ? lanes::WaveInclusiveAdd(n) : 0;
  __syncthreads();
  if (lane == 63) {
    part[wave] = x;
    if (before_n != nullptr) part_n[wave] = c;
  }
  __syncthreads();
  // every wave sums the parts again, a lane for each
  const unsigned long long p = lanes::WaveInclusiveAdd(lane < kParts ? part[lane] : 0ull);
  *total = lanes::ReadLaneT(p, kParts - 1);
  const int up_lane = __builtin_amdgcn_readfirstlane(wave > 0 ? wave - 1 : 0);
  const unsigned long long up = lanes::ReadLaneT(p, up_lane);
  if (before_n != nullptr) {
    const uint32_t pn = lanes::WaveInclusiveAdd(lane < kParts ? part_n[lane] : 0u);
    const uint32_t un = lanes::ReadLaneT(pn, up_lane);
    *before_n = c - n + (wave > 0 ? un : 0);
  }
  return x - q + (wave > 0 ? up : 0);
}

// Where the cut lies, from the row's histogram.
struct Cut {
  int k_bin, p_bin;             // the steps that hold the k-th token and top_p's last one; kBins: none
  uint32_t k_left;              // tokens to keep of k_bin
  uint32_t unused;
  uint64_t k_before, p_before;  // weight of the steps above
  uint64_t all;                 // the row's weight
  // (words: a copy of a struct with padding would go through private memory,
  // which the compiler puts into LDS by reading the dispatch packet, 14 us away)
  uint32_t whole;  // all tokens down to the cut's step are to be listed (there are at most kList), or (2) are already
  uint32_t slow;   // the histogram does not tell
  __device__ __forceinline__ int End() const { return min(k_bin, p_bin); }
};
static_assert(sizeof(Cut) <= 64, "a row's place for its cut");

template <int kN>
__device__ __forceinline__ Cut FindCut(const Row& r, const Bin* bins) {
  __shared__ Cut s;
  __shared__ int bins_of[2];
  __shared__ uint64_t s_through[2];
  __shared__ uint32_t s_ranked;
  constexpr int kEach = kBins / kN;
  const int tid = threadIdx.x;
  uint64_t q[kEach], sum = 0, all;
  uint32_t n[kEach], count = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    q[i] = __hip_atomic_load(&bins[tid * kEach + i].weight, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    n[i] = r.k != 0 ? __hip_atomic_load(&bins[tid * kEach + i].count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                    : r.Most(tid * kEach + i, q[i]);
    sum += q[i];
    count += n[i];
  }
  uint32_t ranked;
  const uint64_t before = Before<kN>(sum, &all, count, &ranked);
  if (tid == 0) s = Cut{kBins, kBins, 0, 0, 0, 0, all, 0, 0}, bins_of[0] = bins_of[1] = kBins;
  if (tid == 0) s_through[0] = s_through[1] = all;
  __syncthreads();
  if (r.k != 0) {
    const uint32_t k = static_cast<uint32_t>(r.k);
    if (ranked < k && ranked + count >= k) {  // one thread's
      uint64_t b = before, q_bin = 0;
      uint32_t c = ranked, n_bin = 0;
      int bin = -1;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (bin < 0 && c + n[i] >= k) bin = tid * kEach + i, q_bin = q[i], n_bin = n[i];
        if (bin < 0) b += q[i], c += n[i];
      }
      if (r.Lean()) {
        s.k_bin = bin;
        s.whole = c + n_bin <= kList;
        s.slow = !s.whole;
      } else if (q_bin != 0) {
        s.k_bin = bin;
        s.k_left = k - c;
        s.k_before = b;
        s.whole = c + n_bin <= kList;
        s_through[0] = b;
        s_through[1] = b + q_bin;
      }  // (else the k-th token has no weight: no limit)
    } else if (tid == kN - 1 && ranked + count < k && r.Lean()) {
      s.k_bin = r.weightless_end ? kBins - 2 : kBins - 1;  // all that are counted
      s.whole = 1;
    }
    __syncthreads();
    if (s.whole || s.slow) return s;
  }
  if (r.p != 0.0) {
    // the first step at which the weight so far reaches p x the weight of the
    // first k tokens, which lies between that above k_bin and that with it
    const double t[2] = {r.p * static_cast<double>(s_through[0]), r.p * static_cast<double>(s_through[1])};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool from = tid == 0 || static_cast<double>(before) < t[j];
      if (from && static_cast<double>(before + sum) >= t[j]) {  // one thread's
        uint64_t b = before;
        uint32_t c = ranked;
        int bin = -1;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (bin < 0) c += n[i];
          if (bin < 0 && static_cast<double>(b + q[i]) >= t[j]) bin = tid * kEach + i;
          if (bin < 0) b += q[i];
        }
        bins_of[j] = bin;
        if (j == 1) s.p_before = b, s_ranked = c;
      }
    }
    __syncthreads();
    if (tid == 0) {
      s.p_bin = bins_of[1];
      s.slow = bins_of[0] != bins_of[1];
      s.whole = r.k == 0 && s_ranked <= kList;
    }
    __syncthreads();
  }
  return s;
}

// Lists the tokens of a slice down to step `last`. They gather in LDS (`found`,
// kList of them) and go to the row's list together: a place in it for each would
// be a round trip to memory.
struct Lister {
  uint64_t* found;
  uint32_t* n_found;
  uint32_t* at;
  __device__ __forceinline__ void Begin() {
    if (threadIdx.x == 0) *n_found = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void Add(float v, int i) {
    const uint32_t k = atomicAdd(n_found, 1u);
    if (k < kList) found[k] = RankKey(v, i);
  }
  __device__ __forceinline__ void End(const Work& w) {
    __syncthreads();
    const uint32_t n = *n_found;
    if (n == 0) return;
    if (threadIdx.x == 0) *at = atomicAdd(w.count, n);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < min(n, static_cast<uint32_t>(kList)); i += kThreads)
      if (*at + i < kList) w.list[*at + i] = found[i];
  }
};
template <typename T>
__device__ __forceinline__ void ListDown(const SampleArgs& a, const Layout& l, const Work& w, const Row& r, const char* x,
                                         int slice, int last, Lister list) {
  list.Begin();
  ForRuns<T>(a, x, slice * l.length, l.length, [&](U4 run, int i, int lo) {
    if (!__any(r.Bin(Top<T>(run)) <= last)) return;  // few runs hold a listed token
    ForTwo<T>(run, i, [&](float y, float z, int at) {
      if (at >= lo && y > kNone && r.Bin(y) <= last) list.Add(y, at);
      if (at + 1 >= lo && z > kNone && r.Bin(z) <= last) list.Add(z, at + 1);
    });
  });
  list.End(w);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void CountKernel(SampleArgs a, Layout l) {
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const Work w(a, l, row);
  const Row r = RowOf(a, l, w, row);
  // no cut to look for (min_p needs none)
  if (r.greedy || r.max == kNone || (r.k == 0 && r.p == 0.0)) return;
  __shared__ unsigned long long weight[kBins];
  __shared__ uint32_t count[kBins];
  __shared__ double pow2[32];
  __shared__ int s_last;
  constexpr int kEach = kBins / kThreads;
  const uint32_t k = static_cast<uint32_t>(r.k);
  LoadPow2(pow2);
  for (int i = tid; i < kBins; i += kThreads) weight[i] = 0, count[i] = 0;
  if (tid == 0) s_last = -1;
  __syncthreads();
  const char* x = a.logits + row * a.row_bytes;
  if (r.Direct(l)) {
    for (int i = tid; i < l.slices * l.groups; i += kThreads) {
      const float top = w.groups[i];
      if (top > kNone) atomicAdd(&count[r.Bin(top)], 1u);
    }
    __syncthreads();
    uint32_t n = 0, before;
    uint64_t unused;
#pragma unroll
    for (int i = 0; i < kEach; ++i) n += count[tid * kEach + i];
    Before<kThreads>(0, &unused, n, &before);
    if (before < k && before + n >= k) {
      uint32_t c = before;
      int bin = -1;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        c += count[tid * kEach + i];
        if (bin < 0 && c >= k) bin = tid * kEach + i;
      }
      // (without weight from there on: no limit)
      s_last = r.weightless_end && bin == kBins - 1 ? kBins - 2 : bin;
    }
    __syncthreads();
    if (s_last >= 0) {
      __shared__ uint32_t n_found, s_at;
      ListDown<T>(a, l, w, r, x, slice, s_last, Lister{reinterpret_cast<uint64_t*>(weight), &n_found, &s_at});
      if (slice == 0 && tid == 0) *w.cut = Cut{s_last, kBins, 0, 0, 0, 0, 0, 2, 0};
      return;
    }
    // fewer groups than k hold a token: the histogram
    for (int i = tid; i < kBins; i += kThreads) count[i] = 0;
    __syncthreads();
  }
  const bool lean = r.Lean();
  ForRuns<T>(a, x, slice * l.length, l.length, [&](U4 run, int i, int lo) {
    ForTwo<T>(run, i, [&](float y, float z, int at) {
      const int by = r.Bin(y), bz = r.Bin(z);
      const bool cy = at >= lo && r.Counted(y, by), cz = at + 1 >= lo && r.Counted(z, bz);
      if (!__any(cy || cz)) return;
      if (!lean) {
        const uint64_t qy = Row::Units(r.Weight(y, pow2)) & Mask(cy), qz = Row::Units(r.Weight(z, pow2)) & Mask(cz);
        if (qy != 0) atomicAdd(&weight[by], static_cast<unsigned long long>(qy));
        if (qz != 0) atomicAdd(&weight[bz], static_cast<unsigned long long>(qz));
      }
      if (r.k == 0) return;  // (see Row::Most)
      if (cy) atomicAdd(&count[by], 1u);
      if (cz) atomicAdd(&count[bz], 1u);
    });
  });
  __syncthreads();
  // For a small top_k the steps down to the slice's own k-th token: the row's
  // lies no further down, and those steps get every slice's counts.
  int last = kBins - 1;
  if (lean) {
    if (tid == 0) s_last = last;
    uint32_t n = 0, before;
    uint64_t unused;
#pragma unroll
    for (int i = 0; i < kEach; ++i) n += count[tid * kEach + i];
    Before<kThreads>(0, &unused, n, &before);
    if (before < k && before + n >= k) s_last = tid * kEach + kEach - 1;
    __syncthreads();
    last = s_last;
  }
  for (int i = tid; i <= last; i += kThreads) {
    if (weight[i] != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&w.bins[i].weight), weight[i]);
    if (count[i] != 0) atomicAdd(&w.bins[i].count, count[i]);
  }
  // The row's last slice to get here finds the cut: every slice's atomics have
  // been carried out, at the device's point of coherence, before it counts
  // itself, and that is where FindCut reads them.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  __shared__ uint32_t s_before;
  if (tid == 0) s_before = atomicAdd(&w.count[1], 1u);
  __syncthreads();
  if (s_before != static_cast<uint32_t>(l.slices - 1)) return;
  const Cut cut = FindCut<kThreads>(r, w.bins);
  if (tid == 0) *w.cut = cut;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void SplitKernel(SampleArgs a, Layout l) {
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const Work w(a, l, row);
  const Row r = RowOf(a, l, w, row);
  if (r.greedy || r.max == kNone) return;
  __shared__ double pow2[32];
  LoadPow2(pow2);
  Cut cut{kBins, kBins, 0, 0, 0, 0, 0, 0, 0};
  if (r.k != 0 || r.p != 0.0) cut = *w.cut;
  __syncthreads();
  if (cut.slow) return;
  const int end_bin = cut.End();
  const char* x = a.logits + row * a.row_bytes;
  if (cut.whole == 2) return;
  __shared__ uint64_t found[kList];
  __shared__ uint32_t n_found, s_at;
  Lister list{found, &n_found, &s_at};
  if (cut.whole) {
    ListDown<T>(a, l, w, r, x, slice, end_bin, list);
    return;
  }
  list.Begin();
  const bool limited = end_bin < kBins;
  const int listed_last = max(cut.k_bin < kBins ? cut.k_bin : -1, cut.p_bin < kBins ? cut.p_bin : -1);
  __shared__ uint64_t part[kThreads / 64];
  for (int start = slice * l.length; start < min(a.vocab, (slice + 1) * l.length); start += kUnit) {
    uint64_t sum = 0;
    ForRuns<T>(a, x, start, kUnit, [&](U4 run, int i, int lo) {
      const float top = Top<T>(run);
      if (!__any(r.MayReach(top) || r.Bin(top) <= listed_last)) return;
      ForTwo<T>(run, i, [&](float y, float z, int at) {
        // (masks, no branches: a branch would take the two weights one after the other)
        const double fy = r.Weight(y, pow2), fz = r.Weight(z, pow2);
        bool ty = at >= lo, tz = at + 1 >= lo;
        if (limited) {
          const int by = r.Bin(y), bz = r.Bin(z);
          const bool ly = ty & (y > kNone) & ((by == cut.k_bin) | (by == cut.p_bin));
          const bool lz = tz & (z > kNone) & ((bz == cut.k_bin) | (bz == cut.p_bin));
          if (__any(ly | lz)) {
            if (ly) list.Add(y, at);
            if (lz) list.Add(z, at + 1);
          }
          ty &= by < end_bin;
          tz &= bz < end_bin;
        }
        sum += Row::Units(fy) & Mask(ty & (fy >= r.floor));
        sum += Row::Units(fz) & Mask(tz & (fz >= r.floor));
      });
    });
    sum = lanes::WaveInclusiveAdd(static_cast<unsigned long long>(sum));
    __syncthreads();
    if ((tid & 63) == 63) part[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) w.weights[start / kUnit] = part[0] + part[1] + part[2] + part[3];
  }
  list.End(w);
}

// The rank key of the last token kept when tokens are taken from the best on
// until `tokens` of them are (limit < 0), or while their weight is below
// `limit`; *weight: the weight of those taken. Over the whole row, a digit of
// 8 bits of the rank key at a time.
template <typename T>
__device__ uint64_t CutByDigits(const SampleArgs& a, const Row& r, const char* x, const double* pow2, uint64_t tokens,
                                double limit, uint64_t* weight) {
  __shared__ unsigned long long q[256];
  __shared__ uint32_t n[256];
  __shared__ uint64_t s_prefix, s_weight, s_count;
  const int tid = threadIdx.x;
  uint64_t prefix = 0, above = 0, above_n = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    if (tid < 256) q[tid] = 0, n[tid] = 0;
    __syncthreads();
    for (int i = tid; i < a.vocab; i += kDrawThreads) {
      const float v = One<T>(x, i);
      const uint64_t key = RankKey(v, i);
      if (shift < 56 && (key >> (shift + 8)) != (prefix >> (shift + 8))) continue;
      const int digit = static_cast<int>(key >> shift) & 255;
      atomicAdd(&q[digit], static_cast<unsigned long long>(Row::Units(r.Weight(v, pow2))));
      atomicAdd(&n[digit], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      int digit = 255, last = -1;
      uint64_t w = above, c = above_n, last_w = above, last_c = above_n;
      for (; digit >= 0; --digit) {
        if (n[digit] == 0) continue;
        last = digit, last_w = w, last_c = c;
        const bool here = limit < 0.0 ? c + n[digit] >= tokens : static_cast<double>(w + q[digit]) >= limit;
        if (here) break;
        w += q[digit];
        c += n[digit];
      }
      // (the whole row when the limit is never reached)
      s_prefix = prefix | static_cast<uint64_t>(last) << shift;
      s_weight = last_w;
      s_count = last_c;
    }
    __syncthreads();
    prefix = s_prefix, above = s_weight, above_n = s_count;
    __syncthreads();
  }
  const int index = static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(prefix));
  *weight = above + Row::Units(r.Weight(One<T>(x, index), pow2));
  return prefix;
}

// The value of the lane whose number differs in bit kBit.
template <int kBit>
__device__ __forceinline__ uint32_t Across(uint32_t v) {
  if constexpr (kBit == 1) return lanes::Dpp<lanes::kQuadXor1>(v);
  if constexpr (kBit == 2) return lanes::Dpp<lanes::kQuadXor2>(v);
  if constexpr (kBit == 4) return lanes::Dpp<0x1B>(lanes::Dpp<lanes::kRowHalfMirror>(v));  // 7 - i, then 3 - i of a quad
  if constexpr (kBit == 8) return lanes::Dpp<lanes::kRowRor8>(v);
  if constexpr (kBit == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  }
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return threadIdx.x & 32 ? r[0] : r[1];
}
template <int kBit>
__device__ __forceinline__ uint64_t Across64(uint64_t v) {
  return Across<kBit>(static_cast<uint32_t>(v)) |
         static_cast<uint64_t>(Across<kBit>(static_cast<uint32_t>(v >> 32))) << 32;
}

// Sorts the first n (a power of two from 64 to kDrawThreads) threads' keys,
// largest first; every thread of the workgroup calls it.
__device__ __forceinline__ uint64_t SortDown(uint64_t key, int n, uint64_t* lds) {
  const int tid = threadIdx.x;
#pragma unroll 1
  for (int size = 2; size <= n; size <<= 1) {
    const bool up = (tid & size) != 0 && size < n;
#pragma unroll 1
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      uint64_t other = 0;
      if (stride >= 64) {
        __syncthreads();
        if (tid < n) lds[tid] = key;
        __syncthreads();
        if (tid < n) other = lds[tid ^ stride];
      } else if (tid < n) {  // (whole waves)
        switch (stride) {
          case 1: other = Across64<1>(key); break;
          case 2: other = Across64<2>(key); break;
          case 4: other = Across64<4>(key); break;
          case 8: other = Across64<8>(key); break;
          case 16: other = Across64<16>(key); break;
          default: other = Across64<32>(key);
        }
      }
      const bool lower = (tid & stride) == 0;
      if (tid < n) key = (lower == up) == (key < other) ? key : other;
    }
  }
  return key;
}
__device__ __forceinline__ int PowerFor(int n) {
  int p = 64;
  while (p < n) p <<= 1;
  return p;
}

__device__ __forceinline__ void Write(const SampleArgs& a, int row, int token, double weight, uint64_t total) {
  a.tokens[row] = token;
  if (a.logprobs != nullptr) a.logprobs[row] = static_cast<float>(log(weight / static_cast<double>(total)));
}

// One workgroup per row.
template <typename T>
__global__ __launch_bounds__(kDrawThreads) void DrawKernel(SampleArgs a, Layout l) {
  const int row = blockIdx.x, tid = threadIdx.x;
  const Work w(a, l, row);
  // All that may be needed, in one round trip (what was not written is not used).
  const int units = (a.vocab + kUnit - 1) / kUnit;
  const uint64_t item = w.list[tid], unit_item = w.weights[tid & (kMaxUnits - 1)];
  const uint32_t listed = w.count[0];
  const Cut stored = *w.cut;
  const float u_given = a.u[row];
  const Row r = RowOf(a, l, w, row);
  if (r.greedy || r.max == kNone) {
    if (tid == 0) {
      a.tokens[row] = r.max == kNone ? -1 : r.best;
      if (a.logprobs != nullptr) a.logprobs[row] = r.max == kNone ? kNone : 0.0f;
    }
    return;
  }
  __shared__ double pow2[32];
  __shared__ uint64_t keys[kDrawThreads];
  __shared__ unsigned long long unit_weight[kMaxUnits];
  __shared__ uint64_t s_taken, s_last;
  __shared__ uint32_t s_there;
  LoadPow2(pow2);
  if (tid < kMaxUnits) unit_weight[tid] = 0;
  if (tid == 0) s_there = 0;
  const char* x = a.logits + row * a.row_bytes;
  Cut cut{kBins, kBins, 0, 0, 0, 0, 0, 0, 0};
  if (r.k != 0 || r.p != 0.0) cut = stored;
  const int end_bin = cut.End();
  const double u = fmax(0.0, fmin(static_cast<double>(u_given), 1.0));
  const uint32_t n = end_bin < kBins && !cut.slow ? listed : 0;
  const bool slow = cut.slow || n > kList;
  __syncthreads();

  // The list, best first: this thread's token and the weight before it.
  uint64_t key = 0, q = 0, before = 0, sum = 0;
  double f = 0.0;
  if (n > 0 && !slow) {
    const int here = static_cast<int>(n);
    key = SortDown(tid < here ? item : 0, PowerFor(here), keys);
    f = tid < here ? r.Weight(ValueOf(key), pow2) : 0.0;
    q = Row::Units(f);
    before = Before<kDrawThreads>(q, &sum);
    if (cut.whole) {
      // It holds all that can be kept. The draw among those that are: the 64th
      // part of the vocabulary that it falls into, then the token there.
      uint64_t taken = cut.all;
      if (r.k != 0) {
        if (tid == min(here, r.k) - 1) s_taken = before + q;
        __syncthreads();
        taken = s_taken;
      }
      const bool in = tid < here && (r.k == 0 || tid < r.k) && q != 0 && f >= r.floor &&
                      (r.p == 0.0 || static_cast<double>(before) < r.p * static_cast<double>(taken));
      const int index = IndexOf(key);
      const int part = min(static_cast<int>(static_cast<float>(index) * (64.0f / static_cast<float>(a.vocab))), 63);
      if (in) atomicAdd(&unit_weight[part], static_cast<unsigned long long>(q));
      __syncthreads();
      const uint64_t mine = unit_weight[tid & 63];
      const uint64_t up_to = lanes::WaveInclusiveAdd(static_cast<unsigned long long>(mine));
      const uint64_t total = lanes::ReadLaneT(up_to, 63);
      const double mark = u * static_cast<double>(total);
      uint64_t hit = __ballot(mine != 0 && static_cast<double>(up_to) > mark);
      if (hit == 0) hit = 1ull << (63 - __clzll(static_cast<long long>(__ballot(mine != 0))));  // u = 1: the last one
      const int at = __builtin_amdgcn_readfirstlane(__ffsll(static_cast<unsigned long long>(hit)) - 1);
      const uint64_t end = lanes::ReadLaneT(up_to, at);
      const bool there = in && part == at;
      if (there) keys[atomicAdd(&s_there, 1u)] = static_cast<uint64_t>(index) << 45 | q;  // (18 bits, 45 bits)
      __syncthreads();
      if (!there) return;
      uint64_t up = end - lanes::ReadLaneT(mine, at);
      for (uint32_t i = 0; i < s_there; ++i)
        if (static_cast<int>(keys[i] >> 45) < index) up += keys[i] & ((uint64_t{1} << 45) - 1);
      if ((static_cast<double>(up + q) > mark || up + q == end) && !(static_cast<double>(up) > mark))
        Write(a, row, index, f, total);
      return;
    }
  }

  if (tid < units) unit_weight[tid] = slow ? 0 : unit_item;
  if (tid == 0) s_last = 0, s_taken = cut.k_before;
  __syncthreads();
  uint64_t last = 0;  // rank key of the last token that top_k and top_p keep; 0: every token
  if (slow) {
    uint64_t taken = cut.all;
    if (r.k != 0) last = CutByDigits<T>(a, r, x, pow2, r.k, -1.0, &taken);
    if (r.p != 0.0) {
      const uint64_t by_p = CutByDigits<T>(a, r, x, pow2, 0, r.p * static_cast<double>(taken), &taken);
      last = max(last, by_p);
    }
    for (int s = 0; s < units; ++s) {
      uint64_t part = 0, all;
      for (int i = s * kUnit + tid; i < min(a.vocab, (s + 1) * kUnit); i += kDrawThreads) {
        const float v = One<T>(x, i);
        const double g = r.Weight(v, pow2);
        if (RankKey(v, i) >= last && g >= r.floor) part += Row::Units(g);
      }
      Before<kDrawThreads>(part, &all);
      if (tid == 0) unit_weight[s] = all;
    }
  } else if (n > 0) {
    // One step's tokens, or top_p's step's and then k_bin's.
    const int bin = tid < static_cast<int>(n) ? r.Bin(ValueOf(key)) : -1;
    const bool both = cut.k_bin < kBins && cut.p_bin < cut.k_bin;
    const int p_tokens = both ? __syncthreads_count(bin == cut.p_bin) : 0;
    if (tid == p_tokens) s_last = before;  // (weight of top_p's step, where k_bin's follow)
    __syncthreads();
    const uint64_t in_step = before - (bin == cut.k_bin ? s_last : 0);
    uint64_t taken = cut.all;
    bool in = bin >= 0 && bin == end_bin;
    if (cut.k_bin < kBins) {
      const uint32_t rank = tid - p_tokens;
      if (bin == cut.k_bin && rank == cut.k_left - 1) s_taken = cut.k_before + in_step + q;
      __syncthreads();
      taken = s_taken;
      if (bin == cut.k_bin) in = in && rank < cut.k_left;
    }
    if (bin == cut.p_bin) in = in && static_cast<double>(cut.p_before + in_step) < r.p * static_cast<double>(taken);
    if (in && f >= r.floor) atomicAdd(&unit_weight[IndexOf(key) / kUnit], static_cast<unsigned long long>(q));
    // the kept ones are the first threads of the step
    const int kept = __syncthreads_count(in);
    if (tid == kept - 1) s_last = key;
    __syncthreads();
    last = s_last;
  }
  __syncthreads();
  // The unit, then the token in it.
  __shared__ int s_unit;
  __shared__ uint64_t s_before, s_total;
  if (tid < 64) {
    const uint64_t mine = tid < units ? unit_weight[tid] : 0;
    const uint64_t up_to = lanes::WaveInclusiveAdd(static_cast<unsigned long long>(mine));
    const uint64_t total = lanes::ReadLaneT(up_to, 63);
    uint64_t hit = __ballot(mine != 0 && static_cast<double>(up_to) > u * static_cast<double>(total));
    if (hit == 0) hit = 1ull << (63 - __clzll(static_cast<long long>(__ballot(mine != 0))));  // u = 1: the last one
    if (tid == __ffsll(static_cast<unsigned long long>(hit)) - 1) s_unit = tid, s_before = up_to - mine, s_total = total;
  }
  __syncthreads();
  constexpr int kEach = kUnit / kDrawThreads;
  const int from = s_unit * kUnit + tid * kEach;
  double weight[kEach];
  sum = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const float v = from + e < a.vocab ? One<T>(x, from + e) : kNone;
    weight[e] = r.Weight(v, pow2);
    if (RankKey(v, from + e) < last || !(weight[e] >= r.floor)) weight[e] = 0.0;
    sum += Row::Units(weight[e]);
  }
  uint64_t all;
  before = s_before + Before<kDrawThreads>(sum, &all);
  const double mark = u * static_cast<double>(s_total);
  // the first thread whose sum passes the mark (or the last with a weight)
  const bool past = sum != 0 && (static_cast<double>(before + sum) > mark || before + sum == s_before + all);
  if (past && !(static_cast<double>(before) > mark)) {
    int token = -1;
    double at = 0.0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const uint64_t q = Row::Units(weight[e]);
      if (q != 0 && !(static_cast<double>(before) > mark)) token = from + e, at = weight[e];
      before += q;
    }
    Write(a, row, token, at, s_total);
  }
}

template <typename T>
void Launch(const SampleArgs& a, hipStream_t s) {
  const Layout l = LayoutOf(a.rows, a.vocab);
  const dim3 grid(l.slices, a.rows);
  MaxKernel<T><<<grid, kThreads, 0, s>>>(a, l);
  // (min_p needs no cut: 8 f32 rows 17 us a call without the launch, 19.5 with it)
  if (a.top_k != nullptr || a.top_p != nullptr) CountKernel<T><<<grid, kThreads, 0, s>>>(a, l);
  SplitKernel<T><<<grid, kThreads, 0, s>>>(a, l);
  DrawKernel<T><<<a.rows, kDrawThreads, 0, s>>>(a, l);
  HIP_CHECK(hipGetLastError());
}

}  // namespace

int64_t WorkBytes(int64_t rows, int64_t vocab) { return LayoutOf(rows, vocab).bytes; }

void Sample(const SampleArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  if (a.type == kF32)
    Launch<F32>(a, s);
  else if (a.type == kF16)
    Launch<F16>(a, s);
  else
    Launch<BF16>(a, s);
}

}  // namespace rows
}  // namespace rpg

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
// polynomial of degree 5, 1.5e-13 relative).
//
// Four launches over (row, slice of the vocabulary), without a sort:
//   Max    largest value (and its first index) and least finite one per slice
//   Count  histogram of 2048 equal steps of x below the row's maximum: count
//          and weight, slices added by atomics
//   Split  the step that holds the cut, from the histogram: weight of the
//          steps above it per slice, and its own tokens as a list
//   Draw   one workgroup a row: the cut inside the list, the slice that the
//          draw falls into, the token inside that slice
// A list of more than kList tokens (thousands of equal values, a temperature
// that flattens everything) or a cut whose step the histogram cannot tell
// (top_k inside one step deciding top_p's) is found by Draw over the whole
// row, digit by digit.
//
// Bound: the logits' bytes, read once from HBM (later launches find them in
// the memory-side cache); a single row is bound by its four launches.

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
constexpr int kMaxSlices = 64;
constexpr int kUnit = 4096;      // a slice's tokens are a multiple of this
constexpr float kNone = -__builtin_inff();

struct Bin {
  uint64_t weight;
  uint32_t count, pad;
};
struct Item {
  float x;
  int32_t index;
};
struct SliceMax {
  float max, min;
  int32_t index, pad;
};

struct Layout {
  int slices, length;  // tokens per slice
  int64_t max_at, bins_at, weights_at, lists_at, counts_at, bytes;
};

__host__ __device__ inline Layout LayoutOf(int64_t rows, int64_t vocab) {
  Layout l;
  // About 1500 workgroups where there are many rows, slices of 4096 tokens
  // where there are few.
  const int64_t most = (vocab + kUnit - 1) / kUnit;
  int64_t want = rows < 1 ? 1 : (1536 + rows - 1) / rows;
  want = want < 1 ? 1 : want > most ? most : want;
  want = want > kMaxSlices ? kMaxSlices : want;
  l.length = static_cast<int>(((vocab + want - 1) / want + kUnit - 1) / kUnit * kUnit);
  l.slices = static_cast<int>((vocab + l.length - 1) / l.length);
  l.bins_at = 0;
  l.max_at = l.bins_at + rows * kBins * static_cast<int64_t>(sizeof(Bin));
  l.weights_at = l.max_at + rows * l.slices * static_cast<int64_t>(sizeof(SliceMax));
  l.lists_at = l.weights_at + rows * l.slices * 8;
  l.counts_at = l.lists_at + rows * kList * static_cast<int64_t>(sizeof(Item));
  l.bytes = (l.counts_at + rows * 4 + 255) / 256 * 256;
  return l;
}

// One row's view of the work buffer.
struct Work {
  Bin* bins;
  SliceMax* max;
  uint64_t* weights;
  Item* list;
  uint32_t* count;
  __device__ Work(const SampleArgs& a, const Layout& l, int row)
      : bins(reinterpret_cast<Bin*>(a.work + l.bins_at) + static_cast<int64_t>(row) * kBins),
        max(reinterpret_cast<SliceMax*>(a.work + l.max_at) + static_cast<int64_t>(row) * l.slices),
        weights(reinterpret_cast<uint64_t*>(a.work + l.weights_at) + static_cast<int64_t>(row) * l.slices),
        list(reinterpret_cast<Item*>(a.work + l.lists_at) + static_cast<int64_t>(row) * kList),
        count(reinterpret_cast<uint32_t*>(a.work + l.counts_at) + row) {}
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

// Values i .. i + kPer - 1 of a row (-inf past its end); wide: the row lies at
// a multiple of 16 bytes.
template <typename T>
__device__ __forceinline__ void Values(const char* row, int i, int vocab, bool wide, float (&x)[kPer<T>]) {
  if (wide && i + kPer<T> <= vocab) {
    const U4 v = paged::Load16(row + static_cast<int64_t>(i) * paged::kBytes<T>);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (paged::kBytes<T> == 4) {
        x[e] = Clean(__uint_as_float(v[e]));
      } else {
        Unpack2<T>(v[e], &x[2 * e], &x[2 * e + 1]);
        x[2 * e] = Clean(x[2 * e]);
        x[2 * e + 1] = Clean(x[2 * e + 1]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e) x[e] = i + e < vocab ? One<T>(row, i + e) : kNone;
  }
}

// 2^(-j / 32)
__device__ const double kPow2[32] = {
    1.0, 0.9785720620877001, 0.9576032806985737, 0.93708381705515,
    0.9170040432046712, 0.8973545375015536, 0.8781260801866497, 0.859309649061239,
    0.8408964152537145, 0.8228777390769825, 0.8052451659746271, 0.7879904225539432,
    0.7711054127039704, 0.7545822137967114, 0.7384130729697497, 0.7225904034885233,
    0.7071067811865476, 0.691954940981916, 0.6771277734684463, 0.6626183215798707,
    0.6484197773255048, 0.6345254785958666, 0.620928906036742, 0.6076236799902345,
    0.5946035575013605, 0.5818624293887887, 0.5693943173783458, 0.5571933712979462,
    0.5452538663326288, 0.5335702003384118, 0.5221368912137069, 0.5109485743270583};

constexpr double kOne = 17592186044416.0;  // 2^44: the largest weight

// A row's parameters, from its slices' maxima.
struct Row {
  float max;     // -inf: nothing to draw from
  int32_t best;  // its first index
  float scale;   // histogram steps per unit of x
  double c;      // log2(e) / T
  bool greedy;
  int32_t k;      // 0: no limit
  double p, floor;  // 0: no limit; min_p in weight units

  // w 2^44, at most half a unit off when rounded; 0 where it would be less
  // than half of one.
  __device__ __forceinline__ double Weight(float x, const double* pow2) const {
    const double d = x == max ? 0.0 : static_cast<double>(max) - static_cast<double>(x);
    const double y = d == 0.0 ? 0.0 : d * c;
    if (!(y < 45.5)) return 0.0;
    const int n = static_cast<int>(y * 32.0);
    const double z = (static_cast<double>(n) * 0.03125 - y) * 0.69314718055994530942;  // (-ln 2 / 32, 0]
    double e = __builtin_fma(z, 1.0 / 120.0, 1.0 / 24.0);
    e = __builtin_fma(z, e, 1.0 / 6.0);
    e = __builtin_fma(z, e, 0.5);
    e = __builtin_fma(z, e, 1.0);
    e = __builtin_fma(z, e, 1.0);
    const uint64_t t = __builtin_bit_cast(uint64_t, pow2[n & 31]) + (static_cast<uint64_t>(44 - (n >> 5)) << 52);
    return e * __builtin_bit_cast(double, t);
  }
  // rounded to an integer (weights are below 2^52)
  static __device__ __forceinline__ uint64_t Units(double w) {
    return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
  }
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
  r.c = 1.4426950408889634074 / static_cast<double>(t);
  const float span = fminf(31.6f * t, max - min);
  r.scale = span > 0.0f ? static_cast<float>(kBins) / span : 0.0f;
  const int32_t k = a.top_k != nullptr ? a.top_k[row] : 0;
  r.k = k > 0 && k < a.vocab ? k : 0;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  r.p = p > 0.0f && p < 1.0f ? static_cast<double>(p) : 0.0;
  const float f = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  r.floor = f > 0.0f ? static_cast<double>(fminf(f, 1.0f)) * kOne : 0.0;
  return r;
}

template <typename T>
__device__ __forceinline__ bool Wide(const SampleArgs& a) {
  return ((reinterpret_cast<uintptr_t>(a.logits) | static_cast<uint64_t>(a.row_bytes)) & 15) == 0;
}

// grid (slice, row)
template <typename T>
__global__ __launch_bounds__(kThreads) void MaxKernel(SampleArgs a, Layout l) {
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const Work w(a, l, row);
  const char* x = a.logits + row * a.row_bytes;
  const bool wide = Wide<T>(a);
  for (int i = slice * kThreads + tid; i < kBins; i += l.slices * kThreads) w.bins[i] = Bin{0, 0, 0};
  if (slice == 0 && tid == 0) *w.count = 0;
  float most = kNone, least = -kNone;
  int at = INT32_MAX;
  const int end = min(a.vocab, (slice + 1) * l.length);
#pragma unroll 4
  for (int i = slice * l.length + tid * kPer<T>; i < end; i += kThreads * kPer<T>) {
    float v[kPer<T>];
    Values<T>(x, i, a.vocab, wide, v);
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e) {
      if (v[e] > most) most = v[e], at = i + e;
      if (v[e] > kNone) least = fminf(least, v[e]);
    }
  }
  __shared__ SliceMax s[kThreads / 64];
  const float top = lanes::WaveMaxF(most);
  const float low = -lanes::WaveMaxF(-least);
  int first = most == top ? at : INT32_MAX;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
  if ((tid & 63) == 0) s[tid >> 6] = SliceMax{top, low, first, 0};
  __syncthreads();
  if (tid != 0) return;
  SliceMax m = s[0];
  for (int i = 1; i < kThreads / 64; ++i) {
    if (s[i].max > m.max || (s[i].max == m.max && s[i].index < m.index)) m.max = s[i].max, m.index = s[i].index;
    m.min = fminf(m.min, s[i].min);
  }
  w.max[slice] = m;
}

__device__ __forceinline__ void LoadPow2(double* pow2) {
  if (threadIdx.x < 32) pow2[threadIdx.x] = kPow2[threadIdx.x];
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
  LoadPow2(pow2);
  for (int i = tid; i < kBins; i += kThreads) weight[i] = 0, count[i] = 0;
  __syncthreads();
  const char* x = a.logits + row * a.row_bytes;
  const bool wide = Wide<T>(a);
  const int end = min(a.vocab, (slice + 1) * l.length);
  for (int i = slice * l.length + tid * kPer<T>; i < end; i += kThreads * kPer<T>) {
    float v[kPer<T>];
    Values<T>(x, i, a.vocab, wide, v);
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e) {
      if (i + e >= a.vocab) continue;
      const int b = r.Bin(v[e]);
      const uint64_t q = Row::Units(r.Weight(v[e], pow2));
      if (q != 0) atomicAdd(&weight[b], static_cast<unsigned long long>(q));
      if (r.k != 0) atomicAdd(&count[b], 1u);
    }
  }
  __syncthreads();
  for (int i = tid; i < kBins; i += kThreads) {
    if (weight[i] != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&w.bins[i].weight), weight[i]);
    if (count[i] != 0) atomicAdd(&w.bins[i].count, count[i]);
  }
}

// Sums over the threads before this one, in a workgroup of kN (every thread
// calls it).
template <int kN, typename V>
__device__ __forceinline__ V Before(V v, V* total) {
  __shared__ V part[kN / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  V x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) part[wave] = x;
  __syncthreads();
  V before = x - v, sum = 0;
  for (int i = 0; i < kN / 64; ++i) {
    if (i < wave) before += part[i];
    sum += part[i];
  }
  *total = sum;
  return before;
}

// Where the cut lies, from the row's histogram.
struct Cut {
  int k_bin, p_bin;        // the steps that hold the k-th token and top_p's last one; kBins: no limit
  uint32_t k_left;         // tokens to keep of k_bin
  uint64_t k_before, p_before;  // weight of the steps above
  uint64_t all;            // the row's weight
  bool unclear;            // p_bin hangs on which tokens of k_bin are kept
  __device__ __forceinline__ int End() const { return min(k_bin, p_bin); }
};

template <int kN>
__device__ __forceinline__ Cut FindCut(const Row& r, const Bin* bins) {
  __shared__ Cut s;
  __shared__ int bins_of[2];
  constexpr int kEach = kBins / kN;
  const int tid = threadIdx.x;
  uint64_t q[kEach], sum = 0, all;
  uint32_t n[kEach], count = 0, unused;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    q[i] = bins[tid * kEach + i].weight;
    n[i] = bins[tid * kEach + i].count;
    sum += q[i];
    count += n[i];
  }
  uint64_t before = Before<kN>(sum, &all);
  uint32_t ranked = Before<kN>(count, &unused);
  __syncthreads();
  if (tid == 0) s = Cut{kBins, kBins, 0, 0, 0, all, false}, bins_of[0] = bins_of[1] = kBins;
  __syncthreads();
  uint64_t lo = all, hi = all;
  if (r.k != 0) {
    uint64_t b = before;
    uint32_t c = ranked;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (c < static_cast<uint32_t>(r.k) && c + n[i] >= static_cast<uint32_t>(r.k)) {
        s.k_bin = tid * kEach + i;
        s.k_left = r.k - c;
        s.k_before = b;
        s.p_before = b + q[i];  // for the others, until they have read it
      }
      b += q[i];
      c += n[i];
    }
    __syncthreads();
    lo = s.k_before, hi = s.p_before;
    __syncthreads();
  }
  if (r.p != 0.0) {
    // the first step with its weight and that above it >= p x the weight
    const double t[2] = {r.p * static_cast<double>(lo), r.p * static_cast<double>(hi)};
    uint64_t b = before;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool first = tid * kEach + i == 0;
        if ((first || static_cast<double>(b) < t[j]) && static_cast<double>(b + q[i]) >= t[j]) {
          if (j == 0) {
            bins_of[0] = tid * kEach + i;
          } else {
            bins_of[1] = tid * kEach + i;
            s.p_before = b;
          }
        }
      }
      b += q[i];
    }
    __syncthreads();
    if (tid == 0) s.p_bin = bins_of[1], s.unclear = bins_of[0] != bins_of[1];
  }
  __syncthreads();
  return s;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void SplitKernel(SampleArgs a, Layout l) {
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const Work w(a, l, row);
  const Row r = RowOf(a, l, w, row);
  if (r.greedy || r.max == kNone) return;
  __shared__ double pow2[32];
  LoadPow2(pow2);
  Cut cut{kBins, kBins, 0, 0, 0, 0, false};
  if (r.k != 0 || r.p != 0.0) cut = FindCut<kThreads>(r, w.bins);
  __syncthreads();
  if (cut.unclear) return;
  const int end_bin = cut.End();
  const char* x = a.logits + row * a.row_bytes;
  const bool wide = Wide<T>(a);
  const int end = min(a.vocab, (slice + 1) * l.length);
  uint64_t sum = 0;
  for (int i = slice * l.length + tid * kPer<T>; i < end; i += kThreads * kPer<T>) {
    float v[kPer<T>];
    Values<T>(x, i, a.vocab, wide, v);
#pragma unroll
    for (int e = 0; e < kPer<T>; ++e) {
      if (i + e >= a.vocab) continue;
      const int b = r.Bin(v[e]);
      if (b < end_bin) {
        const double f = r.Weight(v[e], pow2);
        if (f >= r.floor) sum += Row::Units(f);
      }
      if (b == cut.k_bin || b == cut.p_bin) {
        const uint32_t at = atomicAdd(w.count, 1u);
        if (at < kList) w.list[at] = Item{v[e], i + e};
      }
    }
  }
  uint64_t all;
  Before<kThreads>(sum, &all);
  if (tid == 0) w.weights[slice] = all;
}

// Order of the ranking: x descending, index ascending. The key of x grows with it.
__device__ __forceinline__ uint32_t KeyOf(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t RankKey(float x, int index) {
  return static_cast<uint64_t>(KeyOf(x)) << 32 | (0xFFFFFFFFu - static_cast<uint32_t>(index));
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

// One workgroup per row.
template <typename T>
__global__ __launch_bounds__(kDrawThreads) void DrawKernel(SampleArgs a, Layout l) {
  const int row = blockIdx.x, tid = threadIdx.x;
  const Work w(a, l, row);
  const Row r = RowOf(a, l, w, row);
  if (r.greedy || r.max == kNone) {
    if (tid == 0) {
      a.tokens[row] = r.max == kNone ? -1 : r.best;
      if (a.logprobs != nullptr) a.logprobs[row] = r.max == kNone ? kNone : 0.0f;
    }
    return;
  }
  __shared__ double pow2[32];
  __shared__ float lx[kList];
  __shared__ int li[kList];
  __shared__ uint64_t lq[kList];
  __shared__ unsigned long long slice_weight[kMaxSlices];
  __shared__ uint64_t s_kept;
  LoadPow2(pow2);
  const char* x = a.logits + row * a.row_bytes;
  Cut cut{kBins, kBins, 0, 0, 0, 0, false};
  if (r.k != 0 || r.p != 0.0) cut = FindCut<kDrawThreads>(r, w.bins);
  const int end_bin = cut.End();
  const uint32_t n = end_bin < kBins && !cut.unclear ? *w.count : 0;
  const bool slow = cut.unclear || n > kList;
  if (tid < l.slices) slice_weight[tid] = slow ? 0 : w.weights[tid];
  if (tid == 0) s_kept = 0;
  __syncthreads();
  uint64_t last = 0;  // rank key of the last token before the limits of weight; 0: every token
  if (slow) {
    uint64_t taken = cut.all;
    if (r.k != 0) last = CutByDigits<T>(a, r, x, pow2, r.k, -1.0, &taken);
    if (r.p != 0.0) {
      const uint64_t by_p = CutByDigits<T>(a, r, x, pow2, 0, r.p * static_cast<double>(taken), &taken);
      last = max(last, by_p);
    }
    for (int s = 0; s < l.slices; ++s) {
      uint64_t sum = 0, all;
      for (int i = s * l.length + tid; i < min(a.vocab, (s + 1) * l.length); i += kDrawThreads) {
        const float v = One<T>(x, i);
        const double f = r.Weight(v, pow2);
        if (RankKey(v, i) >= last && f >= r.floor) sum += Row::Units(f);
      }
      Before<kDrawThreads>(sum, &all);
      if (tid == 0) slice_weight[s] = all;
    }
  } else if (n > 0) {
    float v = 0.0f;
    int index = 0, bin = -1;
    uint64_t q = 0;
    double f = 0.0;
    if (tid < static_cast<int>(n)) {
      v = w.list[tid].x, index = w.list[tid].index;
      f = r.Weight(v, pow2);
      q = Row::Units(f);
      bin = r.Bin(v);
      lx[tid] = v, li[tid] = index, lq[tid] = q;
    }
    __syncthreads();
    // rank and weight above within the step
    uint32_t rank = 0;
    uint64_t above = 0;
    if (tid < static_cast<int>(n)) {
      const int other = bin == cut.k_bin ? cut.p_bin : cut.k_bin;
      for (int j = 0; j < static_cast<int>(n); ++j) {
        const float y = lx[j];
        const bool better = y > v || (y == v && li[j] < index);
        if (better && (cut.k_bin == cut.p_bin || other == kBins || r.Bin(y) == bin)) ++rank, above += lq[j];
      }
    }
    bool in = bin >= 0 && bin == end_bin;
    uint64_t taken = cut.all;
    if (cut.k_bin < kBins) {
      const bool in_k = bin == cut.k_bin && rank < cut.k_left;
      if (in_k) atomicAdd(reinterpret_cast<unsigned long long*>(&s_kept), static_cast<unsigned long long>(q));
      __syncthreads();
      taken = cut.k_before + s_kept;
      if (bin == cut.k_bin) in = in && in_k;
    }
    if (cut.p_bin < kBins && bin == cut.p_bin)
      in = in && static_cast<double>(cut.p_before + above) < r.p * static_cast<double>(taken);
    if (in && f >= r.floor) atomicAdd(&slice_weight[index / l.length], static_cast<unsigned long long>(q));
    // the kept token with the smallest key
    uint64_t key = in ? RankKey(v, index) : ~0ull;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) key = min(key, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(key), o, 64)));
    __shared__ uint64_t keys[kDrawThreads / 64];
    if ((tid & 63) == 0) keys[tid >> 6] = key;
    __syncthreads();
    last = keys[0];
    for (int i = 1; i < kDrawThreads / 64; ++i) last = min(last, keys[i]);
  }
  __syncthreads();
  // The slice, then the token in it.
  __shared__ int s_slice;
  __shared__ uint64_t s_before, s_total;
  const double u = fmax(0.0, fmin(static_cast<double>(a.u[row]), 1.0));
  if (tid < 64) {
    const uint64_t mine = tid < l.slices ? slice_weight[tid] : 0;
    uint64_t up_to = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t y = __shfl_up(static_cast<unsigned long long>(up_to), o, 64);
      if (tid >= o) up_to += y;
    }
    const uint64_t total = __shfl(static_cast<unsigned long long>(up_to), 63, 64);
    uint64_t hit = __ballot(mine != 0 && static_cast<double>(up_to) > u * static_cast<double>(total));
    if (hit == 0) hit = 1ull << (63 - __clzll(static_cast<long long>(__ballot(mine != 0))));  // u = 1: the last one
    const int s = __ffsll(static_cast<unsigned long long>(hit)) - 1;
    if (tid == s) s_slice = s, s_before = up_to - mine, s_total = total;
  }
  __syncthreads();
  const int slice = s_slice;
  const uint64_t total = s_total;
  const int each = l.length / kDrawThreads;
  const int from = slice * l.length + tid * each, to = min(from + each, a.vocab);
  auto kept = [&](int i, double* f) {
    const float v = One<T>(x, i);
    *f = r.Weight(v, pow2);
    return RankKey(v, i) >= last && *f >= r.floor ? Row::Units(*f) : 0;
  };
  uint64_t sum = 0, all;
  double f;
  for (int i = from; i < to; ++i) sum += kept(i, &f);
  uint64_t before = s_before + Before<kDrawThreads>(sum, &all);
  const double mark = u * static_cast<double>(total);
  // the first thread whose sum passes the mark (or the last with a weight)
  const bool past = sum != 0 && (static_cast<double>(before + sum) > mark || before + sum == s_before + all);
  const bool first = past && !(static_cast<double>(before) > mark);
  if (first) {
    int token = -1;
    double at = 0.0;
    for (int i = from; i < to; ++i) {
      const uint64_t q = kept(i, &f);
      if (q == 0) continue;
      before += q;
      token = i, at = f;
      if (static_cast<double>(before) > mark) break;
    }
    a.tokens[row] = token;
    if (a.logprobs != nullptr) a.logprobs[row] = static_cast<float>(log(at / static_cast<double>(total)));
  }
}

template <typename T>
void Launch(const SampleArgs& a, hipStream_t s) {
  const Layout l = LayoutOf(a.rows, a.vocab);
  const dim3 grid(l.slices, a.rows);
  MaxKernel<T><<<grid, kThreads, 0, s>>>(a, l);
  CountKernel<T><<<grid, kThreads, 0, s>>>(a, l);
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

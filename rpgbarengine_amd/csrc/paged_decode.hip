// Attention of one new token per sequence over its cache pages
// (rpg_hip_paged_decode, include/rpg_hip.h):
//   out[h] = sum_j p_j v_j,  p = softmax over j < len of scale q[h] . k_j.
//
// One pass over the keys with a running maximum, sum and output. Workgroup
// (sequence, key head, 16 query heads of its group, key range); its four waves
// take the range's key tiles in turn and join their states in LDS at the end.
// Scores and outputs are formed transposed on the matrix cores, S^T = K Q^T
// and O^T = V^T P^T (16 x 16 tiles, columns = query heads), so that a lane
// keeps to one query head: its scores are the B operand of the second product
// as they stand, and maximum, sum and rescaling are per lane. The key index of
// a product is free, so V is taken in the order the scores come in: a lane
// reads 16 bytes of each of its keys' rows (whole rows per load instruction)
// and for the 16-bit types pairs up its keys' values with one v_perm_b32 per
// operand register. K and V go from HBM to registers, LDS is not used on the
// way.
//
// Bound: the K and V bytes, each read once (16 columns are computed for any
// group size: at 8 heads f32 the products would take 1/2 of the time the bytes
// do, the 16-bit types' 1/10). Measured, 32 heads on 8 of 128: 64 sequences of
// 201 to 11167 positions, bf16, 861 MB in 172 us (the rate of a large copy:
// 171); one of 131000, f16, 537 MB in 95 us (107); 8 of about 1073, f32, 70 MB in 18.5
// us (14, and two launches); one of 95, f16: 7.2 us, the call itself (5.4 in a captured
// graph). Ranges: see DecodeSplits.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "lanes.h"
#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {
namespace {

constexpr int kWaves = 4;
constexpr int kCols = 16;  // query heads of a workgroup
// A wave's keys of one step, as 16-key halves (two, in f32 one): K as A operands
// (lane: 16 bytes of key l % 16 per 64 bytes of a row), V as the lane's
// dimensions of keys 4 (l / 16) + r.
template <typename T, int kDim>
struct Tile {
  static constexpr int kHalves = 4 / kBytes<T>;
  static constexpr int kKeys = 16 * kHalves;
  static constexpr int kChunks = kDim * kBytes<T> / 64;  // K: 16-byte pieces; V: dwords per key
  U4 k[kHalves][kChunks];
  uint32_t v[kHalves][4][kChunks];
  bool ok[kHalves];  // its page is there

  // Rows of positions pos .. of the sequence whose last one is `last`; those
  // past it and those of unnamed pages are read from rows that are there.
  __device__ __forceinline__ void Load(const Cache& c, const int32_t* table, int64_t head_off, int pos, int last,
                                       int lane) {
    const int in_page = (1 << c.page_log2) - 1, l16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int p0 = min(pos + 16 * h, last & ~15);
      const int page = PageAt(c, table, p0);
      ok[h] = page >= 0;
      const int64_t at = max(page, 0) * c.page_bytes + head_off + (p0 & in_page) * static_cast<int64_t>(c.row_bytes);
      const char* kb = c.k + at;
      const char* vb = c.v + at;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) k[h][i] = Load16(kb + static_cast<uint32_t>(l16 * c.row_bytes + 64 * i + 16 * g));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const char* row = vb + static_cast<uint32_t>((4 * g + r) * c.row_bytes);
        if constexpr (kChunks == 2) {
          const U2 x = *(const __attribute__((address_space(1))) U2*)(row + 8 * l16);
          v[h][r][0] = x[0], v[h][r][1] = x[1];
        } else {
#pragma unroll
          for (int w = 0; w < kChunks; w += 4) {
            const U4 x = Load16(row + 64 * w + 16 * l16);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[h][r][w + e] = x[e];
          }
        }
      }
    }
  }
};

// The dimension of row m of output block w.
template <typename T, int kDim>
__device__ __forceinline__ int DimOf(int w, int m) {
  if constexpr (kBytes<T> == 4) return 64 * (w / 4) + 4 * m + w % 4;
  return (kDim / 16) * m + w;
}

// Weights are held times 2^kLift, their sums too. f16 has steps of 2^-24 at the
// least: without it, keys whose weight is below 2^-25 of the largest would count
// in the sum and not in the output, and a long cache has many of those.
template <typename T>
constexpr float kLift = __is_same(T, F16) ? 15.0f : 0.0f;

// A query head's running state in a lane: maximum (of scale log2(e) q.k) and
// the output of its column, alike over the lanes of a column; the sum of the
// lane's own keys. 16-bit types: the weights go to the products in two parts, each
// of 8 or 11 bits, and the second parts' products have a sum of their own, `rest`,
// so that a weight which is its first part alone makes no NaN of an infinite value
// (0 x inf). With one part the output is 1.1 to 1.3 times as far from exact as its
// own rounding leaves it; two take hardly longer, for the bytes are what takes the
// time (64 ragged bf16 172 us either way, 131000 f16 95, 8 x 1000 f16 12.6 and 12.8).
template <typename T, int kDim>
struct State {
  static constexpr int kBlocks = kDim / 16, kRest = kBytes<T> == 4 ? 0 : kBlocks;
  float m = kNegInf, l = 0.0f;
  F4 o[kBlocks] = {}, rest[kRest ? kRest : 1] = {};

  // The output, not yet divided by the sum. Where a value that is not finite came
  // in, the first parts' sum says what comes out.
  __device__ __forceinline__ float Out(int w, int e) const {
    if constexpr (kRest == 0) return o[w][e];
    const float x = o[w][e];
    return __builtin_isfinite(x) ? x + rest[w][e] : x;
  }

  // Adds a tile whose first position is pos.
  __device__ __forceinline__ void Add(Tile<T, kDim>& t, const U4 (&q)[Tile<T, kDim>::kChunks], float c, int pos,
                                      int last, int lane) {
    using Tl = Tile<T, kDim>;
    const int g = lane >> 4;
    F4 s[Tl::kHalves];
#pragma unroll
    for (int h = 0; h < Tl::kHalves; ++h) {
      F4 x = {};
#pragma unroll
      for (int i = 0; i < Tl::kChunks; ++i) {
        if constexpr (kBytes<T> == 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x = Mfma16F32(__uint_as_float(t.k[h][i][e]), __uint_as_float(q[i][e]), x);
        } else {
          x = Mfma16<T>(t.k[h][i], q[i], x);
        }
      }
      s[h] = x * c;
    }
    bool whole = pos + Tl::kKeys - 1 <= last;
#pragma unroll
    for (int h = 0; h < Tl::kHalves; ++h) whole = whole && t.ok[h];
    if (!whole) {
      // Masked keys: no weight, and nothing of what their rows hold (which may
      // be anything, NaN among it) reaches the second product.
#pragma unroll
      for (int h = 0; h < Tl::kHalves; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = t.ok[h] && pos + 16 * h + 4 * g + r <= last;
          s[h][r] = in ? s[h][r] : kNegInf;
#pragma unroll
          for (int w = 0; w < Tl::kChunks; ++w) t.v[h][r][w] = in ? t.v[h][r][w] : 0u;
        }
    }
    float top = kNegInf;
#pragma unroll
    for (int h = 0; h < Tl::kHalves; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[h][r]);
    top = lanes::MaxXor32(lanes::MaxXor16(top));
    if (__any(top > m)) {
      const float now = fmaxf(m, top), f = __builtin_amdgcn_exp2f(MaxDiff(m, now));
      m = now;
      l *= f;
#pragma unroll
      for (int w = 0; w < kBlocks; ++w) o[w] *= f;
#pragma unroll
      for (int w = 0; w < kRest; ++w) rest[w] *= f;
    }
    const float base = m == kNegInf ? 0.0f : m - kLift<T>;
#pragma unroll
    for (int h = 0; h < Tl::kHalves; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[h][r] = __builtin_amdgcn_exp2f(s[h][r] - base);
        l += s[h][r];
      }
    if constexpr (kBytes<T> == 4) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int w = 0; w < kDim / 16; ++w) o[w] = Mfma16F32(__uint_as_float(t.v[0][r][w]), s[0][r], o[w]);
    } else {
      // (the sum takes the weights unrounded)
      const U4 p = {Pack2<T>(s[0][0], s[0][1]), Pack2<T>(s[0][2], s[0][3]), Pack2<T>(s[1][0], s[1][1]),
                    Pack2<T>(s[1][2], s[1][3])};
      const U4 p2 = {Rest2<T>(s[0][0], s[0][1], p[0]), Rest2<T>(s[0][2], s[0][3], p[1]),
                     Rest2<T>(s[1][0], s[1][1], p[2]), Rest2<T>(s[1][2], s[1][3], p[3])};
#pragma unroll
      for (int w = 0; w < kDim / 16; ++w) {
        const uint32_t sel = w % 2 ? 0x07060302u : 0x05040100u;
        U4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          a[j] = __builtin_amdgcn_perm(t.v[j / 2][2 * (j % 2) + 1][w / 2], t.v[j / 2][2 * (j % 2)][w / 2], sel);
        o[w] = Mfma16<T>(a, p, o[w]);
        rest[w] = Mfma16<T>(a, p2, rest[w]);
      }
    }
  }
};

// grid (sequence x key head x block of 16 query heads, key range). Four waves to a
// SIMD unit for 16-bit rows of 64, by 128 registers; the compiler alone takes 134
// (64 x 4000 bf16 99 us, 96 so).
template <typename T, int kDim>
__global__ __launch_bounds__(64 * kWaves, kDim == 64 && kBytes<T> == 2 ? 4 : 2) void DecodeKernel(AttentionArgs a) {
  using Tl = Tile<T, kDim>;
  __shared__ float sm[kWaves][kCols], sl[kWaves][kCols];
  __shared__ __align__(16) float so[kWaves][kCols][kDim + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.n_heads / a.c.n_kv, blocks = (group + kCols - 1) / kCols;
  const int hb = blockIdx.x % blocks, kh = blockIdx.x / blocks % a.c.n_kv, seq = blockIdx.x / blocks / a.c.n_kv;
  const int h0 = kh * group + hb * kCols, n_cols = min(kCols, group - hb * kCols);
  const int len = Length(a.s, seq);
  const int range = RangeOf(max(len, 1), a.splits), start = blockIdx.y * range, end = min(len, start + range);
  if (start >= end && blockIdx.y > 0) return;
  State<T, kDim> st;
  if (start < end) {
    const int32_t* table = a.s.table + seq * a.s.table_stride;
    const int64_t head_off = kh * a.c.head_bytes;
    const int col = min(lane & 15, n_cols - 1);
    const char* qp = a.q.p + seq * a.q.token_bytes + (h0 + col) * a.q.head_bytes + 16 * (lane >> 4);
    U4 q[Tl::kChunks];
#pragma unroll
    for (int i = 0; i < Tl::kChunks; ++i) q[i] = Load16(qp + 64 * i);
    const float c = a.scale * 1.44269504088896341f;
    int pos = start + wave * Tl::kKeys;
    Tl now, next;
    if (pos < end) now.Load(a.c, table, head_off, pos, end - 1, lane);
    for (; pos < end; pos += kWaves * Tl::kKeys) {
      next.Load(a.c, table, head_off, pos + kWaves * Tl::kKeys, end - 1, lane);
      st.Add(now, q, c, pos, end - 1, lane);
      now = next;
    }
  }
  st.l = lanes::AddXor32(lanes::AddXor16(st.l));
  const int col = lane & 15, g = lane >> 4;
  if (lane < kCols) sm[wave][lane] = st.m, sl[wave][lane] = st.l;
  __syncthreads();
  float top = sm[0][col];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sm[w][col]);
  const float f = __builtin_amdgcn_exp2f(MaxDiff(st.m, top));
  if (col < n_cols) {
#pragma unroll
    for (int w = 0; w < kDim / 16; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) so[wave][col][DimOf<T, kDim>(w, 4 * g + e)] = st.Out(w, e) * f;
  }
  __syncthreads();
  const bool alone = range >= len;
  const int64_t rows = static_cast<int64_t>(a.s.n_seqs) * a.n_heads;
  for (int i = tid; i < n_cols * (kDim / 4); i += 64 * kWaves) {
    const int h = i / (kDim / 4), d = i % (kDim / 4) * 4;
    float m = sm[0][h], l = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, sm[w][h]);
    F4 o = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      l += sl[w][h] * __builtin_amdgcn_exp2f(MaxDiff(sm[w][h], m));
      o += *reinterpret_cast<const F4*>(&so[w][h][d]);
    }
    if (alone) {
      o *= Inverse(m, l);
      Store4<T>(a.out.p + seq * a.out.token_bytes + (h0 + h) * a.out.head_bytes + d * kBytes<T>, o);
    } else {
      const int64_t row = static_cast<int64_t>(seq) * a.n_heads + h0 + h;
      if (d == 0) PartStats(a, row)[blockIdx.y] = F2{m, l};
      *reinterpret_cast<F4*>(PartOut<kDim>(a, rows, row) + static_cast<int64_t>(blockIdx.y) * kDim + d) = o;
    }
  }
}

template <typename T, int kDim>
__global__ __launch_bounds__(256) void DecodeJoinKernel(AttentionArgs a) {
  const int64_t row = blockIdx.x;
  const int seq = static_cast<int>(row / a.n_heads), head = static_cast<int>(row % a.n_heads);
  const int len = Length(a.s, seq), range = RangeOf(max(len, 1), a.splits);
  if (range >= len) return;  // written by its one range
  JoinRow<T, kDim>(a, static_cast<int64_t>(a.s.n_seqs) * a.n_heads, row, (len + range - 1) / range,
                   a.out.p + seq * a.out.token_bytes + head * a.out.head_bytes);
}

template <typename T, int kDim>
void Launch(const AttentionArgs& a, hipStream_t s) {
  const int group = a.n_heads / a.c.n_kv;
  const int64_t x = static_cast<int64_t>(a.s.n_seqs) * a.c.n_kv * CeilDiv(group, kCols);
  RPG_CHECK(static_cast<int64_t>(a.s.n_seqs) * a.n_heads <= kMaxGroups, "%d x %d query rows in one launch", a.s.n_seqs,
            a.n_heads);
  DecodeKernel<T, kDim><<<dim3(static_cast<uint32_t>(x), a.splits), 64 * kWaves, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
  if (a.splits == 1) return;
  DecodeJoinKernel<T, kDim><<<static_cast<uint32_t>(a.s.n_seqs) * a.n_heads, 256, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
}

template <typename T>
void LaunchDim(const AttentionArgs& a, hipStream_t s) {
  if (a.c.head_dim == 128)
    Launch<T, 128>(a, s);
  else
    Launch<T, 64>(a, s);
}

}  // namespace

// Ranges for a workgroup per compute unit and none with two (9 x 1000 f32: 27.0 us
// with 288 workgroups, 20.0 with 216; 11 x 4000 bf16 51 with 264, 39 with 176), and
// of 2048 positions at most, so that the longest sequence of a ragged batch does not
// end alone: 64 of 200 to 12000 take 152 us, 162 with 1024. Aiming higher only adds
// joins: 32 x 2000 bf16 48.2 us aiming at 256, 52.1 at 512, 53.5 at 1024; 8 x 1088 f32
// 18.7, 22.1, 21.1. Rows of a few steps stay whole, a join takes as long: one of 200
// bf16 12.0 us in ranges, 7.6 whole, 500 11.7 and 8.4, 700 11.9 and 10.3; f32 200 11.7
// and 10.1, 400 11.6 and 13.7. The rule knows the sequences' capacity, not their
// lengths, which are on the device: ranges behind a sequence's end return at once.
// So a table wider than its sequences costs the join's launch: one of 95 positions
// f16 7.8 us a call in a table of its own width, 11.7 in one for 4096 or for 131072
// (5.3 and 6.7 in a captured graph), one of 300 8.3 and 11.8 (8.0 and 8.4).
int DecodeSplits(int64_t n_seqs, int n_heads, int n_kv, int bytes, int64_t capacity) {
  if (capacity * bytes <= 1280) return 1;
  const int64_t base = std::max<int64_t>(1, n_seqs * n_kv * CeilDiv(n_heads / n_kv, kCols));
  const int64_t want = std::max(256 / base, CeilDiv(capacity, 2048));
  return static_cast<int>(std::max<int64_t>(1, std::min({want, CeilDiv(capacity, kRangeUnit), int64_t{kMaxSplits}})));
}

int64_t WorkBytes(int64_t rows, int head_dim, int splits) {
  return splits == 1 ? 0 : (StatFloats(rows, splits) + rows * splits * head_dim) * 4;
}

void Decode(const AttentionArgs& a, hipStream_t s) {
  if (a.s.n_seqs == 0) return;
  if (a.c.type == kF32)
    LaunchDim<F32>(a, s);
  else if (a.c.type == kF16)
    LaunchDim<F16>(a, s);
  else
    LaunchDim<BF16>(a, s);
}

}  // namespace paged
}  // namespace rpg

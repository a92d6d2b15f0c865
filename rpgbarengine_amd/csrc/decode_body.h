// What the kernels of paged_decode.hip, paged_shared.hip and codes_decode.hip have in
// common: attention of one token per sequence, a workgroup for 16 query heads of
// a key head and a range of keys. The method is described in paged_decode.hip.
#pragma once

#include <hip/hip_runtime.h>

#include "lanes.h"
#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {

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

// Weights are held times 2^kDecodeLift, their sums too. f16 has steps of 2^-24 at the
// least: without it, keys whose weight is below 2^-25 of the largest would count
// in the sum and not in the output, and a long cache has many of those.
template <typename T>
constexpr float kDecodeLift = __is_same(T, F16) ? 15.0f : 0.0f;

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
  struct Query {
    U4 x[Tile<T, kDim>::kChunks];
  };
  float m = kNegInf, l = 0.0f;
  F4 o[kBlocks] = {}, rest[kRest ? kRest : 1] = {};

  // The dimension of row m of output block w.
  static __device__ __forceinline__ int DimOf(int w, int m) {
    if constexpr (kBytes<T> == 4) return 64 * (w / 4) + 4 * m + w % 4;
    return (kDim / 16) * m + w;
  }

  // The output, not yet divided by the sum. Where a value that is not finite came
  // in, the first parts' sum says what comes out.
  __device__ __forceinline__ float Out(int w, int e) const {
    if constexpr (kRest == 0) return o[w][e];
    const float x = o[w][e];
    return __builtin_isfinite(x) ? x + rest[w][e] : x;
  }

  // Adds a tile whose first position is pos.
  __device__ __forceinline__ void Add(Tile<T, kDim>& t, const Query& query, float c, int pos, int last, int lane) {
    using Tl = Tile<T, kDim>;
    const int g = lane >> 4;
    const auto& q = query.x;
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
    const float base = m == kNegInf ? 0.0f : m - kDecodeLift<T>;
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

template <int kDim>
struct DecodeLds {
  float so[kWaves][kCols][kDim + 4];
  float sm[kWaves][kCols], sl[kWaves][kCols];
};

struct ColumnPlace {
  int token, head;
};
// Tiles of the range are brought by load(tile, pos), the queries by load_q(q, place(column)),
// and added up in a State; the waves' states are joined in LDS. place(column): the token
// and query head of a column. T: of the rows.
template <typename T, int kDim, typename Tl, typename St, typename Load, typename LoadQ, typename Place>
__device__ __forceinline__ void DecodeBody(const AttentionArgs& a, DecodeLds<kDim>& shared, int n_cols, DecodeRange range,
                                           Load&& load, LoadQ&& load_q, Place&& place) {
  auto& sm = shared.sm;
  auto& sl = shared.sl;
  auto& so = shared.so;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  St st;
  if (range.start < range.end) {
    typename St::Query q;
    load_q(q, place(min(lane & 15, n_cols - 1)));
    const float c = a.scale * 1.44269504088896341f;
    int pos = range.start + wave * Tl::kKeys;
    Tl now, next;
    if (pos < range.end) load(now, pos);
    for (; pos < range.end; pos += kWaves * Tl::kKeys) {
      load(next, pos + kWaves * Tl::kKeys);
      st.Add(now, q, c, pos, range.end - 1, lane);
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
      for (int e = 0; e < 4; ++e) so[wave][col][St::DimOf(w, 4 * g + e)] = st.Out(w, e) * f;
  }
  __syncthreads();
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
    const ColumnPlace at = place(h);
    if (range.alone) {
      o *= Inverse(m, l);
      Store4<T>(a.out.p + at.token * a.out.token_bytes + at.head * a.out.head_bytes + d * kBytes<T>, o);
    } else {
      const int64_t row = static_cast<int64_t>(at.token) * a.n_heads + at.head;
      if (d == 0) PartStats(a, row)[range.slot] = F2{m - range.off, l};
      *reinterpret_cast<F4*>(PartOut<kDim>(a, rows, row) + static_cast<int64_t>(range.slot) * kDim + d) = o;
    }
  }
}

// The workgroup's sequence, key head and query heads: bx counts sequence x key head x
// block of 16 query heads.
struct DecodePlace {
  int seq, kh, h0, n_cols;
  __device__ __forceinline__ ColumnPlace operator()(int column) const { return {seq, h0 + column}; }
};
__device__ __forceinline__ DecodePlace PlaceOf(const AttentionArgs& a, int bx) {
  const int group = a.n_heads / a.c.n_kv, blocks = (group + kCols - 1) / kCols;
  const int hb = bx % blocks, kh = bx / blocks % a.c.n_kv, seq = bx / blocks / a.c.n_kv;
  return {seq, kh, kh * group + hb * kCols, min(kCols, group - hb * kCols)};
}

// Range `y` of all of a sequence's positions; false: there is no such range.
__device__ __forceinline__ bool WholeRange(const AttentionArgs& a, int seq, int y, DecodeRange* out) {
  const int len = Length(a.s, seq);
  const int range = RangeOf(a, max(len, 1), a.splits), start = y * range;
  *out = {start, min(len, start + range), range >= len, y, 0.0f};
  return out->start < out->end || y == 0;
}

// The workgroup's range over a cache of rows, pages by the table of sequence `seq`.
template <typename T, int kDim, typename Place>
__device__ __forceinline__ void DecodeRows(const AttentionArgs& a, DecodeLds<kDim>& shared, int seq, int kh, int n_cols,
                                           DecodeRange range, Place&& place) {
  using Tl = Tile<T, kDim>;
  using St = State<T, kDim>;
  const int lane = threadIdx.x & 63;
  const int32_t* table = a.s.table + seq * a.s.table_stride;
  const int64_t head_off = kh * a.c.head_bytes;
  DecodeBody<T, kDim, Tl, St>(
      a, shared, n_cols, range, [&](Tl& t, int pos) { t.Load(a.c, table, head_off, pos, range.end - 1, lane); },
      [&](typename St::Query& q, ColumnPlace at) {
        const char* qp = a.q.p + at.token * a.q.token_bytes + at.head * a.q.head_bytes + 16 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < Tl::kChunks; ++i) q.x[i] = Load16(qp + 64 * i);
      },
      place);
}

}  // namespace paged
}  // namespace rpg

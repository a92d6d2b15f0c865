// What the kernels of codes_decode.hip and codes_shared.hip have in common: decode
// attention over a cache of 8-bit codes. The method is described in codes_decode.hip.
#pragma once

#include <hip/hip_runtime.h>

#include "codes_dev.h"
#include "decode_body.h"
#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {

// A wave's keys of one step, as two halves of 16: K as 16 codes of key l % 16 per 64
// dimensions, V as the lane's dimensions (kDim / 16) (l % 16) .. of keys 4 (l / 16) + r;
// of key 4 (l / 16) + l % 4 the scales.
template <int kDim>
struct CodesTile {
  static constexpr int kKeys = 32;
  static constexpr int kChunks = kDim / 64;  // K: 16-byte pieces; V: dwords per key
  U4 k[2][kChunks];
  uint32_t v[2][4][kChunks];
  float ks[2], vs[2];
  bool ok[2];  // its page is there

  // Rows of positions pos .. of the sequence whose last one is `last`; those
  // past it and those of unnamed pages are read from rows that are there.
  __device__ __forceinline__ void Load(const Cache& c, const Scales& sc, const int32_t* table, int kh, int pos, int last,
                                       int lane) {
    const int in_page = (1 << c.page_log2) - 1, l16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int p0 = min(pos + 16 * h, last & ~15);
      const int page = PageAt(c, table, p0);
      ok[h] = page >= 0;
      const int64_t at = max(page, 0) * c.page_bytes + kh * c.head_bytes + (p0 & in_page) * static_cast<int64_t>(c.row_bytes);
      const int64_t scale_at = max(page, 0) * sc.page_bytes + kh * sc.head_bytes + 4 * (p0 & in_page);
      const char* kb = c.k + at;
      const char* vb = c.v + at;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) k[h][i] = Load16(kb + static_cast<uint32_t>(l16 * c.row_bytes + 64 * i + 16 * g));
      ks[h] = *(const __attribute__((address_space(1))) float*)(sc.k + scale_at + 16 * g + 4 * (lane & 3));
      vs[h] = *(const __attribute__((address_space(1))) float*)(sc.v + scale_at + 16 * g + 4 * (lane & 3));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const char* row = vb + static_cast<uint32_t>((4 * g + r) * c.row_bytes);
        if constexpr (kChunks == 2) {
          const U2 x = *(const __attribute__((address_space(1))) U2*)(row + 8 * l16);
          v[h][r][0] = x[0], v[h][r][1] = x[1];
        } else {
          v[h][r][0] = *(const __attribute__((address_space(1))) uint32_t*)(row + 4 * l16);
        }
      }
    }
  }
};

// A query head's running state in a lane, as paged_decode.hip has it. The products
// of the weights' parts share a sum: codes are finite, and a scale that is not
// (a row that was not finite) makes NaN of all parts.
template <typename C, typename T, int kDim>
struct CodesState {
  using Tl = CodesTile<kDim>;
  using K = KeyType<T>;
  static constexpr int kBlocks = kDim / 16, kQ = kDim / 32;  // products over a query row
  struct Query {
    U4 x[kQueryParts<T>][kQ];  // dimensions 64 (i / 2) + 16 (l / 16) + 8 (i % 2) ..
  };
  float m = kNegInf, l = 0.0f;
  F4 o[kBlocks] = {};

  static __device__ __forceinline__ int DimOf(int w, int m) { return (kDim / 16) * m + w; }
  __device__ __forceinline__ float Out(int w, int e) const { return o[w][e]; }

  // Adds a tile whose first position is pos.
  __device__ __forceinline__ void Add(Tl& t, const Query& q, float c, int pos, int last, int lane) {
    const int g = lane >> 4;
    F4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      F4 x = {};
#pragma unroll
      for (int i = 0; i < kQ; ++i) {
        const U4 a = Operand8<C, K>(t.k[h][i / 2][i % 2 * 2], t.k[h][i / 2][i % 2 * 2 + 1]);
#pragma unroll
        for (int p = kQueryParts<T> - 1; p >= 0; --p) x = Mfma16<K>(a, q.x[p][i], x);
      }
      s[h] = x;
      ScaleBy<0, 4>(s[h], t.ks[h] * c);
    }
    const bool masked = !(pos + Tl::kKeys - 1 <= last && t.ok[0] && t.ok[1]);
    if (masked) {
      // Masked keys: no weight, and nothing of what their rows hold (which may
      // be anything, NaN among it) reaches the second product.
#pragma unroll
      for (int h = 0; h < 2; ++h)
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
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[h][r]);
    top = lanes::MaxXor32(lanes::MaxXor16(top));
    if (__any(top > m)) {
      const float now = fmaxf(m, top), f = __builtin_amdgcn_exp2f(MaxDiff(m, now));
      m = now;
      l *= f;
#pragma unroll
      for (int w = 0; w < kBlocks; ++w) o[w] *= f;
    }
    const float base = m == kNegInf ? 0.0f : m;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[h][r] = __builtin_amdgcn_exp2f(s[h][r] - base);
        l += s[h][r];  // (the sum takes the weights unrounded)
      }
    if (masked) {  // 0 x NaN must not reach the product
#pragma unroll
      for (int h = 0; h < 2; ++h) t.vs[h] = t.ok[h] && pos + 16 * h + 4 * g + (lane & 3) <= last ? t.vs[h] : 0.0f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) ScaleBy<0, 4>(s[h], t.vs[h]);
    WeightParts<kWeightParts<T>> p;
#pragma unroll
    for (int j = 0; j < 4; ++j) p.Set(j, s[j / 2][2 * (j % 2)], s[j / 2][2 * (j % 2) + 1]);
#pragma unroll
    for (int w = 0; w < kBlocks; w += 4) {
      // bytes of two keys side by side, then as pairs of bf16
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = t.v[j / 2][2 * (j % 2)][w / 4], y = t.v[j / 2][2 * (j % 2) + 1][w / 4];
        lo[j] = __builtin_amdgcn_perm(y, x, 0x05010400u);
        hi[j] = __builtin_amdgcn_perm(y, x, 0x07030602u);
      }
      U4 a[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a[0][j] = Halves2<C, BF16, false>(lo[j]);
        a[1][j] = Halves2<C, BF16, true>(lo[j]);
        a[2][j] = Halves2<C, BF16, false>(hi[j]);
        a[3][j] = Halves2<C, BF16, true>(hi[j]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = kWeightParts<T> - 1; i >= 0; --i) o[w + e] = Mfma16<BF16>(a[e], p.x[i], o[w + e]);
    }
  }
};

// The workgroup's range over a cache of codes, pages by the table of sequence `seq`.
template <typename C, typename T, int kDim, typename Place>
__device__ __forceinline__ void DecodeCodeRows(const CodesAttentionArgs& args, DecodeLds<kDim>& shared, int seq, int kh,
                                               int n_cols, DecodeRange range, Place&& place) {
  using Tl = CodesTile<kDim>;
  using St = CodesState<C, T, kDim>;
  const AttentionArgs& a = args.a;
  const int lane = threadIdx.x & 63;
  const int32_t* table = a.s.table + seq * a.s.table_stride;
  DecodeBody<T, kDim, Tl, St>(
      a, shared, n_cols, range,
      [&](Tl& t, int pos) { t.Load(a.c, args.scales, table, kh, pos, range.end - 1, lane); },
      [&](typename St::Query& q, ColumnPlace at) {
        const char* qp = a.q.p + at.token * a.q.token_bytes + at.head * a.q.head_bytes + 16 * (lane >> 4) * kBytes<T>;
#pragma unroll
        for (int i = 0; i < St::kQ; ++i) LoadQuery<T>(qp + (64 * (i / 2) + 8 * (i % 2)) * kBytes<T>, i, q.x);
      },
      place);
}

}  // namespace paged
}  // namespace rpg

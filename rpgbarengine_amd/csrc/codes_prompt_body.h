// What the kernels of codes_prompt.hip and codes_shared.hip have in common: attention of
// a tile of query rows over a range of a cache of 8-bit codes. The method is
// described in codes_prompt.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "codes_dev.h"
#include "groups.h"
#include "lanes.h"
#include "paged.h"
#include "paged_dev.h"
#include "prompt_body.h"
#include "row_tile.h"

namespace rpg {
namespace paged {

constexpr int kSoloRows = 32;  // query rows of a tile
constexpr int kSoloKeys = 32;  // keys of a wave's step

// A block of 32 keys in a wave: K as 16 codes of key l % 32 per 32 dimensions, V as
// the lane's dimensions (kDim / 32) (l % 32) .. of the keys that its scores come in,
// 8 (e / 4) + 4 (l / 32) + e % 4; the scales of the key that element l % 16 belongs to.
template <int kDim>
struct Block {
  static constexpr int kChunks = kDim / 32;
  U4 k[kChunks];
  uint32_t v[16];
  float ks, vs;
  bool ok[2];  // the page of either 16 positions is there

  // Positions pos .. of a sequence whose last is `last`; those past it and those of
  // unnamed pages are read from rows that are there.
  __device__ __forceinline__ void Load(const Cache& c, const Scales& sc, const int32_t* table, int kh, int pos, int last,
                                       int lane) {
    const int in_page = (1 << c.page_log2) - 1, l32 = lane & 31, h = lane >> 5;
    const char* kb[2];
    const char* vb[2];
    int64_t sb[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int p0 = min(pos + 16 * u, last & ~15);
      const int page = PageAt(c, table, p0);
      ok[u] = page >= 0;
      const int64_t at = max(page, 0) * c.page_bytes + kh * c.head_bytes + (p0 & in_page) * static_cast<int64_t>(c.row_bytes);
      kb[u] = c.k + at;
      vb[u] = c.v + at;
      sb[u] = max(page, 0) * sc.page_bytes + kh * sc.head_bytes + 4 * (p0 & in_page);
    }
    const int u = l32 >> 4;  // key l % 32's half
    const char* row = (u ? kb[1] : kb[0]) + static_cast<uint32_t>((l32 & 15) * c.row_bytes + 16 * h);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) k[i] = Load16(row + 32 * i);
    const int64_t scale_at = (lane & 8 ? sb[1] : sb[0]) + 4 * (8 * (lane / 4 % 2) + 4 * h + lane % 4);
    ks = *(const __attribute__((address_space(1))) float*)(sc.k + scale_at);
    vs = *(const __attribute__((address_space(1))) float*)(sc.v + scale_at);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const char* from = vb[e / 8] + static_cast<uint32_t>((8 * (e / 4 % 2) + 4 * h + e % 4) * c.row_bytes);
      if constexpr (kDim == 128)
        v[e] = *(const __attribute__((address_space(1))) uint32_t*)(from + 4 * l32);
      else
        v[e] = *(const __attribute__((address_space(1))) uint16_t*)(from + 2 * l32);
    }
  }
};

template <int kDim, int kWaves>
struct SoloLds {
  char states[kWaves * kSoloRows * kDim * 4];
  float sm[kWaves][kSoloRows], sl[kWaves][kSoloRows];
};

// Few rows. kPrefix and the last three: as PromptBody's (prompt_body.h).
template <typename C, typename T, int kDim, int kWaves, bool kPrefix>
__device__ __forceinline__ void SoloBody(const CodesAttentionArgs& args, const Seqs& groups, int prefix_splits,
                                         SoloLds<kDim, kWaves>& shared, int bx, int by, int gx) {
  const AttentionArgs& a = args.a;
  using K = KeyType<T>;
  constexpr int kQ = kDim / 16, kBlocks = kDim / 32, kParts = kWeightParts<T>;
  auto& lds = shared.states;
  auto& sm = shared.sm;
  auto& sl = shared.sl;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.n_heads / a.c.n_kv;
  const int kh = bx % a.c.n_kv;
  int seq;
  RowTile t;
  if (!TileOf(kPrefix ? groups : a.s, group, kSoloRows, (gx - 1 - bx) / a.c.n_kv, &seq, &t))
    return;
  if constexpr (kPrefix) {
    const Common common = CommonOf(a.s, t.first, t.n_rows / group, t.len);
    if (common.keys == 0) return;
    seq = common.seq;
    t.len = common.keys;
  }
  const int h = lane >> 5;
  const int row = min(t.row0 + (lane & 31), t.n_rows - 1);
  const int token = row / group, head = kh * group + row % group;
  const int limit = kPrefix ? t.len - 1 : t.pos0 + token;  // the last key that the lane's row sees (< len)
  const int first_limit = kPrefix ? t.len - 1 : t.Position(t.row0, group);
  const int keys = kPrefix ? t.len : t.Position(t.row0 + kSoloRows - 1, group) + 1;
  const int range = RangeOf(max(keys, 1), kPrefix ? prefix_splits : a.splits);
  const int begin = by * range, end = min(max(keys, 0), begin + range);
  if (begin >= end && (kPrefix || by > 0)) return;
  const int32_t* table = a.s.table + seq * a.s.table_stride;

  U4 q[kQueryParts<T>][kQ];  // operand i: dimensions 32 (i / 2) + 16 h + 8 (i % 2) ..
  {
    const char* qp = a.q.p + (t.first + token) * a.q.token_bytes + head * a.q.head_bytes + 16 * h * kBytes<T>;
#pragma unroll
    for (int i = 0; i < kQ; ++i) LoadQuery<T>(qp + (32 * (i / 2) + 8 * (i % 2)) * kBytes<T>, i, q);
  }
  const float c = a.scale * 1.44269504088896341f;
  float m = kNegInf, l = 0.0f;
  F16v o[kBlocks] = {};
  Block<kDim> now, next;
  int pos = begin + wave * kSoloKeys;
  if (pos < end) now.Load(a.c, args.scales, table, kh, pos, t.len - 1, lane);
  for (; pos < end; pos += kWaves * kSoloKeys) {
    next.Load(a.c, args.scales, table, kh, pos + kWaves * kSoloKeys, t.len - 1, lane);
    F16v s;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const U4 x = Operand8<C, K>(now.k[i / 2][i % 2 * 2], now.k[i / 2][i % 2 * 2 + 1]);
#pragma unroll
      for (int p = kQueryParts<T> - 1; p >= 0; --p)
        s = i == 0 && p == kQueryParts<T> - 1 ? Mfma32First<K>(x, q[p][i]) : Mfma32<K>(x, q[p][i], s);
    }
    ScaleBy<0, 16>(s, now.ks * c);
    const bool masked = pos + kSoloKeys - 1 > first_limit || !now.ok[0] || !now.ok[1];
    uint32_t hidden = 0;
    if (masked) {
      // Masked keys: no weight, and nothing of what their scales hold; nor of the
      // codes of rows past the sequence and of unnamed pages, which may be anything.
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = pos + 8 * (e / 4) + 4 * h + e % 4;
        const bool in = key <= limit && now.ok[e / 8];
        s[e] = in ? s[e] : kNegInf;
        hidden |= in ? 0u : 1u << e;
        now.v[e] = now.ok[e / 8] && key < t.len ? now.v[e] : 0u;
      }
      const int key = pos + 8 * (lane / 4 % 4) + 4 * h + lane % 4;
      now.vs = (lane & 8 ? now.ok[1] : now.ok[0]) && key < t.len ? now.vs : 0.0f;
    }
    float top = kNegInf;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
    top = lanes::MaxXor32(top);
    if (__any(top > m + kLazy)) {  // as in paged_prompt.hip
      const float up = fmaxf(m, top), f = __builtin_amdgcn_exp2f(MaxDiff(m, up));
      m = up;
      l *= f;
#pragma unroll
      for (int w = 0; w < kBlocks; ++w) o[w] *= f;
    }
    const float base = m == kNegInf ? 0.0f : m;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = __builtin_amdgcn_exp2f(s[e] - base);
      l += s[e];
    }
    ScaleBy<0, 16>(s, now.vs);
    if (masked) {  // 0 x NaN must not reach the product
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = (hidden >> e) & 1 ? 0.0f : s[e];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      WeightParts<kParts> p;
      U4 x[kBlocks];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 8 * j + 2 * i;  // two keys
        p.Set(i, s[e], s[e + 1]);
        const uint32_t u = now.v[e], v = now.v[e + 1];
        const uint32_t lo = __builtin_amdgcn_perm(v, u, 0x05010400u), hi = __builtin_amdgcn_perm(v, u, 0x07030602u);
        x[0][i] = Halves2<C, BF16, false>(lo);
        x[1][i] = Halves2<C, BF16, true>(lo);
        if constexpr (kDim == 128) x[2][i] = Halves2<C, BF16, false>(hi), x[3][i] = Halves2<C, BF16, true>(hi);
      }
#pragma unroll
      for (int w = 0; w < kBlocks; ++w)
#pragma unroll
        for (int i = kParts - 1; i >= 0; --i) o[w] = Mfma32<BF16>(x[w], p.x[i], o[w]);
    }
    now = next;
  }
  l = lanes::AddXor32(l);

  // The waves' states, joined in LDS: dimension (kDim / 32) m + w in row m of block w;
  // chunk c (four dimensions) of row r at chunk c ^ r % 16.
  const int r = lane & 31;
  if (h == 0) sm[wave][r] = m, sl[wave][r] = l;
  __syncthreads();
  auto at = [&](int w, int row, int chunk) {
    return reinterpret_cast<F4*>(lds + w * kSoloRows * kDim * 4 + row * kDim * 4 + (chunk ^ (row & 15)) * 16);
  };
  float top = sm[0][r];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sm[w][r]);
  const float f = __builtin_amdgcn_exp2f(MaxDiff(m, top));
  if constexpr (kDim == 128) {
#pragma unroll
    for (int e = 0; e < 16; ++e) *at(wave, r, 8 * (e / 4) + 4 * h + e % 4) = F4{o[0][e], o[1][e], o[2][e], o[3][e]} * f;
  } else {
#pragma unroll
    for (int e = 0; e < 16; e += 2)
      *at(wave, r, (8 * (e / 4) + 4 * h + e % 4) / 2) = F4{o[0][e], o[1][e], o[0][e + 1], o[1][e + 1]} * f;
  }
  __syncthreads();
  const bool alone = !kPrefix && range >= keys;
  for (int i = tid; i < kSoloRows * (kDim / 4); i += 64 * kWaves) {
    const int ri = i / (kDim / 4), d = i % (kDim / 4) * 4, row_i = t.row0 + ri;
    if (row_i >= t.n_rows) break;
    float mi = sm[0][ri], li = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mi = fmaxf(mi, sm[w][ri]);
    F4 x = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      li += sl[w][ri] * __builtin_amdgcn_exp2f(MaxDiff(sm[w][ri], mi));
      x += *at(w, ri, d / 4);
    }
    const int token_i = row_i / group, head_i = kh * group + row_i % group;
    if (alone) {
      Store4<T>(a.out.p + (t.first + token_i) * a.out.token_bytes + head_i * a.out.head_bytes + d * kBytes<T>,
                x * Inverse(mi, li));
    } else {
      const int64_t rows = static_cast<int64_t>(kPrefix ? a.s.n_seqs : a.s.n_tokens) * a.n_heads;
      const int64_t out_row = static_cast<int64_t>(t.first + token_i) * a.n_heads + head_i;
      if (d == 0) PartStats(a, out_row)[by] = F2{mi, li};
      *reinterpret_cast<F4*>(PartOut<kDim>(a, rows, out_row) + static_cast<int64_t>(by) * kDim + d) = x;
    }
  }
}

// Many rows: workgroup (tile of 128 rows, key head, key range), a wave for 32 rows.
// A step's 64 keys come as codes to registers while the last step is worked on,
// and go to LDS converted, once for the four waves.
template <typename T, int kDim>
struct Wide {
  static constexpr int kRows = 128, kKeys = 64;
  static constexpr int kRowBytes = 2 * kDim, kTileBytes = kKeys * kRowBytes;
  static constexpr int kLoads = kKeys * kDim / 16 / 256;  // of 16 codes, of K and of V, for a thread
  static constexpr int kLoadRows = 256 / (kDim / 16);     // rows of all threads' loads
  static constexpr int kQ = kDim / 16;
};

template <typename T, int kDim>
struct WideLds {
  char tiles[4 * Wide<T, kDim>::kTileBytes];  // [buffer][K tile, V tile]
  float scales[2][2][Wide<T, kDim>::kKeys];   // per buffer: of the keys, of the values
};

template <typename C, typename T, int kDim, bool kPrefix>
__device__ __forceinline__ void WideBody(const CodesAttentionArgs& args, const Seqs& groups, int prefix_splits,
                                         WideLds<T, kDim>& shared, int bx, int by, int gx) {
  const AttentionArgs& a = args.a;
  using W = Wide<T, kDim>;
  using K = KeyType<T>;
  constexpr int kParts = kWeightParts<T>;
  auto& lds = shared.tiles;
  auto& scales = shared.scales;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.n_heads / a.c.n_kv;
  const int kh = bx % a.c.n_kv;
  int seq;
  RowTile t;
  if (!TileOf(kPrefix ? groups : a.s, group, W::kRows, (gx - 1 - bx) / a.c.n_kv, &seq, &t))
    return;
  if constexpr (kPrefix) {
    const Common common = CommonOf(a.s, t.first, t.n_rows / group, t.len);
    if (common.keys == 0) return;
    seq = common.seq;
    t.len = common.keys;
  }
  const int len = t.len;
  auto position = [&](int row) { return kPrefix ? len - 1 : t.Position(row, group); };
  const int h = lane >> 5;
  const int row = min(t.row0 + 32 * wave + (lane & 31), t.n_rows - 1);
  const int token = row / group, head = kh * group + row % group;
  const int limit = kPrefix ? len - 1 : t.pos0 + token;  // the last key that the lane's row sees (< len)
  const int wave_first = position(t.row0 + 32 * wave), wave_last = position(t.row0 + 32 * wave + 31);
  const int keys = position(t.row0 + W::kRows - 1) + 1;
  int begin = 0, end = max(keys, 0);
  if constexpr (kPrefix) {
    const int range = RangeOf(keys, prefix_splits);
    begin = by * range;
    end = min(end, begin + range);
    if (begin >= end) return;
  }
  const int steps = end <= begin ? 0 : (end - begin - 1) / W::kKeys + 1;
  const int32_t* table = a.s.table + seq * a.s.table_stride;
  const int in_page = (1 << a.c.page_log2) - 1;

  U4 q[kQueryParts<T>][W::kQ];  // operand i: dimensions 16 i + 8 h ..
  {
    const char* qp = a.q.p + (t.first + token) * a.q.token_bytes + head * a.q.head_bytes + 8 * h * kBytes<T>;
#pragma unroll
    for (int i = 0; i < W::kQ; ++i) LoadQuery<T>(qp + 16 * i * kBytes<T>, i, q);
  }

  // Staging: a thread brings codes 16 c .. of rows r0 + i kLoadRows, which of a wave
  // lie in one unit of 16 positions, and a lane of the first two waves a scale.
  constexpr int kPer = kDim / 16;
  const int r0 = tid / kPer, chunk = tid % kPer;
  constexpr int kWaveRows = 64 / kPer;
  U4 kc[W::kLoads], vc[W::kLoads];
  float scale = 0.0f;
  bool scale_ok = false;
  bool ok[W::kLoads];
  int pages[4];  // of the step to come
  auto look_up = [&](int step) {
#pragma unroll
    for (int u = 0; u < 4; ++u) pages[u] = PageAt(a.c, table, max(min(begin + step * W::kKeys + 16 * u, len - 1), 0));
  };
  auto fetch = [&](int step) {
    const int key0 = begin + step * W::kKeys, last = (len - 1) & ~15;  // units that are there
#pragma unroll
    for (int i = 0; i < W::kLoads; ++i) {
      const int u = (wave * kWaveRows + i * W::kLoadRows) / 16;
      const int p0 = min(key0 + 16 * u, last);
      const int page = u == 0 ? pages[0] : u == 1 ? pages[1] : u == 2 ? pages[2] : pages[3];
      ok[i] = page >= 0 && key0 + r0 + i * W::kLoadRows < len;
      const int64_t at = max(page, 0) * a.c.page_bytes + kh * a.c.head_bytes + (p0 & in_page) * static_cast<int64_t>(a.c.row_bytes);
      const uint32_t off = static_cast<uint32_t>(((r0 + i * W::kLoadRows) & 15) * a.c.row_bytes + 16 * chunk);
      kc[i] = Load16(a.c.k + at + off);
      vc[i] = Load16(a.c.v + at + off);
    }
    if (wave < 2) {
      const int u = lane / 16;
      const int p0 = min(key0 + 16 * u, last);
      const int page = u == 0 ? pages[0] : u == 1 ? pages[1] : u == 2 ? pages[2] : pages[3];
      scale = *(const __attribute__((address_space(1))) float*)((wave == 0 ? args.scales.k : args.scales.v) +
                                                                max(page, 0) * args.scales.page_bytes +
                                                                kh * args.scales.head_bytes + 4 * ((p0 & in_page) + lane % 16));
      scale_ok = page >= 0 && key0 + lane < len;
    }
  };
  const float c = a.scale * 1.44269504088896341f;
  auto settle = [&](int step, auto buffer) {
    constexpr int kAt = decltype(buffer)::value;
    char* kt = lds + kAt * 2 * W::kTileBytes;
    char* vt = kt + W::kTileBytes;
#pragma unroll
    for (int i = 0; i < W::kLoads; ++i) {
      const int r = r0 + i * W::kLoadRows;
      // rows past the sequence and of unnamed pages may hold anything
      const U4 x = kc[i], y = ok[i] ? vc[i] : U4{};
      char* kr = kt + r * W::kRowBytes;
      char* vr = vt + r * W::kRowBytes;
      const int ks = KSwizzle<K, kDim>(r), vs = VSwizzle<BF16, kDim>(r);
      *reinterpret_cast<U4*>(kr + 16 * ((2 * chunk) ^ ks)) = Operand8<C, K>(x[0], x[1]);
      *reinterpret_cast<U4*>(kr + 16 * ((2 * chunk + 1) ^ ks)) = Operand8<C, K>(x[2], x[3]);
      *reinterpret_cast<U4*>(vr + 16 * ((2 * chunk) ^ vs)) = Operand8<C, BF16>(y[0], y[1]);
      *reinterpret_cast<U4*>(vr + 16 * ((2 * chunk + 1) ^ vs)) = Operand8<C, BF16>(y[2], y[3]);
    }
    if (wave < 2) scales[kAt][wave][lane] = wave == 0 ? scale * c : scale_ok ? scale : 0.0f;
  };

  const int k_at = (lane & 31) * W::kRowBytes + 16 * (h ^ KSwizzle<K, kDim>(lane & 31));
  int v_at[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = 8 * u + 4 * h + (lane & 15) / 4;
    v_at[u] = r * W::kRowBytes + 16 * ((2 * ((lane >> 4) & 1) + (lane & 3) / 2) ^ VSwizzle<BF16, kDim>(r)) + 8 * (lane & 1);
  }
  float m = kNegInf, l = 0.0f;
  F16v o[kDim / 32] = {};
  if (steps > 0) {
    look_up(0);
    fetch(0);
    settle(0, std::integral_constant<int, 0>{});
  }
  __syncthreads();
  auto work = [&](int step, auto buffer) {
    constexpr int kAt = decltype(buffer)::value;
    const bool more = step + 1 < steps;
    bool named[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) named[u] = pages[u] >= 0;
    if (more) {
      look_up(step + 1);
      fetch(step + 1);
    }
    const int key0 = begin + step * W::kKeys;
    if (key0 <= wave_last && key0 < end) {
      const char* kt = lds + kAt * 2 * W::kTileBytes;
      const char* vt = kt + W::kTileBytes;
      // lane e of each 16: of the key that the lanes' element e belongs to
      const float* of_lane = scales[kAt][0] + 8 * ((lane & 15) / 4) + 4 * h + lane % 4;
      const float ks[2] = {of_lane[0], of_lane[32]};
      const float vs[2] = {of_lane[W::kKeys], of_lane[W::kKeys + 32]};
      F16v s[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int i = 0; i < W::kQ; ++i) {
          const U4 x = *reinterpret_cast<const U4*>(kt + 32 * b * W::kRowBytes + (k_at ^ 32 * i));
#pragma unroll
          for (int p = kQueryParts<T> - 1; p >= 0; --p)
            s[b] = i == 0 && p == kQueryParts<T> - 1 ? Mfma32First<K>(x, q[p][i]) : Mfma32<K>(x, q[p][i], s[b]);
        }
        ScaleBy<0, 16>(s[b], ks[b]);
      }
      uint32_t hidden = 0;
      const bool masked = key0 + W::kKeys - 1 > wave_first || !(named[0] && named[1] && named[2] && named[3]);
      if (masked) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = 32 * b + 8 * (e / 4) + 4 * h + e % 4;
            const bool in = key0 + key <= limit && named[2 * b + e / 8];
            s[b][e] = in ? s[b][e] : kNegInf;
            hidden |= in ? 0u : 1u << (16 * b + e);
          }
      }
      float top = kNegInf;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[b][e]);
      top = lanes::MaxXor32(top);
      // The maximum that weights refer to moves only when one would pass 2^kLazy, as
      // in paged_prompt.hip.
      if (__any(top > m + kLazy)) {
        const float now = fmaxf(m, top), f = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= f;
#pragma unroll
        for (int w = 0; w < kDim / 32; ++w) o[w] *= f;
      }
      const float base = m == kNegInf ? 0.0f : m;
      typedef short S4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[b][e] = __builtin_amdgcn_exp2f(s[b][e] - base);
          l += s[b][e];
        }
        ScaleBy<0, 16>(s[b], vs[b]);
        if (masked) {  // 0 x NaN must not reach the product
#pragma unroll
          for (int e = 0; e < 16; ++e) s[b][e] = (hidden >> (16 * b + e)) & 1 ? 0.0f : s[b][e];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          WeightParts<kParts> p;
#pragma unroll
          for (int e = 0; e < 4; ++e) p.Set(e, s[b][8 * j + 2 * e], s[b][8 * j + 2 * e + 1]);
#pragma unroll
          for (int w = 0; w < kDim / 32; ++w) {
            U4 v;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const char* at = vt + (v_at[u] ^ 64 * w) + (32 * b + 16 * j) * W::kRowBytes;
              const U2 x = __builtin_bit_cast(
                  U2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4*)at));
              v[2 * u] = x[0], v[2 * u + 1] = x[1];
            }
#pragma unroll
            for (int i = kParts - 1; i >= 0; --i) o[w] = Mfma32<BF16>(v, p.x[i], o[w]);
          }
        }
      }
    }
    if (more) settle(step + 1, std::integral_constant<int, 1 - kAt>{});
    __syncthreads();
  };
  for (int step = 0; step < steps; step += 2) {
    work(step, std::integral_constant<int, 0>{});
    if (step + 1 < steps) work(step + 1, std::integral_constant<int, 1>{});
  }

  l = lanes::AddXor32(l);
  if (t.row0 + 32 * wave + (lane & 31) >= t.n_rows) return;
  // dimension 32 w + 8 (e / 4) + 4 h + e % 4 in element e of block w
  if constexpr (kPrefix) {
    const int64_t rows = static_cast<int64_t>(a.s.n_seqs) * a.n_heads;
    const int64_t out_row = static_cast<int64_t>(t.first + token) * a.n_heads + head;
    if (h == 0) PartStats(a, out_row)[by] = F2{m, l};
    float* to = PartOut<kDim>(a, rows, out_row) + static_cast<int64_t>(by) * kDim;
#pragma unroll
    for (int w = 0; w < kDim / 32; ++w)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<F4*>(to + 32 * w + 2 * e + 4 * h) = F4{o[w][e], o[w][e + 1], o[w][e + 2], o[w][e + 3]};
  } else {
    const float inv = Inverse(m, l);
    char* out = a.out.p + (t.first + token) * a.out.token_bytes + head * a.out.head_bytes;
#pragma unroll
    for (int w = 0; w < kDim / 32; ++w)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        Store4<T>(out + kBytes<T> * (32 * w + 2 * e + 4 * h), F4{o[w][e], o[w][e + 1], o[w][e + 2], o[w][e + 3]} * inv);
  }
}

}  // namespace paged
}  // namespace rpg

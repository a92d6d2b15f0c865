// Causal attention of packed new tokens over a cache of 8-bit codes
// (rpg_hip_quant_prompt, include/rpg_hip.h): token i of a sequence at position p,
//   out[h] = sum_{j <= p} p_j vs_j cv_j,  p = softmax over j <= p of scale ks_j (q[h] . ck_j).
//
// The codes are the products' operands and the scales go to scores and weights in
// fp32, as in codes_decode.hip; rows are tiled and scores and outputs formed
// transposed on 32 x 32 tiles, as in paged_prompt.hip.
//
// Few rows (CodesSoloKernel): workgroup (tile of 32 rows, key head, key range), whose
// waves take blocks of 32 keys in turn, from memory to registers, and join their
// states in LDS.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "codes_dev.h"
#include "common.h"
#include "groups.h"
#include "lanes.h"
#include "paged.h"
#include "paged_dev.h"
#include "row_tile.h"

namespace rpg {
namespace paged {
namespace {

constexpr int kRows = 32;  // query rows of a tile
constexpr int kKeys = 32;  // keys of a wave's step

// A block of 32 keys in a wave: K as 16 codes of key l % 32 per 32 dimensions, V as
// the lane's dimensions (kDim / 32) (l % 32) .. of the keys that its scores come in,
// 8 (e / 4) + 4 (l / 32) + e % 4; one scale: of the key (l < 32) or the value of key
// l % 32.
template <int kDim>
struct Block {
  static constexpr int kChunks = kDim / 32;
  U4 k[kChunks];
  uint32_t v[16];
  float scale;
  bool ok[2];  // the page of either 16 positions is there

  // Positions pos .. of a sequence whose last is `last`; those past it and those of
  // unnamed pages are read from rows that are there.
  __device__ __forceinline__ void Load(const Cache& c, const Scales& sc, const int32_t* table, int kh, int pos, int last,
                                       int lane) {
    const int in_page = (1 << c.page_log2) - 1, l32 = lane & 31, h = lane >> 5;
    const char* kb[2];
    const char* vb[2];
    const char* sb[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int p0 = min(pos + 16 * u, last & ~15);
      const int page = PageAt(c, table, p0);
      ok[u] = page >= 0;
      const int64_t at = max(page, 0) * c.page_bytes + kh * c.head_bytes + (p0 & in_page) * static_cast<int64_t>(c.row_bytes);
      kb[u] = c.k + at;
      vb[u] = c.v + at;
      sb[u] = (h == 0 ? sc.k : sc.v) + max(page, 0) * sc.page_bytes + kh * sc.head_bytes + 4 * (p0 & in_page);
    }
    const int u = l32 >> 4;  // key l % 32's half
    const char* row = (u ? kb[1] : kb[0]) + static_cast<uint32_t>((l32 & 15) * c.row_bytes + 16 * h);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) k[i] = Load16(row + 32 * i);
    scale = *(const __attribute__((address_space(1))) float*)((u ? sb[1] : sb[0]) + 4 * (l32 & 15));
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

// grid (row tile x key head, key range): key heads next to each other, the tiles
// with the most keys first. kPrefix: as PromptBody's (prompt_body.h).
template <typename C, typename T, int kDim, int kWaves, bool kPrefix>
__device__ __forceinline__ void SoloBody(const CodesAttentionArgs& args, const Seqs& groups, int prefix_splits) {
  const AttentionArgs& a = args.a;
  using K = KeyType<T>;
  constexpr int kQ = kDim / 16, kBlocks = kDim / 32;
  __shared__ __align__(16) char lds[kWaves * kRows * kDim * 4];  // the waves' states; before, their blocks' scales
  __shared__ float sm[kWaves][kRows], sl[kWaves][kRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.n_heads / a.c.n_kv;
  const int kh = blockIdx.x % a.c.n_kv;
  int seq;
  RowTile t;
  if (!TileOf(kPrefix ? groups : a.s, group, kRows, static_cast<int>((gridDim.x - 1 - blockIdx.x) / a.c.n_kv), &seq, &t))
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
  const int keys = kPrefix ? t.len : t.Position(t.row0 + kRows - 1, group) + 1;
  const int range = RangeOf(max(keys, 1), kPrefix ? prefix_splits : a.splits);
  const int begin = blockIdx.y * range, end = min(max(keys, 0), begin + range);
  if (begin >= end && (kPrefix || blockIdx.y > 0)) return;
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
  float* scales = reinterpret_cast<float*>(lds) + 64 * wave;  // this wave's alone
  Block<kDim> now, next;
  int pos = begin + wave * kKeys;
  if (pos < end) now.Load(a.c, args.scales, table, kh, pos, t.len - 1, lane);
  for (; pos < end; pos += kWaves * kKeys) {
    next.Load(a.c, args.scales, table, kh, pos + kWaves * kKeys, t.len - 1, lane);
    // A wave's LDS operations are done in order; nothing moves past the fences.
    scales[lane] = now.scale;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    F16v s;
#pragma unroll
    for (int i = 0; i < kQ; ++i) {
      const U4 x = Operand8<C, K>(now.k[i / 2][i % 2 * 2], now.k[i / 2][i % 2 * 2 + 1]);
#pragma unroll
      for (int p = kQueryParts<T> - 1; p >= 0; --p)
        s = i == 0 && p == kQueryParts<T> - 1 ? Mfma32First<K>(x, q[p][i]) : Mfma32<K>(x, q[p][i], s);
    }
    float vs[16];
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const F4 x = *reinterpret_cast<const F4*>(scales + 2 * e + 4 * h), y = *reinterpret_cast<const F4*>(scales + 32 + 2 * e + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[e + i] *= x[i] * c, vs[e + i] = y[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (pos + kKeys - 1 > first_limit || !now.ok[0] || !now.ok[1]) {
      // Masked keys: no weight, and nothing of what their scales hold; nor of the
      // codes of rows past the sequence and of unnamed pages, which may be anything.
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = pos + 8 * (e / 4) + 4 * h + e % 4;
        const bool in = key <= limit && now.ok[e / 8];
        s[e] = in ? s[e] : kNegInf;
        vs[e] = in ? vs[e] : 0.0f;
        now.v[e] = now.ok[e / 8] && key < t.len ? now.v[e] : 0u;
      }
    }
    float top = kNegInf;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
    top = lanes::MaxXor32(top);
    if (__any(top > m)) {
      const float up = fmaxf(m, top), f = __builtin_amdgcn_exp2f(MaxDiff(m, up));
      m = up;
      l *= f;
#pragma unroll
      for (int w = 0; w < kBlocks; ++w) o[w] *= f;
    }
    const float base = m == kNegInf ? 0.0f : m;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float p = __builtin_amdgcn_exp2f(s[e] - base);
      l += p;
      s[e] = p * vs[e];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      WeightParts<T> p;
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p.Set(i, s[8 * j + 2 * i], s[8 * j + 2 * i + 1]);
        const uint32_t x = now.v[8 * j + 2 * i], y = now.v[8 * j + 2 * i + 1];
        lo[i] = __builtin_amdgcn_perm(y, x, 0x05010400u);
        if (kDim == 128) hi[i] = __builtin_amdgcn_perm(y, x, 0x07030602u);
      }
#pragma unroll
      for (int w = 0; w < kBlocks; ++w) {
        U4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = w % 2 ? Halves2<C, BF16, true>(w < 2 ? lo[i] : hi[i]) : Halves2<C, BF16, false>(w < 2 ? lo[i] : hi[i]);
#pragma unroll
        for (int i = kWeightParts<T> - 1; i >= 0; --i) o[w] = Mfma32<BF16>(x, p.x[i], o[w]);
      }
    }
    now = next;
  }
  l = lanes::AddXor32(l);

  // The waves' states, joined in LDS: dimension (kDim / 32) m + w in row m of block w;
  // chunk c (four dimensions) of row r at chunk c ^ r % 16.
  const int r = lane & 31;
  if (h == 0) sm[wave][r] = m, sl[wave][r] = l;
  __syncthreads();  // (no wave reads scales any more)
  auto at = [&](int w, int row, int chunk) {
    return reinterpret_cast<F4*>(lds + w * kRows * kDim * 4 + row * kDim * 4 + (chunk ^ (row & 15)) * 16);
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
  for (int i = tid; i < kRows * (kDim / 4); i += 64 * kWaves) {
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
      if (d == 0) PartStats(a, out_row)[blockIdx.y] = F2{mi, li};
      *reinterpret_cast<F4*>(PartOut<kDim>(a, rows, out_row) + static_cast<int64_t>(blockIdx.y) * kDim + d) = x;
    }
  }
}

template <typename C, typename T, int kDim, int kWaves>
__global__ __launch_bounds__(64 * kWaves, 1) void CodesSoloKernel(CodesAttentionArgs a) {
  SoloBody<C, T, kDim, kWaves, false>(a, a.a.s, 1);
}

template <typename C, typename T, int kDim, int kWaves>
__global__ __launch_bounds__(64 * kWaves, 1) void CodesPrefixKernel(CodesSharedArgs a) {
  SoloBody<C, T, kDim, kWaves, true>(a.c, a.groups, static_cast<int>(a.prefix_splits));
}

template <typename C, typename T, int kDim>
void LaunchPrefix(const CodesSharedArgs& args, hipStream_t s) {
  const AttentionArgs& a = args.c.a;
  const int64_t tiles = TilesFor(a.s.n_seqs, args.groups.n_seqs, a.n_heads / a.c.n_kv, kRows);
  RPG_CHECK(tiles * a.c.n_kv <= kMaxGroups, "%d x %d query rows in one launch", a.s.n_seqs, a.n_heads);
  CodesPrefixKernel<C, T, kDim, 4>
      <<<dim3(static_cast<uint32_t>(tiles * a.c.n_kv), static_cast<uint32_t>(args.prefix_splits)), 256, 0, s>>>(args);
  HIP_CHECK(hipGetLastError());
}

template <typename C, typename T, int kDim>
void Launch(const CodesAttentionArgs& args, hipStream_t s) {
  const AttentionArgs& a = args.a;
  const int64_t tiles = TilesFor(a.s.n_tokens, a.s.n_seqs, a.n_heads / a.c.n_kv, kRows);
  RPG_CHECK(tiles * a.c.n_kv <= kMaxGroups &&
                (a.splits == 1 || static_cast<int64_t>(a.s.n_tokens) * a.n_heads <= kMaxGroups),
            "%d x %d query rows in one launch", a.s.n_tokens, a.n_heads);
  CodesSoloKernel<C, T, kDim, 4><<<dim3(static_cast<uint32_t>(tiles * a.c.n_kv), a.splits), 256, 0, s>>>(args);
  HIP_CHECK(hipGetLastError());
  if (a.splits > 1) PromptJoin(a, s);
}

}  // namespace

int CodesPromptSplits(int64_t n_tokens, int64_t n_seqs, int n_heads, int n_kv, int64_t capacity) {
  const int64_t wgs = TilesFor(n_tokens, n_seqs, n_heads / n_kv, kRows) * n_kv;
  if (wgs >= 128) return 1;
  return static_cast<int>(std::max<int64_t>(1, std::min({CeilDiv(256, wgs), CeilDiv(capacity, 512), int64_t{kMaxSplits}})));
}

void PromptCodes(const CodesAttentionArgs& a, hipStream_t s) {
  if (a.a.s.n_tokens == 0 || a.a.s.n_seqs == 0) return;
  ByTypes(a.code, a.a.c, [&](auto code, auto type, auto dim) {
    Launch<decltype(code), decltype(type), decltype(dim)::value>(a, s);
  });
}

void PrefixCodes(const CodesSharedArgs& a, hipStream_t s) {
  ByTypes(a.c.code, a.c.a.c, [&](auto code, auto type, auto dim) {
    LaunchPrefix<decltype(code), decltype(type), decltype(dim)::value>(a, s);
  });
}

}  // namespace paged
}  // namespace rpg

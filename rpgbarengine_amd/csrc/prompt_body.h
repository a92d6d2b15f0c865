// What the kernels of paged_prompt.hip and paged_shared.hip have in common: attention
// of a tile of query rows over a range of keys. The method is described in
// paged_prompt.hip.
#pragma once

#include <hip/hip_runtime.h>

#include "groups.h"
#include "lanes.h"
#include "paged.h"
#include "paged_dev.h"
#include "row_tile.h"

namespace rpg {
namespace paged {

template <typename T, int kDim, int kGroups>
struct Shape {
  static constexpr int kWaves = kGroups == 8 ? 8 : 4;
  static constexpr int kGroupWaves = kWaves / kGroups;
  static constexpr int kRows = 32 * kGroupWaves;              // rows of a workgroup's tile
  static constexpr int kKeys = kBytes<T> == 4 || kGroups > 1 ? 32 : 64;  // keys of a group's step
  static constexpr int kBlocks = kKeys / 32;                  // 32-key score blocks
  static constexpr int kRowBytes = kDim * kBytes<T>;          // a cache row
  static constexpr int kChunks = kRowBytes / 16;              // its 16-byte chunks
  static constexpr int kPerThread = kKeys * kChunks / (64 * kGroupWaves);
  static constexpr int kRowsPerLoad = 64 / kChunks;           // rows of a wave's load instruction
  static constexpr int kWaveRows = kKeys / kGroupWaves;       // rows that a wave stages
  static constexpr int kUnit = kWaveRows < 16 ? kWaveRows : 16;  // rows looked up in the page table together
  static constexpr int kTileBytes = kKeys * kRowBytes;
  static constexpr int kQ = kDim / 16;                        // products over a query row
};

// Chunk c of row r lies at chunk c ^ KSwizzle(r) or VSwizzle(r) of its LDS row.
// K: rows next to each other are read at one chunk; V (16-bit): four rows next
// to each other at four chunks. Both are linear over xor, so that an address
// is one lane's base, xored with a constant.
template <typename T, int kDim>
__device__ __forceinline__ constexpr int KSwizzle(int r) {
  return r & (kDim * kBytes<T> / 16 - 1);
}
template <typename T, int kDim>
__device__ __forceinline__ constexpr int VSwizzle(int r) {
  if constexpr (kBytes<T> == 4) return 0;  // read a row at a time
  return (((r & 3) << 2) | ((r >> 2) & 3)) & (kDim * kBytes<T> / 16 - 1);
}

// A product's operand: eight values, in f32 as three bf16 parts.
template <typename T>
struct OperandOf {
  typedef U4 type;
};
template <>
struct OperandOf<F32> {
  typedef Parts8 type;
};
template <typename T>
using Operand = typename OperandOf<T>::type;
__device__ __forceinline__ Parts8 Split8(U4 x, U4 y) {
  Parts8 p;
  p.Set(0, Split3(__uint_as_float(x[0]), __uint_as_float(x[1])));
  p.Set(1, Split3(__uint_as_float(x[2]), __uint_as_float(x[3])));
  p.Set(2, Split3(__uint_as_float(y[0]), __uint_as_float(y[1])));
  p.Set(3, Split3(__uint_as_float(y[2]), __uint_as_float(y[3])));
  return p;
}

template <typename T>
__device__ __forceinline__ bool NotFinite(uint32_t u) {
  if constexpr (kBytes<T> == 4) return (u & 0x7F800000u) == 0x7F800000u;
  constexpr uint32_t kExp = __is_same(T, BF16) ? 0x7F80u : 0x7C00u;  // of either half
  return (u & kExp) == kExp || ((u >> 16) & kExp) == kExp;
}

// Values that are not finite, in a step where some rows do not see all keys: 0 x
// NaN must not reach those. The product takes zeros in their place; the first
// position of a +inf, a -inf and a NaN in every dimension is kept, and the rows
// that see one have it added at the end.
constexpr int kOddKinds = 3;
template <typename T>
__device__ __forceinline__ int OddKind(uint32_t u) {
  constexpr uint32_t kSign = kBytes<T> == 4 ? 0x80000000u : 0x8000u;
  constexpr uint32_t kInf = kBytes<T> == 4 ? 0x7F800000u : __is_same(T, BF16) ? 0x7F80u : 0x7C00u;
  return (u & (kSign - 1)) != kInf ? 2 : u & kSign ? 1 : 0;
}

// What a row whose last key is `limit` has added in dimension d.
template <int kDim>
__device__ __forceinline__ float OddSum(const int (&first_odd)[kOddKinds][kDim], int d, int limit) {
  const bool plus = first_odd[0][d] <= limit, minus = first_odd[1][d] <= limit, nan = first_odd[2][d] <= limit;
  const float inf = -kNegInf;
  return nan || (plus && minus) ? __builtin_nanf("") : plus ? inf : minus ? -inf : 0.0f;
}

// The dimension of row m of output block w.
template <typename T, int kDim>
__device__ __forceinline__ int DimOf(int w, int m) {
  return kBytes<T> == 4 ? (kDim / 32) * m + w : 32 * w + m;
}

// The maximum that weights refer to moves only when one would pass 2^kLazy: most
// steps raise some row's, and rescaling costs as much as the exponentials (4000
// tokens, bf16: 164 us with a rescaling whenever a maximum rises, 152 without).
// Weights are held times 2^kLift, their sums too: f16 has steps of 2^-24 at the
// least, and keys whose weight is below half of that would count in the sum and
// not in the output. The largest is 2^15.
constexpr float kLazy = 8.0f;
template <typename T>
constexpr float kLift = __is_same(T, F16) ? 15.0f - kLazy : 0.0f;

// A buffer resource (wave-uniform) over `bytes` bytes from p.
__device__ __forceinline__ U4 Resource(const char* p, uint32_t bytes) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  return U4{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(u))),
            static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(u >> 32))) & 0xFFFFu, bytes, 0x00020000u};
}
// 16 bytes per lane from the resource to LDS, a wave's lanes side by side. In
// assembly, since the compiler holds every LDS read after the builtin until the
// load is done, though the reads are of another buffer: the waits are
// written out, before the tile's first read. Of the registers it overwrites m0 alone.
__device__ __forceinline__ void LdsDma(U4 src, char* to, int voff, int soff) {
  const uint32_t at = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)to));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(at), "v"(voff), "s"(src), "s"(soff)
               : "m0");
}

// grid (row tile x key head, key range): key heads next to each other, the tiles
// with the most keys first. kPrefix: the tiles are of the groups of a.s's sequences
// (`groups`), one token each; all rows see the positions that their group has in
// common, and what comes out are partials, of prefix_splits ranges at most.
template <typename T, int kDim, int kGroups, bool kShared>
struct PromptLds {
  using Sh = Shape<T, kDim, kGroups>;
  // A group of one wave needs no barriers: it takes the next K tile in as soon as
  // the scores are done and the next V tile after the second product, each in the
  // place of the last (half the LDS: two workgroups per compute unit). Groups of
  // several waves have two of each in turn.
  static constexpr bool kSolo = Sh::kGroupWaves == 1;
  // kShared: K and V take turns in one place, so that two workgroups fit a compute
  // unit even in f32: the other's products run while a tile is on its way.
  static_assert(kSolo || !kShared, "groups of one wave");
  static constexpr int kTiles = kShared ? 1 : kSolo ? 2 : 4;
  char tiles[kGroups * kTiles * Sh::kTileBytes];  // per group [buffer][K tile, V tile]
  uint32_t page_ok[kGroups][2];                   // per buffer: a byte for each unit of rows
  int any_odd, first_odd[kOddKinds][kDim];
  float sm[kGroups][Sh::kRows], sl[kGroups][Sh::kRows];  // of the groups' join
};

// bx, by, gx: the workgroup's place in the grid and its width.
template <typename T, int kDim, int kGroups, bool kShared, bool kPrefix>
__device__ __forceinline__ void PromptBody(const AttentionArgs& a, const Seqs& groups, int prefix_splits,
                                           PromptLds<T, kDim, kGroups, kShared>& shared, int bx, int by, int gx) {
  using Sh = Shape<T, kDim, kGroups>;
  using Lds = PromptLds<T, kDim, kGroups, kShared>;
  constexpr bool kSolo = Lds::kSolo;
  constexpr int kTiles = Lds::kTiles;
  auto& lds = shared.tiles;
  auto& page_ok = shared.page_ok;
  auto& any_odd = shared.any_odd;
  auto& first_odd = shared.first_odd;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave / Sh::kGroupWaves, gw = wave % Sh::kGroupWaves;  // the wave's group, its place there
  const int group = a.n_heads / a.c.n_kv;
  const int kh = bx % a.c.n_kv;
  int seq;
  RowTile t;
  if (!TileOf(kPrefix ? groups : a.s, group, Sh::kRows, (gx - 1 - bx) / a.c.n_kv, &seq, &t))
    return;
  if constexpr (kPrefix) {
    const Common common = CommonOf(a.s, t.first, t.n_rows / group, t.len);
    if (common.keys == 0) return;
    seq = common.seq;
    t.len = common.keys;
  }
  const int first = t.first, n_rows = t.n_rows, row0 = t.row0, len = t.len, pos0 = t.pos0;
  auto position = [&](int row) { return kPrefix ? len - 1 : t.Position(row, group); };

  // this lane's row: a query token and head, and the last key it sees
  const int h = lane >> 5;
  const int row = min(row0 + 32 * gw + (lane & 31), n_rows - 1);
  const int token = row / group, head = kh * group + row % group;
  const int limit = kPrefix ? len - 1 : pos0 + token;  // (< len)
  const int wave_first = position(row0 + 32 * gw), wave_last = position(row0 + 32 * gw + 31);
  const int tile_first = position(row0), keys = position(row0 + Sh::kRows - 1) + 1;
  int key_begin = 0, key_end = max(keys, 0);
  if constexpr (kGroups >= 4 || kPrefix) {
    const int range = RangeOf(max(keys, 1), kPrefix ? prefix_splits : a.splits);
    key_begin = by * range;
    key_end = min(key_end, key_begin + range);
    if (key_begin >= key_end && (kPrefix || by > 0)) return;
  }
  // steps of the workgroup: a step of every group each
  const int steps = key_end <= key_begin ? 0 : (key_end - key_begin - 1) / (Sh::kKeys * kGroups) + 1;

  // The query row as B operands: dimensions 16 i + 8 h .. + 7 (f32: in parts).
  Operand<T> q[Sh::kQ];
  {
    const char* qp = a.q.p + (first + token) * a.q.token_bytes + head * a.q.head_bytes + 8 * h * kBytes<T>;
#pragma unroll
    for (int i = 0; i < Sh::kQ; ++i) {
      if constexpr (kBytes<T> == 4)
        q[i] = Split8(Load16(qp + 64 * i), Load16(qp + 64 * i + 16));
      else
        q[i] = Load16(qp + 32 * i);
    }
  }
  const int32_t* table = a.s.table + seq * a.s.table_stride;
  const int64_t head_off = kh * a.c.head_bytes;
  const int in_page = (1 << a.c.page_log2) - 1;
  if (tid == 0) any_odd = 0;
  if (tid < 2 * kGroups) page_ok[tid / 2][tid % 2] = 0x01010101u;
  for (int i = tid; i < kOddKinds * kDim; i += 64 * Sh::kWaves) first_odd[i / kDim][i % kDim] = INT32_MAX;
  __syncthreads();

  // Staging by LDS DMA: a wave brings kWaveRows rows, a lane kPerThread chunks
  // of K and of V, in LDS the wave's lanes side by side.
  constexpr int kWaveRows = Sh::kWaveRows, kWaveUnits = kWaveRows / Sh::kUnit;
  const int srow = lane / Sh::kChunks, sc = lane % Sh::kChunks;
  const int row_from = srow * a.c.row_bytes;
  const int k_from = 16 * (sc ^ KSwizzle<T, kDim>(gw * kWaveRows + srow));
  const int v_from = 16 * (sc ^ VSwizzle<T, kDim>(gw * kWaveRows + srow));
  const int to = gw * kWaveRows * Sh::kRowBytes;
  char* tiles = lds + grp * kTiles * Sh::kTileBytes;
  // the first key of the group's part of a step
  auto first_key = [&](int step) { return key_begin + (step * kGroups + grp) * Sh::kKeys; };
  // Where a step's rows of this wave lie. Page numbers are looked up a step ahead.
  struct Place {
    int64_t at[kWaveUnits];
    bool ok[kWaveUnits];
  };
  int ahead[kWaveUnits];
  auto look_up = [&](int step) {
#pragma unroll
    for (int u = 0; u < kWaveUnits; ++u) {
      const int p0 = first_key(step) + gw * kWaveRows + u * Sh::kUnit;
      ahead[u] = PageAt(a.c, table, max(min(p0, len - 1), 0));
    }
  };
  auto place_of = [&](int step) {
    Place x;
#pragma unroll
    for (int u = 0; u < kWaveUnits; ++u) {
      const int p0 = first_key(step) + gw * kWaveRows + u * Sh::kUnit;
      const int p = min(p0, (len - 1) & ~(Sh::kUnit - 1));  // rows that are there
      const int page = __builtin_amdgcn_readfirstlane(ahead[u]);
      x.ok[u] = page >= 0 && p0 < len;
      x.at[u] = max(page, 0) * a.c.page_bytes + head_off + (p & in_page) * static_cast<int64_t>(a.c.row_bytes);
    }
    return x;
  };
  // The wave's rows of a K or V tile: kPerThread loads.
  auto fetch = [&](const char* pool, const Place& x, char* tile, int from, auto swizzle) {
#pragma unroll
    for (int u = 0; u < kWaveUnits; ++u) {
      const U4 src = Resource(pool + x.at[u], (Sh::kUnit - 1) * a.c.row_bytes + Sh::kRowBytes);
      constexpr int kLoads = Sh::kPerThread / kWaveUnits;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int up = i * Sh::kRowsPerLoad;
        LdsDma(src, tile + to + 1024 * (u * kLoads + i), row_from + (from ^ 16 * swizzle(u * Sh::kUnit + up)),
               up * a.c.row_bytes);
      }
    }
  };
  auto fetch_k = [&](const Place& x, char* tile) { fetch(a.c.k, x, tile, k_from, [](int r) { return KSwizzle<T, kDim>(r); }); };
  auto fetch_v = [&](const Place& x, char* tile) { fetch(a.c.v, x, tile, v_from, [](int r) { return VSwizzle<T, kDim>(r); }); };
  // What the wave's rows of a V tile need before they are read: rows past the
  // sequence and of unnamed pages may hold anything, NaN among it, and become
  // zeros (their scores are masked); values that are not finite go to first_odd
  // where some row does not see all of the step's keys (careful: always).
  bool careful = false;
  auto settle_v = [&](int step, const Place& x, char* tile) {
    const int p0 = first_key(step) + gw * kWaveRows;
    bool all = true;
#pragma unroll
    for (int u = 0; u < kWaveUnits; ++u) all = all && x.ok[u];
    if (!careful && first_key(step) + Sh::kKeys <= tile_first && all) return;
    char* vt = tile + to + 16 * lane;
#pragma unroll
    for (int i = 0; i < Sh::kPerThread; ++i) {
      const int r = i * Sh::kRowsPerLoad + srow;
      U4 v = *reinterpret_cast<const U4*>(vt + 1024 * i);
      if (!(x.ok[i * Sh::kRowsPerLoad / Sh::kUnit] && p0 + r < len)) {
        *reinterpret_cast<U4*>(vt + 1024 * i) = U4{};
        v = U4{};
      }
      bool odd = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) odd = odd || NotFinite<T>(v[e]);
      if (odd) {
        const int d0 = (sc ^ VSwizzle<T, kDim>(gw * kWaveRows + r)) * (16 / kBytes<T>);
#pragma unroll 1
        for (int e = 0; e < 16 / kBytes<T>; ++e) {
          const int word = e * kBytes<T> / 4, shift = kBytes<T> == 4 ? 0 : 16 * (e & 1);
          const uint32_t u = kBytes<T> == 4 ? v[word] : (v[word] >> shift) & 0xFFFFu;
          if (NotFinite<T>(u)) {
            atomicMin(&first_odd[OddKind<T>(u)][d0 + e], p0 + r);
            any_odd = 1;
            v[word] &= kBytes<T> == 4 ? 0u : 0xFFFF0000u >> shift;
          }
        }
        *reinterpret_cast<U4*>(vt + 1024 * i) = v;
      }
    }
  };

  // where this lane reads: K row l % 32, chunks 2 i + h; V rows 4 h + 8 u + (0 .. 3),
  // chunk pairs of its 16 lanes' dimensions
  const int k_at = (lane & 31) * Sh::kRowBytes + 16 * (h * (kBytes<T> / 2) ^ KSwizzle<T, kDim>(lane & 31));
  int v_at[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = 8 * u + 4 * h + (lane & 15) / 4;
    v_at[u] = r * Sh::kRowBytes + 16 * ((2 * ((lane >> 4) & 1) + (lane & 3) / 2) ^ VSwizzle<T, kDim>(r)) + 8 * (lane & 1);
  }
  const float c = a.scale * 1.44269504088896341f;
  float m = kNegInf, l = 0.0f;
  F16v o[kDim / 32] = {};
  F16v s[Sh::kBlocks];
  auto scores = [&](const char* kt) {
    if constexpr (kBytes<T> == 4) {
      if (careful) {  // in f32 products: what is infinite stays that
        const char* qp = a.q.p + (first + token) * a.q.token_bytes + head * a.q.head_bytes + 8 * h * kBytes<T>;
        s[0] = F16v{};
#pragma unroll 1
        for (int i = 0; i < Sh::kQ; ++i) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const U4 x = *reinterpret_cast<const U4*>(kt + (k_at ^ (64 * i + 16 * half)));
            const U4 y = Load16(qp + 64 * i + 16 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0] = Mfma32F32(__uint_as_float(x[e]), __uint_as_float(y[e]), s[0]);
          }
        }
        return;
      }
    }
#pragma unroll
    for (int b = 0; b < Sh::kBlocks; ++b) {
#pragma unroll
      for (int i = 0; i < Sh::kQ; ++i) {
        const char* at = kt + 32 * b * Sh::kRowBytes;
        if constexpr (kBytes<T> == 4) {
          const U4 x = *reinterpret_cast<const U4*>(at + (k_at ^ 64 * i));
          const U4 y = *reinterpret_cast<const U4*>(at + (k_at ^ (64 * i + 16)));
          s[b] = i == 0 ? Mfma32x6First(Split8(x, y), q[i]) : Mfma32x6(Split8(x, y), q[i], s[b]);
        } else {
          const U4 x = *reinterpret_cast<const U4*>(at + (k_at ^ 32 * i));
          s[b] = i == 0 ? Mfma32First<T>(x, q[i]) : Mfma32<T>(x, q[i], s[b]);
        }
      }
    }
  };
  // Masks, the running maximum, weights in place of scores.
  auto weigh = [&](int key0, uint32_t pages) {
    if (key0 + Sh::kKeys - 1 > wave_first || pages != 0x01010101u) {
#pragma unroll
      for (int b = 0; b < Sh::kBlocks; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = 32 * b + 8 * (e / 4) + 4 * h + e % 4;
          const bool in = key0 + key <= limit && ((pages >> (8 * (key / Sh::kUnit))) & 1);
          s[b][e] = in ? s[b][e] : kNegInf;
        }
    }
    float top = kNegInf;
#pragma unroll
    for (int b = 0; b < Sh::kBlocks; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[b][e]);
    top = lanes::MaxXor32(top) * c;
    if (__any(top > m + kLazy)) {
      const float now = fmaxf(m, top), f = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= f;
#pragma unroll
      for (int w = 0; w < kDim / 32; ++w) o[w] *= f;
    }
    const float base = m == kNegInf ? 0.0f : m - kLift<T>;
#pragma unroll
    for (int b = 0; b < Sh::kBlocks; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[b][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], c, -base));
        l += s[b][e];
      }
  };
  auto add_values = [&](const char* vt) {
    if constexpr (kBytes<T> == 4) {
      // dimension (kDim / 32) m + w in row m of output block w
      const char* vl = vt + 4 * h * Sh::kRowBytes + (kDim / 8) * (lane & 31);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // keys 16 j + 4 h + {0 .. 3, 8 .. 11}, as the scores come
        Parts8 p, v[kDim / 32];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p.Set(e, Split3(s[0][8 * j + 2 * e], s[0][8 * j + 2 * e + 1]));
          const int key = 16 * j + 8 * (e / 2) + 2 * (e % 2);
          const float* x = reinterpret_cast<const float*>(vl + key * Sh::kRowBytes);
          const float* y = reinterpret_cast<const float*>(vl + (key + 1) * Sh::kRowBytes);
#pragma unroll
          for (int w = 0; w < kDim / 32; ++w) v[w].Set(e, Split3(x[w], y[w]));
        }
#pragma unroll
        for (int w = 0; w < kDim / 32; ++w) o[w] = Mfma32x6(v[w], p, o[w]);
      }
    } else {
      // The weights are rounded to the cache's 16 bits for the product (each
      // by at most half a step, as V itself was); the sum has them unrounded. The
      // output is 1.1 to 1.6 times as far from exact as its own rounding leaves it, the
      // more the flatter the weights (documents bf16: 2.2e-3 relative, 1.6e-3). Weights in two parts, as decode
      // has them, would make that 1.0, for another product: documents 410 -> 538 us,
      // six turns f16 14.1 -> 15.2. Positions that a group of sequences has in common
      // (kPrefix) have two parts, as the decode that they stand for.
      typedef short S4 __attribute__((ext_vector_type(4)));
      // A operand: dimensions 32 w .., keys 32 b + 16 j + 4 h + {0 .. 3, 8 .. 11}
#pragma unroll
      for (int b = 0; b < Sh::kBlocks; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          U4 p, rest;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            p[e] = Pack2<T>(s[b][8 * j + 2 * e], s[b][8 * j + 2 * e + 1]);
            if constexpr (kPrefix) rest[e] = Rest2<T>(s[b][8 * j + 2 * e], s[b][8 * j + 2 * e + 1], p[e]);
          }
#pragma unroll
          for (int w = 0; w < kDim / 32; ++w) {
            U4 v;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const char* at = vt + (v_at[u] ^ 64 * w) + (32 * b + 16 * j) * Sh::kRowBytes;
              const U2 x = __builtin_bit_cast(
                  U2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) S4*)at));
              v[2 * u] = x[0], v[2 * u + 1] = x[1];
            }
            if constexpr (kPrefix) o[w] = Mfma32<T>(v, rest, o[w]);
            o[w] = Mfma32<T>(v, p, o[w]);
          }
        }
    }
  };

  for (;;) {
    if constexpr (kSolo) {
      constexpr int kLoads = Sh::kPerThread;
      char* kt = tiles;
      char* vt = tiles + (kShared ? 0 : Sh::kTileBytes);
      Place now, next;
      if (steps > 0) {
        look_up(0);
        now = place_of(0);
        fetch_k(now, kt);
        if (!kShared) fetch_v(now, vt);
        look_up(1);
      }
      for (int step = 0; step < steps; ++step) {
        const int key0 = first_key(step);
        const bool mine = key0 <= wave_last && key0 < key_end, more = step + 1 < steps;
        next = place_of(step + 1);
        look_up(step + 2);
        // in flight: K, then V of this step (shared: K alone)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kShared ? 0 : kLoads) : "memory");
        if (mine) scores(kt);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read
        if (kShared)
          fetch_v(now, vt);
        else if (more)
          fetch_k(next, kt);
        uint32_t pages = 0;
#pragma unroll
        for (int u = 0; u < kWaveUnits; ++u) pages |= (now.ok[u] ? 1u : 0u) << (8 * u);
#pragma unroll
        for (int u = kWaveUnits; u < 4; ++u) pages |= 1u << (8 * u);
        if (mine) weigh(key0, pages);
        // in flight: V of this step, then K of the next (shared: V alone)
        if (more && !kShared)
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
        else
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (mine) {
          settle_v(step, now, vt);
          add_values(vt);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V is read
        if (more && kShared) fetch_k(next, kt);
        if (more && !kShared) fetch_v(next, vt);
        now = next;
      }
    } else {
      Place x;
      auto tile_of = [&](int step) { return tiles + (step & 1) * 2 * Sh::kTileBytes; };
      auto begin = [&](int step) {
        x = place_of(step);
        fetch_k(x, tile_of(step));
        fetch_v(x, tile_of(step) + Sh::kTileBytes);
        look_up(step + 1);
      };
      // the wave's rows have landed, and then all of the group's
      auto landed = [&](int step) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        settle_v(step, x, tile_of(step) + Sh::kTileBytes);
        if (lane == 0) {
#pragma unroll
          for (int u = 0; u < kWaveUnits; ++u)
            reinterpret_cast<volatile uint8_t*>(&page_ok[grp][step & 1])[gw * kWaveUnits + u] = x.ok[u] ? 1 : 0;
        }
        __syncthreads();
      };
      if (steps > 0) {
        look_up(0);
        begin(0);
        landed(0);
      }
      for (int step = 0; step < steps; ++step) {
        if (step + 1 < steps) begin(step + 1);
        const int key0 = first_key(step);
        if (key0 <= wave_last && key0 < key_end) {
          scores(tile_of(step));
          weigh(key0, page_ok[grp][step & 1]);
          add_values(tile_of(step) + Sh::kTileBytes);
        }
        if (step + 1 < steps) landed(step + 1);
      }
    }
    // In f32 an infinite key, query or value that a row sees comes out as NaN,
    // since the parts of an infinity are not one, and where weights have two parts
    // (kPrefix) an infinite value does, times a second part that is nothing. A tile
    // that ends with a NaN is gone through again, its values looked at and its
    // scores, in f32, in f32 products.
    if ((kBytes<T> == 2 && !kPrefix) || careful) break;
    bool nan = false;
#pragma unroll
    for (int w = 0; w < kDim / 32; ++w)
#pragma unroll
      for (int e = 0; e < 16; ++e) nan = nan || o[w][e] != o[w][e];
    if (!__syncthreads_or(nan)) break;
    careful = true;
    m = kNegInf, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kDim / 32; ++w) o[w] = F16v{};
  }

  l = lanes::AddXor32(l);
  if constexpr (kGroups == 1) {
    if (any_odd) {  // (all of it was found before the last step's barrier)
#pragma unroll
      for (int w = 0; w < kDim / 32; ++w)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[w][e] += OddSum(first_odd, DimOf<T, kDim>(w, 8 * (e / 4) + 4 * h + e % 4), limit);
    }
    const float inv = Inverse(m, l);
    if constexpr (kPrefix) {
      if (row0 + 32 * gw + (lane & 31) < n_rows) {
        const int64_t rows = static_cast<int64_t>(a.s.n_seqs) * a.n_heads;
        const int64_t out_row = static_cast<int64_t>(first + token) * a.n_heads + head;
        if (h == 0) PartStats(a, out_row)[by] = F2{m - kLift<T>, l};
        float* to = PartOut<kDim>(a, rows, out_row) + static_cast<int64_t>(by) * kDim;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if constexpr (kBytes<T> == 4 && kDim == 128)
            *reinterpret_cast<F4*>(to + 4 * (8 * (e / 4) + 4 * h + e % 4)) = F4{o[0][e], o[1][e], o[2][e], o[3][e]};
          else if constexpr (kBytes<T> == 4)
            *reinterpret_cast<F2*>(to + 2 * (8 * (e / 4) + 4 * h + e % 4)) = F2{o[0][e], o[1][e]};
        }
        if constexpr (kBytes<T> == 2) {
#pragma unroll
          for (int w = 0; w < kDim / 32; ++w)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<F4*>(to + 32 * w + 2 * e + 4 * h) = F4{o[w][e], o[w][e + 1], o[w][e + 2], o[w][e + 3]};
        }
      }
    } else if (row0 + 32 * gw + (lane & 31) < n_rows) {
      char* out = a.out.p + (first + token) * a.out.token_bytes + head * a.out.head_bytes;
      if constexpr (kBytes<T> == 4) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float* to = reinterpret_cast<float*>(out) + (kDim / 32) * (8 * (e / 4) + 4 * h + e % 4);
          if constexpr (kDim == 128)
            *reinterpret_cast<F4*>(to) = F4{o[0][e], o[1][e], o[2][e], o[3][e]} * inv;
          else
            *reinterpret_cast<F2*>(to) = F2{o[0][e], o[1][e]} * inv;
        }
      } else {
#pragma unroll
        for (int w = 0; w < kDim / 32; ++w)
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            Store4<T>(out + 2 * (32 * w + 2 * e + 4 * h), F4{o[w][e], o[w][e + 1], o[w][e + 2], o[w][e + 3]} * inv);
      }
    }
  } else {
    // The groups' states, joined in LDS where the tiles were.
    auto& sm = shared.sm;
    auto& sl = shared.sl;
    static_assert(kGroups == 1 || Sh::kRows * kDim * 4 <= kTiles * Sh::kTileBytes, "a group's state fits its tiles");
    // chunk c (four dimensions) of row r of group g
    auto at = [&](int g, int r, int c) {
      return reinterpret_cast<F4*>(lds + g * kTiles * Sh::kTileBytes + r * kDim * 4 + (c ^ (r & 15)) * 16);
    };
    const int r = 32 * gw + (lane & 31);
    if (h == 0) sm[grp][r] = m, sl[grp][r] = l;
    __syncthreads();
    float top = sm[0][r];
#pragma unroll
    for (int i = 1; i < kGroups; ++i) top = fmaxf(top, sm[i][r]);
    const float f = __builtin_amdgcn_exp2f(MaxDiff(m, top));
    if constexpr (kBytes<T> == 4 && kDim == 128) {
#pragma unroll
      for (int e = 0; e < 16; ++e) *at(grp, r, 8 * (e / 4) + 4 * h + e % 4) = F4{o[0][e], o[1][e], o[2][e], o[3][e]} * f;
    } else if constexpr (kBytes<T> == 4) {
#pragma unroll
      for (int e = 0; e < 16; e += 2)
        *at(grp, r, (8 * (e / 4) + 4 * h + e % 4) / 2) = F4{o[0][e], o[1][e], o[0][e + 1], o[1][e + 1]} * f;
    } else {
#pragma unroll
      for (int w = 0; w < kDim / 32; ++w)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *at(grp, r, (32 * w + 2 * e + 4 * h) / 4) = F4{o[w][e], o[w][e + 1], o[w][e + 2], o[w][e + 3]} * f;
    }
    __syncthreads();
    const bool odd = any_odd != 0;
    const bool alone = !kPrefix && (a.splits == 1 || RangeOf(max(keys, 1), a.splits) >= keys);
    for (int i = tid; i < Sh::kRows * (kDim / 4); i += 64 * Sh::kWaves) {
      const int ri = i / (kDim / 4), d = i % (kDim / 4) * 4, row_i = row0 + ri;
      if (row_i >= n_rows) break;
      float mi = sm[0][ri], li = 0.0f;
#pragma unroll
      for (int k = 1; k < kGroups; ++k) mi = fmaxf(mi, sm[k][ri]);
      F4 x = {};
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        li += sl[k][ri] * __builtin_amdgcn_exp2f(MaxDiff(sm[k][ri], mi));
        x += *at(k, ri, d / 4);
      }
      const int token_i = row_i / group, head_i = kh * group + row_i % group;
      if (odd) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += OddSum(first_odd, d + e, kPrefix ? len - 1 : pos0 + token_i);
      }
      if (alone) {
        Store4<T>(a.out.p + (first + token_i) * a.out.token_bytes + head_i * a.out.head_bytes + d * kBytes<T>,
                  x * Inverse(mi, li));
      } else {
        const int64_t rows = static_cast<int64_t>(kPrefix ? a.s.n_seqs : a.s.n_tokens) * a.n_heads;
        const int64_t out_row = static_cast<int64_t>(first + token_i) * a.n_heads + head_i;
        if (d == 0) PartStats(a, out_row)[by] = F2{kPrefix ? mi - kLift<T> : mi, li};
        *reinterpret_cast<F4*>(PartOut<kDim>(a, rows, out_row) + static_cast<int64_t>(by) * kDim + d) = x;
      }
    }
  }
}

}  // namespace paged
}  // namespace rpg

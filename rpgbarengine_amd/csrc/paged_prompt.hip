// Causal attention of packed new tokens over their sequences' cache pages
// (rpg_hip_paged_prompt, include/rpg_hip.h): token i of sequence s at position
// p = len - n_new + i,
//   out[h] = sum_{j <= p} p_j v_j,  p = softmax over j <= p of scale q[h] . k_j.
//
// One pass over the keys with a running maximum, sum and output. The query
// heads of a key head's group are folded into the rows: row r of a sequence is
// (token r / G, head r % G), so a key is staged once for the whole group and a
// few tokens still fill a tile. Workgroup (tile of 128 rows, key head), a wave
// for 32 rows; the key steps are staged in LDS (two buffers, the next step's
// loads in flight over the products). Scores and outputs are formed
// transposed, S^T = K Q^T and O^T = V^T P^T (32 x 32 tiles, columns = rows of
// the query tile): a lane keeps to one row, its scores are the B operand of
// the second product as they stand, and the key order that they come in is
// the one that V is read in (16-bit types: ds_read_b64_tr_b16 reads four keys
// of a dimension).

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
constexpr int kRows = 32 * kWaves;  // rows of a workgroup's tile

template <typename T, int kDim>
struct Shape {
  static constexpr int kKeys = kBytes<T> == 4 ? 32 : 64;      // keys of a step
  static constexpr int kBlocks = kKeys / 32;                  // 32-key score blocks
  static constexpr int kRowBytes = kDim * kBytes<T>;          // a cache row
  static constexpr int kChunks = kRowBytes / 16;              // its 16-byte chunks
  static constexpr int kPerThread = kKeys * kChunks / (64 * kWaves);
  static constexpr int kRowsPerLoad = 64 / kChunks;           // rows of a wave's load instruction
  static constexpr int kTileBytes = kKeys * kRowBytes;
  static constexpr int kQ = kDim * kBytes<T> / 32;            // 16-byte pieces of a query row per lane
};

// Chunk c of row r lies at chunk c ^ KSwizzle(r) or VSwizzle(r) of its LDS row.
// K: rows next to each other are read at one chunk; V (16-bit): four rows next
// to each other at four chunks. Both are linear over xor, so that an address
// is one lane's base, xored with a constant.
template <typename T, int kDim>
__device__ __forceinline__ constexpr int KSwizzle(int r) {
  return r & (Shape<T, kDim>::kChunks - 1);
}
template <typename T, int kDim>
__device__ __forceinline__ constexpr int VSwizzle(int r) {
  if constexpr (kBytes<T> == 4) return 0;  // read a row at a time
  return (((r & 3) << 2) | ((r >> 2) & 3)) & (Shape<T, kDim>::kChunks - 1);
}

// The sequence that row tile b belongs to, -1 for none: tiles of sequence s
// start at floor(starts[s] G / kRows) + s, which leaves each its
// ceil(n_new G / kRows) tiles wherever the starts lie.
__device__ __forceinline__ int SequenceOfTile(const Seqs& s, int group, int b) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int j = 0; j < s.n_seqs; j += 64) {
    const bool le = j + lane < s.n_seqs && s.starts[j + lane] * group / kRows + j + lane <= b;
    n += __popcll(__ballot(le));
  }
  return n - 1;
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

typedef __amdgpu_buffer_rsrc_t Rsrc;
// 16 bytes per lane from the resource to LDS, a wave's lanes side by side
__device__ __forceinline__ void LdsDma(Rsrc src, char* to, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)to, 16, voff, soff, 0, 0);
}

// grid (row tile x key head): key heads next to each other, the tiles with
// the most keys first.
template <typename T, int kDim>
__global__ __launch_bounds__(64 * kWaves, 2) void PromptKernel(AttentionArgs a) {
  using Sh = Shape<T, kDim>;
  __shared__ __align__(256) char lds[4 * Sh::kTileBytes];  // [2][K tile, V tile]
  __shared__ uint32_t page_ok[2];              // per buffer: a byte for each wave's rows
  __shared__ int any_odd, first_odd[kOddKinds][kDim];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = a.n_heads / a.c.n_kv;
  const int kh = blockIdx.x % a.c.n_kv;
  const int tile = static_cast<int>((gridDim.x - 1 - blockIdx.x) / a.c.n_kv);
  const int seq = SequenceOfTile(a.s, group, tile);
  if (seq < 0) return;
  const int first = a.s.starts[seq], n_new = a.s.starts[seq + 1] - first;
  if (first < 0 || n_new <= 0 || first > a.s.n_tokens - n_new) return;
  const int row0 = (tile - (first * group / kRows + seq)) * kRows, n_rows = n_new * group;
  if (row0 < 0 || row0 >= n_rows) return;
  const int len = Length(a.s, seq), pos0 = len - n_new;

  // this lane's row: a query token and head, and the last key it sees
  const int h = lane >> 5;
  const int row = min(row0 + 32 * wave + (lane & 31), n_rows - 1);
  const int token = row / group, head = kh * group + row % group;
  const int limit = pos0 + token;  // (< len)
  const int wave_first = pos0 + min(row0 + 32 * wave, n_rows - 1) / group;
  const int wave_last = pos0 + min(row0 + 32 * wave + 31, n_rows - 1) / group;
  const int tile_first = pos0 + row0 / group, tile_last = pos0 + min(row0 + kRows - 1, n_rows - 1) / group;
  const int steps = tile_last < 0 ? 0 : tile_last / Sh::kKeys + 1;

  U4 q[Sh::kQ];
  {
    const char* qp = a.q.p + (first + token) * a.q.token_bytes + head * a.q.head_bytes + 16 * h;
#pragma unroll
    for (int i = 0; i < Sh::kQ; ++i) q[i] = Load16(qp + 32 * i);
  }
  const int32_t* table = a.s.table + seq * a.s.table_stride;
  const int64_t head_off = kh * a.c.head_bytes;
  const int in_page = (1 << a.c.page_log2) - 1;
  if (tid == 0) any_odd = 0;
  for (int i = tid; i < kOddKinds * kDim; i += 64 * kWaves) first_odd[i / kDim][i % kDim] = INT32_MAX;
  __syncthreads();

  // Staging by LDS DMA: a wave brings kKeys / 4 rows (of one page), a lane
  // kPerThread chunks of K and of V, in LDS the wave's lanes side by side.
  constexpr int kWaveRows = Sh::kKeys / kWaves;
  const int srow = lane / Sh::kChunks, sc = lane % Sh::kChunks;
  const int row_from = srow * a.c.row_bytes;
  const int k_from = 16 * (sc ^ KSwizzle<T, kDim>(wave * kWaveRows + srow));
  const int v_from = 16 * (sc ^ VSwizzle<T, kDim>(wave * kWaveRows + srow));
  const int to = wave * kWaveRows * Sh::kRowBytes;
  bool ok = false;
  auto fetch = [&](int step) {
    const int p0 = step * Sh::kKeys + wave * kWaveRows;
    const int p = min(p0, (len - 1) & ~(kWaveRows - 1));  // rows that are there
    const int page = PageAt(a.c, table, p);
    ok = page >= 0 && p0 < len;
    const int64_t at = max(page, 0) * a.c.page_bytes + head_off + (p & in_page & ~(kWaveRows - 1)) * static_cast<int64_t>(a.c.row_bytes);
    const int bytes = (kWaveRows - 1) * a.c.row_bytes + Sh::kRowBytes;
    const Rsrc kb = __builtin_amdgcn_make_buffer_rsrc(a.c.k + at, 0, bytes, 0x00020000);
    const Rsrc vb = __builtin_amdgcn_make_buffer_rsrc(a.c.v + at, 0, bytes, 0x00020000);
    char* kt = lds + (step & 1) * 2 * Sh::kTileBytes + to;
#pragma unroll
    for (int i = 0; i < Sh::kPerThread; ++i) {
      const int up = i * Sh::kRowsPerLoad;
      LdsDma(kb, kt + 1024 * i, row_from + (k_from ^ 16 * KSwizzle<T, kDim>(up)), up * a.c.row_bytes);
      LdsDma(vb, kt + Sh::kTileBytes + 1024 * i, row_from + (v_from ^ 16 * VSwizzle<T, kDim>(up)), up * a.c.row_bytes);
    }
  };
  // The wave's rows have landed; what they need before the others read them.
  auto landed = [&](int step) {
    const int buf = step & 1, p0 = step * Sh::kKeys + wave * kWaveRows;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if ((step + 1) * Sh::kKeys > tile_first || !ok) {  // some row does not see all keys
      char* vt = lds + buf * 2 * Sh::kTileBytes + Sh::kTileBytes + to + 16 * lane;
#pragma unroll
      for (int i = 0; i < Sh::kPerThread; ++i) {
        // Rows past the sequence and of unnamed pages may hold anything, NaN
        // among it: zeros in place of their values (their scores are masked).
        const int r = i * Sh::kRowsPerLoad + srow;
        U4 v = *reinterpret_cast<const U4*>(vt + 1024 * i);
        const bool in = ok && p0 + r < len;
        bool odd = !in;
#pragma unroll
        for (int e = 0; e < 4; ++e) odd = odd || NotFinite<T>(v[e]);
        if (odd) {
          const int d0 = (sc ^ VSwizzle<T, kDim>(wave * kWaveRows + r)) * (16 / kBytes<T>);
#pragma unroll 1
          for (int e = 0; e < 16 / kBytes<T>; ++e) {
            const int word = e * kBytes<T> / 4, shift = kBytes<T> == 4 ? 0 : 16 * (e & 1);
            const uint32_t u = kBytes<T> == 4 ? v[word] : (v[word] >> shift) & 0xFFFFu;
            if (in && NotFinite<T>(u)) {
              atomicMin(&first_odd[OddKind<T>(u)][d0 + e], p0 + r);
              any_odd = 1;
            }
            if (!in || NotFinite<T>(u)) v[word] &= kBytes<T> == 4 ? 0u : 0xFFFF0000u >> shift;
          }
          *reinterpret_cast<U4*>(vt + 1024 * i) = v;
        }
      }
    }
    if (lane == 0) reinterpret_cast<volatile uint8_t*>(&page_ok[buf])[wave] = ok ? 1 : 0;
    __syncthreads();
  };

  // where this lane reads: K row l % 32, chunks 2 i + h; V rows 4 h + 8 u + (0 .. 3),
  // chunk pairs of its 16 lanes' dimensions
  const int k_at = (lane & 31) * Sh::kRowBytes + 16 * (h ^ KSwizzle<T, kDim>(lane & 31));
  int v_at[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = 8 * u + 4 * h + (lane & 15) / 4;
    v_at[u] = r * Sh::kRowBytes + 16 * ((2 * ((lane >> 4) & 1) + (lane & 3) / 2) ^ VSwizzle<T, kDim>(r)) + 8 * (lane & 1);
  }
  const float c = a.scale * 1.44269504088896341f;
  float m = kNegInf, l = 0.0f;
  F16v o[kDim / 32] = {};
  if (steps > 0) {
    fetch(0);
    landed(0);
  }
  for (int step = 0; step < steps; ++step) {
    if (step + 1 < steps) fetch(step + 1);
    const int key0 = step * Sh::kKeys;
    if (key0 <= wave_last) {
      const int buf = step & 1;
      const char* kt = lds + buf * 2 * Sh::kTileBytes;
      const char* vt = kt + Sh::kTileBytes;
      F16v s[Sh::kBlocks] = {};
#pragma unroll
      for (int b = 0; b < Sh::kBlocks; ++b) {
#pragma unroll
        for (int i = 0; i < Sh::kQ; ++i) {
          const U4 k = *reinterpret_cast<const U4*>(kt + (k_at ^ 32 * i) + 32 * b * Sh::kRowBytes);
          if constexpr (kBytes<T> == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[b] = Mfma32F32(__uint_as_float(k[e]), __uint_as_float(q[i][e]), s[b]);
          } else {
            s[b] = Mfma32<T>(k, q[i], s[b]);
          }
        }
      }
      const uint32_t pages = page_ok[buf];
      if (key0 + Sh::kKeys - 1 > wave_first || pages != 0x01010101u) {
#pragma unroll
        for (int b = 0; b < Sh::kBlocks; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int key = 32 * b + 8 * (e / 4) + 4 * h + e % 4;
            const bool in = key0 + key <= limit && ((pages >> (8 * (key / kWaveRows))) & 1);
            s[b][e] = in ? s[b][e] : kNegInf;
          }
      }
      float top = kNegInf;
#pragma unroll
      for (int b = 0; b < Sh::kBlocks; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, s[b][e]);
      top = lanes::MaxXor32(top) * c;
      if (__any(top > m)) {
        const float now = fmaxf(m, top), f = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= f;
#pragma unroll
        for (int w = 0; w < kDim / 32; ++w) o[w] *= f;
      }
      const float base = m == kNegInf ? 0.0f : m;
#pragma unroll
      for (int b = 0; b < Sh::kBlocks; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          s[b][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], c, -base));
          l += s[b][e];
        }
      if constexpr (kBytes<T> == 4) {
        // dimension (kDim / 32) m + w in row m of output block w
        const char* vl = vt + 4 * h * Sh::kRowBytes + (kDim / 8) * (lane & 31);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float* v = reinterpret_cast<const float*>(vl + (8 * (e / 4) + e % 4) * Sh::kRowBytes);
          float x[kDim / 32];
#pragma unroll
          for (int w = 0; w < kDim / 32; ++w) x[w] = v[w];
#pragma unroll
          for (int w = 0; w < kDim / 32; ++w) o[w] = Mfma32F32(x[w], s[0][e], o[w]);
        }
      } else {
        // The weights are rounded to the cache's 16 bits for the product (each
        // by at most half a step, as V itself was); the sum has them unrounded.
        typedef short S4 __attribute__((ext_vector_type(4)));
        // A operand: dimensions 32 w .., keys 32 b + 16 j + 4 h + {0 .. 3, 8 .. 11}
#pragma unroll
        for (int b = 0; b < Sh::kBlocks; ++b)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            U4 p;
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] = Pack2<T>(s[b][8 * j + 2 * e], s[b][8 * j + 2 * e + 1]);
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
              o[w] = Mfma32<T>(v, p, o[w]);
            }
          }
      }
    }
    if (step + 1 < steps) landed(step + 1);
  }

  l = lanes::AddXor32(l);
  if (any_odd) {
#pragma unroll
    for (int w = 0; w < kDim / 32; ++w)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int mm = 8 * (e / 4) + 4 * h + e % 4, d = kBytes<T> == 4 ? (kDim / 32) * mm + w : 32 * w + mm;
        const float inf = -kNegInf;
        if (first_odd[0][d] <= limit) o[w][e] += inf;
        if (first_odd[1][d] <= limit) o[w][e] -= inf;
        if (first_odd[2][d] <= limit) o[w][e] += __builtin_nanf("");
      }
  }
  // No key (positions before the cache's first, pages that are not there): zeros.
  const float inv = m == kNegInf && l == 0.0f ? 0.0f : 1.0f / l;
  if (row0 + 32 * wave + (lane & 31) < n_rows) {
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
          *reinterpret_cast<U2*>(out + 2 * (32 * w + 2 * e + 4 * h)) =
              U2{Pack2<T>(o[w][e] * inv, o[w][e + 1] * inv), Pack2<T>(o[w][e + 2] * inv, o[w][e + 3] * inv)};
    }
  }
}

template <typename T, int kDim>
void Launch(const AttentionArgs& a, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.s.n_tokens) * (a.n_heads / a.c.n_kv);
  const int64_t tiles = rows / kRows + a.s.n_seqs;
  RPG_CHECK(tiles * a.c.n_kv < (int64_t{1} << 31), "paged_prompt: too many rows for one launch");
  PromptKernel<T, kDim><<<static_cast<uint32_t>(tiles * a.c.n_kv), 64 * kWaves, 0, s>>>(a);
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

void Prompt(const AttentionArgs& a, hipStream_t s) {
  if (a.s.n_tokens == 0 || a.s.n_seqs == 0) return;
  if (a.c.type == kF32)
    LaunchDim<F32>(a, s);
  else if (a.c.type == kF16)
    LaunchDim<F16>(a, s);
  else
    LaunchDim<BF16>(a, s);
}

}  // namespace paged
}  // namespace rpg

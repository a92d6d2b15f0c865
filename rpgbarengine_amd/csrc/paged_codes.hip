// Rows into a cache of 8-bit codes and back (rpg_hip_quant_append,
// rpg_hip_quant_read, include/rpg_hip.h). A row y of a head (keys: normed and
// rotated as in paged_append.hip, in fp32; values as they are) is stored as
//   a = max |y|,  scale = a / M,  code = y M / a to the nearest, even at ties
// with M the largest code (127, 448), and read as code x scale. The quotient is
// fp32's, of the whole product y M: 16-bit rows have many that lie midway between two
// codes, and there y (M / a) would fall to either side. (Where fp32 rounds a quotient onto
// the middle the code is the even one: 16 of 12 million of f32 rows are not the nearest.)
//
// Bound: bytes, or for few tokens the launch and its dependent round trips. A row
// is one 16-byte load of 8, 16 or 32 adjacent lanes; the sum of squares, the
// rotation's partner and the maximum cross lanes by DPP. A wave's rows are of one kind
// (query, key or value), so that none goes through another's steps. Measured, 32 heads on
// 8 of 128, e4m3: 4060 tokens of 12 sequences bf16, 93 MB in 23.1 us (a large copy's rate:
// 18.3; the norm, the rotation and the codes' quotients are the rest: rows of any kind in
// a wave 26.2); 8 tokens f32 3.9 us in the kernel, 11 in the call. Read, 24 sessions, bf16:
// 37.3 us (33); one session of 1100 positions, int8 in f32, 7.4 (4.7 in a captured graph).

#include <hip/hip_runtime.h>

#include "codes_dev.h"
#include "common.h"
#include "lanes.h"
#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {
namespace {

// the largest over aligned groups of kLanes lanes
template <int kLanes>
__device__ __forceinline__ uint32_t GroupMax(uint32_t v) {
  v = max(v, lanes::Dpp<lanes::kQuadXor1>(v));
  v = max(v, lanes::Dpp<lanes::kQuadXor2>(v));
  v = max(v, lanes::Dpp<lanes::kRowHalfMirror>(v));
  if constexpr (kLanes >= 16) v = max(v, lanes::Dpp<lanes::kRowMirror>(v));
  if constexpr (kLanes >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
  }
  return v;
}

// Rows whose largest magnitude is below this are stored as zeros: the quotients
// and scales of all others are normal numbers.
constexpr float kLeast = 0x1p-112f;

// The largest scale with which the largest code is finite: a / M may be rounded up.
template <typename C>
constexpr float MostScale() {
  constexpr double kMax = 0x1.fffffep127;
  const float s = static_cast<float>(kMax / kLargest<C>);
  return static_cast<double>(s) * kLargest<C> <= kMax ? s : static_cast<float>(s * (1.0 - 0x1.8p-24));
}

// The codes of a lane's kPer values of a row, four to a register, and the scale.
template <typename C, int kPer, int kLanes>
__device__ __forceinline__ float Quantise(const float (&y)[kPer], uint32_t (&codes)[kPer / 4]) {
  uint32_t bits = 0;  // magnitudes are ordered as whole numbers, NaN above infinity
#pragma unroll
  for (int i = 0; i < kPer; ++i) bits = max(bits, __float_as_uint(y[i]) & 0x7FFFFFFFu);
  bits = GroupMax<kLanes>(bits);
  const float top = __uint_as_float(bits);
  const bool finite = bits < 0x7F800000u, some = finite && top >= kLeast;
  // by a power of two to where neither products nor reciprocals leave the range
  const float f = top >= 0x1p64f ? 0x1p-64f : top <= 0x1p-48f ? 0x1p64f : 1.0f;
  const float a = some ? top * f : 1.0f, inv = 1.0f / a;
  float q[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    // (y M in two parts: all of it counts)
    const float x = some ? y[i] * f : 0.0f, n = x * kLargest<C>, q0 = n * inv;
    q[i] = __builtin_fmaf(__builtin_fmaf(-q0, a, n) + __builtin_fmaf(x, kLargest<C>, -n), inv, q0);
  }
#pragma unroll
  for (int w = 0; w < kPer / 4; ++w) {
    if constexpr (__is_same(C, E4M3)) {
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * w], q[4 * w + 1], 0, false);
      codes[w] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * w + 2], q[4 * w + 3], c, true));
    } else {
      uint32_t c = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        c |= (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(q[4 * w + e]))) & 0xFFu) << (8 * e);
      codes[w] = c;
    }
  }
  return some ? fminf(top / kLargest<C>, MostScale<C>()) : finite ? 0.0f : __builtin_nanf("");
}

template <typename T, int kPer>
__device__ __forceinline__ void Widen(const U4& raw, float (&y)[kPer]) {
  if constexpr (kPer == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) Unpack2<T>(raw[i], &y[2 * i], &y[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __uint_as_float(raw[i]);
  }
}
template <typename T, int kPer>
__device__ __forceinline__ U4 Narrow(const float (&y)[kPer]) {
  U4 out;
  if constexpr (kPer == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = Pack2<T>(y[2 * i], y[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __float_as_uint(y[i]);
  }
  return out;
}

template <int kPer>
__device__ __forceinline__ void StoreCodes(char* to, const uint32_t (&codes)[kPer / 4]) {
  if constexpr (kPer == 8)
    *reinterpret_cast<U2*>(to) = U2{codes[0], codes[1]};
  else
    *reinterpret_cast<uint32_t*>(to) = codes[0];
}

// A wave's rows of one step: of one kind, so that what differs is decided by scalar
// branches. Rows that there are not are the last one again, not stored.
enum Kind { kQuery, kKey, kValue };
struct Unit {
  Kind kind;
  int head, n;  // the first head, the kind's heads
};
template <int kSub>
__device__ __forceinline__ Unit UnitOf(int u, int nq, int n_kv) {
  const int uq = (nq + kSub - 1) / kSub, uk = (n_kv + kSub - 1) / kSub;
  if (u < uq) return {kQuery, u * kSub, nq};
  if (u < uq + uk) return {kKey, (u - uq) * kSub, n_kv};
  return {kValue, (u - uq - uk) * kSub, n_kv};
}

// grid (token, kEach x 4 units of rows): a token's units are its query heads', then its
// key heads', then its value heads'.
template <typename C, typename T, int kDim, int kEach>
__global__ __launch_bounds__(256) void AppendCodesKernel(CodesAppendArgs args) {
  const AppendArgs& a = args.a;
  constexpr int kPer = 16 / kBytes<T>;  // elements of a lane
  constexpr int kLanes = kDim / kPer;   // lanes of a row
  constexpr int kSub = 64 / kLanes;     // rows of a unit
  const int t = blockIdx.x;
  const int lane = threadIdx.x & 63, c = lane % kLanes, sub = lane / kLanes;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nq = a.q.p != nullptr ? a.n_heads : 0;
  const int u0 = blockIdx.y * (kEach * 4) + wave;
  // The rows are on their way while the token's place is found.
  U4 raw[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const Unit u = UnitOf<kSub>(u0 + 4 * k, nq, a.c.n_kv);
    const Rows& from = u.kind == kQuery ? a.q : u.kind == kKey ? a.k : a.v;
    raw[k] = Load16(from.p + t * from.token_bytes + min(u.head + sub, u.n - 1) * from.head_bytes + 16 * c);
  }
  Sequence x;
  if (!FindSequence(a.s, [&](int end, int) { return end <= t; }, &x)) return;  // behind the last sequence
  const int pos = x.len - x.n_new + (t - x.first);
  // Tokens before the first sequence or at no position of the cache, and those
  // that the rotation table does not reach, are left out.
  if (t < x.first || pos < 0 || (a.rope != nullptr && pos >= a.rope_rows)) return;
  const int page = PageAt(a.c, a.s.table + x.seq * a.s.table_stride, pos);
  const int r = pos & ((1 << a.c.page_log2) - 1);
  const int64_t in_cache = max(page, 0) * a.c.page_bytes + r * static_cast<int64_t>(a.c.row_bytes) + kPer * c;
  const int64_t in_scales = max(page, 0) * args.scales.page_bytes + 4 * r;
  float cs[kPer], sn[kPer];
  if (a.rope != nullptr) {
    const float* p = a.rope + static_cast<int64_t>(pos) * kDim + (kPer * c) % (kDim / 2);
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const F4 u = *reinterpret_cast<const F4*>(p + i), v = *reinterpret_cast<const F4*>(p + kDim / 2 + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) cs[i + e] = u[e], sn[i + e] = c < kLanes / 2 ? -v[e] : v[e];
    }
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const Unit u = UnitOf<kSub>(u0 + 4 * k, nq, a.c.n_kv);
    const int head = u.head + sub;
    float y[kPer];
    Widen<T, kPer>(raw[k], y);
    if (u.kind != kValue) {
      const float* gain = u.kind == kQuery ? a.q_norm : a.k_norm;
      if (gain != nullptr) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum = __builtin_fmaf(y[i], y[i], sum);
        const float mean = GroupSum<kLanes>(sum) * (1.0f / kDim);
        const float scale = 1.0f / __builtin_sqrtf(mean + a.eps);
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
          const F4 g = *reinterpret_cast<const F4*>(gain + kPer * c + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[i + e] = y[i + e] * scale * g[e];
        }
      }
      if (a.rope != nullptr) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const float other = OtherHalf<kLanes>(y[i]);
          y[i] = __builtin_fmaf(y[i], cs[i], other * sn[i]);
        }
      }
    }
    if (u.kind == kQuery) {
      if (head < u.n)
        *reinterpret_cast<U4*>(a.q_out.p + t * a.q_out.token_bytes + head * a.q_out.head_bytes + 16 * c) =
            Narrow<T, kPer>(y);
      continue;
    }
    uint32_t codes[kPer / 4];
    const float scale = Quantise<C, kPer, kLanes>(y, codes);
    if (head >= u.n || page < 0) continue;
    StoreCodes<kPer>((u.kind == kValue ? a.c.v : a.c.k) + head * a.c.head_bytes + in_cache, codes);
    if (c == 0)
      *reinterpret_cast<float*>((u.kind == kValue ? args.scales.v : args.scales.k) + head * args.scales.head_bytes +
                                in_scales) = scale;
  }
}

// Rows of a thread: one for few tokens, whose time is that of their round trips (256
// tokens bf16 6.2 us in a captured graph with one, 6.9 with three), three from where the
// tokens alone fill the card (1040 tokens 11.3 and 10.2, f32 14.6 and 13.7; 4800 of bf16
// 29.5 and 24.8, two 28.0, four 25.4).
constexpr int kManyTokens = 1024;

template <typename C, typename T, int kDim, int kEach>
void LaunchAppendEach(const CodesAppendArgs& args, hipStream_t s) {
  const AppendArgs& a = args.a;
  constexpr int kSub = 64 * 16 / (kDim * kBytes<T>);
  const int64_t units = CeilDiv(a.q.p != nullptr ? a.n_heads : 0, kSub) + 2 * CeilDiv(a.c.n_kv, kSub);
  const uint32_t n = static_cast<uint32_t>(a.s.n_tokens);
  RPG_CHECK(n <= kMaxGroups, "%u new tokens in one launch", n);
  AppendCodesKernel<C, T, kDim, kEach><<<dim3(n, static_cast<uint32_t>(CeilDiv(units, 4 * kEach))), 256, 0, s>>>(args);
  HIP_CHECK(hipGetLastError());
}

template <typename C, typename T, int kDim>
void LaunchAppend(const CodesAppendArgs& a, hipStream_t s) {
  if (a.a.s.n_tokens >= kManyTokens)
    LaunchAppendEach<C, T, kDim, 3>(a, s);
  else
    LaunchAppendEach<C, T, kDim, 1>(a, s);
}

// grid (kEach tokens, 256 / kLanes rows of them): a token's rows are its key heads, then
// its value heads. Positions of unnamed pages give zeros.
template <typename C, typename T, int kDim, int kEach>
__global__ __launch_bounds__(256) void ReadCodesKernel(CodesReadArgs a) {
  constexpr int kPer = 16 / kBytes<T>;
  constexpr int kLanes = kDim / kPer;
  constexpr int kRows = 256 / kLanes;
  const int t0 = blockIdx.x * kEach;
  const int c = threadIdx.x % kLanes;
  const int row = blockIdx.y * kRows + threadIdx.x / kLanes, at_row = min(row, 2 * a.c.n_kv - 1);
  const bool is_v = at_row >= a.c.n_kv;
  const int head = is_v ? at_row - a.c.n_kv : at_row;
  // The tokens' places: mostly of one sequence.
  int pos[kEach];
  const int32_t* table[kEach];
  Sequence x = {};
  bool in = false;
  int end = t0;  // of what is known
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int t = t0 + k;
    if (t >= end && t < a.s.n_tokens) {
      in = FindSequence(a.s, [&](int e, int) { return e <= t; }, &x);
      end = in && t >= x.first ? x.first + x.n_new : t + 1;
    }
    pos[k] = in && t >= x.first && t < a.s.n_tokens ? x.len - x.n_new + (t - x.first) : -1;
    table[k] = a.s.table + x.seq * a.s.table_stride;
  }
  int page[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) page[k] = pos[k] >= 0 ? PageAt(a.c, table[k], pos[k]) : -1;
  uint32_t codes[kEach][kPer / 4];
  float scale[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int r = max(pos[k], 0) & ((1 << a.c.page_log2) - 1);
    const char* from = (is_v ? a.c.v : a.c.k) + head * a.c.head_bytes + max(page[k], 0) * a.c.page_bytes +
                       r * static_cast<int64_t>(a.c.row_bytes) + kPer * c;
    if constexpr (kPer == 8) {
      const U2 u = *reinterpret_cast<const U2*>(from);
      codes[k][0] = u[0], codes[k][1] = u[1];
    } else {
      codes[k][0] = *reinterpret_cast<const uint32_t*>(from);
    }
    scale[k] = *reinterpret_cast<const float*>((is_v ? a.scales.v : a.scales.k) + head * a.scales.head_bytes +
                                               max(page[k], 0) * a.scales.page_bytes + 4 * r);
  }
  const Rows& to = is_v ? a.v : a.k;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    if (pos[k] < 0 || row >= 2 * a.c.n_kv) continue;
    float y[kPer];
#pragma unroll
    for (int w = 0; w < kPer / 4; ++w) {
      const F2 lo = Floats2<C, false>(codes[k][w]), hi = Floats2<C, true>(codes[k][w]);
      y[4 * w] = lo[0], y[4 * w + 1] = lo[1], y[4 * w + 2] = hi[0], y[4 * w + 3] = hi[1];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) y[i] = page[k] >= 0 ? y[i] * scale[k] : 0.0f;
    *reinterpret_cast<U4*>(to.p + (t0 + k) * to.token_bytes + head * to.head_bytes + 16 * c) = Narrow<T, kPer>(y);
  }
}

template <typename C, typename T, int kDim, int kEach>
void LaunchReadEach(const CodesReadArgs& a, hipStream_t s) {
  constexpr int kPass = 256 * 16 / (kDim * kBytes<T>);
  const uint32_t n = static_cast<uint32_t>(CeilDiv(a.s.n_tokens, kEach));
  RPG_CHECK(n <= kMaxGroups, "%d tokens in one launch", a.s.n_tokens);
  ReadCodesKernel<C, T, kDim, kEach><<<dim3(n, static_cast<uint32_t>(CeilDiv(2 * a.c.n_kv, kPass))), 256, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
}

// Tokens of a workgroup: one for few, four for many (1000 tokens bf16 5.8 and 6.3 us in a
// captured graph, 2000 6.6 and 6.9, f32 8.8 and 8.3, 3000 8.4 and 8.1, f32 11.5 and 9.6;
// 48000 94.8 and 62.0, two 68.0, eight 64.1).
constexpr int kManyReads = 2048;

template <typename C, typename T, int kDim>
void LaunchRead(const CodesReadArgs& a, hipStream_t s) {
  if (a.s.n_tokens >= kManyReads)
    LaunchReadEach<C, T, kDim, 4>(a, s);
  else
    LaunchReadEach<C, T, kDim, 1>(a, s);
}

}  // namespace

void AppendCodes(const CodesAppendArgs& a, hipStream_t s) {
  if (a.a.s.n_tokens == 0 || a.a.s.n_seqs == 0) return;
  ByTypes(a.code, a.a.c, [&](auto code, auto type, auto dim) {
    LaunchAppend<decltype(code), decltype(type), decltype(dim)::value>(a, s);
  });
}

void ReadCodes(const CodesReadArgs& a, hipStream_t s) {
  if (a.s.n_tokens == 0 || a.s.n_seqs == 0) return;
  ByTypes(a.code, a.c, [&](auto code, auto type, auto dim) {
    LaunchRead<decltype(code), decltype(type), decltype(dim)::value>(a, s);
  });
}

}  // namespace paged
}  // namespace rpg

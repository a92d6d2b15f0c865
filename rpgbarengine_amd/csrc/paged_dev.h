// Device pieces that the paged attention kernels share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "lanes.h"
#include "paged.h"

namespace rpg {
namespace paged {

typedef float F2 __attribute__((ext_vector_type(2)));
typedef float F4 __attribute__((ext_vector_type(4)));
typedef float F16v __attribute__((ext_vector_type(16)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));
typedef uint32_t U2 __attribute__((ext_vector_type(2)));
typedef _Float16 H8 __attribute__((ext_vector_type(8)));
typedef __bf16 B8 __attribute__((ext_vector_type(8)));

struct F32 {};
struct F16 {};
struct BF16 {};

template <typename T>
constexpr int kBytes = 2;
template <>
inline constexpr int kBytes<F32> = 4;

constexpr float kNegInf = -__builtin_inff();

// Lengths, starts and page tables: nothing writes them while a kernel runs, so a
// wave-uniform one is read by a scalar load.
__device__ __forceinline__ int Uniform(const int32_t* p, int64_t i) {
  return *(const __attribute__((address_space(4))) int32_t*)(p + i);
}

// Positions of sequence s: 0 .. Length - 1.
__device__ __forceinline__ int ClampLength(const Seqs& s, int len) { return max(0, min(len, s.capacity)); }
__device__ __forceinline__ int Length(const Seqs& s, int seq) { return ClampLength(s, Uniform(s.lens, seq)); }

// The first sequence that `skip(its end among the packed tokens, its number)` is
// false for (skip is true up to some sequence): its tokens and length, in one
// round trip for up to 64 sequences, a lane for each. False: there is none, or
// its tokens do not lie in [0, n_tokens).
struct Sequence {
  int seq, first, n_new, len;
};
template <typename F>
__device__ __forceinline__ bool FindSequence(const Seqs& s, F&& skip, Sequence* out) {
  const int lane = threadIdx.x & 63;
  for (int j0 = 0; j0 < s.n_seqs; j0 += 64) {
    const int j = min(j0 + lane, s.n_seqs - 1);
    const int begin = s.starts[j], end = s.starts[j + 1], len = s.lens[j];
    const uint64_t skipped = __ballot(j0 + lane < s.n_seqs && skip(end, j));
    const int n = __popcll(skipped);
    if (n >= min(64, s.n_seqs - j0)) continue;
    out->seq = j0 + n;
    out->first = __builtin_amdgcn_readlane(begin, n);
    out->n_new = __builtin_amdgcn_readlane(end, n) - out->first;
    out->len = ClampLength(s, __builtin_amdgcn_readlane(len, n));
    return out->first >= 0 && out->n_new > 0 && out->first <= s.n_tokens - out->n_new;
  }
  return false;
}

// The page of the 16 positions from pos on (a page holds a multiple of 16), or
// -1 where the table names none: such a page is never read or written, and its
// positions take no part.
__device__ __forceinline__ int PageAt(const Cache& c, const int32_t* row, int pos) {
  const int page = Uniform(row, pos >> c.page_log2);
  return static_cast<uint32_t>(page) < static_cast<uint32_t>(c.n_pages) ? page : -1;
}

__device__ __forceinline__ U4 Load16(const char* p) {
  return *(const __attribute__((address_space(1))) U4*)p;
}

// two floats rounded to nearest even, packed
template <typename T>
__device__ __forceinline__ uint32_t Pack2(float a, float b) {
  if constexpr (__is_same(T, BF16)) {
    typedef __bf16 B2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, B2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
  } else {
    typedef _Float16 H2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, H2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
  }
}
template <typename T>
__device__ __forceinline__ void Unpack2(uint32_t u, float* a, float* b) {
  if constexpr (__is_same(T, BF16)) {
    *a = __uint_as_float(u << 16);
    *b = __uint_as_float(u & 0xFFFF0000u);
  } else {
    typedef _Float16 H2 __attribute__((ext_vector_type(2)));
    const H2 h = __builtin_bit_cast(H2, u);
    *a = static_cast<float>(h[0]);
    *b = static_cast<float>(h[1]);
  }
}

// What rounding to 16 bits took off two floats, rounded and packed the same way.
template <typename T>
__device__ __forceinline__ uint32_t Rest2(float a, float b, uint32_t rounded) {
  float x, y;
  Unpack2<T>(rounded, &x, &y);
  return Pack2<T>(a - x, b - y);
}

// An MFMA whose destination aliases its A or B registers gives wrong sums on
// gfx950, and the compiler allows it where the sum starts or moves to other
// registers. The empty asm behind such a product holds the sources past it. It
// also holds back the loads behind it, so running sums that stay where they are
// go without; a test reads the built kernels for overlaps.
// D[4 (l / 16) + e][l % 16] += sum_k A[l % 16][k] B[k][l % 16]; a lane holds the
// eight k of its l / 16 (16-bit types), the one k = l / 16 (f32).
template <typename T>
__device__ __forceinline__ F4 Mfma16(U4 a, U4 b, F4 c) {
  F4 r;
  if constexpr (__is_same(T, BF16))
    r = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0);
  else
    r = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
  asm volatile("" ::"v"(a), "v"(b), "v"(r));
  return r;
}
__device__ __forceinline__ F4 Mfma16F32(float a, float b, F4 c) {
  const F4 r = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
  asm volatile("" ::"v"(a), "v"(b), "v"(r));
  return r;
}
// D[8 (e / 4) + 4 (l / 32) + e % 4][l % 32] += sum_k A[l % 32][k] B[k][l % 32]; a
// lane holds the eight k of its l / 32 (16-bit types), the one k = l / 32 (f32).
__device__ __forceinline__ F16v Mfma32F32(float a, float b, F16v c) {
  const F16v r = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  asm volatile("" ::"v"(a), "v"(b), "v"(r));
  return r;
}
template <typename T>
__device__ __forceinline__ F16v Mfma32(U4 a, U4 b, F16v c) {
  if constexpr (__is_same(T, BF16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
}
// the first product of a sum
template <typename T>
__device__ __forceinline__ F16v Mfma32First(U4 a, U4 b) {
  const F16v r = Mfma32<T>(a, b, F16v{});
  asm volatile("" ::"v"(a), "v"(b), "v"(r));
  return r;
}

// x = hi + mid + lo exactly: three bf16 parts of 8 bits each (truncated, so that
// no finite value becomes infinite), for a pair of floats. Not for values that
// are not finite: inf - inf.
struct Parts {
  uint32_t hi, mid, lo;
};
__device__ __forceinline__ float Top8(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t Tops(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ Parts Split3(float a, float b) {
  Parts p;
  p.hi = Tops(a, b);
  a -= Top8(a);
  b -= Top8(b);
  p.mid = Tops(a, b);
  a -= Top8(a);
  b -= Top8(b);
  p.lo = Tops(a, b);
  return p;
}
struct Parts8 {
  U4 hi, mid, lo;
  __device__ __forceinline__ void Set(int i, Parts p) { hi[i] = p.hi, mid[i] = p.mid, lo[i] = p.lo; }
};
// f32 products on the bf16 matrix units: the six products of parts down to
// 2^-16 of the whole (the dropped ones, mid lo, lo mid and lo lo, are 2^-23 of it
// on average, less than one rounding of fp32), 192 cycles for 16 keys or
// dimensions where the f32 instruction takes 512. Smallest first.
__device__ __forceinline__ F16v Mfma32x5(const Parts8& a, const Parts8& b, F16v c) {
  c = Mfma32<BF16>(a.hi, b.lo, c);
  c = Mfma32<BF16>(a.mid, b.mid, c);
  c = Mfma32<BF16>(a.mid, b.hi, c);
  c = Mfma32<BF16>(a.hi, b.mid, c);
  return Mfma32<BF16>(a.hi, b.hi, c);
}
__device__ __forceinline__ F16v Mfma32x6(const Parts8& a, const Parts8& b, F16v c) {
  return Mfma32x5(a, b, Mfma32<BF16>(a.lo, b.hi, c));
}
__device__ __forceinline__ F16v Mfma32x6First(const Parts8& a, const Parts8& b) {
  return Mfma32x5(a, b, Mfma32First<BF16>(a.lo, b.hi));
}

// A key range's positions are a multiple of this, a step of a decode workgroup (8 x
// 1088 bf16: 12.4 us, with 64 13.3).
constexpr int kRangeUnit = 128;

// Positions of one key range of a sequence of len positions.
__device__ __forceinline__ int RangeOf(int len, int splits) {
  return ((len - 1) / splits / kRangeUnit + 1) * kRangeUnit;
}

// x - y of maxima that may both be -inf (no key yet): then 0.
__device__ __forceinline__ float MaxDiff(float x, float y) { return x == y ? 0.0f : x - y; }

// Work: [row][splits] (maximum, sum), then (StatFloats) [row][splits][kDim] outputs
// that are not yet divided by the sum; row = query token x head.
__device__ __forceinline__ F2* PartStats(const AttentionArgs& a, int64_t row) {
  return reinterpret_cast<F2*>(a.work) + row * a.splits;
}
template <int kDim>
__device__ __forceinline__ float* PartOut(const AttentionArgs& a, int64_t rows, int64_t row) {
  return a.work + StatFloats(rows, a.splits) + row * a.splits * kDim;
}

template <typename T>
__device__ __forceinline__ void Store4(char* p, F4 x) {
  if constexpr (kBytes<T> == 4)
    *reinterpret_cast<F4*>(p) = x;
  else
    *reinterpret_cast<U2*>(p) = U2{Pack2<T>(x[0], x[1]), Pack2<T>(x[2], x[3])};
}

// 1 / l; no key at all (an empty sequence, pages that are not there): 0.
__device__ __forceinline__ float Inverse(float m, float l) { return m == kNegInf && l == 0.0f ? 0.0f : 1.0f / l; }

// Joins the n ranges of one row: out = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m).
// A workgroup's 256 threads are kDim / 4 columns of four dimensions times the
// parts that take the ranges in turn.
constexpr int kMaxSplits = 512;
template <typename T, int kDim>
__device__ __forceinline__ void JoinRow(const AttentionArgs& a, int64_t rows, int64_t row, int n, char* out) {
  constexpr int kThreadsD = kDim / 4, kParts = 256 / kThreadsD;
  __shared__ float weight[kMaxSplits];
  __shared__ float sm[4], sl[4];
  __shared__ __align__(16) float so[kParts][kDim];
  const int tid = threadIdx.x;
  const F2* stats = PartStats(a, row);
  F2 mine[kMaxSplits / 256];
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 256; ++i) {
    mine[i] = tid + 256 * i < n ? stats[tid + 256 * i] : F2{kNegInf, 0.0f};
    top = fmaxf(top, mine[i][0]);
  }
  top = lanes::WaveMaxF(top);
  if ((tid & 63) == 0) sm[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float l = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxSplits / 256; ++i) {
    const float f = __builtin_amdgcn_exp2f(MaxDiff(mine[i][0], top));
    if (tid + 256 * i < n) weight[tid + 256 * i] = f;
    l += mine[i][1] * f;
  }
  l = lanes::WaveSumF(l);
  if ((tid & 63) == 0) sl[tid >> 6] = l;
  __syncthreads();
  l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
  const int d = tid % kThreadsD * 4, part = tid / kThreadsD;
  const float* po = PartOut<kDim>(a, rows, row) + d;
  F4 o = {};
#pragma unroll 4
  for (int s = part; s < n; s += kParts) o += *reinterpret_cast<const F4*>(po + static_cast<int64_t>(s) * kDim) * weight[s];
  *reinterpret_cast<F4*>(&so[part][d]) = o;
  __syncthreads();
  if (part != 0) return;
#pragma unroll
  for (int p = 1; p < kParts; ++p) o += *reinterpret_cast<const F4*>(&so[p][d]);
  Store4<T>(out + d * kBytes<T>, o * Inverse(top, l));
}

}  // namespace paged
}  // namespace rpg

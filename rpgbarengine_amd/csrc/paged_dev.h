// Device pieces that the paged attention kernels share.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

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

// Positions of sequence s: 0 .. Length - 1.
__device__ __forceinline__ int Length(const Seqs& s, int seq) { return max(0, min(s.lens[seq], s.capacity)); }

// The page of the 16 positions from pos on (a page holds a multiple of 16), or
// -1 where the table names none: such a page is never read or written, and its
// positions take no part.
__device__ __forceinline__ int PageAt(const Cache& c, const int32_t* row, int pos) {
  const int page = row[pos >> c.page_log2];
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

// The empty asm behind a product keeps its sources live past it, so that the
// result is never allocated over them (an MFMA whose destination aliases its
// A or B registers gives wrong sums on gfx950).
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
template <typename T>
__device__ __forceinline__ F16v Mfma32(U4 a, U4 b, F16v c) {
  F16v r;
  if constexpr (__is_same(T, BF16))
    r = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0);
  else
    r = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
  asm volatile("" ::"v"(a), "v"(b), "v"(r));
  return r;
}
__device__ __forceinline__ F16v Mfma32F32(float a, float b, F16v c) {
  const F16v r = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
  asm volatile("" ::"v"(a), "v"(b), "v"(r));
  return r;
}

}  // namespace paged
}  // namespace rpg

// 8-bit codes of a cache (rpg_hip_quant_cache, include/rpg_hip.h) on the device:
// a code's value is exact in f16 and in bf16, so a product with it loses nothing.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "paged_dev.h"

namespace rpg {
namespace paged {

struct I8 {};
struct E4M3 {};

// the largest code
template <typename C>
constexpr float kLargest = __is_same(C, I8) ? 127.0f : 448.0f;

typedef _Float16 H2 __attribute__((ext_vector_type(2)));
typedef __bf16 B2 __attribute__((ext_vector_type(2)));

// codes 2 kHigh and 2 kHigh + 1 of four
template <typename C, bool kHigh>
__device__ __forceinline__ F2 Floats2(uint32_t u) {
  if constexpr (__is_same(C, E4M3)) return __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(u), kHigh);
  const int i = static_cast<int>(kHigh ? u >> 16 : u);
  return F2{static_cast<float>(static_cast<int8_t>(i)), static_cast<float>(static_cast<int8_t>(i >> 8))};
}
// the same as a pair of f16 or bf16
template <typename C, typename T, bool kHigh>
__device__ __forceinline__ uint32_t Halves2(uint32_t u) {
  if constexpr (__is_same(C, E4M3) && __is_same(T, F16)) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, kHigh));
  } else if constexpr (__is_same(C, E4M3)) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, kHigh));
  } else if constexpr (__is_same(T, F16)) {
    // 0x6400 + n is 1024 + n in f16; the code is n - 128
    const uint32_t n = __builtin_amdgcn_perm(0x64646464u, u ^ 0x80808080u, kHigh ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(H2, n) - H2{1152.0f, 1152.0f});
  } else {
    // a whole number up to 128 has its bits in a float's upper half
    const F2 x = Floats2<I8, kHigh>(u);
    return __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x07060302u);
  }
}

}  // namespace paged
}  // namespace rpg

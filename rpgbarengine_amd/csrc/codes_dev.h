// 8-bit codes of a cache (rpg_hip_quant_cache, include/rpg_hip.h) on the device:
// a code's value is exact in f16 and in bf16, so a product with it loses nothing.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {

struct I8 {};
struct E4M3 {};

// the largest code
template <typename C>
constexpr float kLargest = __is_same(C, I8) ? 127.0f : 448.0f;

typedef _Float16 H2 __attribute__((ext_vector_type(2)));

// codes 2 kHigh and 2 kHigh + 1 of four
template <typename C, bool kHigh>
__device__ __forceinline__ F2 Floats2(uint32_t u) {
  if constexpr (__is_same(C, E4M3)) return __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(u), kHigh);
  const int i = static_cast<int>(kHigh ? u >> 16 : u);
  return F2{static_cast<float>(static_cast<int8_t>(i)), static_cast<float>(static_cast<int8_t>(i >> 8))};
}
// codes of I8 plus 1152, as a pair of f16: 0x6400 + n is 1024 + n, the code is n - 128
template <bool kHigh>
__device__ __forceinline__ uint32_t Above1152(uint32_t u) {
  return __builtin_amdgcn_perm(0x64646464u, u ^ 0x80808080u, kHigh ? 0x04030402u : 0x04010400u);
}
// the same as a pair of f16 or bf16
template <typename C, typename T, bool kHigh>
__device__ __forceinline__ uint32_t Halves2(uint32_t u) {
  if constexpr (__is_same(C, E4M3) && __is_same(T, F16)) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, kHigh));
  } else if constexpr (__is_same(C, E4M3)) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, kHigh));
  } else if constexpr (__is_same(T, F16)) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(H2, Above1152<kHigh>(u)) - H2{1152.0f, 1152.0f});
  } else {
    // a whole number up to 128 has its bits in a float's upper half
    const F2 x = Floats2<I8, kHigh>(u);
    return __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x07060302u);
  }
}

// The value of lane i of each 16, to all of them: an operand modifier of the
// instruction that takes it. Scales of the rows that a lane's scores belong to come
// that way, a register for 16 of them.
template <int i>
__device__ __forceinline__ float OfLane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + i, 0xF, 0xF, true));
}
// x[e] * (v of lane e of the 16)
template <int e, int n, typename V>
__device__ __forceinline__ void ScaleBy(V& x, float v) {
  if constexpr (e < n) {
    x[e] *= OfLane<e>(v);
    ScaleBy<e + 1, n>(x, v);
  }
}

// eight codes as a product's operand
template <typename C, typename T>
__device__ __forceinline__ U4 Operand8(uint32_t x, uint32_t y) {
  return U4{Halves2<C, T, false>(x), Halves2<C, T, true>(x), Halves2<C, T, false>(y), Halves2<C, T, true>(y)};
}
// For rows of type T: what the keys' codes are multiplied as, the parts that a query
// takes (f32: three exact bf16 parts, Split3), and those of a weight times a
// value's scale, in bf16: of 8 bits each, so two are as fine as an f16 output's
// rounding, and three are all of an f32.
template <typename T>
struct KeyTypeOf {
  typedef BF16 type;
};
template <>
struct KeyTypeOf<F16> {
  typedef F16 type;
};
template <typename T>
using KeyType = typename KeyTypeOf<T>::type;
template <typename T>
constexpr int kQueryParts = kBytes<T> == 4 ? 3 : 1;
template <typename T>
constexpr int kWeightParts = kBytes<T> == 4 ? 3 : 2;

// eight elements of a query from p on: operand i of its parts
template <typename T, int kParts, int kQ>
__device__ __forceinline__ void LoadQuery(const char* p, int i, U4 (&q)[kParts][kQ]) {
  if constexpr (kBytes<T> == 4) {
    const U4 x = Load16(p), y = Load16(p + 16);
    Parts8 parts;
    parts.Set(0, Split3(__uint_as_float(x[0]), __uint_as_float(x[1])));
    parts.Set(1, Split3(__uint_as_float(x[2]), __uint_as_float(x[3])));
    parts.Set(2, Split3(__uint_as_float(y[0]), __uint_as_float(y[1])));
    parts.Set(3, Split3(__uint_as_float(y[2]), __uint_as_float(y[3])));
    q[0][i] = parts.hi, q[1][i] = parts.mid, q[2][i] = parts.lo;
  } else {
    q[0][i] = Load16(p);
  }
}

// Eight weights (times scales) as the parts of an operand.
template <int kParts>
struct WeightParts {
  U4 x[kParts];
  __device__ __forceinline__ void Set(int j, float a, float b) {
    if constexpr (kParts == 3) {
      const Parts p = Split3(a, b);
      x[0][j] = p.hi, x[1][j] = p.mid, x[2][j] = p.lo;
    } else {
      x[0][j] = Pack2<BF16>(a, b);
      if constexpr (kParts == 2) x[1][j] = Rest2<BF16>(a, b, x[0][j]);
    }
  }
};

// f(code, row type, dimensions) of a cache
template <typename F>
void ByTypes(int64_t code, const Cache& c, F&& f) {
  ByRows(c, [&](auto type, auto dim) {
    if (code == kI8)
      f(I8{}, type, dim);
    else
      f(E4M3{}, type, dim);
  });
}

}  // namespace paged
}  // namespace rpg

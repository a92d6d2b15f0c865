// Edits of logits before the sampler (rpg_hip_edit_logits, include/rpg_hip.h):
// per row, for a token that was seen in the row's history and was made c times
// behind its prompt,
//   x = x > 0 ? x / repetition : x * repetition      (seen)
//   x = x - frequency c - presence                   (c > 0)
//   x = x + bias                                     (listed)
//   x = -inf                                         (masked)
// in f32, rounded once at the store.
//
// Workgroup (slice of the vocabulary, row): it goes through the row's whole
// history and counts, in LDS, the tokens that lie in its slice, so that one
// launch does with no memory of its own; integer counts come out the same in
// any order. The slice's logits are on their way meanwhile.
//
// Bound: the logits, read and written.

#include <hip/hip_runtime.h>

#include "common.h"
#include "edit_rows.h"

namespace rpg {
namespace rows {
namespace {

typedef uint32_t U4 __attribute__((ext_vector_type(4)));

struct F32 {};
struct F16 {};
struct BF16 {};
template <typename T>
constexpr int kBytes = 2;
template <>
inline constexpr int kBytes<F32> = 4;

// element e of 16 bytes
template <typename T>
__device__ __forceinline__ float Get(const U4& u, int e) {
  if constexpr (kBytes<T> == 4) {
    return __uint_as_float(u[e]);
  } else {
    const uint32_t w = u[e / 2];
    if constexpr (__is_same(T, BF16)) return __uint_as_float(e % 2 ? w & 0xFFFF0000u : w << 16);
    const uint16_t h = static_cast<uint16_t>(e % 2 ? w >> 16 : w);
    return static_cast<float>(__builtin_bit_cast(_Float16, h));
  }
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

constexpr int kThreads = 256;
constexpr int kSlice = 4096;                // tokens of a workgroup
constexpr uint32_t kInPrompt = 0x80000000u;  // of a count: seen, whether made or not

// The parameters of a row.
struct Row {
  float repetition, presence, frequency;
};
__device__ __forceinline__ float Edited(float x, uint32_t count, const Row& r) {
  x = x > 0.0f ? x / r.repetition : x * r.repetition;
  const uint32_t made = count & ~kInPrompt;
  return made != 0 ? x - r.frequency * static_cast<float>(made) - r.presence : x;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void EditKernel(EditArgs a) {
  constexpr int kPer = 16 / kBytes<T>;                  // tokens of a load
  constexpr int kLoads = kSlice / (kThreads * kPer);    // loads of a thread
  __shared__ uint32_t count[kSlice];
  __shared__ uint32_t biased[kSlice];  // the last entry of the list that names the token, + 1
  const int row = blockIdx.y, base = blockIdx.x * kSlice, tid = threadIdx.x;
  const int size = min(kSlice, a.vocab - base);
  const char* in = a.logits + row * a.row_bytes + static_cast<int64_t>(base) * kBytes<T>;
  char* out = a.out + row * a.out_bytes + static_cast<int64_t>(base) * kBytes<T>;
  const int mask_row = a.mask == nullptr ? -1 : a.mask_rows != nullptr ? a.mask_rows[row] : row;
  const uint32_t* mask = mask_row >= 0 && mask_row < a.n_masks
                             ? reinterpret_cast<const uint32_t*>(a.mask) + mask_row * a.mask_stride + base / 32
                             : nullptr;
  // Where nothing but single tokens changes and the row stays where it is, only
  // those are touched.
  const bool sparse = in == out && mask == nullptr;
  // Whole 16 bytes where both rows lie at such places, tokens one by one elsewhere.
  const bool wide = ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  U4 x[kLoads];
  if (wide && !sparse) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int at = (j * kThreads + tid) * kPer;
      x[j] = at + kPer <= size ? *reinterpret_cast<const U4*>(in + at * kBytes<T>) : U4{};
    }
  }
  const bool lists = a.history != nullptr || a.bias_ids != nullptr;
  Row r = {1.0f, 0.0f, 0.0f};
  if (lists) {
    for (int i = tid; i < kSlice; i += kThreads) count[i] = 0;
    if (a.bias_ids != nullptr)
      for (int i = tid; i < kSlice; i += kThreads) biased[i] = 0;
    __syncthreads();
    if (a.history != nullptr) {
      if (a.repetition != nullptr) {
        r.repetition = a.repetition[row];
        if (!(r.repetition > 0.0f)) r.repetition = 1.0f;
      }
      if (a.presence != nullptr) r.presence = a.presence[row];
      if (a.frequency != nullptr) r.frequency = a.frequency[row];
      const int n = a.history_lens != nullptr ? max(0, min(a.history_lens[row], a.history_size)) : a.history_size;
      const int prompt = a.prompts != nullptr ? a.prompts[row] : 0;
      const int32_t* ids = a.history + row * a.history_stride;
      constexpr int kIds = 4;  // on their way together
      for (int i0 = tid; i0 < n; i0 += kIds * kThreads) {
        uint32_t at[kIds];
#pragma unroll
        for (int k = 0; k < kIds; ++k) at[k] = static_cast<uint32_t>(ids[min(i0 + k * kThreads, n - 1)]) - base;
#pragma unroll
        for (int k = 0; k < kIds; ++k) {
          const int i = i0 + k * kThreads;
          if (i >= n || at[k] >= static_cast<uint32_t>(size)) continue;
          if (i < prompt)
            atomicOr(&count[at[k]], kInPrompt);
          else
            atomicAdd(&count[at[k]], 1u);
        }
      }
    }
    if (a.bias_ids != nullptr) {
      const int32_t* ids = a.bias_ids + row * a.bias_ids_stride;
      for (int i = tid; i < a.n_biases; i += kThreads) {
        const uint32_t at = static_cast<uint32_t>(ids[i]) - base;
        if (at < static_cast<uint32_t>(size)) atomicMax(&biased[at], static_cast<uint32_t>(i) + 1);
      }
    }
    __syncthreads();
  }
  const float* bias = a.bias + row * a.bias_stride;
  auto edit = [&](float v, int at, uint32_t word) {
    if (lists) {
      const uint32_t c = count[at];
      if (c != 0) v = Edited(v, c, r);
      if (a.bias_ids != nullptr) {
        const uint32_t b = biased[at];
        if (b != 0) v += bias[b - 1];
      }
    }
    return (word >> (at % 32)) & 1 ? v : -__builtin_inff();
  };
  auto untouched = [&](int at) {
    return !lists || (count[at] == 0 && (a.bias_ids == nullptr || biased[at] == 0));
  };
  auto word_of = [&](int at) { return mask != nullptr ? mask[at / 32] : ~0u; };
  if (wide) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int at = (j * kThreads + tid) * kPer;  // (32 tokens of a mask's word hold whole loads)
      if (at + kPer > size) continue;
      if (sparse) {
        bool same = true;
#pragma unroll
        for (int e = 0; e < kPer; ++e) same = same && untouched(at + e);
        if (same) continue;
        x[j] = *reinterpret_cast<const U4*>(in + at * kBytes<T>);
      }
      const uint32_t word = word_of(at);
      U4 y;
      if constexpr (kBytes<T> == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __float_as_uint(edit(Get<T>(x[j], e), at + e, word));
      } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          y[e / 2] = Pack2<T>(edit(Get<T>(x[j], e), at + e, word), edit(Get<T>(x[j], e + 1), at + e + 1, word));
      }
      *reinterpret_cast<U4*>(out + at * kBytes<T>) = y;
    }
  }
  // What is left of a row, or all of it.
  for (int at = (wide ? size / kPer * kPer : 0) + tid; at < size; at += kThreads) {
    if (sparse && untouched(at)) continue;
    const uint32_t word = word_of(at);
    if constexpr (kBytes<T> == 4) {
      reinterpret_cast<float*>(out)[at] = edit(reinterpret_cast<const float*>(in)[at], at, word);
    } else {
      const U4 one = {reinterpret_cast<const uint16_t*>(in)[at], 0, 0, 0};
      reinterpret_cast<uint16_t*>(out)[at] = static_cast<uint16_t>(Pack2<T>(edit(Get<T>(one, 0), at, word), 0.0f));
    }
  }
}

template <typename T>
void Launch(const EditArgs& a, hipStream_t s) {
  EditKernel<T><<<dim3(static_cast<uint32_t>((a.vocab + kSlice - 1) / kSlice), a.rows), kThreads, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
}

}  // namespace

void Edit(const EditArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  if (a.type == kF32)
    Launch<F32>(a, s);
  else if (a.type == kF16)
    Launch<F16>(a, s);
  else
    Launch<BF16>(a, s);
}

}  // namespace rows
}  // namespace rpg

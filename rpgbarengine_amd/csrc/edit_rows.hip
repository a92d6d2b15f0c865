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
// Bound: the logits, read and written; the slices' walks through the history beside it.
// Measured: 192 rows of 151936 bf16, histories of up to 4096, 32 biases, masks on 0.3 of them,
// 117 MB in 27.8 us (a plain copy 23.9; without histories 23.6; 24.2 in a captured graph);
// 8 rows f32 9.6 us a call, 5.1 in a captured graph. Slices of 4096 by 256 threads, which
// walk a history twice as often: 30.2 -> 32.1, of 16384 by 1024: 31.7. Edits one by one,
// by the bits of what was touched: 27.8, 30.2 with all tokens of a load that holds one.
// Biases in their own array in LDS instead of the upper bits of the counts: half the
// workgroups to a compute unit, 44.7 (then 32).

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

constexpr int kThreads = 512;
constexpr int kSlice = 8192;  // tokens of a workgroup
// A token's word in LDS: how often it was made (up to 2^20), whether the prompt has it,
// and above that the last entry of the biases that names it, + 1.
constexpr uint32_t kInPrompt = 1u << 21, kMade = kInPrompt - 1;
constexpr int kBiasShift = 22;
static_assert(kMaxBiases < 1 << (32 - kBiasShift) && kMaxHistory <= kMade, "fields of a word");

// The parameters of a row.
struct Row {
  float repetition, presence, frequency;
};
__device__ __forceinline__ float Edited(float x, uint32_t count, const Row& r) {
  x = x > 0.0f ? x / r.repetition : x * r.repetition;
  const uint32_t made = count & kMade;
  return made != 0 ? x - r.frequency * static_cast<float>(made) - r.presence : x;
}

// -inf, in 16 bits twice
template <typename T>
constexpr uint32_t kLow = __is_same(T, BF16) ? 0xFF80FF80u : __is_same(T, F16) ? 0xFC00FC00u : 0xFF800000u;

template <typename T>
__global__ __launch_bounds__(kThreads) void EditKernel(EditArgs a) {
  constexpr int kPer = 16 / kBytes<T>;                // tokens of a load
  constexpr int kLoads = kSlice / (kThreads * kPer);  // loads of a thread
  __shared__ __align__(16) uint32_t count[kSlice];
  __shared__ float bias_of[kMaxBiases];
  __shared__ uint32_t touched[kSlice / 32];  // a bit for each token that history or biases name
  const int row = blockIdx.y, base = blockIdx.x * kSlice, tid = threadIdx.x;
  const int size = min(kSlice, a.vocab - base);
  const char* in = a.logits + row * a.row_bytes + static_cast<int64_t>(base) * kBytes<T>;
  char* out = a.out + row * a.out_bytes + static_cast<int64_t>(base) * kBytes<T>;
  // Everything that the first round trip can bring is on its way before anything
  // is waited for: logits, the history's first tokens (whatever its length), the
  // list of biases, the row's parameters.
  // Whole 16 bytes where both rows lie at such places, tokens one by one elsewhere.
  const bool wide = ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  auto place = [&](int j) { return (j * kThreads + tid) * kPer; };
  U4 x[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const bool here = wide && (in != out || a.mask != nullptr) && place(j) + kPer <= size;
    x[j] = here ? *reinterpret_cast<const U4*>(in + place(j) * kBytes<T>) : U4{};
  }
  constexpr int kIds = 4;  // tokens of a thread that are on their way together
  const int32_t* ids = a.history + row * a.history_stride;
  uint32_t at[kIds];
  const bool history = a.history_size > 0;
  auto bring = [&](int i0) {
#pragma unroll
    for (int k = 0; k < kIds; ++k) at[k] = static_cast<uint32_t>(ids[min(i0 + k * kThreads + tid, a.history_size - 1)]) - base;
  };
  if (history) bring(0);
  uint32_t bias_at = ~0u;
  float bias_value = 0.0f;
  if (tid < a.n_biases) {
    bias_at = static_cast<uint32_t>(a.bias_ids[row * a.bias_ids_stride + tid]) - base;
    bias_value = a.bias[row * a.bias_stride + tid];
  }
  Row r = {1.0f, 0.0f, 0.0f};
  if (a.repetition != nullptr) r.repetition = a.repetition[row];
  if (a.presence != nullptr) r.presence = a.presence[row];
  if (a.frequency != nullptr) r.frequency = a.frequency[row];
  const int n = a.history_lens != nullptr ? max(0, min(a.history_lens[row], a.history_size)) : a.history_size;
  const int prompt = a.prompts != nullptr ? a.prompts[row] : 0;
  const int mask_row = a.mask == nullptr ? -1 : a.mask_rows != nullptr ? a.mask_rows[row] : row;
#pragma unroll
  for (int i = 0; i < kSlice; i += 4 * kThreads) {
    *reinterpret_cast<U4*>(&count[i + 4 * tid]) = U4{};
  }
  if (tid < kSlice / 32) touched[tid] = 0;
  const uint32_t* mask = mask_row >= 0 && mask_row < a.n_masks
                             ? reinterpret_cast<const uint32_t*>(a.mask) + mask_row * a.mask_stride + base / 32
                             : nullptr;
  // Where nothing but single tokens changes and the row stays where it is, only
  // those are touched.
  const bool sparse = in == out && mask == nullptr;
  uint32_t word[kLoads];  // of the mask (32 tokens hold whole loads)
#pragma unroll
  for (int j = 0; j < kLoads; ++j)
    word[j] = mask != nullptr && wide && place(j) + kPer <= size ? mask[place(j) / 32] : ~0u;
  if (!(r.repetition > 0.0f)) r.repetition = 1.0f;
  __syncthreads();
  if (history) {
    for (int i0 = 0;;) {
#pragma unroll
      for (int k = 0; k < kIds; ++k) {
        const int i = i0 + k * kThreads + tid;
        if (i >= n || at[k] >= static_cast<uint32_t>(size)) continue;
        if (i < prompt)
          atomicOr(&count[at[k]], kInPrompt);
        else
          atomicAdd(&count[at[k]], 1u);
        atomicOr(&touched[at[k] / 32], 1u << (at[k] % 32));
      }
      i0 += kIds * kThreads;
      if (i0 >= n) break;
      bring(i0);
    }
  }
  __syncthreads();
  if (a.n_biases > 0) {
    for (int i = tid; i < a.n_biases; i += kThreads) {
      if (i != tid) {
        bias_at = static_cast<uint32_t>(a.bias_ids[row * a.bias_ids_stride + i]) - base;
        bias_value = a.bias[row * a.bias_stride + i];
      }
      bias_of[i] = bias_value;
      if (bias_at >= static_cast<uint32_t>(size)) continue;
      // (entries of one token differ in the upper bits alone)
      const uint32_t low = count[bias_at] & (kInPrompt | kMade);
      atomicMax(&count[bias_at], static_cast<uint32_t>(i + 1) << kBiasShift | low);
      atomicOr(&touched[bias_at / 32], 1u << (bias_at % 32));
    }
    __syncthreads();
  }
  auto edit = [&](float v, int at) {
    const uint32_t c = count[at];
    if ((c & (kInPrompt | kMade)) != 0) v = Edited(v, c, r);
    return c >> kBiasShift != 0 ? v + bias_of[(c >> kBiasShift) - 1] : v;
  };
  if (wide) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int at = place(j);
      if (at + kPer > size) continue;
      const uint32_t here = touched[at / 32] >> (at % 32) & ((1u << kPer) - 1);
      if (sparse) {
        if (here == 0) continue;
        x[j] = *reinterpret_cast<const U4*>(in + at * kBytes<T>);
      }
      U4 y = x[j];
      for (uint32_t left = here; left != 0; left &= left - 1) {
        const int e = __builtin_ctz(left), i = e * kBytes<T> / 4;
        uint32_t w = i < 2 ? (i == 0 ? y[0] : y[1]) : i == 2 ? y[2] : y[3];
        if constexpr (kBytes<T> == 4) {
          w = __float_as_uint(edit(__uint_as_float(w), at + e));
        } else {
          const int shift = e % 2 * 16;
          const uint32_t v = Pack2<T>(edit(Get<T>(U4{w >> shift, 0, 0, 0}, 0), at + e), 0.0f) & 0xFFFFu;
          w = (w & ~(0xFFFFu << shift)) | v << shift;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = k == i ? w : y[k];
      }
      if (mask != nullptr) {
        const uint32_t bits = word[j] >> (at % 32);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t keep;
          if constexpr (kBytes<T> == 4)
            keep = 0u - (bits >> e & 1);
          else
            keep = ((0u - (bits >> (2 * e) & 1)) & 0xFFFFu) | (0u - (bits >> (2 * e + 1) & 1)) << 16;
          y[e] = (y[e] & keep) | (kLow<T> & ~keep);
        }
      }
      *reinterpret_cast<U4*>(out + at * kBytes<T>) = y;
    }
  }
  // What is left of a row, or all of it.
  for (int at = (wide ? size / kPer * kPer : 0) + tid; at < size; at += kThreads) {
    const bool here = touched[at / 32] >> (at % 32) & 1;
    if (sparse && !here) continue;
    const bool low = mask != nullptr && !(mask[at / 32] >> (at % 32) & 1);
    if constexpr (kBytes<T> == 4) {
      float v = reinterpret_cast<const float*>(in)[at];
      if (here) v = edit(v, at);
      reinterpret_cast<float*>(out)[at] = low ? -__builtin_inff() : v;
    } else {
      uint32_t v = reinterpret_cast<const uint16_t*>(in)[at];
      if (here) v = Pack2<T>(edit(Get<T>(U4{v, 0, 0, 0}, 0), at), 0.0f);
      reinterpret_cast<uint16_t*>(out)[at] = static_cast<uint16_t>(low ? kLow<T> : v);
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

// New tokens of many sequences into their cache pages (rpg_hip_paged_append,
// include/rpg_hip.h): per head row x of a token at position p
//   y = x / sqrt(mean(x^2) + eps) * gain          (keys and queries; optional)
//   out[i] = y[i] c[i] - y[i + D/2] s[i],  out[i + D/2] = y[i + D/2] c[i] + y[i] s[i]
// with (c, s) = row p of the rotation table (optional), as the engine's own
// QK-norm and RoPE (reference src/qwen3.cc:139-167); values are copied.
// Everything between the load and the one rounding at the store is fp32.
//
// Bound: bytes, or for a decode step's few tokens the launch and its two
// dependent round trips (the sequence's place, then the rows and the page). A
// row is one 16-byte load of 8, 16 or 32 adjacent lanes: the sum of squares
// and the rotation's partner half cross lanes by DPP, nothing goes through
// LDS, and a row is stored as it was loaded.

#include <hip/hip_runtime.h>

#include "common.h"
#include "lanes.h"
#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {
namespace {

// the number of j in 1 .. n with starts[j] <= t, over the wave's lanes
__device__ __forceinline__ int SequenceOf(const Seqs& s, int t) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int j = 0; j < s.n_seqs; j += 64) {
    const bool le = j + lane < s.n_seqs && s.starts[j + lane + 1] <= t;
    before += __popcll(__ballot(le));
  }
  return before;
}

// sum over aligned groups of kLanes lanes
template <int kLanes>
__device__ __forceinline__ float GroupSum(float v) {
  v += lanes::DppF<lanes::kQuadXor1>(v);
  v += lanes::DppF<lanes::kQuadXor2>(v);
  v += lanes::DppF<lanes::kRowHalfMirror>(v);
  if constexpr (kLanes >= 16) v += lanes::DppF<lanes::kRowMirror>(v);
  if constexpr (kLanes >= 32) v = lanes::AddXor16(v);
  return v;
}

// the value of the lane kLanes / 2 further in its group of kLanes
template <int kLanes>
__device__ __forceinline__ float OtherHalf(float v) {
  if constexpr (kLanes == 16) return lanes::DppF<lanes::kRowRor8>(v);
  return __shfl_xor(v, kLanes / 2, 64);
}

// grid (token, 256 / kLanes rows of it): the token's rows are its query heads,
// then its key heads, then its value heads.
template <typename T, int kDim>
__global__ __launch_bounds__(256) void AppendKernel(AppendArgs a) {
  constexpr int kPer = 16 / kBytes<T>;      // elements of a lane
  constexpr int kLanes = kDim / kPer;       // lanes of a row
  const int t = blockIdx.x;
  const int row = blockIdx.y * (256 / kLanes) + threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  const int nq = a.q.p != nullptr ? a.n_heads : 0;
  const bool in = row < nq + 2 * a.c.n_kv;
  const bool is_q = row < nq, is_v = row >= nq + a.c.n_kv;
  const int head = is_q ? row : is_v ? row - nq - a.c.n_kv : row - nq;
  const Rows& from = is_q ? a.q : is_v ? a.v : a.k;
  U4 raw = {};
  if (in) raw = Load16(from.p + t * from.token_bytes + head * from.head_bytes + 16 * c);
  const int seq = SequenceOf(a.s, t);
  if (seq >= a.s.n_seqs) return;  // behind the last sequence
  const int first = a.s.starts[seq], n_new = a.s.starts[seq + 1] - first;
  const int pos = Length(a.s, seq) - n_new + (t - first);
  // Tokens before the first sequence or at no position of the cache, and those
  // that the rotation table does not reach, are left out.
  if (t < first || pos < 0 || (a.rope != nullptr && pos >= a.rope_rows)) return;
  const int page = PageAt(a.c, a.s.table + seq * a.s.table_stride, pos);
  U4 out = raw;
  if (!is_v) {
    float x[kPer];
    if constexpr (kPer == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) Unpack2<T>(raw[i], &x[2 * i], &x[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(raw[i]);
    }
    const float* gain = is_q ? a.q_norm : a.k_norm;
    if (gain != nullptr) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) sum = __builtin_fmaf(x[i], x[i], sum);
      const float mean = GroupSum<kLanes>(sum) * (1.0f / kDim);
      const float scale = 1.0f / __builtin_sqrtf(mean + a.eps);
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        const F4 g = *reinterpret_cast<const F4*>(gain + kPer * c + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i + e] = x[i + e] * scale * g[e];
      }
    }
    if (a.rope != nullptr) {
      const float* r = a.rope + static_cast<int64_t>(pos) * kDim + (kPer * c) % (kDim / 2);
      const float sign = c < kLanes / 2 ? -1.0f : 1.0f;
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        const F4 cs = *reinterpret_cast<const F4*>(r + i), sn = *reinterpret_cast<const F4*>(r + kDim / 2 + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float other = OtherHalf<kLanes>(x[i + e]);
          x[i + e] = __builtin_fmaf(x[i + e], cs[e], sign * other * sn[e]);
        }
      }
    }
    if constexpr (kPer == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = Pack2<T>(x[2 * i], x[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = __float_as_uint(x[i]);
    }
  }
  if (!in || (!is_q && page < 0)) return;
  char* to = is_q ? a.q_out.p + t * a.q_out.token_bytes + head * a.q_out.head_bytes
                  : (is_v ? a.c.v : a.c.k) + page * a.c.page_bytes + head * a.c.head_bytes +
                        (pos & ((1 << a.c.page_log2) - 1)) * static_cast<int64_t>(a.c.row_bytes);
  *reinterpret_cast<U4*>(to + 16 * c) = out;
}

template <typename T>
void Launch(const AppendArgs& a, hipStream_t s) {
  const int rows = (a.q.p != nullptr ? a.n_heads : 0) + 2 * a.c.n_kv;
  const int lanes_per_row = a.c.head_dim * kBytes<T> / 16;
  const dim3 grid(static_cast<uint32_t>(a.s.n_tokens), static_cast<uint32_t>(CeilDiv(rows, 256 / lanes_per_row)));
  if (a.c.head_dim == 128)
    AppendKernel<T, 128><<<grid, 256, 0, s>>>(a);
  else
    AppendKernel<T, 64><<<grid, 256, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
}

}  // namespace

void Append(const AppendArgs& a, hipStream_t s) {
  if (a.s.n_tokens == 0 || a.s.n_seqs == 0) return;
  if (a.c.type == kF32)
    Launch<F32>(a, s);
  else if (a.c.type == kF16)
    Launch<F16>(a, s);
  else
    Launch<BF16>(a, s);
}

}  // namespace paged
}  // namespace rpg

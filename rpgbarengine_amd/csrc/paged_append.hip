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
// LDS, and a row is stored as it was loaded. Measured: 4060 tokens of 12
// sequences, 32 heads on 8 of 128, bf16, 101 MB in 24 us (a large copy's rate: 20);
// 8 tokens, f32: 3.5 us in the kernel, 10 in the call.

#include <hip/hip_runtime.h>

#include "common.h"
#include "lanes.h"
#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {
namespace {

// grid (token, kEach x 256 / kLanes rows of it): the token's rows are its query
// heads, then its key heads, then its value heads.
template <typename T, int kDim, int kEach>
__global__ __launch_bounds__(256) void AppendKernel(AppendArgs a) {
  constexpr int kPer = 16 / kBytes<T>;      // elements of a lane
  constexpr int kLanes = kDim / kPer;       // lanes of a row
  constexpr int kRows = 256 / kLanes;       // rows of a pass
  const int t = blockIdx.x;
  const int c = threadIdx.x % kLanes;
  const int nq = a.q.p != nullptr ? a.n_heads : 0, rows = nq + 2 * a.c.n_kv;
  const int row0 = blockIdx.y * (kEach * kRows) + threadIdx.x / kLanes;
  // The rows are on their way while the token's place is found.
  U4 raw[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int row = min(row0 + k * kRows, rows - 1);
    const bool is_q = row < nq, is_v = row >= nq + a.c.n_kv;
    const int head = is_q ? row : is_v ? row - nq - a.c.n_kv : row - nq;
    const Rows& from = is_q ? a.q : is_v ? a.v : a.k;
    raw[k] = Load16(from.p + t * from.token_bytes + head * from.head_bytes + 16 * c);
  }
  Sequence x;
  if (!FindSequence(a.s, [&](int end, int) { return end <= t; }, &x)) return;  // behind the last sequence
  const int pos = x.len - x.n_new + (t - x.first);
  // Tokens before the first sequence or at no position of the cache, and those
  // that the rotation table does not reach, are left out.
  if (t < x.first || pos < 0 || (a.rope != nullptr && pos >= a.rope_rows)) return;
  const int page = PageAt(a.c, a.s.table + x.seq * a.s.table_stride, pos);
  const int64_t in_cache =
      max(page, 0) * a.c.page_bytes + (pos & ((1 << a.c.page_log2) - 1)) * static_cast<int64_t>(a.c.row_bytes) + 16 * c;
  float cs[kPer], sn[kPer];
  if (a.rope != nullptr) {
    const float* r = a.rope + static_cast<int64_t>(pos) * kDim + (kPer * c) % (kDim / 2);
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const F4 u = *reinterpret_cast<const F4*>(r + i), v = *reinterpret_cast<const F4*>(r + kDim / 2 + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) cs[i + e] = u[e], sn[i + e] = c < kLanes / 2 ? -v[e] : v[e];
    }
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int row = row0 + k * kRows;
    const bool is_q = row < nq, is_v = row >= nq + a.c.n_kv;
    const int head = is_q ? row : is_v ? row - nq - a.c.n_kv : row - nq;
    U4 out = raw[k];
    if (!is_v) {
      float y[kPer];
      if constexpr (kPer == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) Unpack2<T>(out[i], &y[2 * i], &y[2 * i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __uint_as_float(out[i]);
      }
      const float* gain = is_q ? a.q_norm : a.k_norm;
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
      if constexpr (kPer == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = Pack2<T>(y[2 * i], y[2 * i + 1]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = __float_as_uint(y[i]);
      }
    }
    if (row >= rows || (!is_q && page < 0)) continue;
    char* to = is_q ? a.q_out.p + t * a.q_out.token_bytes + head * a.q_out.head_bytes + 16 * c
                    : (is_v ? a.c.v : a.c.k) + head * a.c.head_bytes + in_cache;
    *reinterpret_cast<U4*>(to) = out;
  }
}

// Rows of a thread: one for a decode step's few tokens, whose time is that of
// its round trips; three where the tokens alone fill the card, so that a token's
// place is found by a third as many workgroups (12 sequences, 4060 tokens,
// bf16: 28 us with one row, 24 with three).
constexpr int kManyTokens = 1024;

template <typename T, int kDim>
void LaunchDim(const AppendArgs& a, hipStream_t s) {
  const int rows = (a.q.p != nullptr ? a.n_heads : 0) + 2 * a.c.n_kv;
  constexpr int kPass = 256 * 16 / (kDim * kBytes<T>);
  const uint32_t n = static_cast<uint32_t>(a.s.n_tokens);
  RPG_CHECK(n <= kMaxGroups, "%u new tokens in one launch", n);
  if (a.s.n_tokens >= kManyTokens)
    AppendKernel<T, kDim, 3><<<dim3(n, static_cast<uint32_t>(CeilDiv(rows, 3 * kPass))), 256, 0, s>>>(a);
  else
    AppendKernel<T, kDim, 1><<<dim3(n, static_cast<uint32_t>(CeilDiv(rows, kPass))), 256, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
}

template <typename T>
void Launch(const AppendArgs& a, hipStream_t s) {
  if (a.c.head_dim == 128)
    LaunchDim<T, 128>(a, s);
  else
    LaunchDim<T, 64>(a, s);
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

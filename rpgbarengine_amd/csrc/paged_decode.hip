// Attention of one new token per sequence over its cache pages
// (rpg_hip_paged_decode, include/rpg_hip.h):
//   out[h] = sum_j p_j v_j,  p = softmax over j < len of scale q[h] . k_j.
//
// One pass over the keys with a running maximum, sum and output. Workgroup
// (sequence, key head, 16 query heads of its group, key range); its four waves
// take the range's key tiles in turn and join their states in LDS at the end.
// Scores and outputs are formed transposed on the matrix cores, S^T = K Q^T
// and O^T = V^T P^T (16 x 16 tiles, columns = query heads), so that a lane
// keeps to one query head: its scores are the B operand of the second product
// as they stand, and maximum, sum and rescaling are per lane. The key index of
// a product is free, so V is taken in the order the scores come in: a lane
// reads 16 bytes of each of its keys' rows (whole rows per load instruction)
// and for the 16-bit types pairs up its keys' values with one v_perm_b32 per
// operand register. K and V go from HBM to registers, LDS is not used on the
// way.
//
// Bound: the K and V bytes, each read once (16 columns are computed for any
// group size: at 8 heads f32 the products would take 1/2 of the time the bytes
// do, the 16-bit types' 1/10). Measured, 32 heads on 8 of 128: 64 sequences of
// 201 to 11167 positions, bf16, 861 MB in 172 us (the rate of a large copy:
// 171); one of 131000, f16, 537 MB in 95 us (107); 8 of about 1073, f32, 70 MB in 18.5
// us (14, and two launches); one of 95, f16: 7.2 us, the call itself (5.4 in a captured
// graph). Ranges: see DecodeSplits.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "decode_body.h"
#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {
namespace {

// grid (sequence x key head x block of 16 query heads, key range). Four waves to a
// SIMD unit for 16-bit rows of 64, by 128 registers; the compiler alone takes 134
// (64 x 4000 bf16 99 us, 96 so).
template <typename T, int kDim>
__global__ __launch_bounds__(64 * kWaves, kDim == 64 && kBytes<T> == 2 ? 4 : 2) void DecodeKernel(AttentionArgs a) {
  __shared__ __align__(16) DecodeLds<kDim> shared;
  const DecodePlace at = PlaceOf(a, blockIdx.x);
  DecodeRange range;
  if (!WholeRange(a, at.seq, blockIdx.y, &range)) return;
  DecodeRows<T, kDim>(a, shared, at.seq, at.kh, at.n_cols, range, at);
}

template <typename T, int kDim>
__global__ __launch_bounds__(256) void DecodeJoinKernel(AttentionArgs a) {
  const int64_t row = blockIdx.x;
  const int seq = static_cast<int>(row / a.n_heads), head = static_cast<int>(row % a.n_heads);
  const int len = Length(a.s, seq), range = RangeOf(a, max(len, 1), a.splits);
  if (range >= len) return;  // written by its one range
  JoinRow<T, kDim>(a, static_cast<int64_t>(a.s.n_seqs) * a.n_heads, row, (len + range - 1) / range,
                   a.out.p + seq * a.out.token_bytes + head * a.out.head_bytes);
}

template <typename T, int kDim>
void Launch(const AttentionArgs& a, hipStream_t s) {
  const int group = a.n_heads / a.c.n_kv;
  const int64_t x = static_cast<int64_t>(a.s.n_seqs) * a.c.n_kv * CeilDiv(group, kCols);
  RPG_CHECK(static_cast<int64_t>(a.s.n_seqs) * a.n_heads <= kMaxGroups, "%d x %d query rows in one launch", a.s.n_seqs,
            a.n_heads);
  DecodeKernel<T, kDim><<<dim3(static_cast<uint32_t>(x), a.splits), 64 * kWaves, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
  if (a.splits > 1) DecodeJoin(a, s);
}

template <typename T, int kDim>
void LaunchJoin(const AttentionArgs& a, hipStream_t s) {
  DecodeJoinKernel<T, kDim><<<static_cast<uint32_t>(a.s.n_seqs) * a.n_heads, 256, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
}

}  // namespace

// Ranges for a workgroup per compute unit and none with two (9 x 1000 f32: 27.0 us
// with 288 workgroups, 20.0 with 216; 11 x 4000 bf16 51 with 264, 39 with 176), and
// of 2048 positions at most, so that the longest sequence of a ragged batch does not
// end alone: 64 of 200 to 12000 take 152 us, 162 with 1024. Aiming higher only adds
// joins: 32 x 2000 bf16 48.2 us aiming at 256, 52.1 at 512, 53.5 at 1024; 8 x 1088 f32
// 18.7, 22.1, 21.1. Rows of a few steps stay whole, a join takes as long: one of 200
// bf16 12.0 us in ranges, 7.6 whole, 500 11.7 and 8.4, 700 11.9 and 10.3; f32 200 11.7
// and 10.1, 400 11.6 and 13.7. The rule knows the sequences' capacity, not their
// lengths, which are on the device: ranges behind a sequence's end return at once.
// So a table wider than its sequences costs the join's launch: one of 95 positions
// f16 7.8 us a call in a table of its own width, 11.7 in one for 4096 or for 131072
// (5.3 and 6.7 in a captured graph), one of 300 8.3 and 11.8 (8.0 and 8.4).
int DecodeSplits(int64_t n_seqs, int n_heads, int n_kv, int bytes, int64_t capacity) {
  if (capacity * bytes <= 1280) return 1;
  const int64_t base = std::max<int64_t>(1, n_seqs * n_kv * CeilDiv(n_heads / n_kv, kCols));
  const int64_t want = std::max(256 / base, CeilDiv(capacity, 2048));
  return static_cast<int>(std::max<int64_t>(1, std::min({want, CeilDiv(capacity, kRangeUnit), int64_t{kMaxSplits}})));
}

int64_t WorkBytes(int64_t rows, int head_dim, int splits) {
  return splits == 1 ? 0 : (StatFloats(rows, splits) + rows * splits * head_dim) * 4;
}

void Decode(const AttentionArgs& a, hipStream_t s) {
  if (a.s.n_seqs == 0) return;
  ByRows(a.c, [&](auto type, auto dim) { Launch<decltype(type), decltype(dim)::value>(a, s); });
}

void DecodeJoin(const AttentionArgs& a, hipStream_t s) {
  ByRows(a.c, [&](auto type, auto dim) { LaunchJoin<decltype(type), decltype(dim)::value>(a, s); });
}

}  // namespace paged
}  // namespace rpg

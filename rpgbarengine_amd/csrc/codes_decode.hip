// Attention of one new token per sequence over a cache of 8-bit codes
// (rpg_hip_quant_decode, include/rpg_hip.h): with scales ks, vs of the rows,
//   out[h] = sum_j p_j vs_j cv_j,  p = softmax over j < len of scale ks_j (q[h] . ck_j).
//
// The method of paged_decode.hip. A code is exact in 16 bits, so the codes
// themselves are the operands and a row's scale goes to its score or to its
// weight, in fp32: K in the rows' type (f32: bf16, and the query in three exact bf16
// parts), V in bf16, whose range is that of fp32, so that weight x scale needs no
// care whatever the scales are. It goes to the product in two bf16 parts (16 bits;
// f32: three, all of it). What is left of an error is that of fp32 sums.
//
// Bound: the codes' and scales' bytes, each read once. Measured, 32 heads on 8 of 128: 64
// sequences of 201 to 11167 positions, e4m3 in bf16, 382 MB in 86.3 us (a large copy's
// rate: 75; 64 of 2826 each, as many bytes: 83; the join is 4.6 of either); 8
// of about 1090, 16 heads, int8 in f16, 11.5 us, 9.4 of them the kernel's and 3.5 the
// join's. A row's scale is a lane's, and comes to the scores as an operand modifier
// (each lane loading its own keys' scales: 98 us the former, 94.5 so, both then).

#include <hip/hip_runtime.h>

#include <algorithm>

#include "codes_decode_body.h"
#include "codes_dev.h"
#include "common.h"
#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {
namespace {

// Waves to a SIMD unit.
template <typename T, int kDim>
constexpr int kMinWaves = kBytes<T> == 4 ? 2 : kDim == 128 ? 3 : 4;

// grid (sequence x key head x block of 16 query heads, key range), the last ranges first
template <typename C, typename T, int kDim>
__global__ __launch_bounds__(64 * kWaves, (kMinWaves<T, kDim>)) void CodesDecodeKernel(CodesAttentionArgs a) {
  __shared__ __align__(16) DecodeLds<kDim> shared;
  const DecodePlace at = PlaceOf(a.a, blockIdx.x);
  DecodeRange range;
  if (!WholeRange(a.a, at.seq, static_cast<int>(gridDim.y - 1 - blockIdx.y), &range)) return;
  DecodeCodeRows<C, T, kDim>(a, shared, at.seq, at.kh, at.n_cols, range, at);
}

template <typename C, typename T, int kDim>
void Launch(const CodesAttentionArgs& args, hipStream_t s) {
  const AttentionArgs& a = args.a;
  const int group = a.n_heads / a.c.n_kv;
  const int64_t x = static_cast<int64_t>(a.s.n_seqs) * a.c.n_kv * CeilDiv(group, kCols);
  RPG_CHECK(static_cast<int64_t>(a.s.n_seqs) * a.n_heads <= kMaxGroups, "%d x %d query rows in one launch", a.s.n_seqs,
            a.n_heads);
  CodesDecodeKernel<C, T, kDim><<<dim3(static_cast<uint32_t>(x), a.splits), 64 * kWaves, 0, s>>>(args);
  HIP_CHECK(hipGetLastError());
  if (a.splits > 1) DecodeJoin(a, s);
}

}  // namespace

// As DecodeSplits. Where the batch alone fills the card, no range is below 1024
// positions: a table for the longest sequence of a ragged batch would cut all of them
// into as many (64 of 201 to 11167, e4m3: 96.0 us so, 91.8 with 512, 87.9 with 1024, 93.5
// with 2048), and the last ranges, which few sequences have, come first (86.4). Ranges of
// 1024 also for the longest where one workgroup to a sequence and key head is one to two
// for each compute unit, or half of one: 32 of the same lengths 49.8 -> 47.0 us, 16 32.6
// -> 30.7 (f32 34.9 -> 25.5), 16 of 100 to 40000 56.4 -> 49.3; but 8 of them 19.5 -> 20.6,
// 32 of 2826 each 43.5 -> 44.2. Batches below that are cut into one workgroup per compute
// unit, and a table that asks for more ranges than that (one wider than its sequences, as
// a captured graph keeps) cuts none below 384 positions: 8 of 1090, 16 heads, f16, 12.7 us in
// a table of their own width, in one for 8192 and one for 131072 18.7 and 21.7 with ranges of
// 1024, 13.0 and 15.8 with 384, 12.9 and 16.1 with 128 (f32, 32 heads, 13.6; 20.1 and 23.5,
// 13.8 and 17.0, 13.8 and 19.1); 12 ragged in one for 16384 28.4, 24.1 and 24.3; of one or
// two sequences, whose workgroups are few, as the table has it: one of 1000 in one for 131072
// 14.1, 10.7 and 8.8.
int CodesDecodeSplits(int64_t n_seqs, int n_heads, int n_kv, int64_t capacity, int* least) {
  *least = 0;
  if (capacity <= 640) return 1;
  const int64_t base = std::max<int64_t>(1, n_seqs * n_kv * CeilDiv(n_heads / n_kv, kCols));
  const int64_t fill = 256 / base, cap = CeilDiv(capacity, base >= 128 && base < 512 ? 1024 : 2048);
  if (fill <= cap) *least = base >= 128 ? 1024 : base >= 32 ? 384 : 0;
  const int64_t want = std::max(fill, cap);
  return static_cast<int>(std::max<int64_t>(1, std::min({want, CeilDiv(capacity, kRangeUnit), int64_t{kMaxSplits}})));
}

void DecodeCodes(const CodesAttentionArgs& a, hipStream_t s) {
  if (a.a.s.n_seqs == 0) return;
  ByTypes(a.code, a.a.c, [&](auto code, auto type, auto dim) {
    Launch<decltype(code), decltype(type), decltype(dim)::value>(a, s);
  });
}

}  // namespace paged
}  // namespace rpg

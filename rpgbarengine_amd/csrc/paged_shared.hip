// Attention of one token per sequence where the first positions of a group's sequences
// lie in the same pages (rpg_hip_paged_shared, include/rpg_hip.h): as in
// paged_decode.hip,
//   out[h] = sum_j p_j v_j,  p = softmax over j < len of scale q[h] . k_j,
// with the sum over j cut where the group's common positions end. Those are read
// once for the whole group: its sequences' query heads are the rows of tiles, as a
// prompt's tokens are in paged_prompt.hip. A sequence's own positions are attended
// as in paged_decode.hip, and a third kernel joins the ranges of both:
//   out = sum_s o_s 2^(m_s - m) / sum_s l_s 2^(m_s - m).
//
// A group's common positions are its first `shared`, but no more than its shortest
// sequence has and whole units of 16: no row of a tile sees less than another,
// so nothing is masked but behind the last. The rest is a sequence's own.
//
// Bound: the common positions' products (a group of 32 sequences with four heads to a
// key head multiplies each key 128 times), or the own positions' bytes.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "decode_body.h"
#include "groups.h"
#include "paged.h"
#include "paged_dev.h"
#include "prompt_body.h"
#include "row_tile.h"

namespace rpg {
namespace paged {
namespace {

template <typename T, int kDim, int kGroups>
__global__ __launch_bounds__(256, kGroups == 2 || (kGroups == 4 && kBytes<T> == 4) ? 1 : 2) void PrefixKernel(SharedArgs a) {
  PromptBody<T, kDim, kGroups, false, true>(a.a, a.groups, static_cast<int>(a.prefix_splits));
}

// grid (sequence x key head x block of 16 query heads, key range)
template <typename T, int kDim>
__global__ __launch_bounds__(64 * kWaves, kDim == 64 && kBytes<T> == 2 ? 4 : 2) void OwnKernel(SharedArgs a) {
  const DecodePlace at = PlaceOf(a.a);
  DecodeRange range;
  if (!OwnRange(a.a, a.groups, static_cast<int>(a.prefix_splits), at.seq, kDecodeLift<T>, &range)) return;
  DecodeRows<T, kDim>(a.a, at, range);
}

template <typename T, int kDim>
__global__ __launch_bounds__(256) void SharedJoinKernel(SharedArgs args) {
  const AttentionArgs& a = args.a;
  const int splits = static_cast<int>(args.prefix_splits);
  const int64_t row = blockIdx.x;
  const int seq = static_cast<int>(row / a.n_heads), head = static_cast<int>(row % a.n_heads);
  const int len = Length(a.s, seq), from = len > 0 ? CommonKeys(a.s, args.groups, seq) : 0;
  JoinRow<T, kDim>(a, static_cast<int64_t>(a.s.n_seqs) * a.n_heads, row,
                   RangesOf(from, splits) + RangesOf(len - from, a.splits - splits),
                   a.out.p + seq * a.out.token_bytes + head * a.out.head_bytes);
}

template <typename T, int kDim, int kGroups>
void LaunchPrefix(const SharedArgs& args, hipStream_t s) {
  const AttentionArgs& a = args.a;
  const int64_t tiles = TilesFor(a.s.n_seqs, args.groups.n_seqs, a.n_heads / a.c.n_kv, 128 / kGroups);
  RPG_CHECK(tiles * a.c.n_kv <= kMaxGroups, "%d x %d query rows in one launch", a.s.n_seqs, a.n_heads);
  PrefixKernel<T, kDim, kGroups>
      <<<dim3(static_cast<uint32_t>(tiles * a.c.n_kv), static_cast<uint32_t>(args.prefix_splits)), 256, 0, s>>>(args);
  HIP_CHECK(hipGetLastError());
}

template <typename T, int kDim>
void Launch(const SharedArgs& args, hipStream_t s) {
  const AttentionArgs& a = args.a;
  const int group = a.n_heads / a.c.n_kv;
  const int64_t x = static_cast<int64_t>(a.s.n_seqs) * a.c.n_kv * CeilDiv(group, kCols);
  RPG_CHECK(static_cast<int64_t>(a.s.n_seqs) * a.n_heads <= kMaxGroups, "%d x %d query rows in one launch", a.s.n_seqs,
            a.n_heads);
  if (args.groups.n_seqs > 0) {
    const int rows = PrefixRows(a.s.n_seqs, args.groups.n_seqs, group);
    if (rows == 128)
      LaunchPrefix<T, kDim, 1>(args, s);
    else if (rows == 64)
      LaunchPrefix<T, kDim, 2>(args, s);
    else
      LaunchPrefix<T, kDim, 4>(args, s);
  }
  OwnKernel<T, kDim><<<dim3(static_cast<uint32_t>(x), static_cast<uint32_t>(a.splits - args.prefix_splits)), 64 * kWaves, 0, s>>>(args);
  HIP_CHECK(hipGetLastError());
  SharedJoin(args, s);
}

template <typename T, int kDim>
void LaunchJoin(const SharedArgs& a, hipStream_t s) {
  SharedJoinKernel<T, kDim><<<static_cast<uint32_t>(a.a.s.n_seqs) * a.a.n_heads, 256, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
}

}  // namespace

int PrefixRows(int64_t n_seqs, int64_t n_groups, int group) {
  const int64_t rows = n_seqs * group / std::max<int64_t>(n_groups, 1);
  return rows > 64 ? 128 : rows > 32 ? 64 : 32;
}

SharedSplits SplitsOfShared(int64_t n_seqs, int64_t n_groups, int n_heads, int n_kv, int64_t capacity) {
  const int group = n_heads / n_kv;
  const int64_t tiles = TilesFor(n_seqs, n_groups, group, PrefixRows(n_seqs, n_groups, group));
  const int64_t wgs = std::max<int64_t>(1, tiles * n_kv);
  const int64_t prefix = std::min({CeilDiv(512, wgs), CeilDiv(capacity, 256), int64_t{kMaxSplits / 2}});
  const int own = DecodeSplits(n_seqs, n_heads, n_kv, 2, capacity);
  return {static_cast<int>(std::max<int64_t>(1, prefix)), std::min(own, kMaxSplits / 2)};
}

void Shared(const SharedArgs& a, hipStream_t s) {
  if (a.a.s.n_seqs == 0) return;
  ByRows(a.a.c, [&](auto type, auto dim) { Launch<decltype(type), decltype(dim)::value>(a, s); });
}

void SharedJoin(const SharedArgs& a, hipStream_t s) {
  ByRows(a.a.c, [&](auto type, auto dim) { LaunchJoin<decltype(type), decltype(dim)::value>(a, s); });
}

}  // namespace paged
}  // namespace rpg

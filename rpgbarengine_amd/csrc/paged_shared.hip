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
// key head multiplies each key 128 times) beside the own positions' bytes, and the
// join. Measured, 32 heads on 8 of 128: 96 sequences in three groups behind 4000 to
// 12000 positions with 100 to 2500 of their own, bf16, 376 MB, 102 to 107 us (a large copy's
// rate: 74); 8 behind 2000, f32, 21, of which the products take 2 to 4 (4096 cycles of a wave,
// two of which may share a unit) and the second launch 4: what is left, not measured apart, are
// the round trips in front of the first product (starts and counts, lengths, the table, rows)
// and the waves' join. Workgroups of both kinds in turn instead of the common ones first:
// 129 us the former, 28.6 the latter (then 23.6). Weights of common positions in two parts,
// as decode has them: 107 -> 108.8 us the former, 50 -> 61 where own positions are few (both
// then); with one part the output is about 1.4 times as far from exact.

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

// One launch for both, so that the products of the common positions run beside the loads
// of the others. A sequence's last ranges come first. Two workgroups of 128 rows to a compute
// unit, for which f32 rows of 128 keep 34 registers in memory (96 sessions f32 288 us, with all
// in registers and one workgroup 326; 64 behind 4000 89 and 103).
template <typename T, int kDim, int kGroups>
__global__ __launch_bounds__(256, kGroups == 2 || (kGroups == 4 && kBytes<T> == 4) ? 1 : 2) void SharedKernel(SharedArgs args, SharedGrid g) {
  const AttentionArgs& a = args.a;
  __shared__ __align__(256) union {
    PromptLds<T, kDim, kGroups, false> prefix;
    DecodeLds<kDim> own;
  } shared;
  const int prefix_splits = static_cast<int>(args.prefix_splits);
  const int b = blockIdx.x;
  if (b < g.prefix) {
    PromptBody<T, kDim, kGroups, false, true>(a, args.groups, prefix_splits, shared.prefix, b % g.prefix_x,
                                              b / g.prefix_x, g.prefix_x);
  } else {
    const DecodePlace at = PlaceOf(a, (b - g.prefix) % g.own_x);
    const int y = a.splits - prefix_splits - 1 - (b - g.prefix) / g.own_x;
    DecodeRange range;
    if (!OwnRange(a, args.groups, prefix_splits, at.seq, y, kDecodeLift<T>, &range)) return;
    DecodeRows<T, kDim>(a, shared.own, at.seq, at.kh, at.n_cols, range, at);
  }
}

// Short work: tiles of 16 rows, whose common positions are attended as a sequence's own
// are, with the rows of several sequences in the columns. The larger tiles' kernel starts
// later (a workgroup of f32 has the unit to itself) and its tiles end in a longer joining.
template <typename T, int kDim>
__global__ __launch_bounds__(64 * kWaves, 2) void SharedSmallKernel(SharedArgs args, SharedGrid g) {
  __shared__ __align__(16) DecodeLds<kDim> shared;
  SmallPlace at;
  if (!SmallPlaceOf(args.a, args.groups, static_cast<int>(args.prefix_splits), g, blockIdx.x, kDecodeLift<T>, &at)) return;
  DecodeRows<T, kDim>(args.a, shared, at.seq, at.kh, at.n_cols, at.range, at.columns);
}

template <typename T, int kDim>
__global__ __launch_bounds__(256) void SharedJoinKernel(SharedArgs args) {
  const AttentionArgs& a = args.a;
  const int splits = static_cast<int>(args.prefix_splits);
  const int64_t row = blockIdx.x;
  const int seq = static_cast<int>(row / a.n_heads), head = static_cast<int>(row % a.n_heads);
  const int len = Length(a.s, seq), from = len > 0 ? CommonKeys(a.s, args.groups, seq) : 0;
  JoinRow<T, kDim>(a, static_cast<int64_t>(a.s.n_seqs) * a.n_heads, row,
                   RangesOf(from, RangeOf(max(from, 1), splits)) +
                       RangesOf(len - from, RangeOf(a, max(len - from, 1), a.splits - splits)),
                   a.out.p + seq * a.out.token_bytes + head * a.out.head_bytes);
}

// The same for many rows of few ranges, a wave each, without a barrier (96 sequences of 32
// heads, up to 13 ranges: 104.5 us a call with a workgroup for each, 101.6 so; 32 of up to
// 31: 66.2 and 68.0).
constexpr int kManyRows = 1024, kFewRanges = 24;
template <typename T, int kDim>
__global__ __launch_bounds__(256) void SharedJoinWaveKernel(SharedArgs args) {
  const AttentionArgs& a = args.a;
  constexpr int kPer = kDim / 64;  // dimensions of a lane
  const int prefix = static_cast<int>(args.prefix_splits), lane = threadIdx.x & 63;
  const int64_t rows = static_cast<int64_t>(a.s.n_seqs) * a.n_heads;
  static_assert(kFewRanges <= 64, "a lane for each");
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= rows) return;
  const int seq = static_cast<int>(row / a.n_heads), head = static_cast<int>(row % a.n_heads);
  const F2 mine = PartStats(a, row)[min(lane, a.splits - 1)];  // (anything behind the row's last range)
  const int len = Length(a.s, seq), from = len > 0 ? CommonKeys(a.s, args.groups, seq) : 0;
  const int n = RangesOf(from, RangeOf(max(from, 1), prefix)) +
                RangesOf(len - from, RangeOf(a, max(len - from, 1), a.splits - prefix));
  const float m = lane < n ? mine[0] : kNegInf, top = lanes::WaveMaxF(m);
  const float f = lane < n ? __builtin_amdgcn_exp2f(MaxDiff(m, top)) : 0.0f;
  const float l = lanes::WaveSumF(lane < n ? mine[1] * f : 0.0f);
  const float* po = PartOut<kDim>(a, rows, row) + kPer * lane;
  float o[kPer] = {};
  for (int s0 = 0; s0 < n; s0 += 4) {
    float x[4][kPer];  // in flight together
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[j][e] = po[min(s0 + j, n - 1) * kDim + e];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (s0 + j >= n) break;
      const float w = lanes::ReadLaneF(f, s0 + j);
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] += x[j][e] * w;
    }
  }
  const float inv = Inverse(top, l);
  char* out = a.out.p + seq * a.out.token_bytes + head * a.out.head_bytes + kPer * kBytes<T> * lane;
  if constexpr (kBytes<T> == 4 && kPer == 2)
    *reinterpret_cast<F2*>(out) = F2{o[0] * inv, o[1] * inv};
  else if constexpr (kBytes<T> == 4)
    *reinterpret_cast<float*>(out) = o[0] * inv;
  else if constexpr (kPer == 2)
    *reinterpret_cast<uint32_t*>(out) = Pack2<T>(o[0] * inv, o[1] * inv);
  else
    *reinterpret_cast<uint16_t*>(out) = static_cast<uint16_t>(Pack2<T>(o[0] * inv, 0.0f));
}

template <typename T, int kDim>
void Launch(const SharedArgs& args, hipStream_t s) {
  const AttentionArgs& a = args.a;
  const int rows = PrefixRows(a.s.n_seqs, args.groups.n_seqs, a.n_heads, a.c.n_kv, a.s.capacity);
  const SharedGrid g = GridOf(args, rows);
  const uint32_t n = static_cast<uint32_t>(g.prefix + g.own);
  if (rows == 128)
    SharedKernel<T, kDim, 1><<<n, 256, 0, s>>>(args, g);
  else if (rows == 64)
    SharedKernel<T, kDim, 2><<<n, 256, 0, s>>>(args, g);
  else if (rows == 32)
    SharedKernel<T, kDim, 4><<<n, 256, 0, s>>>(args, g);
  else
    SharedSmallKernel<T, kDim><<<n, 64 * kWaves, 0, s>>>(args, g);
  HIP_CHECK(hipGetLastError());
  SharedJoin(args, s);
}

template <typename T, int kDim>
void LaunchJoin(const SharedArgs& a, hipStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.a.s.n_seqs) * a.a.n_heads;
  if (rows >= kManyRows && a.a.splits <= kFewRanges)
    SharedJoinWaveKernel<T, kDim><<<static_cast<uint32_t>(CeilDiv(rows, 4)), 256, 0, s>>>(a);
  else
    SharedJoinKernel<T, kDim><<<static_cast<uint32_t>(rows), 256, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
}

}  // namespace

// By what a group has: of 64 and 32 rows two and all four waves take the keys of the same
// rows in turn. Of 16 where the whole batch is little work: 8 sequences of 32 heads behind
// 2000 positions f32 24.1 us with 32 rows, 21.5 with 16 (bf16 17.4 and 15.2, int8 codes of
// f16 rows 15.6 and 13.5), 16 behind 4000 f32 42.9 and 36.4 (codes 20.8 and 18.8); but 8
// behind 30000 91.3 and 99.4 (codes 34.1 and 38.9), 32 in four groups behind 4000, bf16,
// 30.0 and 38.2.
int PrefixRows(int64_t n_seqs, int64_t n_groups, int n_heads, int n_kv, int64_t capacity) {
  const int64_t rows = n_seqs * (n_heads / n_kv) / std::max<int64_t>(n_groups, 1);
  if (rows <= 64 && n_seqs * n_heads * capacity <= 3 << 20) return kCols;
  return rows > 64 ? 128 : rows > 32 ? 64 : 32;
}

SharedGrid GridOf(const SharedArgs& args, int rows) {
  const AttentionArgs& a = args.a;
  const int group = a.n_heads / a.c.n_kv;
  const int64_t tiles = args.groups.n_seqs == 0 ? 0 : TilesFor(a.s.n_seqs, args.groups.n_seqs, group, rows);
  const int64_t own_x = static_cast<int64_t>(a.s.n_seqs) * a.c.n_kv * CeilDiv(group, kCols);
  const int64_t prefix = tiles * a.c.n_kv * args.prefix_splits, own = own_x * (a.splits - args.prefix_splits);
  RPG_CHECK(prefix + own <= kMaxGroups && static_cast<int64_t>(a.s.n_seqs) * a.n_heads <= kMaxGroups,
            "%d x %d query rows in one launch", a.s.n_seqs, a.n_heads);
  return {static_cast<int32_t>(std::max<int64_t>(1, tiles * a.c.n_kv)), static_cast<int32_t>(prefix),
          static_cast<int32_t>(own_x), static_cast<int32_t>(own)};
}

// Ranges of common positions for one workgroup per compute unit, so that own positions
// run beside them (96 sequences in three groups behind 4000 to 12000, bf16: 103.4 us
// aiming at 512 workgroups, 100.7 at 256, 99.5 at 192; 32 behind 30000 63.1, 57.1, 67.8),
// two in f32, which the products alone keep busy (64 behind 4000: 88.8, 96.9), and none
// above 2560 positions (where the table has up to 655360), so that the longest group does not
// end alone (128 in eight groups
// behind 500 to 8000 91.8 us without, 84.9 so; 64 in 16 behind 100 to 10000 84.8, 76.2; on
// int8 codes of f16 rows the former 72.1, 75.2). Of 256 positions at least (64 behind 64,
// bf16: 29.2, with 128 31.5), 128 in tiles of 16 rows (8 behind 2000, f32: 24.7 us with
// 256, 21.6 with 128). Own ranges as a decode's, none below 512 where the batch fills the
// card (the 96: 114.7 without a least, 110.8 with 512, 115.9 with 1024).
SharedSplits SplitsOfShared(int64_t n_seqs, int64_t n_groups, int n_heads, int n_kv, int bytes, int64_t capacity) {
  const int group = n_heads / n_kv, rows = PrefixRows(n_seqs, n_groups, n_heads, n_kv, capacity);
  const int64_t wgs = std::max<int64_t>(1, TilesFor(n_seqs, n_groups, group, rows) * n_kv);
  const int64_t want = std::max(CeilDiv(bytes == 4 ? 512 : 256, wgs), CeilDiv(capacity, 2560));
  const int64_t prefix = std::min({want, CeilDiv(capacity, rows == kCols ? 128 : 256), int64_t{kMaxSplits / 2}});
  const int own = DecodeSplits(n_seqs, n_heads, n_kv, 2, capacity);
  const bool full = n_seqs * n_kv * CeilDiv(group, kCols) >= 256;
  return {static_cast<int>(std::max<int64_t>(1, prefix)), std::min(own, kMaxSplits / 2), full ? 512 : 0};
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

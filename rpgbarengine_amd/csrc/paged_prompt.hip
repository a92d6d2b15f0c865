// Causal attention of packed new tokens over their sequences' cache pages
// (rpg_hip_paged_prompt, include/rpg_hip.h): token i of sequence s at position
// p = len - n_new + i,
//   out[h] = sum_{j <= p} p_j v_j,  p = softmax over j <= p of scale q[h] . k_j.
//
// One pass over the keys with a running maximum, sum and output. The query
// heads of a key head's group are folded into the rows: row r of a sequence is
// (token r / G, head r % G), so a key is staged once for the whole group and a
// few tokens still fill a tile. Workgroup (tile of 128 rows, key head), a wave
// for 32 rows; the key steps are staged in LDS (two buffers, the next step's
// loads in flight over the products). Scores and outputs are formed
// transposed, S^T = K Q^T and O^T = V^T P^T (32 x 32 tiles, columns = rows of
// the query tile): a lane keeps to one row, its scores are the B operand of
// the second product as they stand, and the key order that they come in is
// the one that V is read in (16-bit types: ds_read_b64_tr_b16 reads four keys
// of a dimension).
//
// Few rows: the waves form 2, 4 or 8 groups (of two waves or of one) that take the
// key steps in turn and join their states in LDS; for fewer still the keys are cut
// into ranges over workgroups, joined by a second kernel.
//
// f32 goes to the bf16 units in three parts a value (Split3): 512 tokens 78 us
// with f32 products, 34 so. Its splitting costs the vector unit as much as the
// products cost the matrix unit.
//
// Bound: the matrix products, for few rows the chain of steps of a tile. Measured,
// 32 heads on 8 of 128: 4000 tokens of one sequence 147 us in bf16 (892 TFLOP/s; a
// large product of a library reaches 1194), 793 in f32 (165; 153 in f32
// instructions); 512 tokens 13 and 34 us; six turns of 13 to 50 tokens behind 400
// to 1000 14 us in f16; four documents of about 3000, 376 GFLOP, bf16, 407 us. Matrix units are
// busy for half the cycles, the exponentials and maxima share the rest; no LDS bank
// conflicts.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.h"
#include "paged.h"
#include "paged_dev.h"
#include "prompt_body.h"
#include "row_tile.h"

namespace rpg {
namespace paged {
namespace {

template <typename T, int kDim, int kGroups, bool kShared>
__global__ __launch_bounds__(kGroups == 8 ? 512 : 256, kGroups == 2 || (kGroups == 4 && kBytes<T> == 4 && !kShared) ? 1 : 2) void PromptKernel(AttentionArgs a) {
  __shared__ __align__(256) PromptLds<T, kDim, kGroups, kShared> shared;
  PromptBody<T, kDim, kGroups, kShared, false>(a, a.s, 1, shared, blockIdx.x, blockIdx.y, gridDim.x);
}

// Joins the key ranges of a tile's rows (four groups, 32 rows): workgroup = row.
template <typename T, int kDim>
__global__ __launch_bounds__(256) void PromptJoinKernel(AttentionArgs a) {
  const int64_t row = blockIdx.x;
  const int token = static_cast<int>(row / a.n_heads), head = static_cast<int>(row % a.n_heads);
  const int group = a.n_heads / a.c.n_kv;
  Sequence x;
  if (!FindSequence(a.s, [&](int end, int) { return end <= token; }, &x) || token < x.first) return;
  const int first = x.first, n_new = x.n_new, pos0 = x.len - x.n_new;
  // the row's tile
  const int tile = ((token - first) * group + head % group) / 32;
  const int keys = pos0 + min(32 * tile + 31, n_new * group - 1) / group + 1;
  const int range = RangeOf(max(keys, 1), a.splits);
  if (range >= keys) return;  // written by its one range
  JoinRow<T, kDim>(a, static_cast<int64_t>(a.s.n_tokens) * a.n_heads, row, (keys + range - 1) / range,
                   a.out.p + token * a.out.token_bytes + head * a.out.head_bytes);
}

int GroupsFor(int64_t n_tokens, int64_t n_seqs, int n_heads, int n_kv, int bytes, int64_t capacity);

// Key ranges where not even half the compute units have a workgroup (12 tokens
// behind 30000: 304 us with one, 37 with ranges; 203 behind 1297, 208 workgroups:
// 20 us with one, 38 with three), of 512 positions at least. In 16 bits eight groups
// go through 1536 positions in the time that the ranges and their join take (100
// behind 1400, 104 workgroups: 24.3 us with three ranges of four groups, 16.3 with
// one of eight; a token each behind 1000, 72: 15.6, 13.3). In f32, a workgroup to a
// compute unit, as many as find one free (40 behind 30000, 48 workgroups: 237 us with
// six, 176 with five), in 16 bits one more (68 and 72).
int RangesFor(int64_t wgs, int bytes, int64_t capacity) {
  if (wgs >= 128 || (bytes == 2 && capacity <= 1536)) return 1;
  const int64_t want = bytes == 4 ? 256 / wgs : CeilDiv(256, wgs);
  return static_cast<int>(std::max<int64_t>(1, std::min({want, CeilDiv(capacity, 512), int64_t{kMaxSplits}})));
}

template <typename T, int kDim, int kGroups, bool kShared = false>
void LaunchGroups(const AttentionArgs& a, hipStream_t s) {
  const int64_t tiles = TilesFor(a.s.n_tokens, a.s.n_seqs, a.n_heads / a.c.n_kv, 128 / std::min(kGroups, 4));
  RPG_CHECK(tiles * a.c.n_kv <= kMaxGroups &&
                (a.splits == 1 || static_cast<int64_t>(a.s.n_tokens) * a.n_heads <= kMaxGroups),
            "%d x %d query rows in one launch", a.s.n_tokens, a.n_heads);
  PromptKernel<T, kDim, kGroups, kShared>
      <<<dim3(static_cast<uint32_t>(tiles * a.c.n_kv), a.splits), 64 * Shape<T, kDim, kGroups>::kWaves, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
  if (a.splits > 1) PromptJoin(a, s);
}

template <typename T, int kDim>
void LaunchJoin(const AttentionArgs& a, hipStream_t s) {
  PromptJoinKernel<T, kDim><<<static_cast<uint32_t>(a.s.n_tokens) * a.n_heads, 256, 0, s>>>(a);
  HIP_CHECK(hipGetLastError());
}

// f32 rows of 128: K and V share a place above this many workgroups, one for each
// compute unit and the few that TilesFor counts too many. With two places / one, us:
// 256 tokens (264 workgroups) 19.0 / 21.9, 350 (352) 31.2 / 27.8, 512 (520) 39.4 /
// 34.5, 700 (704) 65 / 55, 300 behind 1700 (304) 116 / 94; 12 behind 30000 (256 with
// their ranges) 84 / 107.
constexpr int64_t kCrowd = 280;

template <typename T, int kDim>
void Launch(const AttentionArgs& a, hipStream_t s) {
  const int groups = GroupsFor(a.s.n_tokens, a.s.n_seqs, a.n_heads, a.c.n_kv, kBytes<T>, a.s.capacity);
  if constexpr (kBytes<T> == 2) {
    if (groups == 8) return LaunchGroups<T, kDim, 8>(a, s);
  }
  if constexpr (kBytes<T> == 4 && kDim == 128) {
    const int64_t tiles = TilesFor(a.s.n_tokens, a.s.n_seqs, a.n_heads / a.c.n_kv, 32);
    if (groups == 4 && tiles * a.c.n_kv * a.splits > kCrowd) return LaunchGroups<T, kDim, 4, true>(a, s);
  }
  if (groups == 4) return LaunchGroups<T, kDim, 4>(a, s);
  if (groups == 2) return LaunchGroups<T, kDim, 2>(a, s);
  LaunchGroups<T, kDim, 1>(a, s);
}

// Groups of a workgroup (its rows: 128 / groups, 32 at the least): one where that
// makes three workgroups for every two compute units, or else as many as it
// takes. bf16, us with 1 / 2 / 4: 512 tokens 17.9 / 16.5 / 13.8; 1000 30.9 / 28.9 /
// 33.5; 2000 56.8 / 63.5 / 75.7; 4 x 300 18.5 / 21.7 / 28.1; 16 x 60 behind 640 31.3 /
// 26.9 / 34.8; six turns 43.8 / 35.5 / 23.5; 203 behind 1297 38.8 / 31.5 / 20.4.
// 16-bit types: eight, of a wave each, where those workgroups find a compute unit
// to themselves and the keys are many and not cut into ranges (4 / 8: six turns
// 16.8 / 14.9, 200 behind 1300 19.4 / 16.9; 200 alone 10.0 / 10.6, 300 11.9 / 17.7).
constexpr int64_t kUnits = 256;  // compute units
int GroupsFor(int64_t n_tokens, int64_t n_seqs, int n_heads, int n_kv, int bytes, int64_t capacity) {
  const int group = n_heads / n_kv;
  if (TilesFor(n_tokens, n_seqs, group, 128) * n_kv >= 384) return 1;
  if (TilesFor(n_tokens, n_seqs, group, 64) * n_kv >= 384) return 2;
  const int64_t wgs = TilesFor(n_tokens, n_seqs, group, 32) * n_kv;
  return bytes == 2 && wgs <= kUnits && capacity > 512 && RangesFor(wgs, bytes, capacity) == 1 ? 8 : 4;
}

}  // namespace

int PromptSplits(int64_t n_tokens, int64_t n_seqs, int n_heads, int n_kv, int bytes, int64_t capacity) {
  if (GroupsFor(n_tokens, n_seqs, n_heads, n_kv, bytes, capacity) != 4) return 1;
  return RangesFor(TilesFor(n_tokens, n_seqs, n_heads / n_kv, 32) * n_kv, bytes, capacity);
}

void Prompt(const AttentionArgs& a, hipStream_t s) {
  if (a.s.n_tokens == 0 || a.s.n_seqs == 0) return;
  ByRows(a.c, [&](auto type, auto dim) { Launch<decltype(type), decltype(dim)::value>(a, s); });
}

void PromptJoin(const AttentionArgs& a, hipStream_t s) {
  ByRows(a.c, [&](auto type, auto dim) { LaunchJoin<decltype(type), decltype(dim)::value>(a, s); });
}

}  // namespace paged
}  // namespace rpg

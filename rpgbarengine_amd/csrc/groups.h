// Groups of sequences whose first positions lie in the same pages (SharedArgs).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "decode_body.h"
#include "paged.h"
#include "paged_dev.h"
#include "row_tile.h"

namespace rpg {
namespace paged {

// What a group's sequences have in common: `keys` positions, a multiple of 16 (the
// unit that pages are looked up in), read through the table of sequence `seq`.
// Sequences without positions (a batch's empty places) do not count.
struct Common {
  int keys, seq;
};

__device__ __forceinline__ Common CommonOf(const Seqs& s, int first, int n, int shared) {
  const int lane = threadIdx.x & 63;
  int least = shared, seq = -1;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int len = i0 + lane < n ? ClampLength(s, s.lens[first + i0 + lane]) : 0;
    const uint64_t some = __ballot(len > 0);
    if (some == 0) continue;
    if (seq < 0) seq = first + i0 + __builtin_ctzll(some);
    least = min(least, lanes::WaveReduce(len > 0 ? len : INT32_MAX, [](int x, int y) { return min(x, y); }));
  }
  return Common{seq < 0 ? 0 : max(least, 0) & ~15, max(seq, first)};
}

// Of a sequence's group; sequences of no group have nothing in common.
__device__ __forceinline__ int CommonKeys(const Seqs& s, const Seqs& groups, int seq) {
  Sequence x;
  if (!FindSequence(groups, [&](int end, int) { return end <= seq; }, &x) || seq < x.first) return 0;
  return CommonOf(s, x.first, x.n_new, x.len).keys;
}

// The ranges of `range` positions in `len`.
__device__ __forceinline__ int RangesOf(int len, int range) { return len <= 0 ? 0 : (len + range - 1) / range; }

// Range `y` of a sequence's own positions, behind the common ones; false:
// there is no such range. off: DecodeRange's.
__device__ __forceinline__ bool OwnRange(const AttentionArgs& a, const Seqs& groups, int prefix_splits, int seq, int y,
                                         float off, DecodeRange* out) {
  const int len = Length(a.s, seq);
  if (len <= 0) return false;
  const int from = CommonKeys(a.s, groups, seq), own = len - from;
  const int range = RangeOf(a, max(own, 1), a.splits - prefix_splits), start = from + y * range;
  *out = {start, min(len, start + range), false, RangesOf(from, RangeOf(max(from, 1), prefix_splits)) + y, off};
  return out->start < out->end;
}

// 16 query rows as the columns of a decode's tiles: row r is (sequence first + r / group,
// head head0 + r % group), of several sequences or of one.
struct RowColumns {
  int first, head0, row0, group;
  __device__ __forceinline__ ColumnPlace operator()(int column) const {
    const int r = row0 + column;
    return {first + r / group, head0 + r % group};
  }
};

// What workgroup b of a launch of 16-row tiles attends: its rows, their number and key
// head, the sequence whose table is read and the positions. False: there is nothing.
struct SmallPlace {
  RowColumns columns;
  int n_cols, kh, seq;
  DecodeRange range;
};
__device__ __forceinline__ bool SmallPlaceOf(const AttentionArgs& a, const Seqs& groups, int prefix_splits, SharedGrid g,
                                             int b, float off, SmallPlace* out) {
  const int group = a.n_heads / a.c.n_kv;
  if (b >= g.prefix) {
    const DecodePlace at = PlaceOf(a, (b - g.prefix) % g.own_x);
    out->columns = {at.seq, at.kh * group, at.h0 - at.kh * group, group};
    out->n_cols = at.n_cols, out->kh = at.kh, out->seq = at.seq;
    return OwnRange(a, groups, prefix_splits, at.seq, a.splits - prefix_splits - 1 - (b - g.prefix) / g.own_x, off,
                    &out->range);
  }
  RowTile t;
  int of;
  if (!TileOf(groups, group, kCols, b % g.prefix_x / a.c.n_kv, &of, &t)) return false;
  const Common common = CommonOf(a.s, t.first, t.n_rows / group, t.len);
  const int y = b / g.prefix_x, range = RangeOf(max(common.keys, 1), prefix_splits), start = y * range;
  out->kh = b % g.prefix_x % a.c.n_kv;
  out->columns = {t.first, out->kh * group, t.row0, group};
  out->n_cols = min(kCols, t.n_rows - t.row0), out->seq = common.seq;
  out->range = {start, min(common.keys, start + range), false, y, off};
  return start < common.keys;
}

}  // namespace paged
}  // namespace rpg

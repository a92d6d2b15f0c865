// Tiles of query rows: the query heads of a key head's group are folded into the
// rows, row r of a sequence is (token r / G, head r % G). For sequences of packed new
// tokens, and for groups of sequences of one token each.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {

// A row tile: its sequence and rows, and the positions it stands for.
struct RowTile {
  int first, row0, n_rows, len, pos0;  // first: the sequence's first token; row0: of the sequence's n_rows
  __device__ __forceinline__ int Position(int row, int group) const { return pos0 + min(row, n_rows - 1) / group; }
};
// Row tile `tile`: those of sequence s start at floor(starts[s] G / rows) + s,
// which leaves each its ceil(n_new G / rows) tiles wherever the starts lie. False:
// there is no such tile.
__device__ __forceinline__ bool TileOf(const Seqs& s, int group, int rows, int tile, int* seq, RowTile* t) {
  Sequence x;
  if (!FindSequence(s, [&](int end, int j) { return end * group / rows + j + 1 <= tile; }, &x)) return false;
  *seq = x.seq;
  t->first = x.first;
  t->n_rows = x.n_new * group;
  t->row0 = (tile - (x.first * group / rows + x.seq)) * rows;
  t->len = x.len;
  t->pos0 = x.len - x.n_new;
  return t->row0 >= 0 && t->row0 < t->n_rows;
}

// The workgroups that TileOf's tiles take at most.
inline int64_t TilesFor(int64_t n_tokens, int64_t n_seqs, int group, int rows) {
  return n_tokens * group / rows + n_seqs;
}

}  // namespace paged
}  // namespace rpg

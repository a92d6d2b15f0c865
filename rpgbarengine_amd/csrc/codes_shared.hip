// Attention of one token per sequence over a cache of 8-bit codes where the first
// positions of a group's sequences lie in the same pages (rpg_hip_quant_shared,
// include/rpg_hip.h): as paged_shared.hip has it, with the products of
// codes_prompt.hip and codes_decode.hip. Measured, 32 heads on 8 of 128: 8 sessions behind
// 2000, i8 of f16, 14.3 us (their bytes at a large copy's rate: 1.5), e4m3 of f32 14.2 (1.9); 96
// in three groups behind 4000 to 12000, e4m3 of bf16, 89.6 (38), i8 of f32 190 (the products of
// a large f32 one of a library: 101). Large batches: the common positions' products, six for f32
// rows where 16-bit ones take three, beside the own positions' bytes; short ones: the chain of
// look-ups and the join, as paged_shared.hip has it.

#include <hip/hip_runtime.h>

#include "codes_decode_body.h"
#include "codes_dev.h"
#include "codes_prompt_body.h"
#include "common.h"
#include "decode_body.h"
#include "groups.h"
#include "paged.h"
#include "paged_dev.h"

namespace rpg {
namespace paged {
namespace {

// Grid: as SharedKernel's (paged_shared.hip). kWide: tiles of 128 rows, of 32 otherwise. Two
// workgroups to a compute unit, for which f32 rows of 128 keep 40 registers in memory, 16-bit
// ones up to two: 64 sessions behind 4000 i8 of f32 52.3 us, with one workgroup 57.7; 96 in
// three groups i8 191 and 179, e4m3 192 and 173.
template <typename C, typename T, int kDim, bool kWide>
__global__ __launch_bounds__(256, kWide || kBytes<T> == 2 ? 2 : 1) void CodesSharedKernel(CodesSharedArgs args, SharedGrid g) {
  const AttentionArgs& a = args.c.a;
  __shared__ __align__(256) union {
    std::conditional_t<kWide, WideLds<T, kDim>, SoloLds<kDim, 4>> prefix;
    DecodeLds<kDim> own;
  } shared;
  const int prefix_splits = static_cast<int>(args.prefix_splits);
  const int b = blockIdx.x;
  if (b < g.prefix) {
    const int bx = b % g.prefix_x, by = b / g.prefix_x;
    if constexpr (kWide)
      WideBody<C, T, kDim, true>(args.c, args.groups, prefix_splits, shared.prefix, bx, by, g.prefix_x);
    else
      SoloBody<C, T, kDim, 4, true>(args.c, args.groups, prefix_splits, shared.prefix, bx, by, g.prefix_x);
  } else {
    const DecodePlace at = PlaceOf(a, (b - g.prefix) % g.own_x);
    const int y = a.splits - prefix_splits - 1 - (b - g.prefix) / g.own_x;
    DecodeRange range;
    if (!OwnRange(a, args.groups, prefix_splits, at.seq, y, 0.0f, &range)) return;
    DecodeCodeRows<C, T, kDim>(args.c, shared.own, at.seq, at.kh, at.n_cols, range, at);
  }
}

// As SharedSmallKernel (paged_shared.hip).
template <typename C, typename T, int kDim>
__global__ __launch_bounds__(64 * kWaves, 2) void CodesSharedSmallKernel(CodesSharedArgs args, SharedGrid g) {
  __shared__ __align__(16) DecodeLds<kDim> shared;
  SmallPlace at;
  if (!SmallPlaceOf(args.c.a, args.groups, static_cast<int>(args.prefix_splits), g, blockIdx.x, 0.0f, &at)) return;
  DecodeCodeRows<C, T, kDim>(args.c, shared, at.seq, at.kh, at.n_cols, at.range, at.columns);
}

template <typename C, typename T, int kDim>
void Launch(const CodesSharedArgs& args, hipStream_t s) {
  const AttentionArgs& a = args.c.a;
  SharedArgs rows;
  rows.a = a;
  rows.groups = args.groups;
  rows.prefix_splits = args.prefix_splits;
  const int tile = PrefixRows(a.s.n_seqs, args.groups.n_seqs, a.n_heads, a.c.n_kv, a.s.capacity);
  const SharedGrid g = GridOf(rows, tile == 64 ? kSoloRows : tile);
  const uint32_t n = static_cast<uint32_t>(g.prefix + g.own);
  if (tile == 128)
    CodesSharedKernel<C, T, kDim, true><<<n, 256, 0, s>>>(args, g);
  else if (tile == kCols)
    CodesSharedSmallKernel<C, T, kDim><<<n, 64 * kWaves, 0, s>>>(args, g);
  else
    CodesSharedKernel<C, T, kDim, false><<<n, 256, 0, s>>>(args, g);
  HIP_CHECK(hipGetLastError());
  SharedJoin(rows, s);
}

}  // namespace

void SharedCodes(const CodesSharedArgs& a, hipStream_t s) {
  if (a.c.a.s.n_seqs == 0) return;
  ByTypes(a.c.code, a.c.a.c, [&](auto code, auto type, auto dim) {
    Launch<decltype(code), decltype(type), decltype(dim)::value>(a, s);
  });
}

}  // namespace paged
}  // namespace rpg

// Causal attention of packed new tokens over a cache of 8-bit codes
// (rpg_hip_quant_prompt, include/rpg_hip.h): token i of a sequence at position p,
//   out[h] = sum_{j <= p} p_j vs_j cv_j,  p = softmax over j <= p of scale ks_j (q[h] . ck_j).
//
// The codes are the products' operands and the scales go to scores and weights in
// fp32, as in codes_decode.hip; rows are tiled and scores and outputs formed
// transposed on 32 x 32 tiles, as in paged_prompt.hip.
//
// Few rows (CodesSoloKernel): workgroup (tile of 32 rows, key head, key range), whose
// waves take blocks of 32 keys in turn, from memory to registers, and join their
// states in LDS.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "codes_dev.h"
#include "codes_prompt_body.h"
#include "common.h"
#include "paged.h"
#include "paged_dev.h"
#include "row_tile.h"

namespace rpg {
namespace paged {
namespace {

template <typename C, typename T, int kDim>
__global__ __launch_bounds__(256, 2) void CodesWideKernel(CodesAttentionArgs a) {
  __shared__ __align__(256) WideLds<T, kDim> shared;
  WideBody<C, T, kDim, false>(a, a.a.s, 1, shared, blockIdx.x, blockIdx.y, gridDim.x);
}

template <typename C, typename T, int kDim, int kWaves>
__global__ __launch_bounds__(64 * kWaves, 1) void CodesSoloKernel(CodesAttentionArgs a) {
  __shared__ __align__(16) SoloLds<kDim, kWaves> shared;
  SoloBody<C, T, kDim, kWaves, false>(a, a.a.s, 1, shared, blockIdx.x, blockIdx.y, gridDim.x);
}

// Tiles of 128 rows where those fill the compute units.
bool IsWide(int64_t n_tokens, int64_t n_seqs, int group, int n_kv) {
  return TilesFor(n_tokens, n_seqs, group, 128) * n_kv >= 256;
}

template <typename C, typename T, int kDim>
void Launch(const CodesAttentionArgs& args, hipStream_t s) {
  const AttentionArgs& a = args.a;
  const int group = a.n_heads / a.c.n_kv;
  const bool wide = IsWide(a.s.n_tokens, a.s.n_seqs, group, a.c.n_kv);
  const int64_t tiles = TilesFor(a.s.n_tokens, a.s.n_seqs, group, wide ? 128 : kSoloRows);
  RPG_CHECK(tiles * a.c.n_kv <= kMaxGroups &&
                (a.splits == 1 || static_cast<int64_t>(a.s.n_tokens) * a.n_heads <= kMaxGroups),
            "%d x %d query rows in one launch", a.s.n_tokens, a.n_heads);
  if (wide) {
    CodesWideKernel<C, T, kDim><<<dim3(static_cast<uint32_t>(tiles * a.c.n_kv)), 256, 0, s>>>(args);
    HIP_CHECK(hipGetLastError());
    return;
  }
  CodesSoloKernel<C, T, kDim, 4><<<dim3(static_cast<uint32_t>(tiles * a.c.n_kv), a.splits), 256, 0, s>>>(args);
  HIP_CHECK(hipGetLastError());
  if (a.splits > 1) PromptJoin(a, s);
}

}  // namespace

int CodesPromptSplits(int64_t n_tokens, int64_t n_seqs, int n_heads, int n_kv, int64_t capacity) {
  const int64_t wgs = TilesFor(n_tokens, n_seqs, n_heads / n_kv, kSoloRows) * n_kv;
  if (wgs >= 128) return 1;
  return static_cast<int>(std::max<int64_t>(1, std::min({CeilDiv(256, wgs), CeilDiv(capacity, 512), int64_t{kMaxSplits}})));
}

void PromptCodes(const CodesAttentionArgs& a, hipStream_t s) {
  if (a.a.s.n_tokens == 0 || a.a.s.n_seqs == 0) return;
  ByTypes(a.code, a.a.c, [&](auto code, auto type, auto dim) {
    Launch<decltype(code), decltype(type), decltype(dim)::value>(a, s);
  });
}

}  // namespace paged
}  // namespace rpg

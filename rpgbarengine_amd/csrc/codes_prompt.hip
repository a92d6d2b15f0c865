// Causal attention of packed new tokens over a cache of 8-bit codes
// (rpg_hip_quant_prompt, include/rpg_hip.h): token i of a sequence at position p,
//   out[h] = sum_{j <= p} p_j vs_j cv_j,  p = softmax over j <= p of scale ks_j (q[h] . ck_j).
//
// The codes are the products' operands and the scales go to scores and weights in
// fp32, as in codes_decode.hip; rows are tiled and scores and outputs formed
// transposed on 32 x 32 tiles, as in paged_prompt.hip.
//
// Few rows (CodesSoloKernel): workgroup (tile of 32 rows, key head, key range), whose
// four or eight waves take blocks of 32 keys in turn, from memory to registers, and
// join their states in LDS. Many (CodesWideKernel): tiles of 128 rows, a wave for 32;
// a step's 64 keys go to LDS converted, once for the four waves.
//
// Weights times scales go to the product in parts of bf16, whose range is that of fp32, as
// in codes_decode.hip: f16 ones would have to be held over the largest scale, which may be
// a later token's, and the tokens before it would lose their weights' bits to it. Two parts
// (f32 rows: three) leave the output as exact as its own rounding does; rounded to the
// rows' type once, it is 1.40 (bf16) and 1.41 (f16) times as far from exact, and four
// documents e4m3 bf16 take 501 us instead of 645, 2000 tokens 66 instead of 81.5.
//
// Bound: the matrix unit, which the second parts take half as long again, and the vector
// unit, hardly at once (documents: busy for 44 and 54 % of the cycles): per score a product
// with either scale comes to the maximum, the exponential, the sum and the second part,
// and the codes' conversion. Measured, 32 heads on 8 of 128: four documents of about 3000
// tokens, 392 GFLOP, e4m3 in bf16, 613 to 645 us (610 to 640 TFLOP/s, 910 to 960 of the
// products'; a large product of a library reaches 1254); six turns of 13 to 50 tokens behind
// 400 to 1000, i8 in f16, 17 us. Tried on documents with one part: products of one 32-key
// block between the weighing of the other 492 -> 492 (479 without), higher priority around
// products the same, pages looked up another step ahead the same.

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

// Two workgroups to a compute unit: f32 rows of 128 keep 45 (i8) and 60 (e4m3) registers in
// memory for it (documents 1254 and 1315 us; with all in registers and one workgroup 1394
// and 1350; 2000 tokens i8, which have one to a unit anyway, 177 and 131).
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

// Tiles of 128 rows where those make three workgroups for every two compute units,
// of 32 otherwise (1000 tokens 43.2 and 34.3 us, 4 x 300 25.1 and 27.6, 2000 84.4 and
// 91.8).
bool IsWide(int64_t n_tokens, int64_t n_seqs, int group, int n_kv) {
  return TilesFor(n_tokens, n_seqs, group, 128) * n_kv >= 384;
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
  // Eight waves where they find a compute unit to themselves and the keys are many (six
  // turns 18.7 -> 18.0 us, 200 behind 1300 24.2 -> 22.3; 200 alone 9.9 and 10.2).
  const int64_t wgs = tiles * a.c.n_kv * a.splits;
  const dim3 grid(static_cast<uint32_t>(tiles * a.c.n_kv), a.splits);
  bool eight = false;
  if constexpr (kBytes<T> == 2) {
    eight = wgs <= 256 && a.s.capacity > 256;
    if (eight) CodesSoloKernel<C, T, kDim, 8><<<grid, 512, 0, s>>>(args);
  }
  if (!eight) CodesSoloKernel<C, T, kDim, 4><<<grid, 256, 0, s>>>(args);
  HIP_CHECK(hipGetLastError());
  if (a.splits > 1) PromptJoin(a, s);
}

}  // namespace

// Key ranges where not even half the compute units have a workgroup, of 512 positions
// at least, and as many as find one free; none for rows of up to 1536 positions where
// a quarter of them have one (f16: 100 behind 1400, 104 workgroups, 25.4 us with two and
// 21.9 with one, 30 behind 1000, 40 of them, 16.4 with three and 17.1 with one; 12
// behind 30000 32 and 266).
int CodesPromptSplits(int64_t n_tokens, int64_t n_seqs, int n_heads, int n_kv, int64_t capacity) {
  const int64_t wgs = TilesFor(n_tokens, n_seqs, n_heads / n_kv, kSoloRows) * n_kv;
  if (wgs >= 128 || (wgs >= 64 && capacity <= 1536)) return 1;
  return static_cast<int>(std::max<int64_t>(1, std::min({256 / wgs, CeilDiv(capacity, 512), int64_t{kMaxSplits}})));
}

void PromptCodes(const CodesAttentionArgs& a, hipStream_t s) {
  if (a.a.s.n_tokens == 0 || a.a.s.n_seqs == 0) return;
  ByTypes(a.code, a.a.c, [&](auto code, auto type, auto dim) {
    Launch<decltype(code), decltype(type), decltype(dim)::value>(a, s);
  });
}

}  // namespace paged
}  // namespace rpg

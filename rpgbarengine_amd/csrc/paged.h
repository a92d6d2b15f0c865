// Serving operators on device buffers (include/rpg_hip.h): a paged key-value
// cache that many sequences share, the attention that reads it, and the row
// sampler. Launch arguments of the kernels in paged_append.hip,
// paged_decode.hip, paged_prompt.hip and sample_rows.hip; serving_abi.cc
// checks the callers' arguments and fills them in.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rpg {
namespace paged {

// The element type: f32, f16 or bf16 (ggml ids, common.h).
struct Cache {
  char* k = nullptr;
  char* v = nullptr;
  int64_t page_bytes = 0, head_bytes = 0;  // from one page, one head, to the next
  int32_t row_bytes = 0;                   // from one position of a page to the next
  int32_t n_pages = 0, n_kv = 0;
  int32_t page_log2 = 0;  // positions per page: a power of two, at least 16
  int32_t head_dim = 0;
  uint32_t type = 0;
};

// Sequences: sequence s has min(lens[s], capacity) positions, position p in
// page table[s * table_stride + (p >> page_log2)]; its new tokens are the
// packed rows starts[s] .. starts[s + 1], at its last positions.
struct Seqs {
  const int32_t* table = nullptr;
  int64_t table_stride = 0;
  const int32_t* lens = nullptr;
  const int32_t* starts = nullptr;
  int32_t n_seqs = 0, n_tokens = 0;
  int32_t capacity = 0;  // positions that a row of the table covers
};

// [token][head][head_dim] rows, strides in bytes, a head's row contiguous
struct Rows {
  char* p = nullptr;
  int64_t token_bytes = 0, head_bytes = 0;
};

// Workgroups of one launch, at 256 threads each.
constexpr int64_t kMaxGroups = (int64_t{1} << 24) - 1;

struct AppendArgs {
  Cache c;
  Seqs s;
  Rows k, v, q, q_out;  // q.p == nullptr: no queries
  int32_t n_heads = 0;
  const float* q_norm = nullptr;  // [head_dim] gains, or none
  const float* k_norm = nullptr;
  float eps = 0.0f;
  const float* rope = nullptr;  // [rope_rows][head_dim]: cos | sin, or none
  int64_t rope_rows = 0;
};
void Append(const AppendArgs& a, hipStream_t s);

struct AttentionArgs {
  Cache c;
  Seqs s;
  Rows q, out;
  int32_t n_heads = 0;
  float scale = 0.0f;
  int32_t splits = 1;     // key ranges that a query's keys may be cut into
  float* work = nullptr;  // partials of the ranges (WorkBytes)
};

// The key ranges that a batch of this shape is cut into at most, and the bytes
// of their partials (0 for one range).
int DecodeSplits(int64_t n_seqs, int n_heads, int n_kv, int bytes, int64_t capacity);
int PromptSplits(int64_t n_tokens, int64_t n_seqs, int n_heads, int n_kv, int bytes, int64_t capacity);
int64_t WorkBytes(int64_t rows, int head_dim, int splits);

// Floats of the partials' maxima and sums, in front of their outputs, which are
// read and written 16 bytes at a time.
__host__ __device__ inline int64_t StatFloats(int64_t rows, int splits) { return (2 * rows * splits + 3) / 4 * 4; }
void Decode(const AttentionArgs& a, hipStream_t s);

void Prompt(const AttentionArgs& a, hipStream_t s);

}  // namespace paged
}  // namespace rpg

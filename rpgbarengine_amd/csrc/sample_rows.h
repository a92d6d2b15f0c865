// Launch arguments of the row sampler (sample_rows.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rpg {
namespace rows {

struct SampleArgs {
  const char* logits = nullptr;  // [rows][vocab] of f32, f16 or bf16 (ggml ids)
  int64_t row_bytes = 0;
  uint32_t type = 0;
  int32_t rows = 0, vocab = 0;
  const float* temperature = nullptr;  // [rows] each
  const int32_t* top_k = nullptr;      // may be null: no limit
  const float* top_p = nullptr;
  const float* min_p = nullptr;
  const float* u = nullptr;
  int32_t* tokens = nullptr;
  float* logprobs = nullptr;  // may be null
  char* work = nullptr;       // WorkBytes(rows, vocab)
};

int64_t WorkBytes(int64_t rows, int64_t vocab);
void Sample(const SampleArgs& a, hipStream_t s);

}  // namespace rows
}  // namespace rpg

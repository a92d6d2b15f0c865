// Edits of logits before the sampler (rpg_hip_edit_logits, include/rpg_hip.h).
// Launch arguments of the kernel in edit_rows.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rpg {
namespace rows {

constexpr int kMaxHistory = 1 << 20, kMaxBiases = 1023;  // tokens of a row, entries of a row

struct EditArgs {
  const char* logits = nullptr;
  char* out = nullptr;
  int64_t row_bytes = 0, out_bytes = 0;  // from one row to the next
  const int32_t* history = nullptr;      // [rows][history_size], or none
  const int32_t* history_lens = nullptr;
  const int32_t* prompts = nullptr;
  const float* repetition = nullptr;
  const float* presence = nullptr;
  const float* frequency = nullptr;
  const int32_t* bias_ids = nullptr;  // [rows][n_biases], or none
  const float* bias = nullptr;
  const int32_t* mask = nullptr;  // [n_masks][words], or none
  const int32_t* mask_rows = nullptr;
  int64_t history_stride = 0, bias_ids_stride = 0, bias_stride = 0, mask_stride = 0;  // elements
  int32_t history_size = 0, n_biases = 0, n_masks = 0;
  int32_t rows = 0, vocab = 0;
  uint32_t type = 0;  // f32, f16 or bf16 (ggml ids, common.h)
};
void Edit(const EditArgs& a, hipStream_t s);

}  // namespace rows
}  // namespace rpg

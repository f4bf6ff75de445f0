// Filtered sampling of logits rows (filter.cu): one cluster of CTAs per row.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/realm_b200.h"

namespace rb {

constexpr int kFilterMaxVocab = 262144;

struct FilterArgs {
  const void* logits = nullptr;
  int64_t ld = 0;
  int32_t x16 = 0;  // 1: fp16 logits, 0: fp32
  int32_t all = 0;  // 1: the kernel that holds whole rows takes every row, 0: those left to it
  int32_t n_rows = 0, vocab = 0;
  const rb_sampling_filter* params = nullptr;
  const uint32_t* prev = nullptr;
  const uint32_t* prev_off = nullptr;
  const float* uniforms = nullptr;
  uint32_t* tokens = nullptr;
  float* probs = nullptr;  // or null
  float* dist = nullptr;   // not null: the rows' distributions go here instead of a draw
  int64_t ldd = 0;
};

cudaError_t filter_launch(const FilterArgs& a, int num_sms, cudaStream_t s);

}  // namespace rb

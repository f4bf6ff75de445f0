// Norms around a block with its gate and residual (residual.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace rb {

constexpr int kResidualMaxDim = 32768;

struct ResidualArgs {
  const void *y = nullptr, *x = nullptr, *gate = nullptr;  // gate may be null
  void *x_out = nullptr, *out = nullptr;                   // out may be null
  int64_t ldy = 0, ldx = 0, ldg = 0, ldxo = 0, ldo = 0;    // elements between rows
  int32_t y16 = 0, x16 = 0;                                // fp16 (y, gate, out; x, x_out), else fp32
  int32_t n_rows = 0, dim = 0;
  const float *post = nullptr, *pre = nullptr;             // post may be null; pre goes with out
  float scale = 1.f, eps = 0.f;
};

cudaError_t residual_launch(const ResidualArgs& a, cudaStream_t s);

}  // namespace rb

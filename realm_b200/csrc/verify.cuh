// Verification of drafted tokens (verify.cu): one cluster of CTAs per request.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace rb {

struct VerifyArgs {
  int32_t n_requests = 0, n_rows = 0, vocab = 0;
  const uint32_t* offsets = nullptr;
  const float *probs = nullptr, *draft_probs = nullptr;  // draft_probs may be null
  int64_t ldp = 0, ldq = 0;
  const uint32_t* drafts = nullptr;
  const float* uniforms = nullptr;
  uint32_t* tokens = nullptr;
  int32_t* accepted = nullptr;
};

cudaError_t verify_launch(const VerifyArgs& a, int num_sms, cudaStream_t s);

}  // namespace rb

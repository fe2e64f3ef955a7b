// Log-probabilities of given tokens, entropy and top alternatives (nab_logprobs.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace nab {

constexpr int kMaxTopK = 32;

struct LogprobsArgs {
  const void* logits;      // [rows, V], row stride in elements
  int64_t stride;
  const int64_t* tokens;   // [rows]
  int64_t vocab_start;     // token id of column 0
  float* logprob;          // [rows]
  float* entropy;          // [rows]
  float* lse;              // [rows]
  float* top_logprobs;     // [rows, top_k]
  int64_t* top_tokens;     // [rows, top_k]
  float* top_logits;       // [rows, top_k]
  int64_t rows;
  int V, top_k;
};
// dtype: kF32, kF16 or kBF16.
void token_logprobs(cudaStream_t s, const LogprobsArgs& a, int dtype, int sms);

}  // namespace nab

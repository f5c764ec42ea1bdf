// Log probabilities of given tokens (csrc/logprobs.cu).
// The reference has no sampling of its own: it serves that of vLLM and SGLang (README.md:20-33).
#pragma once
#include <cuda_runtime.h>

namespace penny {

constexpr int kLogprobsMaxTop = 32;
enum LogitType { LOGITS_BF16 = 0, LOGITS_FP16 = 1, LOGITS_FP32 = 2 };

struct TokenLogprobs {
  const void* logits;  // [rows, vocab], rows of row_stride elements
  long long row_stride;
  const long long* tokens;
  float *logprobs, *entropy;  // [rows]
  float* top_logprobs;        // [rows, top]
  long long* top_ids;
  int rows, vocab, top;
};
cudaError_t launch_token_logprobs(const TokenLogprobs& a, LogitType type, int sms, cudaStream_t stream);

}  // namespace penny

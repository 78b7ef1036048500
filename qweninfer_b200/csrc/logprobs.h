// Token log probabilities from logits (logprobs.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace qi {

constexpr int kMaxLogprobSlices = 64;

struct LogprobParams {
  const void* logits;
  long long ld;
  const void* targets;  // int32 or int64 (targets64), or null
  int targets64;
  int M, V, top;
  float* logprob;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  float* part_stats;              // M * slices * 4
  unsigned long long* part_list;  // M * slices * 32
  unsigned int* counters;         // M, zero between calls
  int slices;
};

int logprob_slices(int M, int V);
cudaError_t launch_token_logprobs(const LogprobParams& p, int dtype, cudaStream_t s, bool pdl);

}  // namespace qi

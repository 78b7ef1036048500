// Token log probabilities from logits (logprobs.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace qi {

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
  // of rows that several CTAs share, two parts for each CTA: sums (4 floats) and lists (32 words)
  float* part_stats;
  unsigned long long* part_list;
  unsigned int* counters;  // one for each CTA, zero between calls
  int chunks;              // of a row (set by the launch)
};

struct LogprobPlan {
  int ctas, chunks;
  long long scratch;  // bytes
};
LogprobPlan logprob_plan(int M, int V, int dtype);
cudaError_t launch_token_logprobs(const LogprobParams& p, const LogprobPlan& plan, int dtype, cudaStream_t s);

}  // namespace qi

// Attention over one cache layer (cache_attention.cu).
#pragma once

#include "internal.h"
#include "../../include/qi.h"

namespace qi {

struct CacheAttnParams {
  qi_kv_layer c;
  const void* q;
  int dtype;              // of q and out
  long long q_st, q_sh;   // element strides of token and head
  int q_vec;              // q rows can be read 16 bytes at a time (set by the launch)
  int heads, group;       // query heads, and those of one KV head
  const int32_t* rows;
  const int32_t* pos;
  int M;
  int window, sinks;      // window 0: none
  float scale_log2;       // log2(e) / sqrt(head_dim) (set by the launch)
  void* out;              // (M, heads, head_dim), may be null
  uint16_t* out_act;      // activation tiles of token tile out_nt for the o projection, may be null
  int out_nt;
  float* part;            // sums of the per-token kernel's clusters, fp32
  unsigned int* counters; // one per unit, zero between calls
  int splits;             // key splits of the kernel that runs
  int cluster;            // per-token kernel: CTAs of a cluster, which divides splits
  int* err;
  // prompts (cache_attention_prompt.cu)
  int min_tiles;          // key tiles that a split has at least
  int skip_single;        // tokens alone in their tile's cache row are left out
  int only_single;        // the per-token kernel runs for those alone
};

// How a call runs: which kernels, with how many key splits, and the scratch they use.
struct CacheAttnPlan {
  bool prompt;        // the tile kernel (else the per-token one)
  bool singles;       // and then the per-token kernel for single tokens
  int splits, token_splits;
  long long part_floats, counters;
};
CacheAttnPlan cache_attention_plan(const qi_kv_layer& c, int heads, int M, int window, int sinks, int query_run);
// The plan with at most the given scratch.
void cache_attention_fit(CacheAttnPlan& plan, const qi_kv_layer& c, int heads, int M, long long part_floats,
                         long long counters);
cudaError_t launch_cache_attention(const CacheAttnParams& p, const CacheAttnPlan& plan, cudaStream_t s, bool pdl);
// Clusters of `size` CTAs (2..8) of that kernel that run at once on the current device.
int prompt_clusters(int size);
cudaError_t launch_cache_attention_prompt(const CacheAttnParams& p, cudaStream_t s, bool pdl);

}  // namespace qi

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
  int q_vec;              // q rows can be read 16 bytes at a time
  int heads, group;       // query heads, and those of one KV head
  const int32_t* rows;
  const int32_t* pos;
  int M;
  int window, sinks;      // window 0: none
  float scale_log2;       // log2(e) / sqrt(head_dim)
  void* out;              // (M, heads, head_dim), may be null
  uint16_t* out_act;      // activation tiles of token tile out_nt for the o projection, may be null
  int out_nt;
  float* part;            // (M, kv_heads, splits, group, head_dim + 2) fp32
  unsigned int* counters; // M * kv_heads, zero between calls
  int splits;
  int* err;
};

// Key splits of a decode-like call of M tokens over up to max_len keys.
int cache_attention_splits(int M, int kv_heads, int max_len, int window, int sinks);
cudaError_t launch_cache_attention(const CacheAttnParams& p, int query_run, cudaStream_t s, bool pdl);

}  // namespace qi

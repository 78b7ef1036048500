// Log probabilities of given tokens, the entropy and the top alternatives of each row of
// logits, in one pass over the logits.
//
//   m = max x,  Z = sum e^(x - m),  A = sum e^(x - m) (x - m):
//   log p(target) = x_target - m - log Z,  entropy = log Z - A / Z.
//
// Every lane keeps (m, Z, A) of its own elements and rescales them when its maximum grows:
// with f = e^(m - m'), Z' = f Z and A' = f (A + Z (m - m')). A logit of -inf has weight 0.
// The top alternatives: each warp keeps its best 32 as (order of the value, inverted index)
// words, lane i the i-th best, so that equal values go to the lower index; an element can
// enter only if it reaches the top-th best so far, which after a first threshold from the
// lanes' own maxima few do. Two sorted lists merge in 6 exchange steps.
//
// A call reads its logits once and is bound by those bytes. Few rows are cut into slices so
// that all SMs load; the last slice of a row to finish merges the row's slices in order.
#include "cache_layer.cuh"
#include "logprobs.h"

namespace qi {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kList = 32;
constexpr float kLog2e = 1.4426950408889634f;
// e^kFar is 0 in fp32, and a sum of weights times kFar is finite: distances of masked logits
// (-inf, or a type's lowest value) stop there
constexpr float kFar = -1e4f;
constexpr unsigned kAll = 0xffffffffu;

typedef unsigned long long u64;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float key_value(u64 key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

struct Stats {
  float m, z, a;
};
__device__ __forceinline__ void merge(Stats& s, const Stats& t) {
  const float m = fmaxf(s.m, t.m);
  // an empty side (maximum -inf, sum 0) adds nothing; a NaN sum stays one
  const float ds = s.m == -INFINITY ? 0.f : fmaxf(s.m - m, kFar), dt = t.m == -INFINITY ? 0.f : fmaxf(t.m - m, kFar);
  const float fs = ex2(ds * kLog2e), ft = ex2(dt * kLog2e);
  const float a = fs * fmaf(s.z, ds, s.a) + ft * fmaf(t.z, dt, t.a);
  s.z = fs * s.z + ft * t.z;
  s.a = a;
  s.m = m;
}
__device__ __forceinline__ Stats warp_stats(Stats s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stats t = {__shfl_xor_sync(kAll, s.m, o), __shfl_xor_sync(kAll, s.z, o), __shfl_xor_sync(kAll, s.a, o)};
    merge(s, t);
  }
  return s;
}

// list: lane i holds the i-th best. Merge with another sorted list held the same way.
__device__ __forceinline__ u64 merge_lists(u64 list, u64 other, int lane) {
  const u64 rev = __shfl_sync(kAll, other, 31 - lane);
  list = rev > list ? rev : list;  // the 32 best of both, as a bitonic sequence
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 x = __shfl_xor_sync(kAll, list, o);
    list = ((lane & o) == 0) == (x > list) ? x : list;
  }
  return list;
}

// the k-th largest of the lanes' values (1 <= k <= 32)
__device__ __forceinline__ float kth_of_lanes(float v, int k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const float x = __shfl_xor_sync(kAll, v, o);
      const bool down = (lane & size) == 0 || size == 32;
      v = ((lane & o) == 0) == down ? fmaxf(v, x) : fminf(v, x);
    }
  return __shfl_sync(kAll, v, k - 1);
}

template <int DT>
struct Vec {
  static constexpr int N = DT == QI_F32 ? 4 : 8;
};
template <int DT>
__device__ __forceinline__ void unpack(const uint4& u, float* x) {
  if constexpr (DT == QI_F32) {
    x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == QI_BF16) {
        x[2 * i] = bf16lo(w[i]), x[2 * i + 1] = bf16hi(w[i]);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    }
  }
}

template <int DT, bool TOP>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const LogprobParams p) {
  constexpr int VN = Vec<DT>::N, U = 2;  // elements of a 16-byte load, loads per step
  constexpr int ES = DT == QI_F32 ? 4 : 2;
  __shared__ Stats wstats[kWarps];
  __shared__ u64 wlist[kWarps][kList];
  __shared__ int last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.slices, t = blockIdx.x / S, slice = blockIdx.x - t * S;
  const uint8_t* row = static_cast<const uint8_t*>(p.logits) + (long long)t * p.ld * ES;
  // whole 16-byte vectors from the first aligned element on, shared evenly by the slices;
  // the elements before and after them go to the first and the last slice
  const int head = min(p.V, (int)((16 - ((uintptr_t)row & 15)) & 15) / ES);
  const int nvec = (p.V - head) / VN;
  const int v0 = (int)((long long)nvec * slice / S), v1 = (int)((long long)nvec * (slice + 1) / S);
  const uint4* vec = reinterpret_cast<const uint4*>(row + head * ES);

  Stats s = {-INFINITY, 0.f, 0.f};
  u64 list = 0ull;        // TOP: lane i holds the warp's i-th best
  float thr = -INFINITY;  // no element below it can enter
  bool primed = false;

  // N elements of this lane; x[j] has index idx(j), unless it is beyond n
  auto take = [&](auto& x, int n, auto idx) {
    constexpr int N = sizeof(x) / sizeof(float);
    float vm = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) vm = fmaxf(vm, x[j]);
    if (vm > s.m) {
      const float d = s.m == -INFINITY ? 0.f : fmaxf(s.m - vm, kFar), f = ex2(d * kLog2e);
      s.a = f * fmaf(s.z, d, s.a);
      s.z *= f;
      s.m = vm;
    }
    const float mr = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = x[j] - mr, e = ex2(d * kLog2e);
      s.z += e;
      s.a = fmaf(e, fmaxf(d, kFar), s.a);
    }
    if constexpr (TOP) {
      if (!primed) {
        thr = kth_of_lanes(vm, p.top, lane);
        primed = true;
      }
      if (__any_sync(kAll, vm >= thr)) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          unsigned go = __ballot_sync(kAll, j < n && x[j] >= thr);
          const u64 mine = argmax_pack(x[j], idx(j));
          while (go) {
            const int src = __ffs(go) - 1;
            go &= go - 1;
            const u64 key = __shfl_sync(kAll, mine, src);
            const int at = __popc(__ballot_sync(kAll, list > key));
            if (at < p.top) {
              const u64 up = __shfl_up_sync(kAll, list, 1);
              list = lane > at ? up : lane == at ? key : list;
              const u64 kth = __shfl_sync(kAll, list, p.top - 1);
              if (kth) thr = fmaxf(thr, key_value(kth));
            }
          }
        }
      }
    }
  };
  {
    int v = v0 + warp * 32 * U;
    for (; v < v1; v += kThreads * U) {
      float x[U * VN];
      int n = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = v + u * 32 + lane;
        if (i < v1) {
          unpack<DT>(__ldcs(vec + i), x + u * VN);
          n = (u + 1) * VN;
        } else {
#pragma unroll
          for (int j = 0; j < VN; ++j) x[u * VN + j] = -INFINITY;
        }
      }
      take(x, n, [&](int j) { return head + (v + (j / VN) * 32 + lane) * VN + j % VN; });
    }
  }
  if (warp == 0 && (slice == 0 || slice == S - 1)) {  // at most 2 * 15 loose elements
    const int tail = head + nvec * VN;
    float x[1] = {-INFINITY};
    int i = -1;
    if (lane < 16) {
      if (slice == 0 && lane < head) i = lane;
    } else if (slice == S - 1 && tail + lane - 16 < p.V) {
      i = tail + lane - 16;
    }
    if (i >= 0) x[0] = load_elem<DT>(row, i);
    take(x, i >= 0 ? 1 : 0, [&](int) { return i; });
  }

  // warps, then slices
  s = warp_stats(s);
  if (lane == 0) wstats[warp] = s;
  if constexpr (TOP) wlist[warp][lane] = list;
  __syncthreads();
  if (warp == 0) {
    s = wstats[0];
    for (int w = 1; w < kWarps; ++w) merge(s, wstats[w]);
    if constexpr (TOP)
      for (int w = 1; w < kWarps; ++w) list = merge_lists(list, wlist[w][lane], lane);
  }
  if (S > 1) {
    float* st = p.part_stats + ((long long)t * S + slice) * 4;
    u64* ls = p.part_list + ((long long)t * S + slice) * kList;
    if (warp == 0) {
      if (lane == 0) __stcg(reinterpret_cast<float4*>(st), make_float4(s.m, s.z, s.a, 0.f));
      if constexpr (TOP) __stcg(ls + lane, list);
      __syncwarp();
      if (lane == 0) last = atomic_add_acq_rel(p.counters + t, 1u) == (unsigned)(S - 1);
    }
    __syncthreads();
    if (!last) return;
    // warp w takes slices w, w + 8, ..; then warp 0 the warps
    s = {-INFINITY, 0.f, 0.f};
    list = 0ull;
    for (int i = warp; i < S; i += kWarps) {
      const float4 f = __ldcg(reinterpret_cast<const float4*>(p.part_stats + ((long long)t * S + i) * 4));
      merge(s, Stats{f.x, f.y, f.z});
      if constexpr (TOP) list = merge_lists(list, __ldcg(p.part_list + ((long long)t * S + i) * kList + lane), lane);
    }
    if (lane == 0) wstats[warp] = s;
    if constexpr (TOP) wlist[warp][lane] = list;
    __syncthreads();
    if (warp == 0) {
      s = wstats[0];
      for (int w = 1; w < kWarps; ++w) merge(s, wstats[w]);
      if constexpr (TOP)
        for (int w = 1; w < kWarps; ++w) list = merge_lists(list, wlist[w][lane], lane);
    }
    if (tid == 0) p.counters[t] = 0u;
  }
  if (warp != 0) return;
  const float lz = logf(s.z);
  if (lane == 0) {
    if (p.entropy) p.entropy[t] = lz - s.a / s.z;
    if (p.logprob) {
      const long long y = !p.targets   ? -1
                          : p.targets64 ? static_cast<const long long*>(p.targets)[t]
                                        : (long long)static_cast<const int32_t*>(p.targets)[t];
      p.logprob[t] = y < 0 ? 0.f : y >= p.V ? __uint_as_float(0x7fc00000u) : load_elem<DT>(row, y) - s.m - lz;
    }
  }
  if constexpr (TOP) {
    if (lane < p.top) {
      p.top_ids[(long long)t * p.top + lane] = list ? (int)(0xffffffffu - (uint32_t)list) : -1;
      p.top_logprobs[(long long)t * p.top + lane] = list ? key_value(list) - s.m - lz : -INFINITY;
    }
  }
}

template <int DT>
cudaError_t launch(const LogprobParams& p, cudaStream_t s, bool pdl) {
  (void)pdl;
  const dim3 grid((unsigned)(p.slices * p.M), 1, 1);
  if (p.top > 0) token_logprobs_kernel<DT, true><<<grid, kThreads, 0, s>>>(p);
  else token_logprobs_kernel<DT, false><<<grid, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

int logprob_slices(int M, int V) {
  // eight CTAs per SM, and at least 4096 logits for each
  int want = (8 * sm_count() + M - 1) / M, most = V / 4096;
  if (want > most) want = most;
  return want < 1 ? 1 : want > kMaxLogprobSlices ? kMaxLogprobSlices : want;
}

cudaError_t launch_token_logprobs(const LogprobParams& p, int dtype, cudaStream_t s, bool pdl) {
  if (dtype == QI_F32) return launch<QI_F32>(p, s, pdl);
  if (dtype == QI_BF16) return launch<QI_BF16>(p, s, pdl);
  return launch<QI_F16>(p, s, pdl);
}

}  // namespace qi

// Log probabilities of given tokens, the entropy and the top alternatives of each row of
// logits, in one pass over the logits.
//
//   m = max x,  Z = sum e^(x - m),  A = sum e^(x - m) (x - m):
//   log p(target) = x_target - m - log Z,  entropy = log Z - A / Z.
//
// Every lane keeps (m, Z, A) of its own elements and rescales them when its maximum grows:
// with f = e^(m - m'), Z' = f Z and A' = f (A + Z (m - m')). A logit of -inf has weight 0.
// The top alternatives: each warp keeps its best 32 as (order of the value, inverted index)
// words, lane i the i-th best, so that equal values go to the lower index. An element that
// reaches the top-th best so far goes into a buffer; 32 of them are sorted and merged into
// the list at once (15 and 6 exchange steps). The first threshold comes from the lanes' own
// maxima, so that few elements do.
//
// A call reads its logits once and is bound by those bytes. They are cut into chunks of 16 KB
// and the chunks of all rows are shared out evenly, in order, over the CTAs that are
// resident at once, so that all SMs load until the end whatever the number of rows. A
// producer thread keeps a ring of chunks under way with bulk copies, over row ends too: the
// next row streams in while a finished one is summed up. A row that several CTAs have parts
// of is merged by the last of them, in the order of the parts.
#include "cache_layer.cuh"
#include "logprobs.h"

namespace qi {

namespace {

constexpr int kWarps = 8;                     // that compute; one more copies
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kStages = 4;
constexpr int kChunk = 16384;                 // bytes; a warp's share is 4 vectors of every lane
constexpr int kCtas = 3;                      // of an SM
constexpr int kList = 32;
constexpr float kLog2e = 1.4426950408889634f;
// e^kFar is 0 in fp32, and a sum of weights times kFar is finite: distances of masked logits
// (-inf, or a type's lowest value) stop there
constexpr float kFar = -1e4f;
constexpr unsigned kAll = 0xffffffffu;

typedef unsigned long long u64;

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
  const float m = warp_max(s.m);
  const float d = s.m == -INFINITY ? 0.f : fmaxf(s.m - m, kFar), f = ex2(d * kLog2e);
  const float a = f * fmaf(s.z, d, s.a);
  return Stats{m, warp_sum(f * s.z), warp_sum(a)};
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

// the lanes' words in descending order
__device__ __forceinline__ u64 sort_lanes(u64 v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const u64 x = __shfl_xor_sync(kAll, v, o);
      const bool down = (lane & size) == 0 || size == 32;
      v = (((lane & o) == 0) == down) == (x > v) ? x : v;
    }
  return v;
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

// A warp's candidates for the top alternatives: its best 32 so far, and words that may enter.
struct Best {
  u64 list;    // lane i: the i-th best
  float thr;   // nothing below it can enter
  int n;       // words in buf (< 32 between calls)
  u64* buf;    // 64 words of shared memory
  __device__ __forceinline__ void flush(int top, int lane) {
    __syncwarp();
    list = merge_lists(list, sort_lanes(lane < n ? buf[lane] : 0ull, lane), lane);
    const u64 rest = lane + 32 < n ? buf[lane + 32] : 0ull;
    __syncwarp();
    buf[lane] = rest;
    n = max(n - 32, 0);
    const u64 kth = __shfl_sync(kAll, list, top - 1);
    if (kth) thr = fmaxf(thr, key_value(kth));
  }
  // this lane's x (index idx) if `in`
  __device__ __forceinline__ void offer(bool in, float x, int idx, int top, int lane) {
    const unsigned go = __ballot_sync(kAll, in && x >= thr);
    if (!go) return;
    if (in && x >= thr) buf[n + __popc(go & ((1u << lane) - 1u))] = argmax_pack(x, idx);
    n += __popc(go);
    if (n >= 32) flush(top, lane);
  }
};

// chunks [u0, u1) of CTA c, and the CTA that has chunk u, when G CTAs share T chunks evenly
__device__ __forceinline__ int share(int c, long long T, int G) { return (int)(c * T / G); }
__device__ __forceinline__ int owner(long long u, long long T, int G) { return (int)(((u + 1) * G - 1) / T); }

struct Ring {
  uint64_t full[kStages], empty[kStages];
};

template <int DT, bool TOP>
__global__ void __launch_bounds__(kThreads, kCtas) token_logprobs_kernel(const LogprobParams p) {
  constexpr int VN = Vec<DT>::N, ES = DT == QI_F32 ? 4 : 2;
  constexpr int U = DT == QI_F32 ? 4 : 2, N = U * VN;  // vectors and elements of a lane's step
  constexpr int kVecs = kChunk / 16, kSteps = kVecs / (32 * kWarps * U);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Ring ring;
  __shared__ Stats wstats[kWarps];
  __shared__ u64 wlist[kWarps][kList];
  __shared__ u64 wbuf[TOP ? kWarps : 1][2 * kList];
  __shared__ int last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = gridDim.x;
  // chunks of a row: its whole 16-byte vectors, from the first aligned element on
  const int cpr = p.chunks;
  const long long T = (long long)p.M * cpr;
  const int u0 = share(blockIdx.x, T, G), u1 = share(blockIdx.x + 1, T, G);
  auto row_of = [&](int t) { return static_cast<const uint8_t*>(p.logits) + (long long)t * p.ld * ES; };
  auto head_of = [&](const uint8_t* row) { return min(p.V, (int)((16 - ((uintptr_t)row & 15)) & 15) / ES); };
  auto vecs_in = [&](int nvec, int k) { return max(0, min(kVecs, nvec - k * kVecs)); };  // of chunk k

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&ring.full[s], 1);
      mbar_init(&ring.empty[s], kWarps);
    }
    fence_barrier_init();
  }
  __syncthreads();
  if (warp == kWarps) {
    if (lane == 0) {
      for (int u = u0; u < u1; ++u) {
        const int i = u - u0, s = i % kStages, t = u / cpr, k = u - t * cpr;
        const uint8_t* row = row_of(t);
        const int head = head_of(row), n = vecs_in((p.V - head) / VN, k);
        if (i >= kStages && !mbar_wait(&ring.empty[s], (uint32_t)((i / kStages - 1) & 1), nullptr)) break;
        mbar_arrive_expect_tx(&ring.full[s], (uint32_t)n * 16u);
        if (n > 0) bulk_g2s(smem + s * kChunk, row + head * ES + (long long)k * kChunk, (uint32_t)n * 16u, &ring.full[s]);
      }
    }
    return;
  }
  auto bar = [&] { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); };

  int u = u0;
  while (u < u1) {  // a row, or the part of it that is this CTA's
    const int t = u / cpr, k0 = u - t * cpr, k1 = min(cpr, k0 + u1 - u);
    const uint8_t* row = row_of(t);
    const int head = head_of(row), nvec = (p.V - head) / VN;
    Stats s = {-INFINITY, 0.f, 0.f};
    f2 z = 0ull, a = 0ull;  // this lane's sums in pairs
    Best best = {0ull, -INFINITY, 0, wbuf[TOP ? warp : 0]};
    bool primed = false;
    auto rescale = [&](float m) {  // the sums relative to a new maximum
      const float d = s.m == -INFINITY ? 0.f : fmaxf(s.m - m, kFar), f = ex2(d * kLog2e);
      const f2 f_2 = pack2(f, f);
      a = mul2(f_2, fma2(z, pack2(d, d), a));
      z = mul2(f_2, z);
      s.m = m;
    };
    auto add = [&](float x0, float x1, f2 mr) {
      const f2 d = add2(pack2(x0, x1), mr);
      const float2 y = unpack2(mul2(d, pack2(kLog2e, kLog2e))), dd = unpack2(d);
      const f2 e = pack2(ex2(y.x), ex2(y.y));
      z = add2(z, e);
      a = fma2(e, pack2(fmaxf(dd.x, kFar), fmaxf(dd.y, kFar)), a);
    };
    for (int k = k0; k < k1; ++k, ++u) {
      const int i = u - u0, st = i % kStages, n = vecs_in(nvec, k);
      mbar_wait(&ring.full[st], (uint32_t)((i / kStages) & 1), nullptr);
      const uint4* c = reinterpret_cast<const uint4*>(smem + st * kChunk) + warp * (kVecs / kWarps) + lane;
      const int v0 = warp * (kVecs / kWarps) + lane;  // this lane's first vector of the chunk
#pragma unroll
      for (int j0 = 0; j0 < kSteps; ++j0) {
        float x[N];
        const int v = v0 + j0 * 32 * U;
#pragma unroll
        for (int w = 0; w < U; ++w) {
          if (v + w * 32 < n) {
            unpack<DT>(c[j0 * 32 * U + w * 32], x + w * VN);
          } else {
#pragma unroll
            for (int j = 0; j < VN; ++j) x[w * VN + j] = -INFINITY;
          }
        }
        if (j0 == kSteps - 1) {  // the chunk is read
          __syncwarp();
          if (lane == 0) mbar_arrive(&ring.empty[st]);
        }
        float m4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int j = 4; j < N; ++j) m4[j & 3] = fmaxf(m4[j & 3], x[j]);
        const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        if (m > s.m) rescale(m);
        const float mr = s.m == -INFINITY ? 0.f : -s.m;
        const f2 mr2 = pack2(mr, mr);
#pragma unroll
        for (int j = 0; j < N; j += 2) add(x[j], x[j + 1], mr2);
        if constexpr (TOP) {
          if (!primed) {  // the lanes' largest of the first step give a first threshold
            best.thr = kth_of_lanes(m, p.top, lane);
            primed = true;
          }
          if (__any_sync(kAll, m >= best.thr)) {
#pragma unroll
            for (int j = 0; j < N; ++j)
              best.offer(v + (j / VN) * 32 < n, x[j], head + (k * kVecs + v + (j / VN) * 32) * VN + j % VN, p.top, lane);
          }
        }
      }
    }
    if (warp == 0 && (k0 == 0 || k1 == cpr)) {  // at most 2 * 15 loose elements, before and after the vectors
      const int tail = head + nvec * VN;
      int i = -1;
      if (lane < 16) {
        if (k0 == 0 && lane < head) i = lane;
      } else if (k1 == cpr && tail + lane - 16 < p.V) {
        i = tail + lane - 16;
      }
      const float x = i >= 0 ? load_elem<DT>(row, i) : -INFINITY;
      if (x > s.m) rescale(x);
      const float mr = s.m == -INFINITY ? 0.f : -s.m;
      add(x, -INFINITY, pack2(mr, mr));
      if constexpr (TOP) best.offer(i >= 0, x, i, p.top, lane);
    }
    const float2 z2 = unpack2(z), a2 = unpack2(a);
    s.z = z2.x + z2.y, s.a = a2.x + a2.y;
    u64 list = 0ull;
    if constexpr (TOP) {
      if (best.n > 0) best.flush(p.top, lane);
      list = best.list;
    }

    // the warps (halves of them onto the others), then the parts of the row
    auto join = [&] {
      for (int half = kWarps / 2; half > 0; half >>= 1) {
        if (warp >= half && warp < 2 * half) {
          if (lane == 0) wstats[warp] = s;
          if constexpr (TOP) wlist[warp][lane] = list;
        }
        bar();
        if (warp < half) {
          merge(s, wstats[warp + half]);
          if constexpr (TOP) list = merge_lists(list, wlist[warp + half][lane], lane);
        }
      }
    };
    s = warp_stats(s);
    join();
    const int c0 = owner((long long)t * cpr, T, G), parts = owner((long long)(t + 1) * cpr - 1, T, G) - c0 + 1;
    // a CTA has at most two parts of rows: of the row that its share begins in, and of the last
    auto place = [&](int c) { return 2 * c + (share(c, T, G) >= (long long)t * cpr ? 0 : 1); };
    bool mine = true;
    if (parts > 1) {
      if (warp == 0) {
        const int at = place(blockIdx.x);
        if (lane == 0) __stcg(reinterpret_cast<float4*>(p.part_stats) + at, make_float4(s.m, s.z, s.a, 0.f));
        if constexpr (TOP) __stcg(p.part_list + (long long)at * kList + lane, list);
        __syncwarp();
        if (lane == 0) last = atomic_add_acq_rel(p.counters + c0, 1u) == (unsigned)(parts - 1);
      }
      bar();
      mine = last != 0;
      bar();
      if (mine) {
        s = {-INFINITY, 0.f, 0.f};
        list = 0ull;
        for (int i = warp; i < parts; i += kWarps) {
          const int at = place(c0 + i);
          const float4 f = __ldcg(reinterpret_cast<const float4*>(p.part_stats) + at);
          u64 other = 0ull;
          if constexpr (TOP) other = __ldcg(p.part_list + (long long)at * kList + lane);
          merge(s, Stats{f.x, f.y, f.z});
          if constexpr (TOP) list = merge_lists(list, other, lane);
        }
        join();
        if (tid == 0) p.counters[c0] = 0u;  // as the next call expects it
      }
    }
    if (mine && warp == 0) {
      const float lz = logf(s.z);
      if (lane == 0) {
        if (p.entropy) p.entropy[t] = lz - s.a / s.z;
        if (p.logprob) {
          const long long y = !p.targets    ? -1
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
    bar();  // the next row's sums take the same shared memory
  }
}

template <int DT>
cudaError_t launch(const LogprobParams& p, int ctas, cudaStream_t s) {
  constexpr int smem = kStages * kChunk;
  const void* fn = p.top > 0 ? reinterpret_cast<const void*>(token_logprobs_kernel<DT, true>)
                             : reinterpret_cast<const void*>(token_logprobs_kernel<DT, false>);
  const cudaError_t e = set_max_dynamic_smem(fn, smem);
  if (e != cudaSuccess) return e;
  if (p.top > 0) token_logprobs_kernel<DT, true><<<ctas, kThreads, smem, s>>>(p);
  else token_logprobs_kernel<DT, false><<<ctas, kThreads, smem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

LogprobPlan logprob_plan(int M, int V, int dtype) {
  LogprobPlan r;
  const int vn = dtype == QI_F32 ? 4 : 8, kv = kChunk / 16;
  r.chunks = (V / vn + kv - 1) / kv;
  if (r.chunks < 1) r.chunks = 1;
  const long long T = (long long)M * r.chunks, most = (long long)kCtas * sm_count();
  r.ctas = (int)(T < most ? T : most);
  r.scratch = (long long)r.ctas * 2 * (16 + kList * 8);
  return r;
}

cudaError_t launch_token_logprobs(const LogprobParams& args, const LogprobPlan& plan, int dtype, cudaStream_t s) {
  LogprobParams p = args;
  p.chunks = plan.chunks;
  if (dtype == QI_F32) return launch<QI_F32>(p, plan.ctas, s);
  if (dtype == QI_BF16) return launch<QI_BF16>(p, plan.ctas, s);
  return launch<QI_F16>(p, plan.ctas, s);
}

}  // namespace qi

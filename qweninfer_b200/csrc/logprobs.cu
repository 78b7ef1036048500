// Log probabilities of given tokens, the entropy and the top alternatives of each row of
// logits, in one pass over the logits.
//
// with m = max x and y = (x - m) log2(e):
//   Z = sum 2^y,  A = sum 2^y y,  log p(target) = x_target - m - log Z,
//   entropy = log 2 (log2 Z - A / Z).
//
// Every lane keeps (m, Z, A) of its own elements and rescales them when its maximum grows:
// with d = (m - m') log2(e) and f = 2^d, Z' = f Z and A' = f (A + Z d). A logit of -inf has
// weight 0.
// The top alternatives are words (order of the value, inverted index), so that equal values
// go to the lower index. While a row streams by, a lane only keeps its largest logit, and
// which of its steps reached the top-th largest of the lanes' first ones. Of the lanes'
// largest, the top-th is then a bound that hardly more than top elements reach: the steps of
// the lanes that reach it are read again, their elements above it sorted. (More than 64 of
// them or 128 steps, as in a row of equal values: every warp keeps a list of its best 32 instead, 32 candidates
// sorted and merged into it at a time.)
// A call reads its logits once and is bound by those bytes. They are cut into chunks of 32 KB
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
constexpr int kStages = 2;
// Bytes of a chunk (a warp's share is 8 vectors of every lane) and CTAs of an SM. 64 rows of
// 151936 bf16, top 20: 19.8 us, 1000 rows of fp32: 100 (0.94 of the copy rate); with chunks of 16 KB in
// four stages 22.3 and 97, with two CTAs of three stages 25.2 and 101.
constexpr int kChunk = 32768;
constexpr int kCtas = 3;
constexpr int kList = 32;
constexpr int kPairs = 128;                   // steps that are read again
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// 2^kFar is 0 in fp32, and a sum of weights times kFar is finite: distances of masked logits
// (-inf, or a type's lowest value) stop there
constexpr float kFar = -1e4f;
constexpr unsigned kAll = 0xffffffffu;

typedef unsigned long long u64;

__device__ __forceinline__ float key_value(u64 key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

struct Stats {
  float m, z, a;
};
__device__ __forceinline__ void merge(Stats& s, const Stats& t) {
  const float m = fmaxf(s.m, t.m);
  // an empty side (maximum -inf, sum 0) adds nothing; a NaN sum stays one
  const float ds = s.m == -INFINITY ? 0.f : fmaxf((s.m - m) * kLog2e, kFar);
  const float dt = t.m == -INFINITY ? 0.f : fmaxf((t.m - m) * kLog2e, kFar);
  const float fs = ex2(ds), ft = ex2(dt);
  const float a = fs * fmaf(s.z, ds, s.a) + ft * fmaf(t.z, dt, t.a);
  s.z = fs * s.z + ft * t.z;
  s.a = a;
  s.m = m;
}
__device__ __forceinline__ Stats warp_stats(Stats s) {
  const float m = warp_max(s.m);
  const float d = s.m == -INFINITY ? 0.f : fmaxf((s.m - m) * kLog2e, kFar), f = ex2(d);
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
// the lanes' values in descending order
__device__ __forceinline__ float sort_lanes(float v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const float x = __shfl_xor_sync(kAll, v, o);
      const bool down = (lane & size) == 0 || size == 32;
      v = ((lane & o) == 0) == down ? fmaxf(v, x) : fminf(v, x);
    }
  return v;
}
// the 32 largest of two descending sequences, descending
__device__ __forceinline__ float merge_lists(float list, float other, int lane) {
  list = fmaxf(list, __shfl_sync(kAll, other, 31 - lane));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float x = __shfl_xor_sync(kAll, list, o);
    list = (lane & o) == 0 ? fmaxf(list, x) : fminf(list, x);
  }
  return list;
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

// A warp's list of its best 32 so far, and words that may enter.
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

// element i of a vector array in shared memory
template <int DT>
__device__ __forceinline__ float elem(const uint4* v, int i) {
  if constexpr (DT == QI_F32) return reinterpret_cast<const float*>(v)[i];
  else if constexpr (DT == QI_BF16) return bf16_to_f32(reinterpret_cast<const uint16_t*>(v)[i]);
  else return __half2float(reinterpret_cast<const __half*>(v)[i]);
}

struct Yes {
  static constexpr bool value = true;
};
struct No {
  static constexpr bool value = false;
};

struct Ring {
  uint64_t full[kStages], empty[kStages];
};

template <int DT, bool TOP>
__global__ void __launch_bounds__(kThreads, kCtas) token_logprobs_kernel(const LogprobParams p) {
  constexpr int VN = Vec<DT>::N, ES = DT == QI_F32 ? 4 : 2;
  constexpr int U = DT == QI_F32 ? 8 : 4, N = U * VN;  // vectors and elements of a lane's step
  constexpr int kVecs = kChunk / 16, kSteps = kVecs / (32 * kWarps * U);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Ring ring;
  __shared__ Stats wstats[kWarps];
  __shared__ u64 wlist[kWarps][kList];
  __shared__ float wmax[kWarps][kList];
  __shared__ u64 wbuf[TOP ? kWarps : 1][2 * kList];
  __shared__ int last, found, pairs;
  __shared__ int2 again[TOP ? kPairs : 1];
  __shared__ float bound;
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
    uint32_t hot = 0u;      // TOP: bit i: a step i, i + 32, .. of this lane may have a candidate
    float first_bound = -INFINITY;
    auto rescale = [&](float m) {  // the sums relative to a new maximum
      const float d = s.m == -INFINITY ? 0.f : fmaxf((s.m - m) * kLog2e, kFar), f = ex2(d);
      const f2 f_2 = pack2(f, f);
      a = mul2(f_2, fma2(z, pack2(d, d), a));
      z = mul2(f_2, z);
      s.m = m;
    };
    auto add = [&](f2 y) {  // y not below kFar, or 2^y without -inf
      const float2 v = unpack2(y);
      const f2 e = pack2(ex2(v.x), ex2(v.y));
      z = add2(z, e);
      a = fma2(e, y, a);
    };
    auto add_far = [&](f2 y) {
      const float2 v = unpack2(y);
      const f2 e = pack2(ex2(v.x), ex2(v.y));  // (a NaN stays one)
      z = add2(z, e);
      a = fma2(e, pack2(fmaxf(v.x, kFar), fmaxf(v.y, kFar)), a);
    };
    const f2 log2e = pack2(kLog2e, kLog2e);
    for (int k = k0; k < k1; ++k, ++u) {
      const int i = u - u0, st = i % kStages, n = vecs_in(nvec, k);
      // a copy that never came makes the row's results NaN
      if (!mbar_wait(&ring.full[st], (uint32_t)((i / kStages) & 1), nullptr)) z = pack2(NAN, NAN);
      const int v0 = warp * (kVecs / kWarps) + lane;  // this lane's first vector of the chunk
      const uint4* c = reinterpret_cast<const uint4*>(smem + st * kChunk) + v0;
      auto chunk = [&](auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
#pragma unroll 1
        for (int j0 = 0; j0 < kSteps; ++j0) {
          float x[N];
          const int v = v0 + j0 * 32 * U;
#pragma unroll
          for (int w = 0; w < U; ++w) {
            if (kWhole || v + w * 32 < n) {
              unpack<DT>(c[j0 * 32 * U + w * 32], x + w * VN);
            } else {
#pragma unroll
              for (int j = 0; j < VN; ++j) x[w * VN + j] = -INFINITY;
            }
          }
          float m = x[0], lo = x[0];
#pragma unroll
          for (int j = 1; j + 1 < N; j += 2) m = max3(m, x[j], x[j + 1]), lo = min3(lo, x[j], x[j + 1]);
          m = fmaxf(m, x[N - 1]), lo = fminf(lo, x[N - 1]);
          if (m > s.m) rescale(m);
          const float mr = s.m == -INFINITY ? 0.f : -s.m;
          const f2 mr2 = pack2(mr, mr);
          if ((lo + mr) * kLog2e >= kFar) {
#pragma unroll
            for (int j = 0; j < N; j += 2) add(mul2(add2(pack2(x[j], x[j + 1]), mr2), log2e));
          } else {
#pragma unroll
            for (int j = 0; j < N; j += 2) add_far(mul2(add2(pack2(x[j], x[j + 1]), mr2), log2e));
          }
          if constexpr (TOP) {
            const int step = (k - k0) * kSteps + j0;
            // (a step of nothing but NaN has no say: sorted, it would pass another lane's maximum on twice)
            if (step == 0) first_bound = __shfl_sync(kAll, sort_lanes(m == m ? m : -INFINITY, lane), p.top - 1);
            hot |= (m >= first_bound ? 1u : 0u) << (step & 31);
          }
        }
      };
      if (n == kVecs) chunk(Yes{});
      else chunk(No{});
      __syncwarp();
      if (lane == 0) mbar_arrive(&ring.empty[st]);  // the chunk is read
    }
    // at most 2 * 15 loose elements, before and after the vectors
    int loose = -1;
    float xl = -INFINITY;
    if (warp == 0) {
      const int tail = head + nvec * VN;
      if (lane < 16) {
        if (k0 == 0 && lane < head) loose = lane;
      } else if (k1 == cpr && tail + lane - 16 < p.V) {
        loose = tail + lane - 16;
      }
      if (loose >= 0) xl = load_elem<DT>(row, loose);
      if (xl > s.m) rescale(xl);
      const float mr = s.m == -INFINITY ? 0.f : -s.m;
      add_far(mul2(add2(pack2(xl, -INFINITY), pack2(mr, mr)), log2e));
    }
    const float2 z2 = unpack2(z), a2 = unpack2(a);
    s.z = z2.x + z2.y, s.a = a2.x + a2.y;

    // lists and statistics of the warps onto warp 0, halves of them onto the others
    auto join_lists = [&](u64& list) {
      for (int half = kWarps / 2; half > 0; half >>= 1) {
        if (warp >= half && warp < 2 * half) wlist[warp][lane] = list;
        bar();
        if (warp < half) list = merge_lists(list, wlist[warp + half][lane], lane);
      }
    };
    auto join_stats = [&](Stats& x) {  // x of the warps' lanes 0, which warp 0 has after it
      if (lane == 0) wstats[warp] = x;
      bar();
      if (warp == 0) {
        x = wstats[lane & (kWarps - 1)];
#pragma unroll
        for (int o = kWarps / 2; o > 0; o >>= 1) {
          const Stats y = {__shfl_xor_sync(kAll, x.m, o), __shfl_xor_sync(kAll, x.z, o), __shfl_xor_sync(kAll, x.a, o)};
          if ((lane & o) == 0) merge(x, y);  // the upper lane's onto the lower one's
        }
        x = {__shfl_sync(kAll, x.m, 0), __shfl_sync(kAll, x.z, 0), __shfl_sync(kAll, x.a, 0)};
      }
    };
    u64 list = 0ull;
    if constexpr (TOP) {
      float top = sort_lanes(s.m, lane);
      for (int half = kWarps / 2; half > 0; half >>= 1) {
        if (warp >= half && warp < 2 * half) wmax[warp][lane] = top;
        bar();
        if (warp < half) top = merge_lists(top, wmax[warp + half][lane], lane);
      }
      if (tid == p.top - 1) bound = top;
      if (tid == 0) found = pairs = 0;
      bar();
      const float least = bound;
      const int steps = (k1 - k0) * kSteps;
      // every element of this warp that may reach the bound: f(whether it does, value, index)
      auto candidates = [&](auto f) {
        if (warp == 0) f(loose >= 0 && xl >= least, xl, loose);
        for (unsigned go = __ballot_sync(kAll, s.m >= least); go; go &= go - 1) {
          const int from = __ffs(go) - 1;
          for (uint32_t h = __shfl_sync(kAll, hot, from); h; h &= h - 1)
            for (int st = __ffs(h) - 1; st < steps; st += 32) {  // a step's 32 elements, one for each lane
              const int k = k0 + st / kSteps, v = warp * (kVecs / kWarps) + (st % kSteps) * 32 * U + from + lane / VN * 32;
              const int i = head + (k * kVecs + v) * VN + lane % VN;
              const bool in = v < vecs_in(nvec, k);
              const float x = in ? load_elem<DT>(row, i) : 0.f;
              f(in && x >= least, x, i);
            }
        }
      };
      // Steps to read again, as (warp and lane, step), shared out over the warps; their elements
      // that reach the bound go into one buffer.
      if (s.m >= least)
        for (uint32_t h = hot; h; h &= h - 1)
          for (int st = __ffs(h) - 1; st < steps; st += 32) {
            const int at = atomicAdd(&pairs, 1);
            if (at < kPairs) again[at] = make_int2(tid, st);
          }
      bar();
      const int np = pairs;
      auto push = [&](bool in, float x, int i) {
        const unsigned go = __ballot_sync(kAll, in);
        if (!go) return;
        int at = lane == 0 ? atomicAdd(&found, __popc(go)) : 0;
        at = __shfl_sync(kAll, at, 0) + __popc(go & ((1u << lane) - 1u));
        if (in && at < 2 * kList) wbuf[0][at] = argmax_pack(x, i);
      };
      if (np <= kPairs) {
        if (warp == 0) push(loose >= 0 && xl >= least, xl, loose);
        constexpr int B = 4;  // loads under way together
        for (int q = warp; q < np; q += B * kWarps) {
          float x[B];
          int i[B];
#pragma unroll
          for (int b = 0; b < B; ++b) {
            const int2 pr = again[min(q + b * kWarps, kPairs - 1)];
            i[b] = -1, x[b] = 0.f;
            if (q + b * kWarps < np) {
              const int k = k0 + pr.y / kSteps;
              const int v = (pr.x >> 5) * (kVecs / kWarps) + (pr.y % kSteps) * 32 * U + (pr.x & 31) + lane / VN * 32;
              if (v < vecs_in(nvec, k)) {
                i[b] = head + (k * kVecs + v) * VN + lane % VN;
                x[b] = load_elem<DT>(row, i[b]);
              }
            }
          }
#pragma unroll
          for (int b = 0; b < B; ++b) push(i[b] >= 0 && x[b] >= least, x[b], i[b]);
        }
      }
      bar();
      const int n = np <= kPairs ? found : 2 * kList + 1;
      if (n <= 2 * kList) {
        if (warp == 0) {
          list = sort_lanes(lane < n ? wbuf[0][lane] : 0ull, lane);
          if (n > kList) list = merge_lists(list, sort_lanes(lane + kList < n ? wbuf[0][lane + kList] : 0ull, lane), lane);
        }
      } else {
        bar();  // (warp 0's buffer is the one just counted)
        Best best = {0ull, least, 0, wbuf[warp]};
        candidates([&](bool in, float x, int i) { best.offer(in, x, i, p.top, lane); });
        if (best.n > 0) best.flush(p.top, lane);
        list = best.list;
        join_lists(list);
      }
    }
    s = warp_stats(s);
    join_stats(s);
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
        if constexpr (TOP) join_lists(list);
        bar();  // (what the statistics of this CTA's part were joined in)
        join_stats(s);
        if (tid == 0) p.counters[c0] = 0u;  // as the next call expects it
      }
    }
    if (mine && warp == 0) {
      const float lz = log2f(s.z);
      auto logprob = [&](float x) { return fmaf(-lz, kLn2, x - s.m); };
      if (lane == 0) {
        if (p.entropy) p.entropy[t] = (lz - s.a / s.z) * kLn2;
        if (p.logprob) {
          const long long y = !p.targets    ? -1
                              : p.targets64 ? static_cast<const long long*>(p.targets)[t]
                                            : (long long)static_cast<const int32_t*>(p.targets)[t];
          p.logprob[t] = y < 0 ? 0.f : y >= p.V ? __uint_as_float(0x7fc00000u) : logprob(load_elem<DT>(row, y));
        }
      }
      if constexpr (TOP) {
        if (lane < p.top) {
          p.top_ids[(long long)t * p.top + lane] = list ? (int)(0xffffffffu - (uint32_t)list) : -1;
          p.top_logprobs[(long long)t * p.top + lane] = list ? logprob(key_value(list)) : -INFINITY;
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
  // as many chunks for each as the resident CTAs need, then no more CTAs than that takes: an
  // uneven share would only give some CTAs the ends of two rows
  const long long per = (T + most - 1) / most;
  r.ctas = (int)((T + per - 1) / per);
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

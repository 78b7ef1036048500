// Device code shared by the cached-attention kernels: the keys a token sees, wide codes,
// 16-bit parts of fp32 values and output stores.
#pragma once

#include "cache_attention.h"
#include "cache_layer.cuh"
#include "tc_proj.h"

namespace qi {
namespace cattn {

constexpr int kMaxGroup = 8;
// Scores (log2 units) are subtracted from their maximum in the multiplication that scales them, whose
// product is not rounded where the maximum is: all weights are off by one factor, which the
// normalisation takes out again. From this size of the maximum on (a factor of 2^(1/4)) the factor
// could leave the range of the weights: products are rounded before the subtraction.
constexpr float kFarScore = 4194304.f;  // 2^22

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---- parts of fp32 pairs as 16-bit pairs (a in the low half)
__device__ __forceinline__ uint32_t f16x2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t b16x2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// the 16-bit parts of (a, b): part 0 = round(x), each next part = round(rest)
template <bool F16, int N>
__device__ __forceinline__ void split(float a, float b, uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (F16) {
      r[i] = f16x2(a, b);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
      a -= f.x, b -= f.y;
    } else {
      r[i] = b16x2(a, b);
      a -= bf16lo(r[i]), b -= bf16hi(r[i]);
    }
  }
}

// ---- 8-bit codes as fp16 pairs. SEL 0: bytes 0, 1 and 2, 3; SEL 1: bytes 0, 2 and 1, 3
// (where a 16-bit element holds two neighbouring dims of one key). int8: the code plus 128
// as the low byte of 0x6400 is 1024 + 128 + code exactly; minus 1152.
template <int FMT, int SEL>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& p0, uint32_t& p1) {
  if constexpr (FMT == QI_KV_INT8) {
    w ^= 0x80808080u;
    const uint32_t a = __byte_perm(w, 0x64646464u, SEL ? 0x4240 : 0x4140);
    const uint32_t b = __byte_perm(w, 0x64646464u, SEL ? 0x4341 : 0x4342);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    p0 = *reinterpret_cast<const uint32_t*>(&x);
    p1 = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    if constexpr (SEL) w = __byte_perm(w, 0u, 0x3120);
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(p0), "=r"(p1)
        : "r"(w));
  }
}

// Output values of features f .. f + N - 1 (N 2 or 8, f a multiple of N) of a token.
template <int N>
__device__ __forceinline__ void emit(const CacheAttnParams& p, int tok, int f, int width, const float (&v)[N]) {
  static_assert(N == 2 || N == 8, "one store, or a row of 16 bytes");
  if (p.out) {
    const long long o = (long long)tok * width + f;
    if (p.dtype == QI_F32) {
      float* d = static_cast<float*>(p.out) + o;
      if constexpr (N == 2) {
        *reinterpret_cast<float2*>(d) = make_float2(v[0], v[1]);
      } else {
        *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(d + 4) = make_float4(v[4], v[5], v[6], v[7]);
      }
    } else {
      uint16_t* d = static_cast<uint16_t*>(p.out) + o;
      uint32_t w[N / 2];
#pragma unroll
      for (int i = 0; i < N; i += 2) w[i / 2] = p.dtype == QI_BF16 ? b16x2(v[i], v[i + 1]) : f16x2(v[i], v[i + 1]);
      if constexpr (N == 2) *reinterpret_cast<uint32_t*>(d) = w[0];
      else *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (p.out_act) {  // N consecutive features lie side by side in an activation tile
    uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      hi[i / 2] = b16x2(v[i], v[i + 1]);
      lo[i / 2] = b16x2(v[i] - bf16lo(hi[i / 2]), v[i + 1] - bf16hi(hi[i / 2]));
    }
    uint16_t* h = p.out_act + act_offset(tok, f, 0, width, p.out_nt);
    uint16_t* l = p.out_act + act_offset(tok, f, 1, width, p.out_nt);
    if constexpr (N == 2) {
      *reinterpret_cast<uint32_t*>(h) = hi[0];
      *reinterpret_cast<uint32_t*>(l) = lo[0];
    } else {
      *reinterpret_cast<uint4*>(h) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(l) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }
}

// The keys of a token as a list of granules of GRAN aligned positions: the sinks', then the
// window's.
template <int GRAN>
struct Seen {
  int p;      // its position
  int lo;     // first position of the window
  int sinks;  // visible first positions (0 when the window reaches position 0)
  int ns;     // granules of the sinks, before the window's
  int g0;     // first granule of the window
  int n;      // granules in all
  __device__ __forceinline__ int granule(int i) const { return i < ns ? i : g0 + i - ns; }
  __device__ __forceinline__ bool sees(int j) const { return j <= p && (j >= lo || j < sinks); }
  // any of the 16 positions from j on
  __device__ __forceinline__ bool sees16(int j) const { return j <= p && (j + 15 >= lo || j < sinks); }
};
__device__ __forceinline__ int window_start(int p, int window) { return window > 0 && p >= window ? p - window + 1 : 0; }
// positions lo..p and 0..sinks-1
template <int GRAN>
__device__ __forceinline__ Seen<GRAN> seen_range(int p, int lo, int sinks) {
  Seen<GRAN> s;
  s.p = p;
  s.lo = lo;
  s.sinks = min(sinks, lo);
  s.g0 = lo / GRAN;
  s.ns = min((s.sinks + GRAN - 1) / GRAN, s.g0);
  s.n = s.ns + p / GRAN + 1 - s.g0;
  return s;
}

// Whether token t's position and row lie in the cache.
__device__ __forceinline__ bool token_ok(const CacheAttnParams& p, int ps, int row) {
  return ps >= 0 && ps < p.c.max_len && row >= 0 && row < p.c.cache_rows;
}

// Weighted sum of n partials (values relative to a maximum m in log2 units, and the sum l)
// at elements d and d + 1 of a row; load(w, i) is element i of partial w's row, whose m and
// l are elements D and D + 1.
template <int D, class Load>
__device__ __forceinline__ void merge2(Load load, int n, int d, float& m_out, float& l_out, float& a, float& b) {
  float mx = -INFINITY;
  for (int w = 0; w < n; ++w) mx = fmaxf(mx, load(w, D));
  m_out = mx, l_out = 0.f, a = 0.f, b = 0.f;
#pragma unroll 4
  for (int w = 0; w < n; ++w) {
    const float mw = load(w, D), lw = load(w, D + 1);
    // a partial without keys (maximum -inf, sum 0) has nothing to add; a NaN sum stays one
    const float f = mw == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : ex2(mw - mx);
    l_out = fmaf(f, lw, l_out);
    a = fmaf(f, load(w, d), a);
    b = fmaf(f, load(w, d + 1), b);
  }
}

}  // namespace cattn
}  // namespace qi

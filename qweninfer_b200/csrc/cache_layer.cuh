// One layer of a KV cache as the cached-attention and 8-bit kernels address it: bf16 values,
// or 8-bit codes with a power-of-two scale per block of positions and KV head; packed rows
// or pages. Also the element types and fp32 helpers that these kernels and the log
// probabilities share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "internal.h"

namespace qi {

// Element offset of (row, head g, position pos) in a layer of head_dim D, or -1 when the
// position's page is unmapped.
__device__ __forceinline__ long long layer_offset(const qi_kv_layer& c, int D, int row, int g, int pos) {
  if (!c.page_table) return (((long long)row * c.kv_heads + g) * c.max_len + pos) * D;
  const int pg = __ldg(c.page_table + (long long)row * c.pages_per_row + pos / c.page_size);
  if (pg < 0 || pg >= c.n_pages) return -1;
  return (((long long)pg * c.kv_heads + g) * c.page_size + pos % c.page_size) * D;
}

// Index of the scale of (row, head g, the block holding pos), or -1 (unmapped page).
__device__ __forceinline__ long long scale_index(const qi_kv_layer& c, int row, int g, int pos) {
  if (!c.page_table)
    return ((long long)row * c.kv_heads + g) * ((c.max_len + c.block - 1) / c.block) + pos / c.block;
  const int pg = __ldg(c.page_table + (long long)row * c.pages_per_row + pos / c.page_size);
  if (pg < 0 || pg >= c.n_pages) return -1;
  return ((long long)pg * c.kv_heads + g) * (c.page_size / c.block) + (pos % c.page_size) / c.block;
}

// ------------------------------------------------------------- input elements

template <int DT>
__device__ __forceinline__ float load_elem(const void* p, long long i) {
  if constexpr (DT == QI_F32) return __ldcg(static_cast<const float*>(p) + i);
  else if constexpr (DT == QI_BF16) return bf16_to_f32(__ldcg(static_cast<const unsigned short*>(p) + i));
  else return __half2float(__ushort_as_half(__ldcg(static_cast<const unsigned short*>(p) + i)));
}

__device__ __forceinline__ void store_elem(void* p, int dtype, long long i, float v) {
  if (dtype == QI_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == QI_BF16) static_cast<uint16_t*>(p)[i] = f32_to_bf16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// 4 consecutive elements; `vec`: the address is aligned for one load
template <int DT>
__device__ __forceinline__ void load4(const void* p, long long i, bool vec, float (&x)[4]) {
  if (vec) {
    if constexpr (DT == QI_F32) {
      const float4 f = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
      const uint2 u = __ldcg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i));
      if constexpr (DT == QI_BF16) {
        x[0] = bf16lo(u.x), x[1] = bf16hi(u.x), x[2] = bf16lo(u.y), x[3] = bf16hi(u.y);
      } else {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = load_elem<DT>(p, i + e);
  }
}

// ------------------------------------------------------------------ 8-bit codes

// The least power of two s with top * s >= amax (top 127 = 0.9921875 * 2^7 for int8, 448 =
// 0.875 * 2^9 for e4m3), at least 2^-126. amax is finite. With amax = m * 2^e, m in
// [0.5, 1), the exponent is e - 7 (or 9), one more where m exceeds top's own fraction.
template <int FMT>
__device__ __forceinline__ float scale_for(float amax) {
  if (amax == 0.f) return __uint_as_float(0x00800000u);  // 2^-126
  int e;
  const float m = frexpf(amax, &e);
  const int s = FMT == QI_KV_INT8 ? e - 7 + (m > 0.9921875f) : e - 9 + (m > 0.875f);
  return s <= -126 ? __uint_as_float(0x00800000u) : __uint_as_float((uint32_t)(s + 127) << 23);
}

// Code of x given in units of the scale (|x| <= top): nearest, ties to even. A NaN (a
// poisoned block, whose scale is NaN) has code 0.
template <int FMT>
__device__ __forceinline__ uint8_t encode(float x) {
  if constexpr (FMT == QI_KV_INT8) return (uint8_t)(int8_t)(x == x ? __float2int_rn(x) : 0);
  else return x == x ? (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3) : (uint8_t)0;
}

template <int FMT>
__device__ __forceinline__ float decode(uint8_t c) {
  if constexpr (FMT == QI_KV_INT8) return (float)(int8_t)c;
  else return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// ---- pairs of fp32 values in 64 bits: one instruction for two operations
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(f2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Host-side checks of a layer descriptor shared by the entry points.
inline bool bad_layer(const qi_kv_layer* c) {
  if (!c || !c->k || !c->v || c->cache_rows <= 0 || c->kv_heads <= 0 || c->max_len <= 0) return true;
  if (c->head_dim != 64 && c->head_dim != 128) return true;
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return true;
  if (c->page_table && (c->page_size < 128 || c->page_size % 128 != 0 || c->n_pages < 1 || c->pages_per_row < 1 ||
                        (long long)c->pages_per_row * c->page_size < c->max_len))
    return true;
  if (c->format == QI_KV_BF16) return false;
  if (c->format != QI_KV_INT8 && c->format != QI_KV_E4M3) return true;
  if (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3) return true;
  return !c->k_scale || !c->v_scale || (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128);
}
inline bool bad_dtype(int dt) { return dt != QI_F32 && dt != QI_BF16 && dt != QI_F16; }

}  // namespace qi

// The 8-bit KV cache: append with block scales, and the values a layer stands for.
//
// A block is `block` consecutive positions of one cache row and KV head, K and V apart. Its
// scale s is a power of two with top * s >= |x| for all it holds (top = 127 for int8, 448
// for e4m3), and x is held as the code nearest to x / s, ties to even. Multiplying by a
// power of two is exact, so a code depends on nothing but the values; when an append needs
// a larger scale the earlier codes of its block are rounded again to code * old / new, and
// because a scale at least doubles each time, all roundings of one value together stay
// below one step of the final scale.
#include "cache_layer.cuh"

namespace qi {

namespace {

constexpr int kAppendThreads = 256;  // half for K, half for V
constexpr int kHalf = kAppendThreads / 2;
constexpr int kMaxBlock = 128;
constexpr int kMaxSpan = 32;  // tokens of a CTA

struct True {
  static constexpr bool value = true;
};
struct False {
  static constexpr bool value = false;
};

struct Kv8AppendParams {
  qi_kv_layer c;
  const void* k;
  const void* v;
  long long k_st, k_sh, v_st, v_sh;  // element strides of token and head
  const int32_t* rows;
  const int32_t* pos;
  int M, span;
  int* err;
};

// CTA (tokens t0 .. t0 + span - 1, head g). The tokens of one call may come in any order, so
// one of a block's tokens takes all of them: the one with the lowest position. A token right
// behind its predecessor in the same block has nothing to do; for each of the others (run
// starts: one for each block of a prompt, every token of a decode step) the CTA looks through
// rows and positions for the block's tokens. Of two tokens with the same row and position the
// later one is kept.
//
// The bytes are few (a prompt's 4000 tokens of 2 x 64: 2 MB in, 1 MB out, 0.5 us); the time is
// the chain position -> block's tokens -> values -> largest -> codes, so each link's loads are
// under way together, and values are read once and kept in registers (blocks of up to 1024
// quads). `span` is so large that all CTAs run at once, two on an SM (128 registers; at 64 they
// spill and take 1.5 us more), but within a block's positions, so that a prompt gives a
// CTA at most two starts. Those 4000 tokens in blocks of 64: 17.7 us with a CTA for each
// token, which mostly ends at its first test, 11.8 with 8 tokens a CTA, 9.4 with 32; a decode
// step of 32 rows, a CTA for each token: 4.5 us.
template <int FMT, int DT>
__device__ __forceinline__ void append_block(const Kv8AppendParams& p, int t, int g, int ps, int row, int q0, int r0,
                                             int (&slot)[kMaxBlock], float (&red)[kAppendThreads / 32]) {
  const qi_kv_layer& c = p.c;
  const int tid = threadIdx.x, D = c.head_dim, block = c.block;
  const int first = ps - ps % block;  // the block's first position
  const long long base = layer_offset(c, D, row, g, first);
  const long long si = scale_index(c, row, g, first);
  const bool isv = tid >= kHalf;
  float* scale = (isv ? c.v_scale : c.k_scale) + (base < 0 ? 0 : si);
  const float s_held = base < 0 ? 0.f : *scale;
  for (int i = tid; i < block; i += kAppendThreads) slot[i] = -1;
  __syncthreads();
  auto note = [&](int i, int q, int r) {
    if (q >= first && q < first + block && q < c.max_len && r == row) atomicMax(&slot[q - first], i);
  };
  if (tid < p.M) note(tid, q0, r0);
  constexpr int kBatch = 8;  // loads under way together
  const unsigned last = p.M - 1;
  for (unsigned i0 = tid + kAppendThreads; i0 <= last; i0 += kBatch * kAppendThreads) {
    int q[kBatch], r[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const unsigned i = min(i0 + j * kAppendThreads, last);  // the last token more than once does no harm
      q[j] = __ldg(p.pos + i);
      r[j] = __ldg(p.rows + i);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) note((int)min(i0 + j * kAppendThreads, last), q[j], r[j]);
  }
  __syncthreads();
  int f = 0;
  while (f < block && slot[f] < 0) ++f;  // (this token's own slot is taken, unless pos changes meanwhile)
  if (f == block || slot[f] != t) return;
  if (base < 0) {
    if (tid == 0 && p.err) atomicExch(p.err, QI_ERR_INDEX);
    return;
  }
  const int ht = tid & (kHalf - 1);
  const void* x = isv ? p.v : p.k;
  const long long st = isv ? p.v_st : p.k_st;
  const long long xo = (long long)g * (isv ? p.v_sh : p.k_sh);
  uint8_t* codes = static_cast<uint8_t*>(isv ? c.v : c.k) + base;
  const int esz = DT == QI_F32 ? 4 : 2;
  const bool vec = ((uintptr_t)x % (4 * esz)) == 0 && (st & 3) == 0 && (xo & 3) == 0;
  const int qshift = D == 64 ? 4 : 5, quads = 1 << qshift, n = block * quads;  // head_dim is 64 or 128

  // kHeld quads of a thread are in registers at a time; blocks of no more are read once
  constexpr int kHeld = 8;
  float v[kHeld][4];
  int tok[kHeld];
  auto read_as = [&](int i0, auto wide) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0.f;
      const int i = i0 + j * kHalf;
      if (tok[j] >= 0) load4<DT>(x, tok[j] * st + xo + (i & (quads - 1)) * 4, decltype(wide)::value, v[j]);
    }
  };
  auto read = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int i = i0 + j * kHalf;
      tok[j] = i < n ? slot[i >> qshift] : -1;
    }
    if (vec) read_as(i0, True{});
    else read_as(i0, False{});
  };
  float amax = 0.f;
  bool bad = false;
  for (int i = ht; i < n; i += kHeld * kHalf) {
    read(i);
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        bad |= !(fabsf(v[j][e]) <= 3.402823466e38f);
        amax = fmaxf(amax, fabsf(v[j][e]));
      }
  }
  amax = warp_max(bad ? INFINITY : amax);
  if ((tid & 31) == 0) red[tid >> 5] = amax;
  __syncthreads();
  const int w0 = isv ? kHalf / 32 : 0;
  amax = fmaxf(fmaxf(red[w0], red[w0 + 1]), fmaxf(red[w0 + 2], red[w0 + 3]));
  // A value that is not finite makes the block's scale NaN, and with it every result that
  // reads the block, as the value itself would.
  float s_new = amax == INFINITY ? __uint_as_float(0x7fc00000u) : scale_for<FMT>(amax);
  float s_old = s_new;
  if (f > 0) {  // the block keeps its earlier positions
    s_old = s_held;
    s_new = s_old >= s_new || s_old != s_old ? s_old : s_new;
  }
  // 1 / s is exact: s = 2^e with -126 <= e <= 122
  const float inv = 1.0f / s_new, again = s_old * inv;
  // Values next to the largest float would round to 2^128: their code stops at the last
  // one whose value is finite (63 * 2^122 for int8, 240 * 2^120 for e4m3).
  constexpr float kHugeScale = FMT == QI_KV_INT8 ? 0x1p122f : 0x1p120f, kHugeTop = FMT == QI_KV_INT8 ? 63.f : 240.f;
  const float most = s_new >= kHugeScale ? kHugeTop : INFINITY;
  auto code = [&](float x) { return encode<FMT>(x == x ? fminf(fmaxf(x, -most), most) : x); };
  // four new values at once: none is NaN unless the block's scale is
  auto four = [&](const float (&y)[4]) -> uint32_t {
    if (s_new != s_new) return 0u;
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = fminf(fmaxf(y[e] * inv, -most), most);
    if constexpr (FMT == QI_KV_INT8) {
      const int lo = __byte_perm(__float2int_rn(z[0]), __float2int_rn(z[1]), 0x40);
      return __byte_perm(lo, __byte_perm(__float2int_rn(z[2]), __float2int_rn(z[3]), 0x40), 0x5410);
    } else {
      return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(z[0], z[1]), __NV_SATFINITE, __NV_E4M3) |
             (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(z[2], z[3]), __NV_SATFINITE, __NV_E4M3) << 16;
    }
  };
  if (ht == 0) *scale = s_new;
  for (int i0 = ht; i0 < n; i0 += kHeld * kHalf) {
    if (n > kHeld * kHalf) read(i0);
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int i = i0 + j * kHalf;
      if (i >= n) break;
      const int s = i >> qshift, d = (i & (quads - 1)) * 4;
      uchar4* out = reinterpret_cast<uchar4*>(codes + s * D + d);
      if (tok[j] >= 0) {
        *reinterpret_cast<uint32_t*>(out) = four(v[j]);
      } else if (s < f && again != 1.0f) {
        const uchar4 o = *out;
        *out = make_uchar4(code(decode<FMT>(o.x) * again), code(decode<FMT>(o.y) * again),
                           code(decode<FMT>(o.z) * again), code(decode<FMT>(o.w) * again));
      }
    }
  }
}

template <int FMT, int DT>
__global__ void __launch_bounds__(kAppendThreads, 2) kv8_append_kernel(const Kv8AppendParams p) {
  __shared__ int slot[kMaxBlock];  // token that holds the block's position, -1: none
  __shared__ float red[kAppendThreads / 32];
  __shared__ int own_pos[kMaxSpan], own_row[kMaxSpan];
  grid_dep_wait();
  grid_dep_launch();
  const qi_kv_layer& c = p.c;
  const int tid = threadIdx.x, t0 = blockIdx.x * p.span, g = blockIdx.y, nt = min(p.span, p.M - t0);
  // the first tokens of the call, for the search
  const int q0 = tid < p.M ? p.pos[tid] : -1, r0 = tid < p.M ? p.rows[tid] : -1;
  bool start = false;
  if (tid < nt) {
    const int t = t0 + tid, ps = p.pos[t], row = p.rows[t];
    const int before = t > 0 ? p.pos[t - 1] : -1, row_before = t > 0 ? p.rows[t - 1] : -1;
    start = ps != -1;  // not an idle slot
    if (start && (ps < 0 || ps >= c.max_len || row < 0 || row >= c.cache_rows)) {
      if (p.err) atomicExch(p.err, QI_ERR_INDEX);
      start = false;
    }
    if (t > 0 && ps % c.block != 0 && row_before == row && before == ps - 1) start = false;
    own_pos[tid] = ps;
    own_row[tid] = row;
  }
  __shared__ unsigned starts;
  if (tid < 32) {
    const unsigned m = __ballot_sync(0xffffffffu, start);
    if (tid == 0) starts = m;
  }
  __syncthreads();
  for (unsigned m = starts; m != 0u; m &= m - 1u) {
    const int i = __ffs(m) - 1;
    append_block<FMT, DT>(p, t0 + i, g, own_pos[i], own_row[i], q0, r0, slot, red);
    __syncthreads();  // slot and red are free
  }
}

// fp32 values of a layer by (row, head, position): one thread for 4 dims of K and of V.
// Positions on unmapped pages are zero.
template <int FMT>
__global__ void __launch_bounds__(256) kv8_values_kernel(const qi_kv_layer c, float* __restrict__ ko,
                                                         float* __restrict__ vo, long long n) {
  const int quads = c.head_dim / 4;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    const long long cell = i / quads;  // (row, head, position)
    const int d = (int)(i - cell * quads) * 4;
    const long long rg = cell / c.max_len;
    const int pos = (int)(cell - rg * c.max_len), row = (int)(rg / c.kv_heads), g = (int)(rg - (long long)row * c.kv_heads);
    const long long o = layer_offset(c, c.head_dim, row, g, pos);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (o >= 0) {
      const long long si = scale_index(c, row, g, pos);
      const uchar4 x = *reinterpret_cast<const uchar4*>(static_cast<const uint8_t*>(c.k) + o + d);
      const uchar4 y = *reinterpret_cast<const uchar4*>(static_cast<const uint8_t*>(c.v) + o + d);
      const float s = __ldg(c.k_scale + si), u = __ldg(c.v_scale + si);
      a = make_float4(decode<FMT>(x.x) * s, decode<FMT>(x.y) * s, decode<FMT>(x.z) * s, decode<FMT>(x.w) * s);
      b = make_float4(decode<FMT>(y.x) * u, decode<FMT>(y.y) * u, decode<FMT>(y.z) * u, decode<FMT>(y.w) * u);
    }
    reinterpret_cast<float4*>(ko)[i] = a;
    reinterpret_cast<float4*>(vo)[i] = b;
  }
}

template <int FMT>
cudaError_t launch_append(const Kv8AppendParams& p, int dtype, cudaStream_t s, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.M + p.span - 1) / p.span, p.c.kv_heads, 1);
  cfg.blockDim = dim3(kAppendThreads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  if (dtype == QI_F32) return cudaLaunchKernelEx(&cfg, kv8_append_kernel<FMT, QI_F32>, p);
  if (dtype == QI_BF16) return cudaLaunchKernelEx(&cfg, kv8_append_kernel<FMT, QI_BF16>, p);
  return cudaLaunchKernelEx(&cfg, kv8_append_kernel<FMT, QI_F16>, p);
}

}  // namespace

cudaError_t launch_kv8_append(const qi_kv_layer& c, const void* k, const void* v, int dtype, long long k_st,
                              long long k_sh, long long v_st, long long v_sh, const int32_t* rows, const int32_t* pos,
                              int M, int* err, cudaStream_t s, bool pdl) {
  int span = 1;
  while (span < kMaxSpan && span < c.block && (long long)((M - 1) / span + 1) * c.kv_heads > 2LL * sm_count()) span *= 2;
  const Kv8AppendParams p = {c, k, v, k_st, k_sh, v_st, v_sh, rows, pos, M, span, err};
  return c.format == QI_KV_INT8 ? launch_append<QI_KV_INT8>(p, dtype, s, pdl)
                                : launch_append<QI_KV_E4M3>(p, dtype, s, pdl);
}

cudaError_t launch_kv8_values(const qi_kv_layer& c, float* k_out, float* v_out, cudaStream_t s) {
  const long long n = (long long)c.cache_rows * c.kv_heads * c.max_len * (c.head_dim / 4);
  const long long want = (n + 255) / 256, most = 16LL * sm_count();
  const int grid = (int)(want < most ? want : most);
  if (c.format == QI_KV_INT8) kv8_values_kernel<QI_KV_INT8><<<grid, 256, 0, s>>>(c, k_out, v_out, n);
  else kv8_values_kernel<QI_KV_E4M3><<<grid, 256, 0, s>>>(c, k_out, v_out, n);
  return cudaGetLastError();
}

}  // namespace qi

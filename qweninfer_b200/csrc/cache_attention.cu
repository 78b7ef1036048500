// Grouped-query attention over one cache layer for query tokens that each read their own
// row: bf16, int8 or e4m3 keys and values, packed or paged, with an optional sliding
// window and first tokens ("sinks") that stay visible.
//
//   o[t, h] = sum_j w_j v_j,  w = softmax over the seen j of q[t, h] . k_j / sqrt(D),
//   seen: 0 <= j <= p and (no window, or j > p - window, or j < sinks), p = pos[t].
//
// One CTA per (key split, KV head, token), 4 warps. The seen keys of a token form a list of
// granules of 32 aligned positions (the sinks' granules, then the window's); a split takes
// a contiguous run of the list, of whatever length the token really has, and its warps take
// the run's granules in turn. Nothing but seen keys is read: a granule's other keys are
// zero-filled, so what dead positions hold (NaN included) never enters a product.
//
// Each warp streams its own granules through a private ring of shared memory with cp.async
// and never waits for another warp before the sums. A call is bound by the cache's bytes,
// so what counts is bytes in flight: 16 warps of an SM with two granules each requested.
//
// The group's query heads (at most 8) are rows of m16n8k16 MMAs. Row h holds the high part
// of q_h, row h + 8 the next part: their products land in the same thread, which adds
// them. 8-bit codes are exact in fp16, so both products run in fp16: q is scaled by a power
// of two to a maximum in [1, 2) and split into two fp16 parts (22 bits), the probabilities
// are computed as 2^12 p (the factor cancels in the normalisation) and split the same
// way. A bf16 cache multiplies in bf16 with three parts of q and p for fp32 callers (24
// bits) and two for 16-bit ones; the third part is a second MMA. Scores, softmax statistics
// and outputs are fp32; the block scales multiply scores and products of 16 keys in fp32.
//
// The dims of a k-step are permuted: a thread's share of a key is 16 contiguous bytes (one
// shared-memory load gives 4 k-steps of 8-bit codes or 2 of bf16), and the query fragments
// are loaded in the same order, which leaves the dot product unchanged. V goes through
// ldmatrix.trans; for 8-bit codes its 16-bit elements are pairs of neighbouring dims, taken
// apart into an even and an odd n-tile.
#include "cache_attention.cuh"

namespace qi {

namespace {

using namespace cattn;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kGran = 32;  // keys per granule
constexpr int kPromptRows = 128, kPromptKeys = 128;  // cache_attention_prompt.cu's tiles

template <int FMT, int D>
struct Shape {
  static constexpr int kRow = D * (FMT == QI_KV_BF16 ? 2 : 1);  // bytes of one key
  static constexpr int kChunks = kRow / 16;
  static constexpr int kTensor = kGran * kRow;                   // K or V of a granule
  static constexpr int kStage = 2 * kTensor + 16;                // + 2 K scales, 2 V scales
  static constexpr int kStages = 2;
  static constexpr size_t kRing = (size_t)kWarps * kStages * kStage;
  // CTAs of an SM: by registers for 8-bit codes (head_dim 64: 26.7 us on two rows of 131072, with
  // 5 CTAs 29.5, with 3 27.3; 128: 3 CTAs 29.4 us on 64 rows of 4096, with 2 34.8), by shared
  // memory otherwise
  static constexpr int kCtas = FMT == QI_KV_BF16 ? (D == 64 ? 3 : 1) : (D == 64 ? 4 : 3);
  static_assert((kRing + 6 * 1024) * kCtas <= 228 * 1024, "shared memory of an SM");
};

// physical 16-byte chunk c of key r: 8 keys at one chunk (ldmatrix) and 2 keys at 4
// chunks of one quad (K loads) both cover all banks
template <int CH>
__device__ __forceinline__ int swizzle(int r, int c) {
  if constexpr (CH == 4) return c ^ ((r >> 1) & 3);
  else return c ^ (((r & 1) << 2) | ((r >> 1) & 3));
}

__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
  return r;
}
// d = a b + c of m16n8k16
template <bool F16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, "
        "%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, "
        "%12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Granules a split has at least: one for each warp. (One row of 700 keys: 6.2 us, with twice as
// many 7.5.)
constexpr int kMinSplit = kWarps;
constexpr int kMaxCluster = 8;

// What the CTAs of a cluster push to each other, apart from the rings that are still in use:
// maximum and sum of the heads, and a share of the outputs as pairs of dims.
template <int D>
struct Inbox {
  float2 ml[kMaxCluster][kMaxGroup];
  float2 pairs[kMaxGroup * D / 2 + kMaxCluster];  // [split][the share]
};
// into the shared memory of CTA w of the cluster
__device__ __forceinline__ void put2(float2* to, int w, float a, float b) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(map_rank(to, (uint32_t)w)), "f"(a), "f"(b) : "memory");
}

// F16 products for 8-bit codes, bf16 for a bf16 cache; P3: three parts of q and p (bf16).
template <int FMT, int D, bool P3>
__global__ void __launch_bounds__(kThreads, Shape<FMT, D>::kCtas) cache_attention_kernel(const CacheAttnParams p) {
  using S = Shape<FMT, D>;
  constexpr bool F16 = FMT != QI_KV_BF16;
  constexpr int kParts = P3 ? 3 : 2, kA = P3 ? 2 : 1;  // parts, A operands
  constexpr int kSteps = D / 16;                       // k-steps of a key
  constexpr int kPer = F16 ? 4 : 2;                    // k-steps in 16 bytes
  constexpr int kOut = D / 4;                          // output dims of a thread
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int last;
  __shared__ Inbox<D> in;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, qd = lane & 3;
  const int tok = blockIdx.x / p.splits, split_i = blockIdx.x - tok * p.splits, g = blockIdx.y;
  const qi_kv_layer& c = p.c;
  const int G = p.group, width = p.heads * D;
  grid_dep_wait();
  grid_dep_launch();
  if (p.cluster > 1) cluster_arrive();  // this CTA's shared memory may be written by the others
  const int ps = p.pos[tok], row = p.rows[tok];
  // the query of head gq: dims 16 bytes apart per quad, in the keys' chunk order (loaded
  // before the keys, whose addresses wait for the position)
  float x[D / 4];
  {
    const long long qo = (long long)tok * p.q_st + (long long)(g * G + (gq < G ? gq : 0)) * p.q_sh;
#pragma unroll
    for (int i = 0; i < D / 4; i += 4) {
      // i-th value of this thread: k-step i / 4 lies in chunk 4 * (i / 4 / kPer) + qd
      const int d = (4 * (i / 4 / kPer) + qd) * 4 * kPer + (i / 4 % kPer) * 4;
      if (p.dtype == QI_F32) load4<QI_F32>(p.q, qo + d, p.q_vec, *reinterpret_cast<float(*)[4]>(x + i));
      else if (p.dtype == QI_BF16) load4<QI_BF16>(p.q, qo + d, p.q_vec, *reinterpret_cast<float(*)[4]>(x + i));
      else load4<QI_F16>(p.q, qo + d, p.q_vec, *reinterpret_cast<float(*)[4]>(x + i));
    }
    if (gq >= G) {
#pragma unroll
      for (int i = 0; i < D / 4; ++i) x[i] = 0.f;
    }
  }
  auto leave = [&] {  // nothing to do: the cluster's first barrier is still to be met
    if (p.cluster > 1) cluster_wait();
  };
  if (!token_ok(p, ps, row)) {  // nothing seen: zeros; a position or row outside the cache is reported
    if (split_i == 0 && !p.only_single) {
      if (ps != -1 && tid == 0 && p.err) atomicExch(p.err, QI_ERR_INDEX);
      const float z[2] = {0.f, 0.f};
      for (int e = tid; e < G * D / 2; e += kThreads) emit<2>(p, tok, g * G * D + 2 * e, width, z);
    }
    return leave();
  }
  if (p.only_single) {  // the tokens that the prompt kernel left out: alone in their row of a CTA's
    const int n = (D == 64 ? 2 : 1) * (kPromptRows / G), t0 = tok / n * n;
    int same = 0;
    for (int j = 0; j < n; j += kThreads) {
      const int t = t0 + j + tid;
      same += __syncthreads_count(j + tid < n && t < p.M && p.rows[t] == row && token_ok(p, p.pos[t], row));
    }
    if (same != 1) return leave();
  }
  const Seen<kGran> seen = seen_range<kGran>(ps, window_start(ps, p.window), p.sinks);
  const int nsplit = min(p.splits, (seen.n + kMinSplit - 1) / kMinSplit);
  if (nsplit == 1 ? split_i > 0 : split_i / p.cluster * p.cluster >= nsplit) return leave();  // without keys
  // (a split without keys in a cluster that has some gets an empty run)
  const int gbeg = (int)((long long)seen.n * split_i / nsplit), gend = split_i < nsplit ? (int)((long long)seen.n * (split_i + 1) / nsplit) : gbeg;

  const uint32_t ring = smem_u32(smem) + (uint32_t)(warp * S::kStages * S::kStage);
  // The row's keys and values of this head, in bytes, and its scales (of a packed layer; a
  // paged one looks every granule's page up). Lanes 0..3 take the granule's scales, of K in
  // its two halves and of V.
  const bool paged = c.page_table != nullptr;
  const uint8_t* krow = static_cast<const uint8_t*>(c.k);
  const uint8_t* vrow = static_cast<const uint8_t*>(c.v);
  const float* srow = lane < 2 ? c.k_scale : c.v_scale;
  const int lg_block = F16 ? __ffs(c.block) - 1 : 0;
  if (!paged) {
    const long long rg = (long long)row * c.kv_heads + g;
    krow += rg * c.max_len * S::kRow;
    vrow += rg * c.max_len * S::kRow;
    if constexpr (F16) srow += rg * ((c.max_len + c.block - 1) >> lg_block);
  }
  // Chunk x = lane + 32 j of a granule is chunk x % kChunks of key x / kChunks.
  auto place = [&](int j) -> uint32_t {
    constexpr int kStep = 32 / S::kChunks;  // keys of 32 chunks: the next j is 512 bytes on
    const int r0 = lane / S::kChunks, ch = lane % S::kChunks;
    if constexpr (S::kChunks == 4) return r0 * S::kRow + swizzle<4>(r0, ch) * 16 + j * 512;  // swizzled alike
    else if constexpr (S::kChunks == 8) return ((r0 * S::kRow + swizzle<8>(r0, ch) * 16) ^ ((j & 1) * 32)) + j * 512;
    else return (r0 + j * kStep) * S::kRow + swizzle<S::kChunks>(r0 + j * kStep, ch) * 16;
  };
  // granule i (its place in the list) into ring stage st; nothing for i >= gend
  auto issue = [&](int i, int st) {
    if (i < gend) {
      const int k0 = seen.granule(i) * kGran;
      const uint32_t dst = ring + (uint32_t)(st * S::kStage);
      long long ko = (long long)k0 * S::kRow, so = k0;  // of the first key: bytes, and position
      bool mapped = true;
      if (paged) {
        const long long o = layer_offset(c, D, row, g, k0);
        mapped = o >= 0;
        ko = (mapped ? o : 0) * (S::kRow / D);
        if constexpr (F16) so = mapped ? scale_index(c, row, g, k0) << lg_block | (k0 & (c.block - 1)) : 0;
        // an unmapped page: reported, read as zeros
        if (!mapped && lane == 0 && p.err) atomicExch(p.err, QI_ERR_INDEX);
      }
      const uint8_t* kp = krow + ko + lane * 16;
      const uint8_t* vp = vrow + ko + lane * 16;
      if (mapped && k0 + kGran - 1 <= seen.p && (k0 >= seen.lo || k0 + kGran <= seen.sinks)) {
#pragma unroll
        for (int j = 0; j < S::kChunks; ++j) {
          cp16(dst + place(j), kp + j * 512);
          cp16(dst + S::kTensor + place(j), vp + j * 512);
        }
        if constexpr (F16) {
          if (lane < 4) cp4(dst + 2 * S::kTensor + 4 * lane, srow + ((so + 16 * (lane & 1)) >> lg_block), 4u);
        }
      } else {
#pragma unroll
        for (int j = 0; j < S::kChunks; ++j) {
          // a key that is not seen reads nothing; its address stays in the granule's page
          const uint32_t n = mapped && seen.sees(k0 + (lane + 32 * j) / S::kChunks) ? 16u : 0u;
          cp16(dst + place(j), n ? kp + j * 512 : krow + ko, n);
          cp16(dst + S::kTensor + place(j), n ? vp + j * 512 : vrow + ko, n);
        }
        if constexpr (F16) {
          if (lane < 4) {
            const int h0 = k0 + 16 * (lane & 1);
            const bool any = mapped && seen.sees16(h0);
            cp4(dst + 2 * S::kTensor + 4 * lane, srow + (any ? (so + 16 * (lane & 1)) >> lg_block : 0), any ? 4u : 0u);
          }
        }
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) issue(gbeg + warp + s * kWarps, s);

  uint32_t qa[kA][kSteps][4];
  float qscale = p.scale_log2;
  {
    if constexpr (F16) {
      // q * 2^-e in [1, 2) at its largest: fp16 parts keep 22 bits of every head's scale
      float am = 0.f;
#pragma unroll
      for (int i = 0; i < D / 4; ++i) am = fmaxf(am, fabsf(x[i]));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
      const uint32_t e = __float_as_uint(am) >> 23;  // biased exponent (am >= 0)
      if (e > 0 && e < 253) {
        const float inv = __uint_as_float((254u - e) << 23);
        qscale *= __uint_as_float(e << 23);
#pragma unroll
        for (int i = 0; i < D / 4; ++i) x[i] *= inv;
      }
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      uint32_t a[kParts], b[kParts];
      split<F16, kParts>(x[4 * s], x[4 * s + 1], a);
      split<F16, kParts>(x[4 * s + 2], x[4 * s + 3], b);
      qa[0][s][0] = a[0], qa[0][s][1] = a[1], qa[0][s][2] = b[0], qa[0][s][3] = b[1];
      if constexpr (P3) qa[1][s][0] = a[2], qa[1][s][1] = 0u, qa[1][s][2] = b[2], qa[1][s][3] = 0u;
    }
  }

  float m = -INFINITY, l = 0.f, o[kOut];
  bool far = false;  // a maximum of this warp's is beyond kFarScore
#pragma unroll
  for (int i = 0; i < kOut; ++i) o[i] = 0.f;

  int st = 0;
  for (int i = gbeg + warp; i < gend; i += kWarps) {
    cp_wait<S::kStages - 2>();
    __syncwarp();  // the granule is in place for every lane, and the last one is read
    issue(i + (S::kStages - 1) * kWarps, st == 0 ? S::kStages - 1 : st - 1);
    const uint32_t kt = ring + (uint32_t)(st * S::kStage), vt = kt + S::kTensor;
    st = st + 1 == S::kStages ? 0 : st + 1;
    const int k0 = seen.granule(i) * kGran;

    // scores of head gq for keys 8 t + 2 qd + e, without the factor f[t] > 0
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    float sc[4][2], f[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float acc[4];
#pragma unroll
      for (int h = 0; h < S::kChunks / 4; ++h) {
        const uint4 w = lds128(kt + (uint32_t)((8 * t + gq) * S::kRow + swizzle<S::kChunks>(8 * t + gq, 4 * h + qd) * 16));
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          uint32_t b0, b1;
          if constexpr (F16) widen<FMT, 0>(ws[j], b0, b1);
          else b0 = ws[2 * j], b1 = ws[2 * j + 1];
          if (h + j == 0) mma<F16>(acc, qa[0][0], b0, b1, zero);
          else mma<F16>(acc, qa[0][kPer * h + j], b0, b1, acc);
          if constexpr (P3) mma<F16>(acc, qa[1][kPer * h + j], b0, b1, acc);
        }
      }
      sc[t][0] = acc[0] + acc[2];
      sc[t][1] = acc[1] + acc[3];
    }
    float2 sv = make_float2(1.f, 1.f);  // V scales of the halves
    if constexpr (F16) {
      const uint4 w = lds128(kt + 2 * S::kTensor);
      f[0] = f[1] = qscale * __uint_as_float(w.x);
      f[2] = f[3] = qscale * __uint_as_float(w.y);
      sv = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
    } else {
      f[0] = f[1] = f[2] = f[3] = qscale;
    }
    if (k0 + kGran - 1 > seen.p || (k0 < seen.lo && k0 + kGran > seen.sinks)) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // (0 * f would be NaN for a scale that is not finite)
          const bool in = seen.sees(k0 + 8 * t + 2 * qd + e);
          sc[t][e] = in ? sc[t][e] * f[t] : -INFINITY;
        }
      f[0] = f[1] = f[2] = f[3] = 1.f;
    }
    float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1])) * f[0],
                     fmaxf(fmaxf(sc[2][0], sc[2][1]), fmaxf(sc[3][0], sc[3][1])) * f[2]);
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    if (__any_sync(0xffffffffu, mx > m)) {  // a new maximum: rescale what is summed so far
      const float mn = fmaxf(m, mx);
      const float alpha = m == -INFINITY ? 0.f : ex2(m - mn);
      m = mn;
      far = __any_sync(0xffffffffu, m != -INFINITY && fabsf(m) >= kFarScore);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < kOut; ++d) o[d] *= alpha;
    }
    // probabilities relative to the running maximum (8-bit: times 2^12, which keeps the
    // second fp16 part of small ones above the subnormal range)
    const float mref = (F16 ? 12.f : 0.f) - (m == -INFINITY ? 0.f : m);
    uint32_t pa[2][kA][4];
    if (far) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          sc[t][e] = __fmul_rn(sc[t][e], f[t]) - (m == -INFINITY ? 0.f : m) + (F16 ? 12.f : 0.f);
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) sc[t][e] = fmaf(sc[t][e], f[t], mref);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float p0 = ex2(sc[t][0]), p1 = ex2(sc[t][1]);
      l += p0 + p1;
      uint32_t r[kParts];
      split<F16, kParts>(p0, p1, r);
      pa[t >> 1][0][2 * (t & 1)] = r[0];
      pa[t >> 1][0][2 * (t & 1) + 1] = r[1];
      if constexpr (P3) pa[t >> 1][1][2 * (t & 1)] = r[2], pa[t >> 1][1][2 * (t & 1) + 1] = 0u;
    }
    // O += P V: 16 keys have one V scale; where the two halves share it (blocks of 32 and
    // more), or have none, both go into one sum before it is multiplied
    const bool one = !F16 || sv.x == sv.y;
#pragma unroll
    for (int h = 0; h < S::kChunks / 2; ++h) {
      // matrices: keys 16 hf + 8 (j & 1) .., chunk 2 h + (j >> 1)
      uint32_t b[2][4];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int lj = lane >> 3, r = 16 * hf + 8 * (lj & 1) + (lane & 7), ch = 2 * h + (lj >> 1);
        ldsm4t(vt + (uint32_t)(r * S::kRow + swizzle<S::kChunks>(r, ch) * 16), b[hf]);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if constexpr (F16) {
          // chunk of 16 dims: this thread's columns are dims 4 qd + {0, 2} of the even and
          // {1, 3} of the odd n-tile
          float* oo = o + 4 * (2 * h + u);
          uint32_t e[2][2], d[2][2];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            widen<FMT, 1>(b[hf][2 * u], e[hf][0], d[hf][0]);
            widen<FMT, 1>(b[hf][2 * u + 1], e[hf][1], d[hf][1]);
          }
          float ae[4], ad[4];
          mma<F16>(ae, pa[0][0], e[0][0], e[0][1], zero);
          mma<F16>(ad, pa[0][0], d[0][0], d[0][1], zero);
          if (one) {
            mma<F16>(ae, pa[1][0], e[1][0], e[1][1], ae);
            mma<F16>(ad, pa[1][0], d[1][0], d[1][1], ad);
          } else {
            float be[4], bd[4];
            mma<F16>(be, pa[1][0], e[1][0], e[1][1], zero);
            mma<F16>(bd, pa[1][0], d[1][0], d[1][1], zero);
            oo[0] = fmaf(sv.y, be[0] + be[2], oo[0]);
            oo[1] = fmaf(sv.y, bd[0] + bd[2], oo[1]);
            oo[2] = fmaf(sv.y, be[1] + be[3], oo[2]);
            oo[3] = fmaf(sv.y, bd[1] + bd[3], oo[3]);
          }
          oo[0] = fmaf(sv.x, ae[0] + ae[2], oo[0]);
          oo[1] = fmaf(sv.x, ad[0] + ad[2], oo[1]);
          oo[2] = fmaf(sv.x, ae[1] + ae[3], oo[2]);
          oo[3] = fmaf(sv.x, ad[1] + ad[3], oo[3]);
        } else {
          float acc[4];
          mma<F16>(acc, pa[0][0], b[0][2 * u], b[0][2 * u + 1], zero);
          if constexpr (P3) mma<F16>(acc, pa[0][1], b[0][2 * u], b[0][2 * u + 1], acc);
          mma<F16>(acc, pa[1][0], b[1][2 * u], b[1][2 * u + 1], acc);
          if constexpr (P3) mma<F16>(acc, pa[1][1], b[1][2 * u], b[1][2 * u + 1], acc);
          float* oo = o + 2 * (2 * h + u);
          oo[0] += acc[0] + acc[2];
          oo[1] += acc[1] + acc[3];
        }
      }
    }
  }
  cp_wait<0>();
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);

  // merge of the warps, in shared memory that the rings no longer need
  constexpr int kPart = D + 2;
  float* wp = reinterpret_cast<float*>(smem);  // [warp][head][D values, m, l]
  __syncthreads();
  if (gq < G) {
    float* w = wp + (warp * G + gq) * kPart;
#pragma unroll
    for (int i = 0; i < kOut; ++i) {
      const int d = F16 ? 16 * (i / 4) + 4 * qd + i % 4 : 8 * (i / 2) + 2 * qd + i % 2;
      w[d] = o[i];
    }
    if (qd == 0) w[D] = m, w[D + 1] = l;
  }
  __syncthreads();
  // The splits of a unit are clusters of p.cluster CTAs. Every CTA adds up a share of the
  // outputs: the others push theirs into its shared memory, and it sums them in split order.
  // Over more than one cluster the clusters' sums go through global memory to the CTA that
  // arrives last.
  const long long unit = (long long)tok * c.kv_heads + g;
  const int C = p.cluster, rank = split_i % C, first = split_i - rank;
  const int here = min(C, nsplit - first);  // splits of this cluster with keys
  const int clusters = (nsplit + C - 1) / C;
  constexpr int kPairs = D / 2;
  const int E = G * kPairs, per = (E + C - 1) / C;  // pairs of outputs, and a CTA's share of them
  if (nsplit > 1) cluster_wait();                   // every CTA of the cluster has started
  for (int e = tid; e < E; e += kThreads) {
    const int h = e / kPairs, d = 2 * (e - h * kPairs);
    float mm, ll, a, b;
    merge2<D>([&](int w, int i) { return wp[(w * G + h) * kPart + i]; }, kWarps, d, mm, ll, a, b);
    if (nsplit == 1) {
      const float inv = ll != 0.f ? 1.f / ll : 0.f;
      const float v[2] = {a * inv, b * inv};
      emit<2>(p, tok, g * G * D + h * D + d, width, v);
    } else if (rank < here) {
      const int to = e / per;
      put2(&in.pairs[rank * per + e - to * per], to, a, b);
      // maximum and sum of the head, for the first pair of it in each share
      if (d == 0 || e % per == 0) put2(&in.ml[rank][h], to, mm, ll);
    }
  }
  if (nsplit == 1) return leave();
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  float* part = p.part + unit * (p.splits / C) * (long long)(G * kPart);  // [cluster][head][D + 2]
  for (int e = rank * per + tid; e < min(E, (rank + 1) * per); e += kThreads) {
    const int h = e / kPairs, d = 2 * (e - h * kPairs);
    float mm, ll, a, b;
    merge2<0>([&](int w, int i) { return i < 2 ? (i ? in.ml[w][h].y : in.ml[w][h].x)
                                               : (i == 2 ? in.pairs[(w - rank) * per + e].x : in.pairs[(w - rank) * per + e].y); },
              here, 2, mm, ll, a, b);
    if (clusters == 1) {
      const float inv = ll != 0.f ? 1.f / ll : 0.f;
      const float v[2] = {a * inv, b * inv};
      emit<2>(p, tok, g * G * D + h * D + d, width, v);
    } else {
      float* y = part + (long long)(first / C) * (G * kPart) + h * kPart;
      __stcg(reinterpret_cast<float2*>(y + d), make_float2(a, b));
      if (d == 0) __stcg(reinterpret_cast<float2*>(y + D), make_float2(mm, ll));
    }
  }
  if (clusters == 1) return;
  __syncthreads();
  if (tid == 0) last = atomic_add_acq_rel(p.counters + unit, 1u) == (unsigned)(C * clusters - 1);
  __syncthreads();
  if (!last) return;
  for (int e = tid; e < E; e += kThreads) {
    const int h = e / kPairs, d = 2 * (e - h * kPairs);
    float mm, ll, a, b;
    merge2<D>([&](int w, int i) { return __ldcg(part + ((long long)w * G + h) * kPart + i); }, clusters, d, mm, ll, a, b);
    const float inv = ll != 0.f ? 1.f / ll : 0.f;
    const float v[2] = {a * inv, b * inv};
    emit<2>(p, tok, g * G * D + h * D + d, width, v);
  }
  if (tid == 0) p.counters[unit] = 0u;  // as the next call expects it
}

template <int FMT, int D, bool P3>
cudaError_t launch_token(const CacheAttnParams& p, cudaStream_t s, bool pdl) {
  auto kernel = cache_attention_kernel<FMT, D, P3>;
  constexpr size_t merge = sizeof(float) * (kWarps + 1) * kMaxGroup * (D + 2);
  constexpr size_t smem = Shape<FMT, D>::kRing > merge ? Shape<FMT, D>::kRing : merge;
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.M * p.splits), p.c.kv_heads, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)p.cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int D>
cudaError_t launch_dim(const CacheAttnParams& p, cudaStream_t s, bool pdl) {
  if (p.c.format == QI_KV_INT8) return launch_token<QI_KV_INT8, D, false>(p, s, pdl);
  if (p.c.format == QI_KV_E4M3) return launch_token<QI_KV_E4M3, D, false>(p, s, pdl);
  return p.dtype == QI_F32 ? launch_token<QI_KV_BF16, D, true>(p, s, pdl) : launch_token<QI_KV_BF16, D, false>(p, s, pdl);
}

}  // namespace

namespace {

// Key tiles a CTA of the tile kernel has at least: the exchange in a cluster costs less than
// another tile's softmax. 128 tokens, 14 heads on 2 of 64, int8, rows of 512 keys: 19.7 us, with
// two tiles 21.7, four 27.3; 1500 keys: 24.4, 26.2, 34.4.
constexpr int kMinTiles = 1;

// The tile kernel takes runs of kMinRun tokens and more of calls whose work, were every row
// full, is at least kMinWork (tokens x KV heads x dims x keys). It starts at 13 to 27 us
// whatever the work (tensor memory, the softmax chain of a CTA's few tiles, the cluster's
// exchange), the per-token kernel at 7; but that reads and widens every key for each
// token. Where positions are is known on the device only, so the choice goes by what the
// layer lets them be. Measured at 4096 positions, us, per token / tiles, rows of 512 and of
// 4000 keys; 14 heads on 2 of 64, int8, one row of 128 tokens (2^26): 10/20, 32/32; 256 (2^27):
// 13/20, 57/38; 512: 16/21, 98/45; 16 on 2 of 128, bf16, 64 tokens (2^26): 13/26, 53/42; 128
// (2^27): 23/27, 100/51; 8 on 8 of 64, int8, 32 tokens (2^26): 9/13, 31/20; 64 (2^27): 12/13, 54/21.
constexpr int kMinRun = 16;
constexpr long long kMinWork = 1LL << 27;

long long seen_at_most(const qi_kv_layer& c, int window, int sinks) {
  const long long w = (long long)window + sinks;
  return window > 0 && w < c.max_len ? w : c.max_len;
}

constexpr int kMaxTokenSplits = 256;

// Key splits of the per-token kernel: as many CTAs as are resident at once, as far as rows
// are long enough to give each split kMinSplit granules; whole clusters when there are more
// than fit one.
int token_splits(const qi_kv_layer& c, int M, int window, int sinks) {
  const int ctas = c.format == QI_KV_BF16 ? (c.head_dim == 64 ? Shape<QI_KV_BF16, 64>::kCtas : Shape<QI_KV_BF16, 128>::kCtas)
                                          : (c.head_dim == 64 ? Shape<QI_KV_INT8, 64>::kCtas : Shape<QI_KV_INT8, 128>::kCtas);
  const long long gran = seen_at_most(c, window, sinks) / kGran + 2, units = (long long)M * c.kv_heads;
  const long long most = (gran + kMinSplit - 1) / kMinSplit;
  // (nine tenths of them: clusters do not fill every GPC)
  long long want = (long long)ctas * sm_count() * 9 / 10 / units;
  want = want > most ? most : want;
  want = want > kMaxTokenSplits ? kMaxTokenSplits : want < 1 ? 1 : want;
  // Sums of several clusters go through global memory, 3 us: up to 9 rounds of a cluster's warps
  // (9216 keys) cost less. 8 rows of 4096, int8, 2 heads of 64: 8.8 us in one cluster, 12.9 in
  // two; one row of 16384 (16 rounds): 17.0 in one, 14.3 in several.
  if (want > kMaxCluster && gran <= 9 * kMaxCluster * kWarps) want = kMaxCluster;
  return (int)(want > kMaxCluster ? want / kMaxCluster * kMaxCluster : want);
}

// Key splits of the prompt kernel, the CTAs of a cluster: the most whose clusters all run at
// once (a CTA takes an SM, and a cluster the SMs of one GPC, so large ones leave some idle:
// 16 clusters of 8 do not fit, and took two rounds).
int prompt_splits(const qi_kv_layer& c, int M, int group, int window, int sinks) {
  const int tokens = kPromptRows / group * (c.head_dim == 64 ? 2 : 1);  // of a CTA
  const long long clusters = (long long)((M - 1) / tokens + 1) * c.kv_heads;
  const long long most = (seen_at_most(c, window, sinks) / kPromptKeys + 2) / kMinTiles;
  int n = (int)(most > 8 ? 8 : most);
  while (n > 1 && prompt_clusters(n) < clusters) --n;
  return n < 1 ? 1 : n;
}

void sizes(CacheAttnPlan& r, const qi_kv_layer& c, int heads, int M) {
  r.part_floats = r.counters = 0;
  if ((!r.prompt || r.singles) && r.token_splits > kMaxCluster) {  // sums of more than one cluster
    r.part_floats = (long long)M * heads * (r.token_splits / kMaxCluster) * (c.head_dim + 2);
    r.counters = (long long)M * c.kv_heads;
  }
}

}  // namespace

CacheAttnPlan cache_attention_plan(const qi_kv_layer& c, int heads, int M, int window, int sinks, int query_run) {
  CacheAttnPlan r = {};
  const bool tiles = (query_run & QI_RUN_TILES) != 0;
  query_run &= QI_RUN_TILES - 1;
  const long long work = (long long)M * c.kv_heads * c.head_dim * seen_at_most(c, window, sinks);
  r.prompt = tiles || ((query_run > 0 ? query_run >= kMinRun : M > 128) && work >= kMinWork);
  r.singles = r.prompt && query_run != M;
  r.splits = r.prompt ? prompt_splits(c, M, heads / c.kv_heads, window, sinks) : 1;
  r.token_splits = token_splits(c, M, window, sinks);
  sizes(r, c, heads, M);
  return r;
}

void cache_attention_fit(CacheAttnPlan& r, const qi_kv_layer& c, int heads, int M, long long part_floats,
                         long long counters) {
  while (r.part_floats > part_floats || r.counters > counters) {
    r.token_splits -= kMaxCluster;  // (with one cluster there is no scratch)
    sizes(r, c, heads, M);
  }
}

cudaError_t launch_cache_attention(const CacheAttnParams& args, const CacheAttnPlan& plan, cudaStream_t s, bool pdl) {
  CacheAttnParams p = args;
  p.scale_log2 = 1.4426950408889634f / sqrtf((float)p.c.head_dim);
  const int per = p.dtype == QI_F32 ? 4 : 8;
  p.q_vec = ((uintptr_t)p.q & 15) == 0 && p.q_st % per == 0 && p.q_sh % per == 0;
  if (plan.prompt) {
    p.min_tiles = kMinTiles;
    p.splits = plan.splits;
    p.skip_single = plan.singles;
    const cudaError_t e = launch_cache_attention_prompt(p, s, pdl);
    if (e != cudaSuccess || !plan.singles) return e;
    p.only_single = 1;
  }
  p.splits = plan.token_splits;
  p.cluster = p.splits > kMaxCluster ? kMaxCluster : p.splits;
  return p.c.head_dim == 64 ? launch_dim<64>(p, s, pdl) : launch_dim<128>(p, s, pdl);
}

}  // namespace qi

// Attention over one cache layer for prompts: tiles of consecutive query tokens share their
// keys on the 5th-generation tensor cores (the formula is in cache_attention.cu).
//
// A CTA takes the query rows of 128 / group consecutive tokens and one KV head (row = token
// x head of the group), at head_dim 64 two such tiles, and a share of the 128-key tiles that
// any of them sees:
//   S = Q K^T     M 128 x N 128 x K D, fp32 in TMEM; Q in shared memory
//   T = P V       M 128 x N D x K 128, fp32 in TMEM; P in TMEM, where it takes the place of S
// Threads r and r + 128 of the softmax warps share query row r (TMEM lane r), 64 keys and
// half of the output dims each: two passes over their scores (maximum, then exponentials),
// and O += T of the tile before in registers: the tensor cores' own accumulation truncates,
// so it stays within a tile and sums over tiles are rounded fp32 additions. The passes are
// chains of dependent instructions; the two threads of a row hide each other's latencies,
// as do the two tiles of a CTA, which share the keys that producer warps bring into the
// K-major layout of UMMA descriptors as fp16. The widening costs about as much as a tile's
// softmax: eight warps for bf16 values (4000 tokens, window 1024, head_dim 64: 119 us, with
// four 130; 2048 tokens on 4000 keys of 128 dims: 377, with four 724; the eight have become faster
// since), four for 8-bit codes, whose registers the softmax warps use better (1024 tokens on 4096
// keys: 54 us, with eight 56). V in the same layout is the MN-major operand of the second product, so nothing
// is transposed. One warp issues the MMAs.
//
// Measured: 1024 tokens on 4096 keys, 14 heads on 2 of 64, int8, bf16 queries: 54 us, 0.15 of
// the tensor cores' rate (8.1 us at the measured peak is the floor of 13.2 GFLOP); 4000 tokens
// under a window of 1024 on bf16 keys, fp32 queries: 111 us (floor 7.9 us, each product is
// two). What bounds it is the softmax: a pair of tiles takes 5300 to 6400 cycles for 128
// keys, of which the 64 exponentials of each of the 512 threads need 2048 of the one unit
// that makes them; the two products need 1500 (3000 in two parts).
//
// Every format is multiplied in fp16 with a scale for 16 keys: 8-bit codes are exact and
// have their block's scale; bf16 values get a power of two that puts the largest of 16 keys
// in [2^14, 2^15), which leaves all within 2^-28 of it exact and the others off by less than
// that. Where that is too coarse for one of the 16 (its own largest value more than 2^kSpread below;
// the large one may be masked for a row, or have no weight), each key gets a scale of its own, and
// the softmax applies them key by key: a row's result does not depend on what the keys beside its own
// hold. q is scaled per row to a maximum in [1, 2). fp32 callers: q and p in two fp16
// parts (22 bits), each part one UMMA chain into the same accumulator, the small ones first.
// 16-bit callers: q in one part, exact for it (to 2^-25 of the row's largest). p in two for fp16, whose
// outputs have 11 bits themselves, and in one for bf16: off by 2^-11, an eighth of the output's own
// rounding. (1024 tokens on 4096 keys, int8: 64 us in two parts, 55 in one, where the error of bf16 outputs
// against 64 bits is 1.66e-3, as that of their rounding alone is.)
//
// The K scale multiplies scores, the V scale of a block its probabilities: P holds 2^(x_j +
// log2 s_j - R + 14), where R is the largest x + log2 s of the row in the tile, so that what
// counts uses fp16's range whatever the scales are; T is brought back to the running maximum
// of the softmax when it is added to O.
//
// With few tiles the keys are split over the CTAs of a cluster, which exchange their partials
// through distributed shared memory: no scratch in global memory, no waiting CTA.
//
// Tokens of several cache rows in one tile are segments, worked off one after another with
// the other rows masked. Tokens alone in their tile's segment (a batched prefill's last
// tokens) are left to the per-token kernel in a second launch.
//
// What masked keys hold must not reach a row. Scores are replaced, keys that no row of the
// tile sees are zero-filled; but in P V a zero weight times a NaN or infinity that another
// row does see would be NaN. A row that ends up not finite is therefore computed again, key
// by key (8-bit codes are always finite: only the bf16 cache needs it), and so is one whose scores
// are as far from 0 as kFarScore says. That costs milliseconds a row of some thousand keys; neither
// comes up in a working model.
#include <atomic>

#include "cache_attention.cuh"
#include "tc_device.cuh"

namespace qi {

namespace {

using namespace cattn;
using namespace tc;

constexpr int kRows = 128;   // query rows of a tile
constexpr int kKeys = 128;   // keys of a tile
constexpr float kLift = 14.f;
constexpr uint32_t kMag = 0x7fff7fffu;  // magnitudes of a bf16 pair
// Exponents that the largest values of 16 bf16 keys may lie apart under one scale: all of the smallest
// key's are then known to 2^-22 of its largest. (4000 tokens, window 1024, head_dim 64, fp32 queries:
// 113 us where none lies further apart, 236 with such keys in every tile.)
constexpr uint32_t kSpread = 7;
constexpr unsigned kAll = 0xffffffffu;

struct True {
  static constexpr bool value = true;
};
struct False {
  static constexpr bool value = false;
};

template <int FMT, int D, int QP>
struct Shape {
  static constexpr int kTiles = D == 64 ? 2 : 1;  // query tiles of a CTA
  // warpgroups: two of softmax for each tile, producers, and one whose first warp issues MMAs
  static constexpr int kSoftWarps = 8 * kTiles, kLoadWarp = kSoftWarps, kLoadWarps = FMT == QI_KV_BF16 ? 8 : 4, kMmaWarp = kLoadWarp + kLoadWarps;
  static constexpr int kThreads = 32 * (kMmaWarp + 4);
  static constexpr uint32_t kQ = kRows * D * 2;   // one part of a tile's Q
  static constexpr uint32_t kT = kKeys * D * 2;   // K or V tile, two stages each
  static constexpr uint32_t kOffK = kTiles * QP * kQ, kOffV = kOffK + 2 * kT, kOffMisc = kOffV + 2 * kT;
  // TMEM columns: three S (each with its P in its place) that the tiles take in turn, then T
  static constexpr uint32_t kColT = 3 * 128, kCols = 512;
  static_assert(kColT + kTiles * D <= kCols, "tensor memory");
  // Registers of a thread: of the launch, and of the warpgroups, which together have no more.
  static constexpr int kRegLaunch = kLoadWarps == 8 ? (D == 64 ? 72 : 96) : (D == 64 ? 80 : 128);
  static constexpr int kRegSoft = D == 64 ? (FMT == QI_KV_BF16 ? 88 : 96) : 152;
  static constexpr int kRegLoad = D == 64 ? 56 : kLoadWarps == 8 ? 64 : 160, kRegMma = D == 64 ? 40 : 48;
  static_assert(kSoftWarps * kRegSoft + kLoadWarps * kRegLoad + 4 * kRegMma <= kThreads / 32 * kRegLaunch, "the increase must be covered");
};

constexpr int kMaxTok = 2 * kRows;  // tokens of a CTA

// the part of a CTA's tokens that lies in one cache row
struct Seg {
  int row, lo, hi, sinks, first;  // positions lo..hi and 0..sinks-1 seen; first tile in the list
};

struct Misc {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[3], p_full[3], t_full[2], done;
  uint32_t tmem;
  int nseg, ntiles;
  int abort;  // a wait of this CTA gave up: the others do not wait any more
  int pos[kMaxTok], row[kMaxTok], seg[kMaxTok];  // per token
  Seg segs[kMaxTok];
  Seg one;  // of tokens that all have one cache row (first: how many)
  // of 16 keys, by stage: K scale, exponent and significand of the V scale (s = 2^e * f; a
  // scale that is not finite has f = NaN)
  float ks[2][8], ve[2][8], vf[2][8];
  // bf16 layers: whether the 16 keys have scales of their own, of K (bit 0) and V (bit 1); then K scale
  // and exponent of the V scale of each
  __align__(4) uint8_t wide[2][8];
  __align__(16) float kk[2][kKeys], vk[2][kKeys];
  int k0[2], sg[2];  // first position and segment of the stage's keys
  float2 pair[2][2][2 * kRows];  // what the two threads of a row tell each other, by turns
  float2 ml[2 * kRows];       // maximum and sum of the rows' partials
};
constexpr uint32_t kMiscBytes = (sizeof(Misc) + 15) / 16 * 16;

__device__ __forceinline__ uint64_t desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46);
}
// kind::f16 instruction: fp16 operands, fp32 accumulator; bit 16: B is MN-major
__device__ __forceinline__ uint32_t idesc_f16(bool b_mn, int N) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
// One UMMA, issued by the lane whose `lead` is not 0. Executed by the whole warp, so that
// descriptors and addresses stay in uniform registers. A in shared memory, or (ts) in TMEM.
__device__ __forceinline__ void umma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
// 16 columns of this thread's lane, asynchronously: valid after tmem_ready on them
__device__ __forceinline__ void tmem_get16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// every load so far is complete; the registers pass through so that no use moves before it
__device__ __forceinline__ void tmem_ready(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
// f(j, columns 16 j .. 16 j + 15) for j < N, the next load under way meanwhile
template <int N, class F>
__device__ __forceinline__ void tmem_each16(uint32_t taddr, F f) {
  uint32_t r[2][16];
  tmem_get16(taddr, r[0]);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    tmem_ready(r[j & 1]);
    if (j + 1 < N) tmem_get16(taddr + 16 * (j + 1), r[(j + 1) & 1]);
    f(j, r[j & 1]);
  }
}
__device__ __forceinline__ void tmem_put8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// byte offset of (row r, 8-element chunk c) of an operand with D elements a row: 8x8 core
// matrices of 128 bytes, chunks 128 bytes apart, groups of 8 rows D * 16
template <int D>
__device__ __forceinline__ uint32_t core(int r, int c) {
  return (uint32_t)((r >> 3) * (D * 16) + c * 128 + (r & 7) * 16);
}

// Bounded wait that ends at once when another wait of the CTA has given up. The thread is
// suspended for up to kNap ns at a time: polling warps would take issue slots from the
// others.
constexpr uint32_t kNap = 20000;
__device__ __forceinline__ bool nap(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(kNap)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, Misc& X, int* err) {
  if (nap(bar, parity)) return;
  const uint64_t t0 = global_timer_ns();
  while (!nap(bar, parity)) {
    if (*reinterpret_cast<volatile int*>(&X.abort)) return;
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      *reinterpret_cast<volatile int*>(&X.abort) = 1;
      if (err) atomicExch(err, QI_ERR_TIMEOUT);
      return;
    }
  }
}

// N 16-byte pieces of a query row (fp32, or a 16-bit type) from element o on, as they are
template <int N, bool F32>
__device__ __forceinline__ void load_row(const CacheAttnParams& p, long long o, uint4 (&x)[N]) {
  if (p.q_vec) {
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.q) + o * (F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __ldcg(q + i);
  } else {
    for (int i = 0; i < N; ++i) {
      uint32_t w[4];
      for (int e = 0; e < 4; ++e) {
        if constexpr (F32) {
          w[e] = __ldcg(static_cast<const uint32_t*>(p.q) + o + 4 * i + e);
        } else {
          const unsigned short* h = static_cast<const unsigned short*>(p.q) + o + 8 * i + 2 * e;
          w[e] = (uint32_t)__ldcg(h) | (uint32_t)__ldcg(h + 1) << 16;
        }
      }
      x[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
// values 2 i and 2 i + 1 of such a row
template <bool F32>
__device__ __forceinline__ float2 row_pair(const uint4* x, int i, int dtype) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
  if constexpr (F32) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  else if (dtype == QI_BF16) return make_float2(bf16lo(w[i]), bf16hi(w[i]));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
}
// one element of q
__device__ __forceinline__ float load_q(const CacheAttnParams& p, long long i) {
  return p.dtype == QI_F32 ? load_elem<QI_F32>(p.q, i) : p.dtype == QI_BF16 ? load_elem<QI_BF16>(p.q, i) : load_elem<QI_F16>(p.q, i);
}

// Key by key: the partial of token t's head over the given tiles of its segment, dims d0 .. d0 + D / 2 - 1 of
// the output into o (shared memory); returns its maximum and sum. The weights of masked keys are left out, not
// multiplied by zero.
template <int FMT, int D>
__device__ __noinline__ float2 plain_row(const CacheAttnParams& p, const Seg& sg, int tbeg, int tend, int tok, int head, int g,
                                         int ps, int d0, float* o) {
  auto value = [](const void* x, long long i) -> float {
    if constexpr (FMT == QI_KV_BF16) return bf16_to_f32(static_cast<const uint16_t*>(x)[i]);
    else return decode<FMT>(static_cast<const uint8_t*>(x)[i]);
  };
  const Seen<kKeys> list = seen_range<kKeys>(sg.hi, sg.lo, sg.sinks);
  const Seen<kKeys> mine = seen_range<kKeys>(ps, window_start(ps, p.window), p.sinks);
  const long long qo = (long long)tok * p.q_st + (long long)head * p.q_sh;
  float m = -INFINITY, l = 0.f;
  for (int d = 0; d < D / 2; ++d) o[d] = 0.f;
  for (int i = tbeg; i < tend; ++i) {
    const int k0 = list.granule(i) * kKeys;
    const long long base = layer_offset(p.c, D, sg.row, g, k0);
    for (int j = 0; j < kKeys; ++j) {
      if (!mine.sees(k0 + j)) continue;
      float s = 0.f, fv = 0.f;
      const long long at = base + j * D;
      if (base >= 0) {
        float fk = 1.f;
        fv = 1.f;
        if constexpr (FMT != QI_KV_BF16) {
          const long long si = scale_index(p.c, sg.row, g, k0 + j);
          fk = __ldcg(p.c.k_scale + si), fv = __ldcg(p.c.v_scale + si);
        }
        for (int d = 0; d < D; ++d) s = fmaf(load_q(p, qo + d), value(p.c.k, at + d) * fk, s);
      }
      s = __fmul_rn(s, p.scale_log2);  // rounded, as the maximum is
      if (s > m) {
        const float a = m == -INFINITY ? 0.f : ex2(m - s);
        l *= a;
        for (int d = 0; d < D / 2; ++d) o[d] *= a;
        m = s;
      }
      const float w = ex2(s - (m == -INFINITY ? 0.f : m));
      l += w;
      if (base >= 0)
        for (int d = 0; d < D / 2; ++d) o[d] = fmaf(w, value(p.c.v, at + d0 + d) * fv, o[d]);
    }
  }
  return make_float2(m, l);
}

// The two passes of the softmax over a thread's 64 scores where some of the keys have scales of their
// own (`wide`: Misc's bytes); bit j of `seen`: key j is seen. Out of line: rare, and the registers of the
// passes without them stay as they are.
struct KeyScales {
  const float *k, *v;
  int ks, vs;  // steps from key to key
  __device__ __forceinline__ KeyScales(const Misc& X, int st, int hf, uint32_t wide, int c) {
    const uint32_t w = wide >> (8 * c);
    ks = w & 1u, vs = (w >> 1) & 1u;
    k = ks ? &X.kk[st][64 * hf + 16 * c] : &X.ks[st][4 * hf + c];
    v = vs ? &X.vk[st][64 * hf + 16 * c] : &X.ve[st][4 * hf + c];
  }
};
// The maxima of the scores and of score + exponent of the V scale.
__device__ __noinline__ float2 key_maxima(const Misc& X, int st, int hf, uint32_t wide, uint32_t srow, uint64_t seen, float qs) {
  float mx = -INFINITY, R = -INFINITY;
  tmem_each16<4>(srow, [&](int c, const uint32_t(&s)[16]) {
    const KeyScales y(X, st, hf, wide, c);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float x = (seen >> (16 * c + j)) & 1u ? __uint_as_float(s[j]) * (qs * y.k[j * y.ks]) : -INFINITY;
      R = fmaxf(R, x + y.v[j * y.vs]);
      mx = fmaxf(mx, x);
    }
  });
  return make_float2(mx, R);
}
// P into the place of the scores; returns the weights' sum.
template <int PARTS>
__device__ __noinline__ float key_weights(const Misc& X, int st, int hf, uint32_t wide, uint32_t srow, uint64_t seen, float qs,
                                          float mr, float rest) {
  float sum[2] = {0.f, 0.f};
  tmem_each16<4>(srow, [&](int c, const uint32_t(&s)[16]) {
    const KeyScales y(X, st, hf, wide, c);
    uint32_t part[PARTS][8];
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      float u[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = (seen >> (16 * c + j + i)) & 1u;
        const float x = fmaf(__uint_as_float(s[j + i]), qs * y.k[(j + i) * y.ks], -mr);
        sum[i] += in ? ex2(x) : 0.f;
        // (not as weight times factor: a weight that underflows may have the largest product)
        u[i] = in ? ex2(x + (y.v[(j + i) * y.vs] + rest)) : 0.f;
      }
      uint32_t h[PARTS];
      split<true, PARTS>(u[0], u[1], h);
#pragma unroll
      for (int q = 0; q < PARTS; ++q) part[q][j / 2] = h[q];
    }
    // the 16 columns of S are read: their P takes them
#pragma unroll
    for (int q = 0; q < PARTS; ++q) tmem_put8(srow + 16 * c + 8 * q, part[q]);
  });
  return sum[0] + sum[1];
}
// the same shared memory of CTA w of the cluster (of C CTAs)
__device__ __forceinline__ float peer(const float* x, int w, int C) {
  if (C == 1) return *x;
  float r;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(r) : "r"(map_rank(x, (uint32_t)w)) : "memory");
  return r;
}
__device__ __forceinline__ float4 peer4(const float* x, int w, int C) {
  if (C == 1) return *reinterpret_cast<const float4*>(x);
  float4 r;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w)
               : "r"(map_rank(x, (uint32_t)w))
               : "memory");
  return r;
}

template <int N>
__device__ __forceinline__ void more_regs() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_regs() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int FMT, int D, int QP, int PP>
__global__ void __launch_bounds__(Shape<FMT, D, QP>::kThreads, 1) prompt_kernel(const __grid_constant__ CacheAttnParams p) {
  using H = Shape<FMT, D, QP>;
  constexpr bool BF = FMT == QI_KV_BF16;
  constexpr int kPitch = D + 4;  // floats of a row of partial outputs
  extern __shared__ __align__(1024) uint8_t smem[];
  Misc& X = *reinterpret_cast<Misc*>(smem + H::kOffMisc);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const qi_kv_layer& c = p.c;
  const int G = p.group, TT = kRows / G, width = p.heads * D;  // TT: tokens of a tile
  const int CT = H::kTiles * TT;
  const int ctas_m = (p.M + CT - 1) / CT;
  // the last tokens see most: they start first
  const int split_i = blockIdx.x % p.splits, g = blockIdx.y;
  const int t0 = (ctas_m - 1 - (int)(blockIdx.x / p.splits)) * CT, ntok = min(CT, p.M - t0);
  const int ntl = ntok > TT ? 2 : 1;  // tiles with tokens

  grid_dep_wait();
  if (warp == H::kMmaWarp) {
    tmem_alloc(&X.tmem, H::kCols);
    tmem_relinquish();
  }
  grid_dep_launch();
  // Threads r and r + 128 of a tile's softmax warps: query row r = (token, head), half of
  // its dims (and 64 of a tile's keys). The loads overlap the setup.
  constexpr int DH = D / 2, kRaw = DH / (QP == 2 ? 4 : 8);
  const int qt = tid >> 8, r = tid & (kRows - 1), hf = (tid >> 7) & 1;
  const int rr = qt * kRows + r;  // row of the CTA
  // its token of the CTA, none (ntok) for rows past the tile's last whole token
  const int tl = r / G < TT ? min(qt * TT + r / G, ntok) : ntok, head = g * G + r % G;
  uint4 raw[kRaw];
  if (warp < H::kSoftWarps)
    load_row<kRaw, QP == 2>(p, (long long)(t0 + min(tl, ntok - 1)) * p.q_st + (long long)head * p.q_sh + hf * DH, raw);
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&X.k_full[s], H::kLoadWarps);
      mbar_init(&X.v_full[s], H::kLoadWarps);
      mbar_init(&X.k_empty[s], 1);
      mbar_init(&X.v_empty[s], 1);
      mbar_init(&X.t_full[s], 1);
    }
    for (int s = 0; s < 3; ++s) {
      mbar_init(&X.s_full[s], 1);
      mbar_init(&X.p_full[s], 8);
    }
    mbar_init(&X.done, 1);
    X.abort = 0;
    X.one = Seg{0, 0x7fffffff, -1, 0, 0};
    fence_barrier_init();
  }
  if (tid < kMaxTok) {
    int ps = -1, rw = -1;
    if (tid < ntok) {
      ps = p.pos[t0 + tid], rw = p.rows[t0 + tid];
      if (!token_ok(p, ps, rw)) {
        if (ps != -1 && g == 0 && split_i == 0 && p.err) atomicExch(p.err, QI_ERR_INDEX);
        ps = -1;
      }
    }
    X.pos[tid] = ps;
    X.row[tid] = rw;
  }
  __syncthreads();
  // The tokens' segments. Mostly there is one: all of one cache row.
  const bool valid = tid < ntok && X.pos[tid] >= 0;
  if (!__syncthreads_or(valid && X.row[tid] != X.row[0])) {
    if (valid) {
      const int ps = X.pos[tid], lo = window_start(ps, p.window);
      atomicMin(&X.one.lo, lo);
      atomicMax(&X.one.hi, ps);
      atomicMax(&X.one.sinks, min(p.sinks, lo));
      atomicAdd(&X.one.first, 1);
    }
    __syncthreads();
    if (tid == 0) {
      const int tokens = X.one.first;
      X.segs[0] = Seg{X.row[0], X.one.lo, X.one.hi, X.one.sinks, 0};
      X.nseg = tokens > (p.skip_single ? 1 : 0);  // a single token is left to the per-token kernel
      X.ntiles = X.nseg ? seen_range<kKeys>(X.one.hi, X.one.lo, X.one.sinks).n : 0;
    }
  } else {
    // the first token of each cache row gathers what its tokens see
    if (tid < ntok) {
      int first = -1;
      Seg s = {0, 0x7fffffff, -1, 0, 0};
      if (X.pos[tid] >= 0) {
        int n = 0;
        for (int i = 0; i < ntok; ++i) {
          if (X.pos[i] < 0 || X.row[i] != X.row[tid]) continue;
          if (first < 0) first = i;
          if (first != tid) break;
          const int ps = X.pos[i], lo = window_start(ps, p.window);
          ++n;
          s.lo = min(s.lo, lo);
          s.hi = max(s.hi, ps);
          s.sinks = max(s.sinks, min(p.sinks, lo));
        }
        s.row = X.row[tid];
        if (p.skip_single && first == tid && n == 1) s.hi = -1;  // left to the per-token kernel
      }
      X.seg[tid] = first;
      X.segs[tid] = s;
    }
    __syncthreads();
    if (tid == 0) {  // the list of key tiles: segment after segment
      int n = 0, t = 0;
      for (int i = 0; i < ntok; ++i) {
        if (X.seg[i] != i || X.segs[i].hi < 0) continue;
        Seg s = X.segs[i];
        s.first = t;
        t += seen_range<kKeys>(s.hi, s.lo, s.sinks).n;
        // compacted in place: the segments before it are at places up to i
        X.segs[n++] = s;
      }
      X.nseg = n;
      X.ntiles = t;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = X.tmem;
  const int nsplit = max(1, min(p.splits, X.ntiles / p.min_tiles));
  const bool work = split_i < nsplit;
  const int tbeg = work ? (int)((long long)X.ntiles * split_i / nsplit) : 0;
  const int tend = work ? (int)((long long)X.ntiles * (split_i + 1) / nsplit) : 0;
  const int n = tend - tbeg;
  if (warp >= H::kMmaWarp) {
    // ------------------------------------------------------------------- MMA
    fewer_regs<H::kRegMma>();
    if (warp == H::kMmaWarp) {
      asm volatile("bar.sync 1, %0;" ::"n"(32 * (H::kSoftWarps + 1)) : "memory");  // Q is in place
      const uint32_t sb = smem_u32(smem), lead = lane == 0;
      const uint32_t id_s = idesc_f16(false, kKeys), id_t = idesc_f16(true, D);
      // Products of the key tiles i, of each for the query tiles t: number x = i ntl + t. S of x
      // goes to buffer x % 3, where S of x - 3 was, whose P the product T of x - 3, issued
      // before, has read. Scores run `ahead` products before T, so that those of a tile's next
      // keys are ready when it is done with these; with one query tile only 2, since its third
      // would wait for keys whose stage the first T has to free.
      const int lg = ntl - 1, total = n << lg;
      auto scores = [&](int x, int buf) {
        const int i = x >> lg, t = x & lg;
        wait(&X.k_full[i & 1], (uint32_t)(i >> 1) & 1u, X, p.err);
        tc_fence_after();
        const uint64_t qd = desc(sb + t * QP * H::kQ, 128, D * 16);
        const uint64_t kd = desc(sb + H::kOffK + (i & 1) * H::kT, 128, D * 16);
#pragma unroll
        for (int q = QP - 1; q >= 0; --q)
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_ss(lead, tmem + 128 * buf, qd + (uint64_t)(q * (H::kQ >> 4) + k * 16), kd + (uint64_t)(k * 16), id_s,
                    q < QP - 1 || k > 0 ? 1u : 0u);
        commit(lead, &X.s_full[buf]);
        if (t == lg) commit(lead, &X.k_empty[i & 1]);
      };
      const int ahead = 2 + lg;
      for (int x = 0; x < min(ahead, total); ++x) scores(x, x);
      int buf = 0;
      uint32_t ph = 0u;
      for (int x = 0; x < total; ++x) {
        const int i = x >> lg, t = x & lg, st = i & 1;
        wait(&X.v_full[st], (uint32_t)(i >> 1) & 1u, X, p.err);
        wait(&X.p_full[buf], ph, X, p.err);
        tc_fence_after();
        const uint64_t vd = desc(sb + H::kOffV + st * H::kT, D * 16, 128);
#pragma unroll
        for (int q = PP - 1; q >= 0; --q)
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k)
            // 16 keys: 8 columns of P for each part; 2 key groups of V
            umma_ts(lead, tmem + H::kColT + D * t, tmem + 128 * buf + 16 * k + 8 * q, vd + (uint64_t)(k * 2 * D), id_t,
                    q < PP - 1 || k > 0 ? 1u : 0u);
        commit(lead, &X.t_full[t]);
        if (t == lg) commit(lead, &X.v_empty[st]);
        if (x + ahead < total) scores(x + ahead, buf + ahead >= 3 ? buf + ahead - 3 : buf + ahead);
        if (++buf == 3) buf = 0, ph ^= 1u;
      }
      commit(lead, &X.done);
      __syncwarp();
    }
    __syncthreads();
  } else if (warp >= H::kLoadWarp) {
    // ------------------------------------------------------------- producers
    if constexpr (H::kRegLoad > H::kRegLaunch) more_regs<H::kRegLoad>();
    else fewer_regs<H::kRegLoad>();
    const int lt = tid - 32 * H::kLoadWarp, lw = warp - H::kLoadWarp;
    constexpr int kCh = D * (BF ? 2 : 1) / 16;        // 16-byte chunks of a key
    constexpr int kN = kKeys * kCh / (32 * H::kLoadWarps);    // of a thread
    // a warp takes 32 keys; one of its loads is 8 keys x 4 chunks: whole lines, and the
    // lanes of a store phase hold 8 keys
    auto place = [&](int j, int& r, int& ch) {
      r = lw * (kKeys / H::kLoadWarps) + (j / (kCh / 4)) * 8 + (lane & 7);
      ch = (j % (kCh / 4)) * 4 + (lane >> 3);
    };
    constexpr bool kBoth = !BF || D == 64;  // else V follows K in the same registers
    uint4 kr[kN], vr[kBoth ? kN : 1];
    float sc = 1.f;
    int si = 0, first_key = 0;  // segment of the tile at hand (entries come in order), its first key
    auto fetch = [&](int i, bool k_side) {
      while (si + 1 < X.nseg && i >= X.segs[si + 1].first) ++si;
      const Seg& sg = X.segs[si];
      const Seen<kKeys> list = seen_range<kKeys>(sg.hi, sg.lo, sg.sinks);
      const int k0 = list.granule(i - sg.first) * kKeys;
      first_key = k0;
      const long long o = layer_offset(c, D, sg.row, g, k0);
      if (o < 0 && lt == 0 && p.err) atomicExch(p.err, QI_ERR_INDEX);
      const long long base = (o < 0 ? 0 : o) * (BF ? 2 : 1);
      const uint8_t* kb = static_cast<const uint8_t*>(c.k) + base;
      const uint8_t* vb = static_cast<const uint8_t*>(c.v) + base;
      const uint4 z = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        int r, ch;
        place(j, r, ch);
        const bool in = o >= 0 && list.sees(k0 + r);
        const int x = (r * kCh + ch) * 16;
        if constexpr (!kBoth) {
          kr[j] = in ? __ldcg(reinterpret_cast<const uint4*>((k_side ? kb : vb) + x)) : z;
        } else {
          kr[j] = in ? __ldcg(reinterpret_cast<const uint4*>(kb + x)) : z;
          vr[j] = in ? __ldcg(reinterpret_cast<const uint4*>(vb + x)) : z;
        }
      }
      if constexpr (!BF) {
        if (lt < 16) {
          const int h0 = k0 + 16 * (lt & 7);
          const bool any = o >= 0 && list.sees16(h0);
          // (not a read-only load: this kernel may have been launched before the append wrote them)
          sc = any ? __ldcg((lt < 8 ? c.k_scale : c.v_scale) + scale_index(c, sg.row, g, h0)) : 1.f;
        }
      }
    };
    // 8-bit codes in registers -> fp16 operand rows
    auto store8 = [&](const uint4* regs, uint8_t* t) {
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        int r, ch;
        place(j, r, ch);
        const uint32_t w[4] = {regs[j].x, regs[j].y, regs[j].z, regs[j].w};
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) widen<BF ? QI_KV_INT8 : FMT, 0>(w[e], h[2 * e], h[2 * e + 1]);
        *reinterpret_cast<uint4*>(t + core<D>(r, 2 * ch)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(t + core<D>(r, 2 * ch + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
    };
    // bf16 values -> fp16 operand rows, and the scales of the warp's 16 keys, or of each of them
    // (returned: whether they are wide)
    auto store16 = [&](const uint4* regs, uint8_t* t, int st, bool k_side) -> bool {
      static_assert(!BF || H::kLoadWarps == 8, "a warp has 16 keys");
      constexpr int kHalf = kN / 2;  // chunks of the thread's keys lane & 7 and 8 + (lane & 7)
      // Largest magnitudes of the two keys' chunks here (of the low and the high halves, then of both):
      // where every lane's lie within the spread, all keys do; else the lanes that have the keys' other
      // chunks are asked.
      uint32_t m2[2] = {0u, 0u};
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        uint32_t& m = m2[j / kHalf];
        m = __vmaxu2(__vmaxu2(m, __vmaxu2(regs[j].x & kMag, regs[j].y & kMag)),
                     __vmaxu2(regs[j].z & kMag, regs[j].w & kMag));
      }
      uint32_t k0 = max(m2[0] >> 16, m2[0] & 0xffffu), k1 = max(m2[1] >> 16, m2[1] & 0xffffu);
      // the exponent e of a largest value 2^(e - 127) * [1, 2), whose scale is 2^(e - 127 - 14): in
      // 15..253 (the scale and its reciprocal are normal); tiny keys are left with a smaller maximum
      auto exponent = [](uint32_t m) { return min(max(m >> 7, 15u), 253u); };
      uint32_t mx = __reduce_max_sync(kAll, max(k0, k1)), e = exponent(mx);
      bool wide = false;
      if (!__any_sync(kAll, mx >= 0x7f80u || e < 29u || exponent(min(k0, k1)) + kSpread < e)) {
        // bf16 to fp16 at that scale: the exponent field moves by e - 29 (from e to 29, that
        // of 2^14) and the significand gains three zeros; values below fp16's normal range, 2^-28
        // of the largest, come out off by less than that. Both halves at once: neither borrows
        // nor overflows.
        const uint32_t off2 = ((e - 29u) << 7) * 0x10001u;
        auto half2_of = [&](uint32_t w) -> uint32_t { return ((__vmaxu2(w & kMag, off2) - off2) << 3) | (w & ~kMag); };
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          int r, ch;
          place(j, r, ch);
          *reinterpret_cast<uint4*>(t + core<D>(r, ch)) =
              make_uint4(half2_of(regs[j].x), half2_of(regs[j].y), half2_of(regs[j].z), half2_of(regs[j].w));
        }
      } else {  // wide blocks, those with infinities or NaN (scaled by the finite values) and tiny ones: by way of fp32
        if (mx >= 0x7f80u) {
          k0 = k1 = 0u;
#pragma unroll
          for (int j = 0; j < kN; ++j) {
            const uint32_t w[4] = {regs[j].x, regs[j].y, regs[j].z, regs[j].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t lo = w[x] & 0x7fffu, hi = (w[x] >> 16) & 0x7fffu;
              uint32_t& m = j < kHalf ? k0 : k1;
              m = max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
            }
          }
        }
        uint32_t km = k0 | k1 << 16;
        km = __vmaxu2(km, __shfl_xor_sync(kAll, km, 8));
        km = __vmaxu2(km, __shfl_xor_sync(kAll, km, 16));
        k0 = km & 0xffffu, k1 = km >> 16;
        e = exponent(__reduce_max_sync(kAll, max(k0, k1)));
        wide = __any_sync(kAll, (k0 != 0u && exponent(k0) + kSpread < e) || (k1 != 0u && exponent(k1) + kSpread < e));
        const uint32_t e0 = wide ? exponent(k0) : e, e1 = wide ? exponent(k1) : e;
        if (wide && lane < 8) {
          const int i = lw * 16 + lane;
          if (k_side) X.kk[st][i] = __uint_as_float((e0 - 14u) << 23), X.kk[st][i + 8] = __uint_as_float((e1 - 14u) << 23);
          else X.vk[st][i] = (float)((int)e0 - 141), X.vk[st][i + 8] = (float)((int)e1 - 141);
        }
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          int r, ch;
          place(j, r, ch);
          const float inv = __uint_as_float((268u - (j < kHalf ? e0 : e1)) << 23);
          const uint32_t w[4] = {regs[j].x, regs[j].y, regs[j].z, regs[j].w};
          uint32_t h[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) h[x] = f16x2(bf16lo(w[x]) * inv, bf16hi(w[x]) * inv);
          *reinterpret_cast<uint4*>(t + core<D>(r, ch)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
      }
      if (lane == 0) {
        if (k_side) X.ks[st][lw] = __uint_as_float((e - 14u) << 23);
        else X.ve[st][lw] = (float)((int)e - 141), X.vf[st][lw] = 1.f;
      }
      return wide;
    };
    auto publish = [&](uint64_t* bar) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    if (n > 0) fetch(tbeg, true);
    for (int i = 0; i < n; ++i) {
      const int st = i & 1;
      const uint32_t ph = (uint32_t)((i >> 1) - 1) & 1u;
      uint8_t* kt = smem + H::kOffK + st * H::kT;
      uint8_t* vt = smem + H::kOffV + st * H::kT;
      // tile i - 2 is done with: its products, and its scales (all of them after the last T)
      if (i >= 2) {
        wait(&X.k_empty[st], ph, X, p.err);
        wait(&X.v_empty[st], ph, X, p.err);
      }
      if (lt == 0) X.k0[st] = first_key, X.sg[st] = si;
      if constexpr (BF) {
        const bool wide_k = store16(kr, kt, st, true);
        publish(&X.k_full[st]);
        if constexpr (!kBoth) fetch(tbeg + i, false);
        const bool wide_v = store16(kBoth ? vr : kr, vt, st, false);
        if (lane == 0) X.wide[st][lw] = (uint8_t)((wide_k ? 1 : 0) | (wide_v ? 2 : 0));
        publish(&X.v_full[st]);
      } else {
        if (lt < 8) X.ks[st][lt] = sc;
        else if (lt < 16) {
          const uint32_t bits = __float_as_uint(sc);
          X.ve[st][lt - 8] = (float)((int)(bits >> 23) - 127);
          X.vf[st][lt - 8] = bits < 0x7f800000u ? __uint_as_float((bits & 0x7fffffu) | 0x3f800000u)
                                                : __uint_as_float(0x7fc00000u);
        }
        store8(kr, kt);
        publish(&X.k_full[st]);
        store8(vr, vt);
        publish(&X.v_full[st]);
      }
      if (i + 1 < n) fetch(tbeg + i + 1, true);
    }
    __syncthreads();
  } else {
    // --------------------------------------------------------------- softmax
    more_regs<H::kRegSoft>();
    auto pair_bar = [&] { asm volatile("bar.sync %0, 64;" ::"r"(2 + 4 * qt + (warp & 3)) : "memory"); };
    const int ps = tl < ntok ? X.pos[tl] : -1;
    // the row's segment, by cache row (segments left out have no entry)
    int seg = -1;
    for (int s = 0; s < X.nseg && ps >= 0; ++s)
      if (X.segs[s].row == X.row[tl]) seg = s;
    const bool live = ps >= 0 && seg >= 0;
    float qs = p.scale_log2;
    {
      float am = 0.f;
#pragma unroll
      for (int i = 0; i < DH / 2; ++i) {
        const float2 x = row_pair<QP == 2>(raw, i, p.dtype);
        am = fmaxf(am, fmaxf(fabsf(x.x), fabsf(x.y)));
      }
      X.pair[1][hf][rr].x = am;
      pair_bar();
      am = fmaxf(am, X.pair[1][hf ^ 1][rr].x);
      float inv = live ? 1.f : 0.f;
      const uint32_t e = __float_as_uint(am) >> 23;
      if (live && e > 0 && e < 253) {
        inv = __uint_as_float((254u - e) << 23);
        qs *= __uint_as_float(e << 23);
      }
#pragma unroll
      for (int ch = 0; ch < DH / 8; ++ch) {
        uint32_t w[4][QP];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = row_pair<QP == 2>(raw, 4 * ch + i, p.dtype);
          split<true, QP>(live ? x.x * inv : 0.f, live ? x.y * inv : 0.f, w[i]);
        }
#pragma unroll
        for (int q = 0; q < QP; ++q)
          *reinterpret_cast<uint4*>(smem + (qt * QP + q) * H::kQ + core<D>(r, hf * (DH / 8) + ch)) =
              make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
      }
      fence_async_smem();
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * (H::kSoftWarps + 1)) : "memory");
    const Seen<kKeys> mine = seen_range<kKeys>(live ? ps : 0, live ? window_start(ps, p.window) : 0, p.sinks);
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t orow = trow + H::kColT + D * qt + DH * hf;  // and dims

    float m = -INFINITY, l = 0.f;  // maximum of the scores (log2 units), sum of 2^(x - m)
    float size = 0.f;              // the largest that |m| was
    f2 o[DH / 2];                  // sum of 2^(x - m) v (this half's dims; l: this half's keys)
#pragma unroll
    for (int d = 0; d < DH / 2; ++d) o[d] = 0ull;
    // the last tile: O = O * oa + T * ob
    float oa = 1.f, ob = 0.f;
    auto add_tile = [&] {
      if (__any_sync(kAll, oa != 1.f)) {
        const f2 f = pack2(oa, oa);
#pragma unroll
        for (int d = 0; d < DH / 2; ++d) o[d] = mul2(o[d], f);
      }
      const f2 f = pack2(ob, ob);
      tmem_each16<DH / 16>(orow, [&](int c, const uint32_t(&t)[16]) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          o[8 * c + j] = fma2(pack2(__uint_as_float(t[2 * j]), __uint_as_float(t[2 * j + 1])), f, o[8 * c + j]);
      });
    };
    const int n_mine = qt < ntl ? n : 0;
    int buf = qt;  // S of the tile at hand, and its phase
    uint32_t sph = 0u;
    for (int i = 0; i < n_mine; ++i) {
      const int st = i & 1;
      wait(&X.v_full[st], (uint32_t)(i >> 1) & 1u, X, p.err);  // the scales and the place of the keys
      const int k0 = X.k0[st];
      // the row's keys of this tile: [a, b] and [0, s0)
      const int b = live && seg == X.sg[st] ? min(mine.p - k0, kKeys - 1) : -1;
      const int a = mine.lo - k0, s0 = min(mine.sinks - k0, b + 1);
      // (what rows without a token do is not used)
      const bool whole = !live || (b == kKeys - 1 && (a <= 0 || s0 >= kKeys));
      const bool masked = __any_sync(kAll, !whole);
      auto mask16 = [&](int c0) -> uint32_t {  // bit j < 16: key c0 + j is seen
        auto below = [](int x) { return x <= 0 ? 0u : x >= 16 ? 0xffffu : (1u << x) - 1u; };
        return (below(b + 1 - c0) & ~below(a - c0)) | below(s0 - c0);
      };
      auto seen64 = [&]() -> uint64_t {
        uint64_t m = 0ull;
        for (int c = 3; c >= 0; --c) m = m << 16 | mask16(64 * hf + 16 * c);
        return m;
      };
      float ks[4], ve[4];  // of this half's 4 blocks
#pragma unroll
      for (int c = 0; c < 4; ++c) ks[c] = qs * X.ks[st][4 * hf + c], ve[c] = X.ve[st][4 * hf + c];
      const uint32_t wide = BF ? *reinterpret_cast<const uint32_t*>(&X.wide[st][4 * hf]) : 0u;  // a byte for each
      wait(&X.s_full[buf], sph, X, p.err);
      tc_fence_after();
      const uint32_t srow = trow + 128 * buf + 64 * hf;  // this half's scores
      // pass 1: the maxima of the scores and of score + log2(V scale)
      float mx = -INFINITY, R = -INFINITY;
      auto maxima = [&](auto some_masked) {
        tmem_each16<4>(srow, [&](int c, const uint32_t(&s)[16]) {
          float a4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          const uint32_t mk = decltype(some_masked)::value ? mask16(64 * hf + 16 * c) : 0u;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float x = __uint_as_float(s[j]);
            if constexpr (decltype(some_masked)::value) a4[j & 3] = fmaxf(a4[j & 3], (mk >> j) & 1u ? x : -INFINITY);
            else a4[j & 3] = fmaxf(a4[j & 3], x);
          }
          float v = fmaxf(fmaxf(a4[0], a4[1]), fmaxf(a4[2], a4[3]));
          // a block without seen keys has no say; its scale may be anything
          v = v == -INFINITY ? v : v * ks[c];
          R = fmaxf(R, v + ve[c]);
          mx = fmaxf(mx, v);
        });
      };
      if (wide) {
        const float2 r = key_maxima(X, st, hf, wide, srow, seen64(), qs);
        mx = r.x, R = r.y;
      } else if (masked) maxima(True{});
      else maxima(False{});
      X.pair[st][hf][rr] = make_float2(mx, R);
      pair_bar();
      const float2 other = X.pair[st][hf ^ 1][rr];
      R = fmaxf(R, other.y);
      const float mn = fmaxf(m, fmaxf(mx, other.x));
      if (i > 0) {  // T of the tile before, with its factors
        wait(&X.t_full[qt], (uint32_t)(i - 1) & 1u, X, p.err);
        tc_fence_after();
        add_tile();
      }
      oa = m == -INFINITY ? 1.f : ex2(m - mn);  // nothing summed yet: nothing to rescale
      l *= oa;
      m = mn;
      // (a tile of which the row sees nothing: P is zero, and T's factor stays finite whatever the maximum is)
      const float mr = m == -INFINITY ? 0.f : m, Rr = R == -INFINITY ? mr : R;
      // (one rounded exponent both ways: what P is raised by, T is lowered by)
      const float rest = mr - Rr + kLift;
      ob = ex2(-rest);
      size = fmaxf(size, fabsf(mr));
      // pass 2: weights and their parts
      f2 sum[2] = {0ull, 0ull};
      auto weights = [&](auto some_masked) {
        tmem_each16<4>(srow, [&](int c, const uint32_t(&s)[16]) {
          // 2^(x - m) * fv = 2^(x + log2(V scale) - R + lift)
          const float fv = X.vf[st][4 * hf + c] * ex2(fminf(ve[c] + rest, 126.f));
          const f2 fk2 = pack2(ks[c], ks[c]), fv2 = pack2(fv, fv), mr2 = pack2(-mr, -mr);
          const uint32_t mk = decltype(some_masked)::value ? mask16(64 * hf + 16 * c) : 0u;
          uint32_t part[PP][8];
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const float2 x = unpack2(fma2(pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), fk2, mr2));
            float w0 = ex2(x.x), w1 = ex2(x.y);
            if constexpr (decltype(some_masked)::value) {
              w0 = (mk >> j) & 1u ? w0 : 0.f;
              w1 = (mk >> (j + 1)) & 1u ? w1 : 0.f;
            }
            const f2 w = pack2(w0, w1);
            sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], w);
            float2 u = unpack2(mul2(w, fv2));
            if constexpr (decltype(some_masked)::value) {  // the scale of a block without seen keys may be NaN
              u.x = (mk >> j) & 1u ? u.x : 0.f;
              u.y = (mk >> (j + 1)) & 1u ? u.y : 0.f;
            }
            uint32_t y[PP];
            split<true, PP>(u.x, u.y, y);
#pragma unroll
            for (int q = 0; q < PP; ++q) part[q][j / 2] = y[q];
          }
          // the block's 16 columns of S are read: its P takes them
#pragma unroll
          for (int q = 0; q < PP; ++q) tmem_put8(srow + 16 * c + 8 * q, part[q]);
        });
      };
      if (wide) {
        l += key_weights<PP>(X, st, hf, wide, srow, seen64(), qs, mr, rest);
      } else if (masked) weights(True{});
      else weights(False{});
      const float2 sum2 = unpack2(add2(sum[0], sum[1]));
      l += sum2.x + sum2.y;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&X.p_full[buf]);
      buf += ntl;
      if (buf >= 3) buf -= 3, sph ^= 1u;
    }
    if (n_mine > 0) {
      wait(&X.t_full[qt], (uint32_t)(n - 1) & 1u, X, p.err);
      tc_fence_after();
      add_tile();
    }

    // ---------------------------------------------------------------- output
    const bool row_in = tl < ntok && work && !(ps >= 0 && seg < 0);  // rows left out write nothing
    float of[DH];
#pragma unroll
    for (int d = 0; d < DH; d += 2) {
      const float2 x = unpack2(o[d / 2]);
      of[d] = live ? x.x : 0.f, of[d + 1] = live ? x.y : 0.f;
    }
    if (!live) m = -INFINITY, l = 0.f;
    bool bad = size >= kFarScore;
    if constexpr (BF) {
#pragma unroll
      for (int d = 0; d < DH; ++d) bad |= !(fabsf(of[d]) <= 3.402823466e38f);
    }
    pair_bar();
    X.pair[0][hf][rr] = make_float2(l, bad ? 1.f : 0.f);
    pair_bar();
    const float2 other = X.pair[0][hf ^ 1][rr];
    l = hf ? other.x + l : l + other.x;
    // The split's partial (relative to m) into shared memory, in the place of Q and K, which
    // all products are done with: rows of D + 4 floats, so that rows 8 apart share a bank.
    wait(&X.done, 0u, X, p.err);
    float* po = reinterpret_cast<float*>(smem) + rr * kPitch + hf * DH;
    if (row_in && live && (bad || other.y != 0.f)) {
      const Seg sg = X.segs[seg];
      const int end = sg.first + seen_range<kKeys>(sg.hi, sg.lo, sg.sinks).n;
      const float2 y = plain_row<FMT, D>(p, sg, max(tbeg, sg.first) - sg.first, min(tend, end) - sg.first, t0 + tl, head, g, ps,
                                         hf * DH, po);
      m = y.x, l = y.y;
    } else {
#pragma unroll
      for (int d = 0; d < DH; d += 4) *reinterpret_cast<float4*>(po + d) = make_float4(of[d], of[d + 1], of[d + 2], of[d + 3]);
    }
    if (hf == 0) X.ml[rr] = make_float2(m, l);
    tc_fence_before();
    __syncthreads();
  }
  if (warp == H::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, H::kCols);
  }
  // The splits of a tile are one cluster: each takes a share of the rows, sums the partials
  // in split order out of the others' shared memory, and writes them out.
  const int C = p.splits;
  if (C > 1) {
    cluster_arrive();
    cluster_wait();
  }
  const int rows_in = ntok * G, r0 = rows_in * split_i / C, r1 = rows_in * (split_i + 1) / C;
  for (int e = tid; e < (r1 - r0) * (D / 8); e += H::kThreads) {
    const int x = r0 + e / (D / 8), d = e % (D / 8) * 8, tt = x / G, hh = x - tt * G;
    const int rr = tt < TT ? x : kRows + x - TT * G;  // its row of the CTA
    if (X.pos[tt] >= 0) {  // a row that was left out
      bool in = false;
      for (int s = 0; s < X.nseg; ++s) in |= X.segs[s].row == X.row[tt];
      if (!in) continue;
    }
    float mx = -INFINITY;
    for (int w = 0; w < nsplit; ++w) mx = fmaxf(mx, peer(&X.ml[rr].x, w, C));
    float ll = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < nsplit; ++w) {
      const float mw = peer(&X.ml[rr].x, w, C), lw = peer(&X.ml[rr].y, w, C);
      // a partial without keys (maximum -inf, sum 0) has nothing to add; a NaN sum stays one
      const float f = mw == -INFINITY ? (lw == 0.f ? 0.f : 1.f) : ex2(mw - mx);
      ll = fmaf(f, lw, ll);
      const float* po = reinterpret_cast<const float*>(smem) + rr * kPitch + d;
      const float4 a = peer4(po, w, C), b = peer4(po + 4, w, C);
      v[0] = fmaf(f, a.x, v[0]), v[1] = fmaf(f, a.y, v[1]), v[2] = fmaf(f, a.z, v[2]), v[3] = fmaf(f, a.w, v[3]);
      v[4] = fmaf(f, b.x, v[4]), v[5] = fmaf(f, b.y, v[5]), v[6] = fmaf(f, b.z, v[6]), v[7] = fmaf(f, b.w, v[7]);
    }
    const float inv = ll != 0.f ? 1.f / ll : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= inv;
    emit<8>(p, t0 + tt, (g * G + hh) * D + d, width, v);
  }
  if (C > 1) {  // the others are done with this CTA's shared memory
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
}

template <int FMT, int D, int QP, int PP>
cudaError_t launch(const CacheAttnParams& p, cudaStream_t s, bool pdl) {
  using H = Shape<FMT, D, QP>;
  auto kernel = prompt_kernel<FMT, D, QP, PP>;
  constexpr int smem = H::kOffMisc + kMiscBytes;
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  cudaError_t e = set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  // the warpgroups' register counts are made for this launch size
  static const cudaError_t regs = [&] {
    cudaFuncAttributes a;
    const cudaError_t r = cudaFuncGetAttributes(&a, reinterpret_cast<const void*>(kernel));
    return r != cudaSuccess ? r : a.numRegs < H::kRegLaunch ? cudaErrorInvalidConfiguration : cudaSuccess;
  }();
  if (regs != cudaSuccess) return regs;
  const int CT = H::kTiles * (kRows / p.group);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.M + CT - 1) / CT * p.splits), p.c.kv_heads, 1);
  cfg.blockDim = dim3(H::kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (pdl) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.splits > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = (unsigned)p.splits;
    attr[na].val.clusterDim.y = 1;
    attr[na++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int FMT, int D>
cudaError_t launch_parts(const CacheAttnParams& p, cudaStream_t s, bool pdl) {
  if (p.dtype == QI_F32) return launch<FMT, D, 2, 2>(p, s, pdl);
  return p.dtype == QI_F16 ? launch<FMT, D, 1, 2>(p, s, pdl) : launch<FMT, D, 1, 1>(p, s, pdl);
}

template <int D>
cudaError_t launch_dim(const CacheAttnParams& p, cudaStream_t s, bool pdl) {
  if (p.c.format == QI_KV_INT8) return launch_parts<QI_KV_INT8, D>(p, s, pdl);
  if (p.c.format == QI_KV_E4M3) return launch_parts<QI_KV_E4M3, D>(p, s, pdl);
  return launch_parts<QI_KV_BF16, D>(p, s, pdl);
}

}  // namespace

int prompt_clusters(int size) {
  static std::atomic<int> known[kMaxDevices][9];  // 0: not yet queried
  const int guess = sm_count() / size;
  int dev = 0;
  if (size < 2 || size > 8 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    (void)cudaGetLastError();
    return guess;
  }
  int n = known[dev][size].load(std::memory_order_relaxed);
  if (n > 0) return n;
  // one CTA on an SM in every variant; this one stands for all
  using H = Shape<QI_KV_BF16, 128, 1>;
  auto kernel = prompt_kernel<QI_KV_BF16, 128, 1, 1>;
  constexpr int smem = H::kOffMisc + kMiscBytes;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)size, 1, 1);
  cfg.blockDim = dim3(H::kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    return guess;
  }
  known[dev][size].store(n, std::memory_order_relaxed);
  return n;
}

cudaError_t launch_cache_attention_prompt(const CacheAttnParams& p, cudaStream_t s, bool pdl) {
  return p.c.head_dim == 64 ? launch_dim<64>(p, s, pdl) : launch_dim<128>(p, s, pdl);
}

}  // namespace qi

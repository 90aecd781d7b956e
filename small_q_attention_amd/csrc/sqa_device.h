// Device code that the kernels of several files share: element types, the MFMA page
// steps, the walk of a work item over its pages, the way results leave. The layouts
// these rest on are described at the top of sqa_kernels.hip.
#pragma once

#include "sqa_internal.h"

#include <math.h>

namespace sqa {
namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));

// Element types of Q, K, V and the output. Operands travel as raw 16-bit
// lanes (u4 = 8 elements, u2 = 4); the traits pick the MFMA and the rounding.
struct ElemF16 {
  // Split partials leave as fp16 rows normalised by their sum (a convex
  // combination of V rows, so within V's fp16 range), with (max, sum) in fp32:
  // half the partial bytes written and merged.
  static constexpr bool kHalfPartials = true;
  // S^T += K . Q^T over 32 head dims.
  static __device__ __forceinline__ f4 mma_qk(u4 k, u4 q, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, k),
                                                  __builtin_bit_cast(h8, q), c, 0, 0, 0);
  }
  // O^T += V^T . P^T over 16 tokens; P is one fp16 operand (relative error
  // 2^-11), with no low part.
  static __device__ __forceinline__ f4 mma_pv(u2 v, u2 p, u2 /*lo*/, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4, v),
                                                 __builtin_bit_cast(h4, p), c, 0, 0, 0);
  }
  // Rounds four probabilities once; adds the rounded values to l (v_dot2
  // against ones) so O stays an exact convex combination.
  static __device__ __forceinline__ u2 round_p(float p0, float p1, float p2, float p3, float& l,
                                               u2& /*lo*/) {
    const h2 ones = {(_Float16)1.0f, (_Float16)1.0f};
    const h2 lo = {(_Float16)p0, (_Float16)p1};
    const h2 hi = {(_Float16)p2, (_Float16)p3};
    l = __builtin_amdgcn_fdot2(hi, ones, __builtin_amdgcn_fdot2(lo, ones, l, false), false);
    return __builtin_bit_cast(u2, h4{lo[0], lo[1], hi[0], hi[1]});
  }
  static __device__ __forceinline__ u4 pack8(const float (&x)[8]) {
    h8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (_Float16)x[i];
    return __builtin_bit_cast(u4, o);
  }
  static __device__ __forceinline__ unsigned pack2(float x, float y) {
    return __builtin_bit_cast(unsigned, h2{(_Float16)x, (_Float16)y});
  }
  static __device__ __forceinline__ u2 pack4(const float (&x)[4]) {
    return __builtin_bit_cast(u2, h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2],
                                     (_Float16)x[3]});
  }
  static __device__ __forceinline__ unsigned short pack1(float x) {
    return __builtin_bit_cast(unsigned short, (_Float16)x);
  }
  // Four OCP e4m3 values (bytes of w, low first) -> four fp16 (exact).
  static __device__ __forceinline__ u2 widen_fp8x4(unsigned w) {
    return u2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))};
  }
  // Eight OCP e4m3 values (bytes of w, low first) -> eight fp16 (exact).
  static __device__ __forceinline__ u4 widen_fp8(u2 w) {
    return u4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], 1.f, false)),
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], 1.f, true)),
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], 1.f, false)),
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], 1.f, true))};
  }
};

// fp16 queries and outputs whose split partials stay unnormalised fp32.
struct ElemF16Wide : ElemF16 {
  static constexpr bool kHalfPartials = false;
};

struct ElemBF16 {
  // bf16 V can exceed fp16's range and bf16's 8 bits would cost accuracy:
  // partials stay unnormalised fp32.
  static constexpr bool kHalfPartials = false;
  // One bf16 P (relative error 2^-9) would cost up to ~1% on rows that average
  // a few keys; P goes in as hi + lo bf16 parts (~2^-17), both in one PV
  // product.
  static __device__ __forceinline__ f4 mma_qk(u4 k, u4 q, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, k),
                                                   __builtin_bit_cast(b8, q), c, 0, 0, 0);
  }
  // O^T += V^T . (P_hi + P_lo)^T in one 16x16x32 MFMA (on gfx950 as many
  // cycles as the 16x16x16 one): k-slots 0-3 of a lane group take its four
  // tokens with P_hi, slots 4-7 the same tokens with P_lo, so every operand is
  // already in the lane (bf16 q16: 395 -> 358 us against two 16x16x16
  // products).
  static __device__ __forceinline__ f4 mma_pv(u2 v, u2 hi, u2 lo, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(b8, u4{v[0], v[1], v[0], v[1]}),
        __builtin_bit_cast(b8, u4{hi[0], hi[1], lo[0], lo[1]}), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u2 round_p(float p0, float p1, float p2, float p3, float& l,
                                               u2& lo) {
    const b4 hi = {(__bf16)p0, (__bf16)p1, (__bf16)p2, (__bf16)p3};
    const float h0 = (float)hi[0], h1 = (float)hi[1], h2v = (float)hi[2], h3 = (float)hi[3];
    const b4 lw = {(__bf16)(p0 - h0), (__bf16)(p1 - h1), (__bf16)(p2 - h2v), (__bf16)(p3 - h3)};
    // The row sum takes p itself: hi + lo is within 2^-17 of p, and summing p
    // saves the conversions back (bf16 q16: 363 -> 350 us).
    l += (p0 + p1) + (p2 + p3);
    lo = __builtin_bit_cast(u2, lw);
    return __builtin_bit_cast(u2, hi);
  }
  static __device__ __forceinline__ u4 pack8(const float (&x)[8]) {
    b8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (__bf16)x[i];
    return __builtin_bit_cast(u4, o);
  }
  static __device__ __forceinline__ unsigned pack2(float x, float y) {
    typedef __bf16 bb2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, bb2{(__bf16)x, (__bf16)y});
  }
  static __device__ __forceinline__ u2 pack4(const float (&x)[4]) {
    return __builtin_bit_cast(u2, b4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]});
  }
  static __device__ __forceinline__ unsigned short pack1(float x) {
    return __builtin_bit_cast(unsigned short, (__bf16)x);
  }
  static __device__ __forceinline__ u2 widen_fp8x4(unsigned w) {
    return u2{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))};
  }
  static __device__ __forceinline__ u4 widen_fp8(u2 w) {
    return u4{__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], 1.f, false)),
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], 1.f, true)),
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], 1.f, false)),
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], 1.f, true))};
  }
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Split partials leave as write-through stores (relaxed agent-scope atomics:
// global_store with sc1, which the XCD's L2 passes on to memory) rather than
// write-back ones: the merge kernel reads them from other XCDs anyway, and
// dirty lines left in the L2s would be written back at the end of the partial
// kernel, before the merge kernel can start (stamped on one box: the merge
// began 1.6 us after the last partial workgroup at 2 MB of partials, 4.5 us at
// 8 MB). Whole calls back to back: one sequence of 32K keys, q_len 8, 34.6 ->
// 31.8 us; 4 x 8K, q_len 4, 30.6 -> 29.7 us; 16 x 32K +-0.7 us.
__device__ __forceinline__ void store_through(void* p, unsigned long long x) {
  __hip_atomic_store((unsigned long long*)p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// x of the lower and the upper of two 16-lane rows (kOff 16: rows 0 and 1, and 2
// and 3) or of two 32-lane halves (kOff 32), each in all of their lanes: one
// v_permlane swap of x with itself, no LDS permute.
struct LanePair {
  float lo, hi;
};
template <int kOff>
__device__ __forceinline__ LanePair lane_pair(float x) {
  static_assert(kOff == 16 || kOff == 32, "rows or halves of a wave");
  const unsigned v = __builtin_bit_cast(unsigned, x);
  unsigned lo, hi;
  if constexpr (kOff == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    lo = r[0];
    hi = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    lo = r[0];
    hi = r[1];
  }
  return {__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}

__device__ __forceinline__ float xor_max(float x) {
  const LanePair a = lane_pair<16>(x);
  const LanePair b = lane_pair<32>(fmaxf(a.lo, a.hi));
  return fmaxf(b.lo, b.hi);
}

__device__ __forceinline__ float xor_sum(float x) {
  const LanePair a = lane_pair<16>(x);
  const LanePair b = lane_pair<32>(a.lo + a.hi);
  return b.lo + b.hi;
}

// Buffer-resource word 3 for gfx9-family raw (untyped, 32-bit) accesses.
constexpr int kBufferFlags = 0x00020000;
// Cache-policy operand of the K/V buffer loads: non-temporal (read once).
constexpr int kStreamAux = 2;
// Cache-policy operand of the partials' buffer stores: device scope (sc1), a
// write-through store, as store_through.
constexpr int kThroughAux = 16;
// A buffer-store offset past every bounded resource here (their sizes stay
// below it): the hardware drops such a store.
constexpr unsigned kDroppedOffset = 0xFFFFFFF0u;

// Per-lane shapes for head dim HD (64, 128 or 256): KK = HD/32 K fragments of
// 8 dims, MB = HD/16 output dim blocks, VW = HD/32 dwords of V per token (HD/16
// dims of one token in 16-bit elements), each lane owning HD/4 output dims.
template <int HD>
struct Dims {
  static constexpr int KK = HD / 32;
  static constexpr int MB = HD / 16;
  static constexpr int VW = HD / 32;
};

// K/V storage. Per page a lane holds K for token l%16 and V for tokens
// 4*(l/16) + 0..3, dims (HD/16)*(l%16) + 0..HD/16-1. The head dims of K
// fragment kk are q_dims(kk, l/16) + 0..7 (Q is loaded with the same map, so
// the QK contraction is unchanged); V and the output mapping are the same for
// every storage type. expand_k() / expand_v() hand the MFMAs 16-bit elements.

template <int HD>
struct KvNative {  // the query's 16-bit type
  static constexpr int kBytes = 2;
  static constexpr int KK = Dims<HD>::KK, VW = Dims<HD>::VW;
  static constexpr int kLoads = KK + 4 * (VW > 4 ? VW / 4 : 1);  // instructions per page
  // One 16-byte load per fragment: dims 32*kk + 8*g.
  static __device__ __forceinline__ int q_dims(int kk, int g) { return 32 * kk + 8 * g; }
  static __device__ __forceinline__ unsigned k_lane_bytes(int g) { return 16 * g; }
  static __device__ __forceinline__ unsigned v_lane_bytes(int l16) { return 4 * VW * l16; }
  struct Regs {
    u4 k[KK];
    unsigned v[4][VW];
  };
  static __device__ __forceinline__ void load(Regs& r, __amdgpu_buffer_rsrc_t kr,
                                              __amdgpu_buffer_rsrc_t vr, unsigned k_lane,
                                              unsigned v_lane, unsigned tok) {
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      r.k[kk] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_lane + 64 * kk, 0, kStreamAux);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (VW == 2) {
        const u2 x = __builtin_amdgcn_raw_buffer_load_b64(vr, v_lane, e * tok, kStreamAux);
        r.v[e][0] = x[0];
        r.v[e][1] = x[1];
      } else {
#pragma unroll
        for (int h = 0; h < VW / 4; ++h) {
          const u4 x = __builtin_amdgcn_raw_buffer_load_b128(vr, v_lane + 16 * h, e * tok,
                                                             kStreamAux);
#pragma unroll
          for (int i = 0; i < 4; ++i) r.v[e][4 * h + i] = x[i];
        }
      }
    }
  }
  template <typename E>
  static __device__ __forceinline__ void expand_k(const Regs& r, u4 (&k)[KK]) {
#pragma unroll
    for (int i = 0; i < KK; ++i) k[i] = r.k[i];
  }
  template <typename E>
  static __device__ __forceinline__ void expand_v(const Regs& r, unsigned (&v)[4][VW]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < VW; ++i) v[e][i] = r.v[e][i];
  }
};

template <int HD>
struct KvFp8 {  // OCP e4m3 bytes, widened exactly to the query's type
  static constexpr int kBytes = 1;
  static constexpr int KK = Dims<HD>::KK, VW = Dims<HD>::VW;
  static constexpr int kLoads = KK / 2 + 4;  // instructions per page
  // K rows are HD bytes: 16-byte loads per lane (64 bytes of a row per
  // instruction, as for the 16-bit types; 8-byte loads used 32 bytes per row
  // request and ran at 58% of peak instead of 78%). Load i holds dims
  // 64*i + 16*g + 0..15, i.e. fragments kk = 2i, 2i+1.
  static __device__ __forceinline__ int q_dims(int kk, int g) {
    return 64 * (kk >> 1) + 16 * g + 8 * (kk & 1);
  }
  static __device__ __forceinline__ unsigned k_lane_bytes(int g) { return 16 * g; }
  static __device__ __forceinline__ unsigned v_lane_bytes(int l16) { return 2 * VW * l16; }
  struct Regs {
    u4 k[KK / 2];
    unsigned v[4][VW / 2];  // HD/16 e4m3 bytes per token
  };
  static __device__ __forceinline__ void load(Regs& r, __amdgpu_buffer_rsrc_t kr,
                                              __amdgpu_buffer_rsrc_t vr, unsigned k_lane,
                                              unsigned v_lane, unsigned tok) {
#pragma unroll
    for (int i = 0; i < KK / 2; ++i)
      r.k[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_lane + 64 * i, 0, kStreamAux);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (VW == 2) {
        r.v[e][0] = __builtin_amdgcn_raw_buffer_load_b32(vr, v_lane, e * tok, kStreamAux);
      } else if constexpr (VW == 4) {
        const u2 x = __builtin_amdgcn_raw_buffer_load_b64(vr, v_lane, e * tok, kStreamAux);
        r.v[e][0] = x[0];
        r.v[e][1] = x[1];
      } else {
        const u4 x = __builtin_amdgcn_raw_buffer_load_b128(vr, v_lane, e * tok, kStreamAux);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[e][i] = x[i];
      }
    }
  }
  template <typename E>
  static __device__ __forceinline__ void expand_k(const Regs& r, u4 (&k)[KK]) {
#pragma unroll
    for (int i = 0; i < KK / 2; ++i) {
      k[2 * i] = E::widen_fp8(u2{r.k[i][0], r.k[i][1]});
      k[2 * i + 1] = E::widen_fp8(u2{r.k[i][2], r.k[i][3]});
    }
  }
  template <typename E>
  static __device__ __forceinline__ void expand_v(const Regs& r, unsigned (&v)[4][VW]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < VW / 2; ++i) {
        const u2 w = E::widen_fp8x4(r.v[e][i]);
        v[e][2 * i] = w[0];
        v[e][2 * i + 1] = w[1];
      }
  }
};

template <int NB, int HD>
struct WaveState {
  f4 acc[Dims<HD>::MB][NB];  // O^T blocks: lane l holds dims (HD/4)*(l/16)+(HD/16)*r+mb of row 16*nb+l%16
  float m[NB];     // reference max (log2 units, within kMaxLag of the true row max), same in all 4 lane groups
  float l[NB];     // partial row sum over this lane's tokens
  // Kept with m by the page-pair steps (pair_finish): m + kMaxLag, and the
  // exponent offset -(m, or 0 while m is -inf).
  float thr[NB];
  float nmu[NB];
};

// Padding of the LDS page-id table beyond the split's last page: covers the
// ring's look-ahead (at most 2 * D + 1 entries past the end).
constexpr int kIdPad = 64;

__device__ __forceinline__ int clamp_page(int pid, long long num_pages) {
  return (pid >= 0 && (long long)pid < num_pages) ? pid : 0;
}

// The running row max may trail the true max by up to this many log2 units
// (probabilities up to 2^8 = 256, still exact to fp16 precision in P and far
// from any fp32 range limit in the sums). Rows only pay for the cross-lane max
// and the accumulator rescale when a new score exceeds the running max by
// more than this, which after the first page is rare.
constexpr float kMaxLag = 8.0f;

// max(a, b, c) as one v_maximum3_f32 (IEEE maximum: a NaN operand gives NaN).
// fmaxf (maxnum) makes the compiler quiet every operand it cannot prove
// canonical, MFMA results among them, with an extra v_max_f32 x, x, x first,
// which doubled the instructions of the per-page score maxima. The two agree
// except where a score is NaN, and such a score's row is NaN either way (its
// probability enters the row's sums). Invisible tokens are masked to -inf
// before any maximum is taken.
__device__ __forceinline__ float max3_raw(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
__device__ __forceinline__ float max4(f4 v) { return max3_raw(max3_raw(v[0], v[1], v[2]), v[3], v[3]); }

// Bytes {a.lo16, b.lo16} and {a.hi16, b.hi16} of two dwords (v_perm_b32).
__device__ __forceinline__ unsigned pack_lo(unsigned a, unsigned b) {
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ unsigned pack_hi(unsigned a, unsigned b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// One 16-token page for one wave, in two steps: page_scores() runs the QK
// products, page_finish() masks, updates the softmax state and runs the PV
// products. The pipelined loop issues the next page's scores before this
// page's finish, so those MFMAs run under the softmax.
// sm_q: Q fragments in LDS, [nb][kk][lane] (the B-operand layout).
// HPW = 2 with NB = 1 (one 16-row block, rows 0-7 of kv head 0 of the wave
// and rows 8-15 of head 1): the QK and PV products run once per head over all
// 16 rows; each lane keeps the scores of its own row's head (`upper`: row >=
// 8), and each head's PV product gets the probabilities of its own rows only,
// so both land in the one set of accumulators. HPW = 2 with NB = 2 or 4:
// blocks nb of head nb / (NB / 2) take only that head's K and V.
// A page's K and V widened to the MFMAs' 16-bit type (a register copy for
// 16-bit caches).
template <int HD, int HPW>
struct PageK {
  u4 k[HPW][Dims<HD>::KK];
};
template <int HD, int HPW>
struct PageV {
  unsigned v[HPW][4][Dims<HD>::VW];
};

template <typename E, typename KV, int HD, int HPW>
__device__ __forceinline__ PageK<HD, HPW> widen_k(const typename KV::Regs (&raw)[HPW]) {
  PageK<HD, HPW> kf;
#pragma unroll
  for (int h = 0; h < HPW; ++h) KV::template expand_k<E>(raw[h], kf.k[h]);
  return kf;
}
template <typename E, typename KV, int HD, int HPW>
__device__ __forceinline__ PageV<HD, HPW> widen_v(const typename KV::Regs (&raw)[HPW]) {
  PageV<HD, HPW> pv;
#pragma unroll
  for (int h = 0; h < HPW; ++h) KV::template expand_v<E>(raw[h], pv.v[h]);
  return pv;
}

template <int NB, int HD, typename E, typename KV, int HPW>
__device__ __forceinline__ void page_scores(f4 (&s)[NB], const PageK<HD, HPW>& kf,
                                            const u4* sm_q, int lane, bool upper) {
  constexpr int KK = Dims<HD>::KK;
  static_assert(HPW == 1 || NB <= 4, "two heads per wave: one shared block or NB / 2 each");
  // Raw scores S^T[token][row] = K . Q^T for this page.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    s[nb] = f4{0.f, 0.f, 0.f, 0.f};
    f4 s1 = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const u4 qf = sm_q[(nb * KK + kk) * 64 + lane];
      if constexpr (HPW == 2 && NB >= 2) {
        s[nb] = E::mma_qk(kf.k[nb / (NB / 2)][kk], qf, s[nb]);  // head nb / (NB / 2)
      } else {
        s[nb] = E::mma_qk(kf.k[0][kk], qf, s[nb]);
        if constexpr (HPW == 2) s1 = E::mma_qk(kf.k[HPW - 1][kk], qf, s1);
      }
    }
    if constexpr (HPW == 2 && NB == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nb][e] = upper ? s1[e] : s[nb][e];
    }
  }
}

// c = softmax scale * log2(e); scores stay raw until the exponent, where the
// scale and the running max meet in one FMA. Visibility on masked pages: token
// t < len is seen by a row when it lies before the draft block
// (t < draft_base = len - q_len) or when bit t - draft_base of the row's draft
// bits is set.
// Scores of tokens a row does not see set to -inf; tok0 = absolute index of
// this lane's first token (4 consecutive tokens).
template <int NB>
__device__ __forceinline__ void mask_scores(f4 (&s)[NB], const unsigned long long (&dbits)[NB],
                                            int draft_base, int tok0, int len) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // Bitwise, not short-circuit, logic: one select per score, no
      // lane-divergent control flow around the scores.
      const int t = tok0 + e;
      const int j = t - draft_base;  // < q_len <= 64 whenever t < len
      const unsigned bit = (unsigned)(dbits[nb] >> (j & 63)) & 1u;
      const unsigned seen = (unsigned)(t < len) & ((unsigned)(j < 0) | bit);
      s[nb][e] = seen ? s[nb][e] : -INFINITY;
    }
  }
}

// Masked pages: scores of tokens a row does not see become -inf, and V rows
// past the sequence end may hold anything (even NaN; 0 * NaN would poison the
// product), so they are zeroed.
template <int NB, int HD, int HPW>
__device__ __forceinline__ void mask_page(f4 (&s)[NB], PageV<HD, HPW>& pv,
                                          const unsigned long long (&dbits)[NB], int draft_base,
                                          int tok0, int len) {
  constexpr int VW = Dims<HD>::VW;
  mask_scores<NB>(s, dbits, draft_base, tok0, len);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (tok0 + e >= len) {
#pragma unroll
      for (int h = 0; h < HPW; ++h)
#pragma unroll
        for (int i = 0; i < VW; ++i) pv.v[h][e][i] = 0u;
    }
  }
}

// The running max: lm[nb] holds this lane's max of its new scores (times c); the
// row max is only reduced across the four 16-lane groups when some lane runs
// ahead of its running max.
template <int NB, int HD>
__device__ __forceinline__ void raise_max(WaveState<NB, HD>& st, const float (&lm)[NB]) {
  constexpr int MB = Dims<HD>::MB;
  bool grow = false;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) grow |= lm[nb] > st.m[nb] + kMaxLag;
  if (__any(grow)) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float mn = fmaxf(st.m[nb], xor_max(lm[nb]));
      const float alpha = fast_exp2(st.m[nb] - (mn == -INFINITY ? 0.f : mn));
      st.m[nb] = mn;
      st.l[nb] *= alpha;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) st.acc[mb][nb] *= alpha;
    }
  }
}

// One page's probabilities against the running max and its PV products.
template <int NB, int HD, typename E, typename KV, int HPW>
__device__ __forceinline__ void page_pv(WaveState<NB, HD>& st, const f4 (&s)[NB],
                                        const PageV<HD, HPW>& pv, bool upper, float c) {
  constexpr int MB = Dims<HD>::MB;
  // P = 2^(c*s - m), rounded once to the element type; with fp16 the row sum
  // is taken over the rounded values so O is an exact convex combination (with
  // bf16, P is hi + lo and the sum is within 2^-17 of it).
  u2 ph[NB], pl[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float mu = st.m[nb] == -INFINITY ? 0.f : st.m[nb];
    pl[nb] = u2{0u, 0u};  // stays zero where P has no low part
    ph[nb] = E::round_p(fast_exp2(fmaf(s[nb][0], c, -mu)), fast_exp2(fmaf(s[nb][1], c, -mu)),
                        fast_exp2(fmaf(s[nb][2], c, -mu)), fast_exp2(fmaf(s[nb][3], c, -mu)),
                        st.l[nb], pl[nb]);
  }

  // O^T += V^T . P^T, one 16x16x16 MFMA per (dim block, row block, head). Dim
  // block mb takes half mb%2 of dword mb/2 from the four token rows this lane
  // holds.
  const u2 zero = {0u, 0u};
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    const int j = mb >> 1;
#pragma unroll
    for (int h = 0; h < HPW; ++h) {
      const unsigned w0 = pv.v[h][0][j], w1 = pv.v[h][1][j], w2 = pv.v[h][2][j],
                     w3 = pv.v[h][3][j];
      const u2 av = (mb & 1) == 0 ? u2{pack_lo(w0, w1), pack_lo(w2, w3)}
                                  : u2{pack_hi(w0, w1), pack_hi(w2, w3)};
      // With two heads, head h's product takes only the probabilities of its
      // own rows (the other rows' lanes pass zeros).
      const bool mine = HPW == 1 || NB >= 2 || (h == 1) == upper;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (HPW == 2 && NB >= 2 && h != nb / (NB / 2)) continue;  // its own head's V only
        st.acc[mb][nb] =
            E::mma_pv(av, mine ? ph[nb] : zero, mine ? pl[nb] : zero, st.acc[mb][nb]);
      }
    }
  }
}

// bits.get(dbits): the draft bits of the lane's rows, asked for on masked pages only.
template <int NB, int HD, typename E, typename KV, int HPW, typename Bits>
__device__ __forceinline__ void page_finish(WaveState<NB, HD>& st, f4 (&s)[NB],
                                            PageV<HD, HPW>& pv, bool upper, const Bits& bits,
                                            int draft_base, int tok0, int len, bool masked,
                                            float c) {
  if (masked) {
    unsigned long long dbits[NB];
    bits.get(dbits);
    mask_page<NB, HD, HPW>(s, pv, dbits, draft_base, tok0, len);
  }
  float lm[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) lm[nb] = max4(s[nb]) * c;
  raise_max<NB, HD>(st, lm);
  page_pv<NB, HD, E, KV, HPW>(st, s, pv, upper, c);
}

// threadIdx.x through an empty asm statement: what a piece of work, or a rare branch
// of one, derives from it is computed there, not hoisted by the compiler in front of
// the loop over pieces, where it would hold registers through every page loop.
__device__ __forceinline__ int piece_tid() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// Two pages in one softmax step: fp16 queries over an e4m3 cache at head dim
// 128, one kv head per wave (the 64-row kernel, where the math, not the bytes,
// sets the time). s0 / s1: the raw scores of pages p and p + 1; r0 / r1 their
// raw K/V registers. One running-max update covers the 32 tokens, and each PV
// product is one v_mfma_f32_16x16x32_f16 over both pages (k-slots 0-3 of a lane
// group take its four tokens of page p, slots 4-7 the same tokens of page
// p + 1), which costs the cycles of one 16x16x16 product over one page: half
// the PV MFMA time. V is widened per dim block from its bytes, after the bytes
// of tokens past the sequence end are zeroed (they may hold NaN). have1 false:
// page p + 1 is past the piece (its slot holds a zero page); its scores become
// -inf. Same sums as two page_finish steps up to fp32 rounding and the point
// at which the lagging max is raised.
template <int NB, typename Bits>
__device__ __forceinline__ void pair_finish(WaveState<NB, 128>& st, f4 (&s0)[NB], f4 (&s1)[NB],
                                            KvFp8<128>::Regs r0, KvFp8<128>::Regs r1,
                                            bool have1, const Bits& bits, int draft_base,
                                            int tok_base, int len, bool masked, float c) {
  using E = ElemF16;
  constexpr int MB = Dims<128>::MB;
  // Both conditions are uniform over the wave and rare (pages at the draft
  // block or the sequence end; the last pair of a piece of odd length): one
  // branch keeps their selects out of the common step.
  if (masked || !have1) {
    if (masked) {
      unsigned long long dbits[NB];
      bits.get(dbits);
      const int tok0 = tok_base + 4 * ((piece_tid() & 63) >> 4);
      mask_scores<NB>(s0, dbits, draft_base, tok0, len);
      mask_scores<NB>(s1, dbits, draft_base, tok0 + kPageSize, len);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (tok0 + e >= len) r0.v[e][0] = r0.v[e][1] = 0u;
        if (tok0 + kPageSize + e >= len) r1.v[e][0] = r1.v[e][1] = 0u;
      }
    }
    if (!have1) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s1[nb] = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    }
  }

  // The step is VALU-bound (fp8 widening, 32 exponentials per lane): the
  // pair's maxima as four v_maximum3 (no operand quieting), and the threshold and
  // exponent offset kept with the running max instead of recomputed per step
  // (cfg3 shape q16: 214.0 -> 205.0 us, bit-identical).
  float lm[NB];
  bool grow = false;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    lm[nb] = max3_raw(max3_raw(s0[nb][0], s0[nb][1], s0[nb][2]),
                      max3_raw(s0[nb][3], s1[nb][0], s1[nb][1]),
                      max3_raw(s1[nb][2], s1[nb][3], s1[nb][3])) * c;
    grow |= lm[nb] > st.thr[nb];
  }
  if (__any(grow)) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float mn = fmaxf(st.m[nb], xor_max(lm[nb]));
      const float alpha = fast_exp2(st.m[nb] - (mn == -INFINITY ? 0.f : mn));
      st.m[nb] = mn;
      st.thr[nb] = mn + kMaxLag;
      st.nmu[nb] = -(mn == -INFINITY ? 0.f : mn);
      st.l[nb] *= alpha;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) st.acc[mb][nb] *= alpha;
    }
  }

  u4 pp[NB];  // P^T of both pages: this lane's 4 tokens of page p, then of p + 1
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float nmu = st.nmu[nb];
    u2 unused;
    const u2 a0 = E::round_p(fast_exp2(fmaf(s0[nb][0], c, nmu)), fast_exp2(fmaf(s0[nb][1], c, nmu)),
                             fast_exp2(fmaf(s0[nb][2], c, nmu)), fast_exp2(fmaf(s0[nb][3], c, nmu)),
                             st.l[nb], unused);
    const u2 a1 = E::round_p(fast_exp2(fmaf(s1[nb][0], c, nmu)), fast_exp2(fmaf(s1[nb][1], c, nmu)),
                             fast_exp2(fmaf(s1[nb][2], c, nmu)), fast_exp2(fmaf(s1[nb][3], c, nmu)),
                             st.l[nb], unused);
    pp[nb] = u4{a0[0], a0[1], a1[0], a1[1]};
  }

  // Dim block mb = 2 j + h takes byte 2 (j % 2) + h of the lane's e4m3 dword
  // j / 2 from each of its four token rows of each page. The
  // bytes of token rows 2i and 2i + 1 are interleaved first (one v_perm_b32:
  // {t0 b, t1 b, t0 b+1, t1 b+1}), so each fp8 -> fp16 conversion of a 16-bit
  // word yields the MFMA operand dword itself (tokens 2i, 2i + 1 at one dim):
  // 8 conversions and 4 permutes per j instead of 8 conversions and 8 permutes
  // (widen each token row, then pair the rows' halves). Same values, same bits.
  const unsigned sel = 0x05010400u;  // bytes {t0.b0, t1.b0, t0.b1, t1.b1}; + 0x02020202: b2, b3
#pragma unroll
  for (int j = 0; j < MB / 2; ++j) {
    const unsigned sj = (j & 1) ? sel + 0x02020202u : sel;
    const int d = j >> 1;
    const unsigned x[4] = {__builtin_amdgcn_perm(r0.v[1][d], r0.v[0][d], sj),
                           __builtin_amdgcn_perm(r0.v[3][d], r0.v[2][d], sj),
                           __builtin_amdgcn_perm(r1.v[1][d], r1.v[0][d], sj),
                           __builtin_amdgcn_perm(r1.v[3][d], r1.v[2][d], sj)};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int mb = 2 * j + h;
      u4 av;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        av[i] = __builtin_bit_cast(
            unsigned, h == 0 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i], 1.f, false)
                             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i], 1.f, true));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        st.acc[mb][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            __builtin_bit_cast(h8, av), __builtin_bit_cast(h8, pp[nb]), st.acc[mb][nb], 0, 0, 0);
    }
  }
}

// The page range one workgroup owns and where its sequence's result goes.
struct ItemRange {
  int b;        // sequence (-1: no work item for this workgroup)
  int split;    // split index within the sequence
  int p_begin;  // first page (logical index within the sequence)
  int p_end;    // one past the last page
  int len;      // seq_lens[b], clamped to >= 0
  int n_valid;  // splits of this sequence that own pages: 0, 1 or more (then 2)
  int slot0;    // partial slot of split 0 of this sequence
  int g_end;    // balanced plan: where the piece ends along the item's pages
  int paired;   // a paired item of the expected-page plan (its loop time is timed)
};

// A value every lane needs from memory no workgroup of the call writes, at an
// address the same in every lane: read through the scalar cache into a scalar
// register (the compiler picks the vector path for plain loads here: it cannot see
// that nothing writes there), without a place in the vector loads' order.
__device__ __forceinline__ int scalar_load(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*)p;
}

// Fixed plan: sequence b owns slots b * num_splits + s.
__device__ __forceinline__ ItemRange fixed_item(const PartialArgs& a, int item) {
  ItemRange r;
  r.b = item / a.by_splits;
  r.split = item - r.b * a.num_splits;
  r.p_begin = r.split * a.pages_per_split;
  r.len = max(scalar_load(a.seq_lens + r.b), 0);
  const int pages = min((r.len + kPageSize - 1) / kPageSize, a.max_pages);
  r.p_end = min(r.p_begin + a.pages_per_split, pages);
  r.n_valid = min(pages > a.pages_per_split ? 2 : (int)(pages > 0), a.num_splits);
  r.slot0 = r.b * a.num_splits;
  r.g_end = 0;
  r.paired = 0;
  return r;
}

// Inclusive prefix sum over the wave's 64 lanes with DPP: within rows of 16
// lanes by shifts of 1, 2, 4 and 8 (lanes past the row start add 0), then each
// row's total broadcast into the rows after it (lane 15 into rows 1 and 3, lane
// 31 into rows 2 and 3). Six VALU operations instead of six LDS permutes.
__device__ __forceinline__ int wave_inclusive_scan_int(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// Balanced plan (batch <= kMaxBalancedBatch = 4 x 64), packed: num_splits =
// T + batch slots, T = the work items one wave of resident workgroups holds. The
// pages of all sequences, concatenated in batch order (sequence b's pages start
// at start_b, the sum of the page counts before it), are cut into items of
// P = ceil(total / T) pages (clamped to [kMinSplitPages, kMaxSplitPages]):
// item i is global pages [i P, min((i + 1) P, total)), whatever the lengths,
// so every workgroup streams the same number of pages and none waits for a
// second wave. An item visits each sequence it overlaps as a piece, with its own
// softmax state, rows and partial slot i + b (unique: walking the pages in
// order, each next piece has the next item or the next sequence and neither
// index ever falls, so i + b grows strictly). Sequence b thus owns slots
// [i0_b + b, i1_b + b], i0_b = start_b / P, i1_b = (start_b + pages_b - 1) / P;
// a sequence inside one item is finished by the partial kernel. In a ragged
// batch the positions include the seam gaps (start_b then counts the gaps
// before sequence b too; an item may end inside a gap). Lane l holds
// sequences l, l + 64, l + 128, l + 192: every wave derives the plan on its own
// with wave reductions (no LDS, no barrier), and wave 0 of workgroup 0 writes
// each sequence's (first slot, count) for the merge kernel.
constexpr int kSeqPerLane = kMaxBalancedBatch / 64;

// The per-lane view of the batch a packed plan works from (lane l: sequences
// l + 64 k). Page counts are recomputed from the lengths where needed, which
// keeps the view at two registers per sequence slot: it stays live through the
// item's pieces.
struct PackedBatch {
  int start[kSeqPerLane];  // first global page of each sequence
  int len[kSeqPerLane];    // lengths (0 past the batch)
  int P;                   // pages per item
  int total;               // pages of the batch
};

// A workgroup's view of the balanced plan: its head group's slot count, merge
// table and item size, and whether it writes that table (the first workgroup of
// the call, or with items per head group the first of its group).
struct PlanView {
  int num_splits;
  SeqSplits* table;
  int spec_pps;
  bool writer;
};
__device__ __forceinline__ PlanView plan_view(const PartialArgs& a) {
  return PlanView{a.num_splits, a.seq_splits, a.spec_pps, blockIdx.x == 0};
}
__device__ __forceinline__ PlanView plan_view(const PartialArgs& a, const HeadGroupItems& h) {
  return PlanView{h.slots, a.seq_splits + h.group * a.batch, h.spec_pps, h.item == 0};
}

// Kernel pages of a sequence of `len` tokens within a block-table row.
__device__ __forceinline__ int pages_of(const PartialArgs& a, int len) {
  return min((len + kPageSize - 1) / kPageSize, a.max_pages);
}

// Prefix sums of the page counts and the item size; with write_table, the
// merge kernel's table.
__device__ __forceinline__ void packed_plan(const PartialArgs& a, const PlanView& v,
                                            PackedBatch& pb, bool write_table) {
  const int lane = threadIdx.x & 63;
  // Groups of 64 sequences past the batch hold no pages: their scans are skipped
  // (a uniform branch), and a group's sum is the last lane of its scan.
  const int groups = (a.batch + 63) / 64;
  int base = 0;  // pages of the groups of 64 sequences before this one
  int pages[kSeqPerLane];
#pragma unroll
  for (int k = 0; k < kSeqPerLane; ++k) {
    pages[k] = pages_of(a, pb.len[k]);
    pb.start[k] = base;
    if (k < groups) {
      const int incl = wave_inclusive_scan_int(pages[k]);
      pb.start[k] += incl - pages[k];
      base += __builtin_amdgcn_readlane(incl, 63);
    }
  }
  // Wave sums are the same in every lane; readfirstlane says so to the
  // compiler, which keeps the loop over pieces (and the page ids loaded in it)
  // uniform rather than wrapping each buffer load in a waterfall loop.
  pb.total = __builtin_amdgcn_readfirstlane(base);
  const int target = v.num_splits - a.batch;
  pb.P = packed_item_pages(pb.total, target);
  // Seams (ragged batches): seam_pages of nothing before every sequence start
  // that is not on an item boundary of the layout without them, so an item that
  // spans the start carries fewer pages; skipped where the gaps would need
  // items over kMaxSplitPages pages, or items are too short for them to matter.
  const int first_pages = __builtin_amdgcn_readfirstlane(pages[0]);
  bool ragged = false;
#pragma unroll
  for (int k = 0; k < kSeqPerLane; ++k) ragged |= 64 * k + lane < a.batch && pages[k] != first_pages;
  const int seam = a.seam_pages;
  if (seam > 0 && pb.P >= 4 * seam && __any(ragged)) {  // uniform
    int gap_base = 0;
    int vstart[kSeqPerLane];
#pragma unroll
    for (int k = 0; k < kSeqPerLane; ++k) {
      vstart[k] = pb.start[k] + gap_base;
      if (k < groups) {
        const int gap = pages[k] > 0 && pb.start[k] % pb.P != 0 ? seam : 0;
        const int incl = wave_inclusive_scan_int(gap);
        vstart[k] += incl;
        gap_base += __builtin_amdgcn_readlane(incl, 63);
      }
    }
    const int total = pb.total + __builtin_amdgcn_readfirstlane(gap_base);
    if (total <= target * kMaxSplitPages) {  // uniform
#pragma unroll
      for (int k = 0; k < kSeqPerLane; ++k) pb.start[k] = vstart[k];
      pb.total = total;
      pb.P = packed_item_pages(total, target);
    }
  }
  if (write_table && threadIdx.x < 64) {
#pragma unroll
    for (int k = 0; k < kSeqPerLane; ++k) {
      const int sq = 64 * k + lane;
      if (sq < a.batch) {
        const int i0 = pb.start[k] / pb.P;
        const int count = pages[k] > 0 ? (pb.start[k] + pages[k] - 1) / pb.P - i0 + 1 : 0;
        v.table[sq] = SeqSplits{min(i0 + sq, v.num_splits - 1), count};
      }
    }
  }
}

// The piece of item `item` from position g on (g inside the item): the first
// sequence with pages that end after g (the one holding g, or the next one if g
// lies in the gap before a sequence start), its page range (within the
// sequence), length, split count and slot, and where the piece ends. The wave
// finds the lane holding that sequence with one ballot per sequence slot;
// everything after is scalar.
__device__ __forceinline__ ItemRange packed_piece(const PartialArgs& a, const PackedBatch& pb,
                                                 int item, int g, int item_end) {
  int b = -1, st = 0, len = 0;
#pragma unroll
  for (int k = 0; k < kSeqPerLane; ++k) {
    // Lengths are 0 past the batch: those slots have no pages.
    const int np = pages_of(a, pb.len[k]);
    const bool mine = np > 0 && g < pb.start[k] + np;
    const unsigned long long hit = __ballot(mine);
    if (hit && b < 0) {
      const int src = __builtin_ctzll(hit);
      b = 64 * k + src;
      st = __builtin_amdgcn_readlane(pb.start[k], src);  // src is uniform
      len = __builtin_amdgcn_readlane(pb.len[k], src);
    }
  }
  ItemRange r;
  const int np = pages_of(a, len);
  const int g_end = min(item_end, pb.total);
  r.b = b;
  r.split = 0;
  r.len = len;
  r.p_begin = max(g - st, 0);
  r.p_end = min(g_end, st + np) - st;  // <= p_begin: the item ends in the gap
  // One split: the sequence lies within this item.
  r.n_valid = st >= item * pb.P && st + np <= (item + 1) * pb.P ? 1 : 2;
  r.slot0 = item + b;
  r.g_end = st + r.p_end;
  r.paired = 0;
  return r;
}

// Lengths of sequences l, l + 64, l + 128, l + 192 in lane l (0 past the
// batch). The loads are unconditional, from clamped in-bounds addresses, and
// selected afterwards: a load under a branch is waited for where the branch
// joins, which would put a full memory round trip in front of whatever follows.
__device__ __forceinline__ void load_lengths(const PartialArgs& a, int (&len)[kSeqPerLane]) {
  const int lane = threadIdx.x & 63;
  int raw[kSeqPerLane];
#pragma unroll
  for (int k = 0; k < kSeqPerLane; ++k) raw[k] = a.seq_lens[min(64 * k + lane, a.batch - 1)];
#pragma unroll
  for (int k = 0; k < kSeqPerLane; ++k) len[k] = 64 * k + lane < a.batch ? max(raw[k], 0) : 0;
}

// The rows of a wave: row slot r (0..15) of 16-row block nb is row row(nb, r)
// (= qi * group + g) of kv head head(nb, r), real() unless it is padding (past
// the rows of a head, or a head past the last). One kv head per wave (HPW = 1):
// blocks nb hold rows 16 nb + r. Two (HPW = 2, head dim 64): one shared block,
// rows 0-7 of the first head in slots 0-7 and of the second in 8-15, or NB / 2
// blocks per head.
template <int NB, int HPW>
struct WaveRows {
  int kvh, rows, hkv;  // the wave's first kv head; rows per kv head; kv heads
  static constexpr int kBlocksPerHead = NB >= 2 ? NB / HPW : 1;
  __device__ __forceinline__ int head(int nb, int r) const {
    return kvh + (HPW == 1 ? 0 : (NB == 1 ? r >> 3 : nb / kBlocksPerHead));
  }
  __device__ __forceinline__ int row(int nb, int r) const {
    return HPW == 1 ? nb * 16 + r : (NB == 1 ? (r & 7) : (nb % kBlocksPerHead) * 16 + r);
  }
  __device__ __forceinline__ bool real(int nb, int r) const {
    return head(nb, r) < hkv && row(nb, r) < rows;
  }
};

// The same in every lane (readfirstlane tells the compiler): the piece, and the
// buffer-resource addresses built from it, stay in scalar registers.
__device__ __forceinline__ void make_uniform(ItemRange& it) {
  it.b = __builtin_amdgcn_readfirstlane(it.b);
  it.split = __builtin_amdgcn_readfirstlane(it.split);
  it.p_begin = __builtin_amdgcn_readfirstlane(it.p_begin);
  it.p_end = __builtin_amdgcn_readfirstlane(it.p_end);
  it.len = __builtin_amdgcn_readfirstlane(it.len);
  it.n_valid = __builtin_amdgcn_readfirstlane(it.n_valid);
  it.slot0 = __builtin_amdgcn_readfirstlane(it.slot0);
  it.g_end = __builtin_amdgcn_readfirstlane(it.g_end);
}

// A work item on its way through its pieces: a fixed plan has one (g 0, g_end 1),
// a balanced item the pieces packed_piece() finds from global page g to g_end.
struct ItemWalk {
  PackedBatch pb;
  ItemRange it;     // the current piece
  int g_end;        // balanced: where the item's pages end
  int item_end;     // balanced: where the item ends
  bool paired;      // the item runs as a paired item
};

template <int D>
__device__ __forceinline__ void load_first_ids(const PartialArgs& a, int seq, int p0,
                                               int (&first_id)[D]) {
  const int32_t* row = a.block_tables + (size_t)max(seq, 0) * a.bt_stride;
#pragma unroll
  for (int j = 0; j < D; ++j)
    first_id[j] = scalar_load(row + (min(max(p0 + j, 0), a.max_pages - 1) >> a.page_shift));
}

// A balanced item's piece from global page g on; false if the item has none there.
// A piece has a sequence and at least one page unless the item ends in the gap
// before a sequence start (no further pieces then); the check also keeps every
// walk finite whatever the inputs.
__device__ __forceinline__ bool piece_at(const PartialArgs& a, ItemWalk& w, int item, int g) {
  if (g >= w.g_end) return false;  // uniform
  w.it = packed_piece(a, w.pb, item, g, w.item_end);
  make_uniform(w.it);
  w.it.paired = w.paired;
  return w.it.b >= 0 && w.it.p_end > w.it.p_begin;
}

// Finds the first piece of workgroup item `item` and loads the ids of its first D
// pages (index clamped into the block-table row; ids past the piece are never
// used); false if the item has no piece. Fixed plan: one piece whose page range
// follows from `item` alone, so its ids are issued before the sequence length is
// read and both arrive in one round trip. Balanced plan: all lengths, the packed
// plan's wave reductions, then the ids; with an expected page count (every
// sequence spec_pages pages, item size spec_pps from the host) the plan needs no
// lengths, so the ids go out with them, and a length that does not match falls
// back to the plan from the loaded lengths.
// kPairs: paired items may be asked for; kBalanced: the plan is a balanced one.
template <int D, bool kPairs, bool kBalanced>
__device__ __forceinline__ bool first_piece(const PartialArgs& a, const PlanView& v, int item,
                                            ItemWalk& w, int (&first_id)[D]) {
  const int lane = threadIdx.x & 63;
  PackedBatch& pb = w.pb;
  w.paired = false;
  if constexpr (!kBalanced) {
    const int seq = item / a.by_splits;
    load_first_ids<D>(a, seq, (item - seq * a.num_splits) * a.pages_per_split, first_id);
    w.it = fixed_item(a, item);
    make_uniform(w.it);
    w.item_end = 1;
    w.g_end = 1;
    return w.it.b >= 0;
  } else {
  bool ids_loaded = false;
  int g = 0;
  if (a.spec_pages > 0) {
    // Every sequence spec_pages pages: sequence b starts at b * spec_pages;
    // the item size comes from the host. The first piece's ids go out with
    // the lengths (index clamped: an item past the batch never uses them).
    const int P = a.spec_pages;
#pragma unroll
    for (int k = 0; k < kSeqPerLane; ++k) pb.start[k] = min(64 * k + lane, a.batch) * P;
    pb.total = a.batch * P;
    pb.P = v.spec_pps;
    if (v.writer && threadIdx.x < 64) {
#pragma unroll
      for (int k = 0; k < kSeqPerLane; ++k) {
        const int sq = 64 * k + lane;
        if (sq < a.batch) {
          const int i0 = pb.start[k] / pb.P;
          v.table[sq] = SeqSplits{i0 + sq, (pb.start[k] + P - 1) / pb.P - i0 + 1};
        }
      }
    }
    // Paired items: the shared boundary of items 2k and 2k + 1 moves by d
    // pages; delta is the fixed one, or (adaptive pairs) the record's, read
    // with the lengths, the first ids after.
    w.paired = kPairs && a.pair_items != 0;
    int g0 = item * pb.P;
    w.item_end = g0 + pb.P;
    if (w.paired) {
      float dl = kPairDeltaFixed;
      if (a.pair_items == kPairsAdaptive) {
        const float2 rec = *(const float2*)a.tune;
        dl = __float_as_uint(rec.x) == kTuneMagic ? rec.y : 0.f;
      }
      load_lengths(a, pb.len);
      dl = dl == dl ? fminf(fmaxf(dl, -kPairDeltaMax), kPairDeltaMax) : 0.f;
      // Both items of a pair stay within kMaxSplitPages (the page-id table).
      const int dmax = kMaxSplitPages - pb.P;
      const int d = __builtin_amdgcn_readfirstlane(
          min(max((int)rintf((float)pb.P * dl), -dmax), dmax));
      g0 = (item >> 1) * 2 * pb.P + ((item & 1) ? pb.P + d : 0);
      w.item_end = (item >> 1) * 2 * pb.P + ((item & 1) ? 2 * pb.P : pb.P + d);
    }
    g0 = __builtin_amdgcn_readfirstlane(g0);
    const int b0 = min(g0 / a.by_spec_pages, a.batch - 1);
    load_first_ids<D>(a, b0, g0 - b0 * P, first_id);
    if (!w.paired) load_lengths(a, pb.len);
    bool differs = false;
#pragma unroll
    for (int k = 0; k < kSeqPerLane; ++k)
      differs |= 64 * k + lane < a.batch && pages_of(a, pb.len[k]) != P;
    if (__any(differs)) {
      packed_plan(a, v, pb, v.writer);  // rewrites the table
      w.paired = false;
    } else {
      ids_loaded = true;
    }
    if (w.paired) g = g0;
  } else {
    load_lengths(a, pb.len);
    packed_plan(a, v, pb, v.writer);
  }
  if (!w.paired) {
    g = item * pb.P;
    w.item_end = g + pb.P;
  }
  g = __builtin_amdgcn_readfirstlane(g);
  w.g_end = __builtin_amdgcn_readfirstlane(min(w.item_end, pb.total));
  if (!piece_at(a, w, item, g)) return false;  // uniform
  if (!ids_loaded) load_first_ids<D>(a, w.it.b, w.it.p_begin, first_id);
  return true;
  }
}

// Runs `piece(range, first_id)` for every piece of workgroup item `item`.
// Consecutive pieces are separated by a barrier (they reuse the workgroup's LDS).
// Returns whether the item ran as a paired item (every workgroup of a call
// returns the same).
template <int D, bool kBalanced, typename Piece>
__device__ __forceinline__ bool for_each_piece(const PartialArgs& a, const PlanView& v, int item,
                                               Piece&& piece) {
  int first_id[D];
  ItemWalk w;
  bool more = first_piece<D, true, kBalanced>(a, v, item, w, first_id);
  while (more) {  // uniform
    piece(w.it, first_id);
    more = kBalanced && piece_at(a, w, item, w.it.g_end);
    if (more) {
      load_first_ids<D>(a, w.it.b, w.it.p_begin, first_id);
      __syncthreads();  // the previous piece is done with the LDS
    }
  }
  return w.paired;
}

// Draft bits of a row of sequence b, draft row qi: bit j = the row sees draft
// token j (the caller's mask, or the causal chain j <= qi); 0 for padding rows.
// Both mask words are loaded unconditionally (without a mask: from seq_lens,
// never used) and selected by bit masks, not by branches on loaded values, so
// the compiler need not wait for them before later loads are issued.
__device__ __forceinline__ unsigned long long draft_bits(const PartialArgs& a, int b, int qi,
                                                         bool real) {
  const bool has_mask = a.draft_mask != nullptr;
  const uint32_t* mp = has_mask ? a.draft_mask + (size_t)(b * a.q_len + qi) * a.mask_words
                                : (const uint32_t*)a.seq_lens;
  const unsigned long long lo = mp[0];
  const unsigned long long hi = mp[a.mask_words > 1 ? 1 : 0];
  const unsigned long long causal = qi >= 63 ? ~0ull : (2ull << qi) - 1ull;
  const unsigned long long use_mask = 0ull - (unsigned long long)(has_mask && real);
  const unsigned long long use_hi = 0ull - (unsigned long long)(a.mask_words > 1);
  const unsigned long long use_causal = 0ull - (unsigned long long)(!has_mask && real);
  return ((lo | ((hi << 32) & use_hi)) & use_mask) | (causal & use_causal);
}

// Leaves one wave's results: normalised rows of the output (`direct`: the
// sequence's pages fit one split) or the unnormalised partial sums and (max in
// log2 units, sum) of each row at partial slot `slot`. Row slot r of block nb is
// map.real(nb, r), kv head map.head(nb, r), row map.row(nb, r) of that head.
// `mark_done` (a fixed plan with several splits, finished here) also writes
// l = -1 at the slot, which tells the merge kernel the row is in the output.
// The results leave through LDS one 16-row block at a time: every lane writes
// its dims (HD/4) (l/16) + (HD/16) rr + mb of row l % 16 row-major into the
// wave's `stage` (16 rows of HD + 4 floats; the pad spreads rows over banks),
// then reads back 4 contiguous values of a row, so a store instruction writes
// whole rows (1 KiB runs of partial sums) instead of 64 scattered 16-byte
// pieces, which ran at a quarter of the store rate (the epilogue of a 64-row
// wave took 5 us).
template <int NB, int HD, typename E, typename Map>
__device__ __forceinline__ void write_results(const PartialArgs& a, WaveState<NB, HD>& st,
                                              float* stage, const Map& map, bool direct,
                                              bool mark_done, int b, size_t slot,
                                              int slot_heads, int head0) {
  constexpr int MB = Dims<HD>::MB;
  constexpr int kStageRow = HD + 4;  // floats per staged row
  constexpr int CPR = HD / 4;        // 4-value chunks per row
  const int lane = piece_tid() & 63;
  const int g16 = lane >> 4, l16 = lane & 15;
  // Partial slots of slot_heads kv heads from head0 on: all of them (hkv, 0), or
  // with items per head group the group's four (4, 4 group; slot counts from
  // the start of the group's region).
  auto item_of = [&](int nb, int r) {
    return (slot * slot_heads + map.head(nb, r) - head0) * a.rows;
  };
  // Row sums over the four lane groups.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) st.l[nb] = xor_sum(st.l[nb]);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    if (map.row(nb, 0) >= a.rows) break;  // uniform
    // l = 0: the row saw no key (written as 0). A NaN l (a NaN score or
    // probability the row saw) passes, so the NaN reaches the row's output.
    const float inv_l = !(st.l[nb] <= 0.f) ? 1.f / st.l[nb] : 0.f;
    const float sc = direct ? a.out_scale * inv_l : (E::kHalfPartials ? inv_l : 1.f);
    if (map.real(nb, l16)) {
      float* dst = stage + l16 * kStageRow + (HD / 4) * g16;
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
#pragma unroll
        for (int h = 0; h < MB / 4; ++h) {
          f4 o;
#pragma unroll
          for (int mb = 0; mb < 4; ++mb) o[mb] = st.acc[4 * h + mb][nb][rr] * sc;
          *(f4*)(dst + MB * rr + 4 * h) = o;
        }
      }
    }
    // The staging rows are this wave's own: LDS keeps a wave's accesses in
    // order, the fences keep the compiler from moving them. All reads are
    // issued before the first store, so the block pays one LDS latency.
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    if (direct) {
      f4 v[CPR / 4];
#pragma unroll
      for (int i = 0; i < CPR / 4; ++i) {
        const int e = i * 64 + lane;  // row e / CPR (< 16), chunk e % CPR
        v[i] = *(const f4*)(stage + (e / CPR) * kStageRow + 4 * (e % CPR));
      }
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      if (mark_done && g16 == 0 && map.real(nb, l16)) {
        const size_t pitem = item_of(nb, l16) + map.row(nb, l16);
        a.part_ml[pitem * 2 + 0] = -INFINITY;
        a.part_ml[pitem * 2 + 1] = -1.f;
      }
#pragma unroll
      for (int i = 0; i < CPR / 4; ++i) {
        const int e = i * 64 + lane;
        const int rs = e / CPR;
        if (map.real(nb, rs)) {
          const int r = map.row(nb, rs);
          const int qi = r / a.by_group;
          const int gg = r - qi * a.group;
          _Float16* op = a.out + ((size_t)(b * a.q_len + qi) * a.hq +
                                  map.head(nb, rs) * a.group + gg) * HD + 4 * (e % CPR);
          const float o[4] = {v[i][0], v[i][1], v[i][2], v[i][3]};
          *(u2*)op = E::pack4(o);
        }
      }
    } else {
      // Partial rows: 16 bytes per lane (8 fp16 or 4 fp32 values), each store
      // a write-through buffer store (sc1) through a resource bounded to the
      // partials, with padding rows sent past its end, where the hardware drops
      // them: no branch per store, and half the store instructions of 8-byte
      // stores, whose issue took 0.9 us per 16-row block (stamped; whole calls
      // back to back: 16 x 32K keys q_len 8 320.9 -> 319.5 us, 16 x 8K 89.8 ->
      // 88.8 us, one sequence of 8K keys q_len 8 19.3 -> 18.8 us).
      constexpr int DPL = E::kHalfPartials ? 8 : 4;  // values per lane and store
      constexpr int PPR = HD / DPL;                   // 16-byte pieces per row
      constexpr int esz = E::kHalfPartials ? 2 : 4;
      f4 w[PPR / 4][DPL / 4];
#pragma unroll
      for (int i = 0; i < PPR / 4; ++i) {
        const int e = i * 64 + lane;  // row e / PPR (< 16), piece e % PPR
#pragma unroll
        for (int h = 0; h < DPL / 4; ++h)
          w[i][h] = *(const f4*)(stage + (e / PPR) * kStageRow + DPL * (e % PPR) + 4 * h);
      }
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
          (void*)a.part_o, (short)0, (int)a.part_o_bytes, kBufferFlags);
#pragma unroll
      for (int i = 0; i < PPR / 4; ++i) {
        const int e = i * 64 + lane;
        const int rs = e / PPR;
        const unsigned at =
            (unsigned)(((item_of(nb, rs) + map.row(nb, rs)) * HD + DPL * (e % PPR)) * esz);
        const unsigned off = map.real(nb, rs) ? at : kDroppedOffset;
        u4 data;
        if constexpr (E::kHalfPartials) {
          const float o[8] = {w[i][0][0], w[i][0][1], w[i][0][2], w[i][0][3],
                              w[i][1][0], w[i][1][1], w[i][1][2], w[i][1][3]};
          data = E::pack8(o);
        } else {
          data = __builtin_bit_cast(u4, w[i][0]);
        }
        __builtin_amdgcn_raw_buffer_store_b128(data, pr, off, 0, kThroughAux);
      }
      if (g16 == 0 && map.real(nb, l16)) {
        const size_t pitem = item_of(nb, l16) + map.row(nb, l16);
        // A NaN sum travels with a finite max, so the merge counts the split.
        const float m_out = st.l[nb] == st.l[nb] ? st.m[nb] : 0.f;
        store_through(a.part_ml + pitem * 2,
                      __builtin_bit_cast(unsigned long long, float2{m_out, st.l[nb]}));
      }
    }
  }
}

// A fixed-plan split past its sequence's pages (the balanced plan has none):
// the merge reads every split of a sequence without its length, so the split's
// rows say "no keys" (l = 0), or, when the sequence fitted one split and is
// already in the output, "done" (l = -1).
template <int NB, typename Map>
__device__ __forceinline__ void write_empty_split(const PartialArgs& a, const Map& map,
                                                  size_t slot, float mark) {
  const int lane = piece_tid() & 63;
  if ((lane >> 4) != 0) return;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    if (map.real(nb, lane)) {
      const size_t pitem = (slot * a.hkv + map.head(nb, lane)) * a.rows + map.row(nb, lane);
      a.part_ml[pitem * 2 + 0] = -INFINITY;
      a.part_ml[pitem * 2 + 1] = mark;
    }
  }
}

// s_waitcnt vmcnt(n) that no memory access is moved across.
template <int N>
__device__ __forceinline__ void wait_vmcnt_fence() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N < 63 ? N : 63) : "memory");
}

// One load per lane straight into LDS (gfx950 global_load_lds_*): lane l's 16 (or
// 4) bytes land at LDS byte address lds + 16 l (4 l). Inline asm for the reason
// given at load_to_lds: the compiler's wait-count pass must not drain the page
// ring for it. The callers wait themselves (wait_vmcnt_fence). The s_nop is the wait
// state the hardware asks for between a scalar write of m0 and a load into LDS, which
// the compiler's hazard pass does not put into inline asm.
__device__ __forceinline__ void copy16_to_lds(const void* src, unsigned lds) {
  unsigned saved;
  asm volatile(
      "s_mov_b32 %[saved], m0\n\t"
      "s_mov_b32 m0, %[lds]\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %[src], off\n\t"
      "s_mov_b32 m0, %[saved]"
      : [saved] "=&s"(saved)
      : [lds] "s"(lds), [src] "v"(src)
      : "memory");
}
__device__ __forceinline__ void copy4_to_lds(const void* src, unsigned lds) {
  unsigned saved;
  asm volatile(
      "s_mov_b32 %[saved], m0\n\t"
      "s_mov_b32 m0, %[lds]\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %[src], off\n\t"
      "s_mov_b32 m0, %[saved]"
      : [saved] "=&s"(saved)
      : [lds] "s"(lds), [src] "v"(src)
      : "memory");
}

// Draft bits held in registers (loaded with draft_bits()).
template <int NB>
struct RegBits {
  unsigned long long b[NB];
  __device__ __forceinline__ void get(unsigned long long (&dbits)[NB]) const {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) dbits[nb] = b[nb];
  }
};

// Draft bits of a wave's rows: the caller's mask words, copied to LDS with the
// piece's Q (block nb's row r: word w at 32 nb + 16 w + r), or the causal chain.
// Padding rows get some row's bits; they are never stored. FIND: get() finds the
// lane for itself. The e4m3 64-row kernel needs that: held through its page loop, the
// lane and what follows from it took a pair of ring registers, whose copies waited for
// a load just issued (16 x 32K keys, q_len 16, per call: 212.8 against 193.0 us). At
// 32 rows the branch around it costs the pipelined loop its overlap (e4m3 q_len 8
// 172.4 -> 195.3 us).
template <int NB, int HPW, bool FIND>
struct StagedBits {
  const unsigned* words;
  bool masked;            // the caller's words; else the causal chain
  bool two;               // two words per row
  FastDiv by_group;
  int lane16;
  WaveRows<NB, HPW> map;
  __device__ __forceinline__ void get(unsigned long long (&dbits)[NB]) const {
    const int l16 = FIND ? piece_tid() & 15 : lane16;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if (masked) {  // uniform
        dbits[nb] = words[32 * nb + l16];
        if (two) dbits[nb] |= (unsigned long long)words[32 * nb + 16 + l16] << 32;
      } else {
        const int qi = map.row(nb, l16) / by_group;
        dbits[nb] = qi >= 63 ? ~0ull : (2ull << qi) - 1ull;
      }
    }
  }
};

}  // namespace
}  // namespace sqa

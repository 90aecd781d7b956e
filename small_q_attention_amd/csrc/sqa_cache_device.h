// Device code of the kernels around the paged cache: the cut of a batch of sequences into
// work items, and the codes of 8-bit caches as they are written and as the products take
// them.
#pragma once

#include "sqa_device.h"

#include <type_traits>

namespace sqa {
namespace {

// A split of one sequence.
struct Split {
  int b, len;          // sequence and its length
  int p_begin, p_end;  // kernel pages
  int count;           // splits of the sequence
  int slot;            // its work item, and partial slot
  int first;           // work item of the sequence's first split
};

__device__ __forceinline__ int wave_sum_int(int x) {
  return __builtin_amdgcn_readlane(wave_inclusive_scan_int(x), 63);
}

// ceil(n / d) for 0 <= n < 2^27, 0 < d, by the reciprocal: the first estimate is off by a
// few at most, the second by one. A dozen instructions; a division by a run-time value is
// three times that, and a wave's way to its first load had up to ten.
__device__ __forceinline__ int ceil_quotient(int n, int d, float inv) {
  int q = (int)((float)n * inv);
  q += (int)((float)(n - q * d) * inv);
  int r = n - q * d;
  q -= r < 0 ? 1 : 0;
  r += r < 0 ? d : 0;
  return q + (r > 0 ? 1 : 0) + (r > d ? 1 : 0);
}

// The cut of the batch into work items, found by every wave for itself from the lengths:
// sequence b takes n_b = max(1, ceil(pages_b / P)) items of nearly equal size, with P the
// smallest page count of at least kMinSplitPages for which they sum to at most `items`
// (or P the longest sequence, one item each, where the batch has as many sequences as
// that or more). Up to there all items are resident at once, and the longest, P pages,
// sets the time. Items do not cross sequence ends, so a batch near the number of items
// leaves some of the chip idle, and one past it is not cut at all: attention, e4m3, 8 kv
// heads (128 items), q_len 4, 8K keys each, whole calls beside those of the e4m3 kernel with
// one scale per tensor, whose items do cross: 64 sequences 177 and 172 us, 65 289 and 176,
// 100 316 and 265, 128 344 and 333, 129 593 and 336; 100 of 1K to 16K 474 and 309.
// Returns whether item `item` exists; `table` (one wave of the grid) also receives each
// sequence's first item and count for the merge kernel. ONE: at most 64 sequences, one
// per lane, whose page counts stay in a register.
template <bool ONE>
__device__ __forceinline__ bool find_split_of(const PartialArgs& a, int items, int item,
                                              SeqSplits* table, Split& out) {
  const int lane = threadIdx.x & 63;
  const int groups = ONE ? 1 : (a.batch + 63) / 64;
  auto length_of = [&](int k) {
    const int i = 64 * k + lane;
    return i < a.batch ? max(a.seq_lens[i], 0) : 0;
  };
  const int len0 = length_of(0);
  auto len_at = [&](int k) { return ONE || k == 0 ? len0 : length_of(k); };
  auto pages_at = [&](int k) {  // unsigned: a length may be the largest there is
    return min((int)(((unsigned)len_at(k) + kPageSize - 1) / kPageSize), a.max_pages);
  };
  auto splits_of = [&](int k, int P, float inv) {
    return 64 * k + lane < a.batch ? max(ceil_quotient(pages_at(k), P, inv), 1) : 0;
  };
  int total = 0;
  for (int k = 0; k < groups; ++k) total += wave_sum_int(pages_at(k));
  auto fits = [&](int P) {
    const float inv = __builtin_amdgcn_rcpf((float)P);
    int n = 0;
    for (int k = 0; k < groups; ++k) n += wave_sum_int(splits_of(k, P, inv));
    return n <= items;
  };
  int P = max(kMinSplitPages, (total + items - 1) / a.by_splits);  // by_splits: items
  if (!fits(P)) {
    // ceil(pages_b / P) sum to at most total / P + batch.
    int lo = P, hi = items > a.batch ? max(P, (total + items - a.batch - 1) / (items - a.batch))
                                     : max(a.max_pages, 1);
    while (lo + 1 < hi) {  // lo does not fit, hi does (or is one item each)
      const int mid = lo + (hi - lo) / 2;
      if (fits(mid))
        hi = mid;
      else
        lo = mid;
    }
    P = hi;
  }
  const float inv = __builtin_amdgcn_rcpf((float)P);
  int base = 0;
  bool found = false;
  for (int k = 0; k < groups; ++k) {
    const int n = splits_of(k, P, inv);
    const int incl = wave_inclusive_scan_int(n);
    const int first = base + incl - n;
    if (table != nullptr && 64 * k + lane < a.batch) table[64 * k + lane] = SeqSplits{first, n};
    const unsigned long long hit = __ballot(item >= first && item < first + n);
    if (hit && !found) {
      const int src = __builtin_ctzll(hit);
      const int pages = __builtin_amdgcn_readlane(pages_at(k), src);
      out.b = 64 * k + src;
      out.len = __builtin_amdgcn_readlane(len_at(k), src);
      out.count = __builtin_amdgcn_readlane(n, src);
      out.slot = item;
      out.first = __builtin_amdgcn_readlane(first, src);
      const int size = __builtin_amdgcn_readfirstlane(
          ceil_quotient(pages, out.count, __builtin_amdgcn_rcpf((float)out.count)));
      out.p_begin = (item - out.first) * size;
      out.p_end = min(out.p_begin + size, pages);
      found = true;
      if (table == nullptr) return true;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return found;
}
__device__ __forceinline__ bool find_split(const PartialArgs& a, int items, int item,
                                           SeqSplits* table, Split& out) {
  return a.batch <= 64 ? find_split_of<true>(a, items, item, table, out)
                       : find_split_of<false>(a, items, item, table, out);
}

// x / s for many x, rounded as the division is. With r = 1/s rounded to nearest, two
// corrections q += r (x - q s), the remainders exact in an fma, leave the quotient
// correctly rounded (Markstein's division) while nothing under- or overflows: s within
// 2^+-100, as all but freak scales are, and x no larger than 448 s (a remainder of an x so
// small that it underflows belongs to a quotient far below the smallest code). Five
// operations in place of the division's dozen.
struct Quotient {
  float s, r;
  bool fast;
};
__device__ __forceinline__ Quotient quotient(float s) {
  return {s, 1.f / s, s >= 0x1p-100f && s <= 0x1p100f};
}
__device__ __forceinline__ float divide_fast(float x, const Quotient& d) {
  // The remainder as -(q s - x): so written, -0 / s stays -0.
  float q = x * d.r;
  q = fmaf(-fmaf(q, d.s, -x), d.r, q);
  return fmaf(-fmaf(q, d.s, -x), d.r, q);
}

// Four values in units of the scale -> four codes (bytes, low first). e4m3: no magnitude
// exceeds 448 by more than a rounding of the quotient, which rounds to 448.
template <bool INT8>
__device__ __forceinline__ unsigned encode4(const float (&y)[4]) {
  if constexpr (INT8) {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float r = fminf(fmaxf(rintf(y[i] == y[i] ? y[i] : 0.f), -127.f), 127.f);
      w |= ((unsigned)(int)r & 0xffu) << (8 * i);
    }
    return w;
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  }
}

template <bool INT8>
__device__ __forceinline__ float decode(unsigned w, int i) {
  if constexpr (INT8) {
    return (float)(signed char)(w >> (8 * i));
  } else {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return i < 2 ? lo[i] : hi[i - 2];
  }
}

// V of a page as the PV product's A operand: av[mb] = this lane's dim mb of its four
// tokens in fp16, which holds every e4m3 value and every 8-bit integer exactly.
template <int HD>
struct CodesFp8 : KvFp8<HD> {
  using Regs = typename KvFp8<HD>::Regs;
  static constexpr int MB = Dims<HD>::MB, VW = Dims<HD>::VW;
  static constexpr bool kNan = true;  // codes may be NaN
  static __device__ __forceinline__ void operand_v(const Regs& r, u2 (&av)[MB]) {
#pragma unroll
    for (int i = 0; i < VW / 2; ++i) {
      // Bytes of two token rows interleaved, so that a conversion yields two tokens of
      // one dim.
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const unsigned sel = half ? 0x07030602u : 0x05010400u;
        const unsigned t01 = __builtin_amdgcn_perm(r.v[1][i], r.v[0][i], sel);
        const unsigned t23 = __builtin_amdgcn_perm(r.v[3][i], r.v[2][i], sel);
        const u2 a = ElemF16::widen_fp8x4(t01), b = ElemF16::widen_fp8x4(t23);
        av[4 * i + 2 * half] = u2{a[0], b[0]};
        av[4 * i + 2 * half + 1] = u2{a[1], b[1]};
      }
    }
  }
};

template <int HD>
struct CodesInt8 : KvFp8<HD> {
  using Regs = typename KvFp8<HD>::Regs;
  static constexpr int KK = Dims<HD>::KK, MB = Dims<HD>::MB, VW = Dims<HD>::VW;
  static constexpr bool kNan = false;
  static __device__ __forceinline__ float byte(unsigned w, int i) {
    return (float)(signed char)(w >> (8 * i));
  }
  template <typename E>
  static __device__ __forceinline__ void expand_k(const Regs& r, u4 (&k)[KK]) {
#pragma unroll
    for (int i = 0; i < KK; ++i) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const unsigned x = r.k[i / 2][2 * (i & 1) + w];
        k[i][2 * w] = E::pack2(byte(x, 0), byte(x, 1));
        k[i][2 * w + 1] = E::pack2(byte(x, 2), byte(x, 3));
      }
    }
  }
  static __device__ __forceinline__ void operand_v(const Regs& r, u2 (&av)[MB]) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int i = mb / 4, e = mb % 4;
      av[mb] = u2{ElemF16::pack2(byte(r.v[0][i], e), byte(r.v[1][i], e)),
                  ElemF16::pack2(byte(r.v[2][i], e), byte(r.v[3][i], e))};
    }
  }
};

// Partial rows are fp32 for both types of queries: fp16 ones, as the 16-bit kernels leave,
// added a rounding of the size of the output's own (error against 64 bits 1.45 times that
// of a rounded 32-bit result; so 1.1 times). It costs 16 x 32K keys, q_len 8, 178 -> 181 us
// a call, 4 x 8K 22 -> 27.
template <typename E>
using PartialRows = std::conditional_t<E::kHalfPartials, ElemF16Wide, E>;

// Raw scores of a page, K code . Q^T. Where Q does not fit the vector registers beside
// the accumulators (64 rows, head dim 256) it lives in accumulation registers, which the
// MFMAs read as they are; the empty asm says so, or the compiler copies it over for every
// page.
template <int NB, int HD, typename E, typename KV>
__device__ __forceinline__ void code_scores(f4 (&s)[NB], const typename KV::Regs& r,
                                            u4 (&q)[NB][Dims<HD>::KK]) {
  constexpr int KK = Dims<HD>::KK;
  u4 k[KK];
  KV::template expand_k<E>(r, k);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    if constexpr (NB * HD >= 512) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) asm volatile("" : "+a"(q[nb][kk]));
    }
    s[nb] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) s[nb] = E::mma_qk(k[kk], q[nb][kk], s[nb]);
  }
}

// A masked page's NaN codes of V: in the PV product one would reach every row of its
// block, those that do not see its token too (0 * NaN). They become 0 here, and NaN the
// sums of the rows that do see them. Rare: decoding pages without one costs a few
// instructions on the pages of the draft block only.
template <int NB, int HD, typename KV>
__device__ __forceinline__ void nan_values(WaveState<NB, HD>& st, typename KV::Regs& r,
                                           const f4 (&s)[NB]) {
  constexpr int MB = Dims<HD>::MB, VW = Dims<HD>::VW;
  typename KV::Regs marks;
  unsigned any = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int w = 0; w < VW / 2; ++w) {
      // Bytes of magnitude 0x7f, as 0x80.
      const unsigned nan = ((r.v[e][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
      any |= nan;
      marks.v[e][w] = (nan >> 7) * 0x38u;  // 1.0 in e4m3
      r.v[e][w] &= ~((nan >> 7) * 0xffu);
    }
  if (!__any(any != 0u)) return;  // uniform
  u2 av[MB];
  KV::operand_v(marks, av);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float seen[4], sum = 0.f;
    u2 none;
#pragma unroll
    for (int e = 0; e < 4; ++e) seen[e] = s[nb][e] == -INFINITY ? 0.f : 1.f;
    const u2 rows = ElemF16::round_p(seen[0], seen[1], seen[2], seen[3], sum, none);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const f4 hits = ElemF16::mma_pv(av[mb], rows, none, f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int e = 0; e < 4; ++e)
        st.acc[mb][nb][e] = hits[e] > 0.f ? __builtin_nanf("") : st.acc[mb][nb][e];
    }
  }
}

}  // namespace
}  // namespace sqa

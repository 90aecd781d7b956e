// Device code of the kernels around the paged cache: the cut of a batch of sequences into
// work items, and the codes of 8-bit caches.
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

}  // namespace
}  // namespace sqa

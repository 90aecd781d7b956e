// Device code of the kernels over parts of sequences: which pages a sequence's own splits
// cover, values that are not finite beside tokens a row does not see, partial rows.
#pragma once

#include "sqa_part.h"
#include "sqa_cache_device.h"

namespace sqa {
namespace {

// ceil(n / d) with d the same in every lane.
__device__ __forceinline__ int ceil_over(int n, int d) {
  return ceil_quotient(n, d, __builtin_amdgcn_rcpf((float)d));
}

// even_splits() on the device (0 <= pages < 2^26, size > 0).
__device__ __forceinline__ void even_splits(int pages, int size, int* count, int* each) {
  const int n = ceil_over(pages, size);
  *each = n > 0 ? ceil_quotient(pages, n, __builtin_amdgcn_rcpf((float)n)) : 1;
  *count = ceil_quotient(pages, *each, __builtin_amdgcn_rcpf((float)*each));
}

// A group as the kernels use it: within the batch, its pages in 16 tokens; a group of one
// sequence shares nothing (pages 0).
struct Group {
  int first, count, pages;
};
__device__ __forceinline__ Group load_group(const PartArgs& a, int i) {
  const int32_t* g = a.groups + 3 * min(i, a.n_groups - 1);
  Group x{g[0], g[1], g[2]};
  x.first = min(max(x.first, 0), a.p.batch);
  x.count = min(max(x.count, 0), a.p.batch - x.first);
  x.pages = x.count > 1 && i < a.n_groups ? min(max(x.pages, 0), a.p.bt_stride) << a.p.page_shift
                                          : 0;
  return x;
}
__device__ __forceinline__ Group from_lane(const Group& g, int src) {
  return {__builtin_amdgcn_readlane(g.first, src), __builtin_amdgcn_readlane(g.count, src),
          __builtin_amdgcn_readlane(g.pages, src)};
}

// Whether all rows of a sequence of `len` tokens lie behind `pages` shared pages.
__device__ __forceinline__ bool reaches(const PartArgs& a, int len, int pages) {
  return len >= a.p.q_len && (len - a.p.q_len) / kPageSize >= pages;
}

// The first sequence of a group that reaches past the shared pages, -1: none (then nobody
// reads the group's partials). Its table row names the pages: a padded sequence's need not.
__device__ __forceinline__ int leader_of(const PartArgs& a, const Group& g) {
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < g.count; i += 64) {
    const int b = g.first + min(i + lane, g.count - 1);
    const unsigned long long hit = __ballot(reaches(a, a.p.seq_lens[b], g.pages));
    if (hit) return g.first + min(i + (int)__builtin_ctzll(hit), g.count - 1);
  }
  return -1;
}

// The kernel pages that a sequence goes over by itself: [0, head) and from `tail` on, n in
// all, page v of them at v or, past `head`, v - head + tail.
struct Span {
  int head, tail, n;
  int before;  // of seq_groups, where `shared` pages of its group lie before `tail`; -1: none
  int shared;
};

// The slot of the first split of its group for sequence b; further ones follow slot_step apart.
// Held to what there is: a table that is not the plan's names wrong places, and none outside.
__device__ __forceinline__ int shared_slot(const PartArgs& a, int b, int before) {
  if (!a.packed) return b;  // uniform
  return min(max(b + before / a.by_shared_size, 0), a.shared_slots - 1);
}

// Window: of the pages before row 0's window (the earliest) only those of the first `sink`
// tokens. Shared prefix: what follows it, provided that every row lies behind it; a shorter
// sequence goes over all of its pages by itself. Any lane's sequence.
__device__ __forceinline__ Span span_of(const PartArgs& a, int b, int len) {
  const int pages = min((int)(((unsigned)len + kPageSize - 1) / kPageSize), a.p.max_pages);
  Span s{0, 0, 0, -1, 0};
  if (a.window > 0) {
    const long long from = (long long)len - a.p.q_len + 1 - a.window;
    s.head = min((int)(((unsigned)a.sink + kPageSize - 1) / kPageSize), pages);
    s.tail = from > 0 ? (int)min(from / kPageSize, (long long)pages) : 0;
    s.tail = max(s.tail, s.head);
  }
  if (a.n_groups > 0) {
    const int before = a.seq_groups[2 * b];
    const int shared = min(max(a.seq_groups[2 * b + 1], 0), a.p.bt_stride) << a.p.page_shift;
    if (before >= 0 && shared > 0 && reaches(a, len, shared)) {
      s.before = before;
      s.shared = s.tail = shared;
    }
  }
  s.n = s.head + max(pages - s.tail, 0);
  return s;
}

// Equal splits of one sequence's n pages, none under kMinSplitPages while there are two.
__device__ __forceinline__ void own_splits(const PartArgs& a, int n, int* count, int* size) {
  const int most = max(min(a.splits, n / kMinSplitPages), 1);
  *size = max(ceil_over(n, most), 1);
  *count = ceil_over(n, *size);
}

// The batch's own pages end to end, cut into own_items items of `size` pages: every wave
// finds that for itself, a lane to a sequence, 64 at a time. Workgroups of one item each
// then take the same time whatever the lengths (an extra workgroup on a compute unit waits
// for the first: 128 sequences of 34 pages, 8 kv heads, 256 workgroups, 49 us; 130 of them,
// one sequence to a workgroup, 77).
// Every sequence counts kSeamPages more than it has, before its first one.
struct OwnCut {
  int size, total;
  // The 64 sequences from k on, after `base` pages: the lane's, its pages and length.
  int k, base, n, len;
};
__device__ __forceinline__ int own_pages(const PartArgs& a, int b, int* len) {
  if (b >= a.p.batch) return 0;
  *len = max(a.p.seq_lens[b], 0);
  const int n = span_of(a, b, *len).n;
  return n > 0 ? n + kSeamPages : 0;
}
__device__ __forceinline__ OwnCut own_cut(const PartArgs& a, bool writer) {
  const int lane = threadIdx.x & 63;
  OwnCut c{0, 0, 0, 0, 0, 0};
  c.n = own_pages(a, lane, &c.len);
  int sum = c.n;  // of every 64th sequence from the lane's on
#pragma unroll 4
  for (int k = 64; k < a.p.batch; k += 64) {
    int len;
    sum += own_pages(a, k + lane, &len);
  }
  c.total = wave_sum_int(sum);
  c.size = max(ceil_over(c.total, a.own_items), kMinSplitPages);
  if (!writer) return c;
  int base = 0;  // the join's table
  for (int k = 0; k < a.p.batch; k += 64) {
    int len;
    const int n = k == 0 ? c.n : own_pages(a, k + lane, &len);
    const int incl = wave_inclusive_scan_int(n);
    const int start = base + incl - n, first = (start + kSeamPages) / c.size;
    if (k + lane < a.p.batch)
      a.p.seq_splits[k + lane] =
          SeqSplits{first + k + lane, n > 0 ? (start + n - 1) / c.size - first + 1 : 0};
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return c;
}
// The sequence with page `at` of the batch, the first of its pages (past the seam) and how
// many it has (b < 0: none). For pages in ascending order.
struct OwnPiece {
  int b, len, start, n;
};
__device__ __forceinline__ OwnPiece own_piece(const PartArgs& a, OwnCut& c, int at) {
  const int lane = threadIdx.x & 63;
  for (;;) {
    const int incl = wave_inclusive_scan_int(c.n);
    const unsigned long long hit = __ballot(c.n > 0 && at < c.base + incl);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      return {c.k + src, __builtin_amdgcn_readlane(c.len, src),
              c.base + __builtin_amdgcn_readlane(incl - c.n, src) + kSeamPages,
              __builtin_amdgcn_readlane(c.n, src) - kSeamPages};
    }
    c.base += __builtin_amdgcn_readlane(incl, 63);
    c.k += 64;
    if (c.k >= a.p.batch) return {-1, 0, 0, 0};
    c.n = own_pages(a, c.k + lane, &c.len);
  }
}

// One item of the groups: a block of a group's rows over a split of its pages.
struct SharedItem {
  Group group;  // pages 0: no such item
  int split, block, begin, n;  // pages begin .. begin + n
};
__device__ __forceinline__ SharedItem item_of(const PartArgs& a, int item) {
  const int lane = threadIdx.x & 63;
  SharedItem it{{0, 0, 0}, 0, 0, 0, 0};
  int base = 0;
  for (int k = 0; k < a.n_groups; k += 64) {
    const Group g = load_group(a, k + lane);
    int count, size;
    even_splits(g.pages, a.shared_size, &count, &size);
    const int blocks = (g.count * a.p.rows + a.block_rows - 1) / a.block_rows;
    const int items = g.pages > 0 ? blocks * count : 0;
    const int incl = wave_inclusive_scan_int(items);
    const int first = base + incl - items;
    const unsigned long long hit = __ballot(item >= first && item < first + items);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      it.group = from_lane(g, src);
      const int at = item - __builtin_amdgcn_readlane(first, src);
      const int per = __builtin_amdgcn_readlane(blocks, src);
      it.split = __builtin_amdgcn_readfirstlane(at / per);
      it.block = at - it.split * per;
      const int each = __builtin_amdgcn_readlane(size, src);
      it.begin = it.split * each;
      it.n = max(min(each, it.group.pages - it.begin), 0);
      return it;
    }
    base += __builtin_amdgcn_readlane(incl, 63);
  }
  return it;
}

// Values of a page that are not finite, added up in `to` as the rows see them (tokens of a
// score of -infinity are not seen). Returns whether there are any. INF: there may be infinities,
// and not NaN alone.
template <int NB, int HD, typename E, bool INF>
__device__ __forceinline__ bool add_wild(f4 (&to)[Dims<HD>::MB][NB], const PageV<HD, 1>& pv,
                                         const f4 (&s)[NB], bool bf16) {
  constexpr int VW = Dims<HD>::VW;
  static_assert(Dims<HD>::MB == 2 * VW, "two blocks of dims to a word");
  const unsigned inf = bf16 ? 0x7f80u : 0x7c00u, one = bf16 ? 0x3f80u : 0x3c00u;
  const unsigned up = (0x8000u - inf) * 0x10001u;
  unsigned any = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int w = 0; w < VW; ++w) any |= (pv.v[0][e][w] & 0x7fff7fffu) + up;
  if (__builtin_expect(!__any((any & 0x80008000u) != 0u), 1)) return false;  // uniform
  u2 rows[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float seen[4], sum = 0.f;
    u2 none;
#pragma unroll
    for (int e = 0; e < 4; ++e) seen[e] = s[nb][e] == -INFINITY ? 0.f : 1.f;
    rows[nb] = E::round_p(seen[0], seen[1], seen[2], seen[3], sum, none);
  }
  // Sums of ones: over what is NaN or +infinity, then over what is NaN or -infinity; where there
  // are no infinities, over what is NaN. (By bits of both halves of a word at once: compares, two
  // to an element, took a hundred scalars.)
#pragma unroll 1
  for (int sign = 0; sign < (INF ? 2 : 1); ++sign) {
    const float value = INF ? (sign ? -INFINITY : INFINITY) : __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      unsigned mark[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned x = pv.v[0][e][j];
        unsigned bad = (x & 0x7fff7fffu) + up;
        if constexpr (INF) {
          const unsigned y = x ^ (sign ? inf : inf | 0x8000u) * 0x10001u;  // 0: the other infinity
          bad &= ((y & 0x7fff7fffu) + 0x7fff7fffu) | y;
        }
        mark[e] = ((bad & 0x80008000u) >> 15) * one;
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const u2 av = half == 0 ? u2{pack_lo(mark[0], mark[1]), pack_lo(mark[2], mark[3])}
                                : u2{pack_hi(mark[0], mark[1]), pack_hi(mark[2], mark[3])};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const f4 hits = E::mma_pv(av, rows[nb], u2{0u, 0u}, f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int e = 0; e < 4; ++e) to[2 * j + half][nb][e] += hits[e] > 0.f ? value : 0.f;
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // few registers rather than few waits
    }
  }
  return true;
}

// Values of a masked page that are not finite: in the PV product one would reach every row
// of its block, those that do not see its token too (0 * NaN). They become 0 here, and what
// they are in the sums of the rows that do see them. Rare: pages without one pay a few
// instructions, on masked pages only.
template <int NB, int HD, typename E, bool INF>
__device__ __forceinline__ void wild_values(WaveState<NB, HD>& st, PageV<HD, 1>& pv,
                                            const f4 (&s)[NB], bool bf16) {
  constexpr int VW = Dims<HD>::VW;
  if (!add_wild<NB, HD, E, INF>(st.acc, pv, s, bf16)) return;
  const unsigned up = (0x8000u - (bf16 ? 0x7f80u : 0x7c00u)) * 0x10001u;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      const unsigned x = pv.v[0][e][w];
      const unsigned bad = (((x & 0x7fff7fffu) + up) & 0x80008000u) >> 15;
      pv.v[0][e][w] = x & ~(bad * 0xffffu);
    }
}

// Whether sums are NaN somewhere in the wave: maxima that pass one on, in four chains.
struct NanOf {
  float top[4] = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(int i, f4 x) {
    top[i % 4] = max3_raw(max3_raw(top[i % 4], x[0], x[1]), x[2], x[3]);
  }
  __device__ __forceinline__ bool any() const {
    const float x = max3_raw(max3_raw(top[0], top[1], top[2]), top[3], top[3]);
    return __any(x != x);
  }
};

// 2^x for a sum's weight, never 0: an infinity stays one however far its token's score lies
// behind. (The smallest number there is, so that finite sums do not notice.)
__device__ __forceinline__ float weight_of(float x) { return fmaxf(fast_exp2(x), 0x1p-149f); }

// Where row x of a share is: x counts the rows of one kv head of the sequences from `first`
// on, Q * (Hq / Hkv) each.
struct RowMap {
  int first, kvh;
  long long at;  // partial row of row 0
  // Of a group's share where its slots are packed (else pages is 0): the split, the first
  // sequence's entry in seq_groups, the group's pages.
  int split = 0, before = 0, pages = 0;
  struct Place {
    int b, y;  // sequence, row of its kv head
  };
  __device__ __forceinline__ Place place(const PartArgs& a, int x) const {
    const int i = x / a.by_rows;
    return {first + i, x - i * a.p.rows};
  }
  // In query and output, in rows of HD.
  __device__ __forceinline__ long long out_row(const PartArgs& a, int x) const {
    const Place p = place(a, x);
    const int qi = p.y / a.p.by_group;
    return ((long long)p.b * a.p.q_len + qi) * a.p.hq + kvh * a.p.group + (p.y - qi * a.p.group);
  }
  __device__ __forceinline__ long long part_row(const PartArgs& a, int x) const {
    const Place p = place(a, x);
    if (__builtin_expect(pages == 0, 1))
      return at + (long long)(p.b - first) * a.p.hkv * a.p.rows + p.y;
    const unsigned slot = shared_slot(a, p.b, before + (p.b - first) * pages) + split;
    return a.shared_at +
           ((long long)min(slot, (unsigned)a.shared_slots - 1) * a.p.hkv + kvh) * a.p.rows + p.y;
  }
};

// Chunk c (of HD / 4) of partial row `at`, where `is`. Past 32-bit offsets two stores by
// address take the place of one through the buffer.
template <int HD>
__device__ __forceinline__ void store_partial(const PartArgs& args, __amdgpu_buffer_rsrc_t pr,
                                              f4 v, long long at, int c, bool is) {
  if (__builtin_expect(args.far_rows, 0)) {  // uniform
    const u4 x = __builtin_bit_cast(u4, v);
    float* to = args.p.part_o + at * HD + 4 * c;
    if (is) {
      store_through(to, __builtin_bit_cast(unsigned long long, u2{x[0], x[1]}));
      store_through(to + 2, __builtin_bit_cast(unsigned long long, u2{x[2], x[3]}));
    }
    return;
  }
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), pr,
                                         is ? (unsigned)((at * HD + 4 * c) * 4) : kDroppedOffset, 0,
                                         kThroughAux);
}

// The map of a group's share for kv head kvh.
__device__ __forceinline__ RowMap shared_map(const PartArgs& a, int first, int split, int pages,
                                             int kvh) {
  RowMap map{first, kvh,
             a.shared_at + (((long long)split * a.p.batch + first) * a.p.hkv + kvh) * a.p.rows};
  if (__builtin_expect(a.packed, 0)) {  // uniform
    map.split = split;
    map.before = scalar_load(a.seq_groups + 2 * first);
    map.pages = pages;
  }
  return map;
}

// Leaves the rows of one wave, or of the `waves` ones that have gone over pages of one share
// (wave `mine` of them; their stages follow one another): normalised rows of the output, or
// fp32 sums and (max, sum) at partial rows. Through LDS one block of 16 rows at a time, so
// that a store instruction writes whole rows (write_results() in sqa_device.h has the
// figures); partial rows are fp32 for both types of queries, as after block scales. Rows
// row0 + 16 nb + r below n_rows are there; without `store` nothing is written.
template <int NB, int HD, typename E>
__device__ __forceinline__ void leave_rows(const PartArgs& args, WaveState<NB, HD>& st,
                                           float* stage, int waves, int mine, bool direct,
                                           const RowMap& map, int row0, int n_rows, bool store) {
  const PartialArgs& a = args.p;
  constexpr int MB = Dims<HD>::MB;
  constexpr int kStageRow = HD + 4;
  constexpr int kStage = 16 * kStageRow;
  constexpr int CPR = HD / 4;  // 4-value chunks per row
  const int lane = piece_tid() & 63;
  const int g16 = lane >> 4, l16 = lane & 15;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) st.l[nb] = xor_sum(st.l[nb]);
  const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
      (void*)a.part_o, (short)0, (int)a.part_o_bytes, kBufferFlags);
  float* own = stage + mine * kStage;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int x0 = row0 + 16 * nb;
    if (x0 >= n_rows) break;  // uniform over the waves of a share
    float* dst = own + l16 * kStageRow + (HD / 4) * g16;
#pragma unroll
    for (int rr = 0; rr < 4; ++rr)
#pragma unroll
      for (int h = 0; h < MB / 4; ++h) {
        f4 o;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) o[mb] = st.acc[4 * h + mb][nb][rr];
        *(f4*)(dst + MB * rr + 4 * h) = o;
      }
    // (max, sum) beside the row, where its padding is. A NaN sum travels with a finite max,
    // so that it counts.
    const float m_out = st.l[nb] == st.l[nb] ? st.m[nb] : 0.f;
    if (g16 == 0) *(float2*)(own + l16 * kStageRow + HD) = float2{m_out, st.l[nb]};
    if (waves > 1)  // uniform
      __syncthreads();
    else
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    // Where the lane's row goes, in rows of HD (less than 2^31 of either), -1: nowhere.
    const int to = !store || x0 + l16 >= n_rows ? -1
                   : direct                     ? (int)map.out_row(args, x0 + l16)
                                                : (int)map.part_row(args, x0 + l16);
    // Chunk e % CPR of row e / CPR (< 16), the waves in turn.
    for (int i = waves > 1 ? mine : 0; i < CPR / 4; i += waves) {
      const int e = i * 64 + lane;
      const int rs = e / CPR;
      const float* row = stage + (waves > 1 ? 0 : mine * kStage) + rs * kStageRow;
      float m = -INFINITY, l = 0.f;
      f4 v = {0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < waves; ++w) {
        const float2 ml = *(const float2*)(row + w * kStage + HD);
        m = ml.y != 0.f ? fmaxf(m, ml.x) : m;
      }
      const float base = m == -INFINITY ? 0.f : m;
      for (int w = 0; w < waves; ++w) {
        const float2 ml = *(const float2*)(row + w * kStage + HD);
        const f4 o = *(const f4*)(row + w * kStage + 4 * (e % CPR));
        const float f = waves == 1 || ml.y != ml.y ? 1.f : weight_of(ml.x - base);
        v += o * f;
        l += ml.y * f;
      }
      const long long at = __shfl(to, rs);
      const bool is = at >= 0;
      if (direct) {
        // l = 0: the row saw no key (written as 0). A NaN l passes.
        const float sc = !(l <= 0.f) ? a.out_scale / l : 0.f;
        const float o[4] = {v[0] * sc, v[1] * sc, v[2] * sc, v[3] * sc};
        if (is) *(u2*)(a.out + at * HD + 4 * (e % CPR)) = E::pack4(o);
      } else {
        store_partial<HD>(args, pr, v, at, e % CPR, is);
        if (is && e % CPR == 0)
          store_through(a.part_ml + at * 2, __builtin_bit_cast(unsigned long long, float2{m, l}));
      }
    }
    if (waves > 1)  // uniform
      __syncthreads();
    else
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  }
}

// The kernel's (first and only) argument, where the compiler cannot know that it was asked
// for before: what a branch or a piece of work takes from it is loaded there, and not held in
// scalar registers through all others (a third to a half more of them spilled otherwise).
__device__ __forceinline__ const PartArgs& own_args() {
  auto* p = (const __attribute__((address_space(4))) PartArgs*)
      __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const PartArgs*)p;
}

// How a cache's elements go to the products. kScaled: codes with block scales.
// kInf: elements may be infinite.
template <int HD>
struct PartNative : KvNative<HD> {
  static constexpr bool kScaled = false, kInf = true;
};
template <int HD>
struct PartFp8 : KvFp8<HD> {
  static constexpr bool kScaled = false, kInf = false;
};
template <int HD>
struct PartCodesFp8 : CodesFp8<HD> {
  static constexpr bool kScaled = true, kInf = false;
};
template <int HD>
struct PartCodesInt8 : CodesInt8<HD> {
  static constexpr bool kScaled = true, kInf = false;
};

// The softmax step of one page without block scales: P = 2^(c s - m) against a maximum that
// may lag, one PV product.
template <int NB, int HD, typename E, typename KV>
__device__ __forceinline__ void plain_page(WaveState<NB, HD>& st, const typename KV::Regs& r,
                                           const f4 (&s)[NB], bool masked, float c, bool bf16) {
  PageV<HD, 1> pv;
  KV::template expand_v<E>(r, pv.v[0]);
  float lm[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) lm[nb] = max4(s[nb]) * c;
  raise_max<NB, HD>(st, lm);
  // After the first maximum, whose factor is 0.
  if (masked) wild_values<NB, HD, E, KV::kInf>(st, pv, s, bf16);
  page_pv<NB, HD, E, KV, 1>(st, s, pv, false, c);
}

// The same with a scale for K (in c) and V (in the exponent, as P weighs codes): see
// sqa_scaled_attention_kernel.
template <int NB, int HD, typename KV>
__device__ __forceinline__ void scaled_page(WaveState<NB, HD>& st, const typename KV::Regs& r,
                                            const f4 (&s)[NB], bool masked, float c, float add,
                                            float inv_vs, bool loud) {
  constexpr int MB = Dims<HD>::MB;
  float lm[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) lm[nb] = fmaf(max4(s[nb]), c, add);
  raise_max<NB, HD>(st, lm);
  u2 ph[NB];
  u2 none = {0u, 0u};
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float off = add - (st.m[nb] == -INFINITY ? 0.f : st.m[nb]);
    float pr[4], rounded = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) pr[e] = fast_exp2(fmaf(s[nb][e], c, off));
    const float sum = (pr[0] + pr[1]) + (pr[2] + pr[3]);
    const float l = st.l[nb];
    st.l[nb] = fmaf(sum, inv_vs, l);
    // A V scale that is not finite stays with the rows that see its page.
    if (masked) st.l[nb] = sum == 0.f ? l : st.l[nb];  // uniform
    ph[nb] = ElemF16::round_p(pr[0], pr[1], pr[2], pr[3], rounded, none);
  }
  if (loud) {  // uniform
    u2 av[MB];
    KV::operand_v(r, av);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        st.acc[mb][nb] = ElemF16::mma_pv(av[mb], ph[nb], none, st.acc[mb][nb]);
  }
}

// One workgroup = W waves, wave w with kv head w % wg_heads of the workgroup's heads; the
// W / wg_heads waves of a head divide the pages of one share, each on its own, and join
// their rows at the end. A share is a split of a sequence's own pages, or (`shared`) a block
// of a group's rows over a split of the shared pages. A wave holds all rows of its share (NB
// blocks of 16) and keeps a ring of D pages in flight in registers.
//
// Memory bounds it where there is enough of it: 64 windows of 4K tokens, q_len 8, fp16,
// 176 us for 1.09 GB (6.2 TB/s of the 7.25 that reads alone reach); 100 of e4m3, one
// token, 149 us a call for 0.84 GB, where a page's chain of products, maximum and exponentials (0.55
// us a wave) takes as long as its half as many bytes. Short calls are start-up: the length,
// the page ids, the pages and the way out through LDS follow one another (one sequence of a
// single token 6.6 us in a graph, of 1K tokens 8.2; a kernel that does nothing 1.8).
template <int NB, int D, int HD, int W, typename E, typename KV>
__device__ __forceinline__ void part_share(float* sm_stage, int block, bool shared) {
  constexpr int KK = Dims<HD>::KK, MB = Dims<HD>::MB;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int g16 = lane >> 4, l16 = lane & 15;
  const PartArgs& first_args = own_args();
  const int wgh = first_args.wg_heads;
  const int log_heads = wgh >> 1;  // of 1, 2 and 4
  const int waves = W >> log_heads;
  const int mine = wave >> log_heads;
  const int head_in = wave & (wgh - 1);
  const int share = block / first_args.p.by_head_groups;
  const int hkv = first_args.p.hkv;
  const int kvh = (block - share * ((hkv + wgh - 1) / wgh)) * wgh + head_in;

  // No such head: nothing to do, but to wait with the other heads' waves.
  const bool is_head = kvh < hkv;
  const int head_at = is_head ? kvh : 0;

  // What the wave goes over: pages v0 .. v0 + n_pages of table row b (page v of the sequence
  // at v, or past `head` at v + skip), for n_rows rows from row0 on.
  int b, len, head = 0, skip = 0, v0, n_pages, row0 = 0, n_rows = first_args.p.rows;
  RowMap map;
  map.kvh = head_at;
  bool direct = false;
  OwnCut cut;
  int at = 0, end = 0;  // of an item that may cross sequence ends
  const bool crosses = !shared && first_args.splits == 0;
  auto piece = [&] {  // of the item, from page `at` on
    const PartArgs& args = own_args();
    const OwnPiece x = own_piece(args, cut, at);
    b = __builtin_amdgcn_readfirstlane(max(x.b, 0));
    len = __builtin_amdgcn_readfirstlane(x.len);
    const Span span = span_of(args, b, len);
    const int start = __builtin_amdgcn_readfirstlane(x.start);
    const int n = __builtin_amdgcn_readfirstlane(x.n);
    head = span.head;
    skip = span.tail - span.head;
    v0 = max(at - start, 0);
    n_pages = max(min(end - start, n) - v0, 0);  // 0: the item ends in the seam
    direct = span.before < 0 && n_pages == n;
    map.first = b;
    map.at = ((long long)(share + b) * args.p.hkv + head_at) * args.p.rows;
    at = x.b < 0 ? end : start + n;
  };
  if (shared) {  // uniform
    const PartArgs& args = own_args();
    const PartialArgs& a = args.p;
    const SharedItem it = item_of(args, share);
    b = it.group.pages > 0 ? leader_of(args, it.group) : -1;
    if (b < 0 || it.split >= args.most_splits) return;  // uniform over the workgroup
    len = 0x7fffffff;
    row0 = it.block * (16 * NB);
    n_rows = it.group.count * a.rows;
    v0 = it.begin;
    n_pages = it.n;
    map = shared_map(args, it.group.first, it.split, it.group.pages, head_at);
  } else if (crosses) {
    const PartArgs& args = own_args();
    cut = own_cut(args, block == 0 && wave == 0);
    at = __builtin_amdgcn_readfirstlane(share * cut.size);
    end = __builtin_amdgcn_readfirstlane(min(at + cut.size, cut.total));
    if (share >= args.own_items || at >= end) return;  // uniform over the workgroup
  } else {
    const PartArgs& args = own_args();
    const PartialArgs& a = args.p;
    b = share / a.by_splits;
    if (b >= a.batch) return;  // uniform over the workgroup
    const int split = share - b * args.splits;
    len = max(scalar_load(a.seq_lens + b), 0);
    const Span span = span_of(args, b, len);
    int count, size;
    own_splits(args, span.n, &count, &size);
    if (split >= max(count, 1)) return;  // uniform over the workgroup
    direct = span.before < 0 && count <= 1;
    head = span.head;
    skip = span.tail - span.head;
    v0 = split * size;
    n_pages = max(min(v0 + size, span.n) - v0, 0);
    map.first = b;
    map.at = ((long long)share * a.hkv + head_at) * a.rows;
  }
  for (;;) {  // pieces
  if (crosses) {
    piece();
    if (n_pages <= 0) return;  // uniform over the workgroup
  }
  const PartArgs& args = own_args();
  const PartialArgs& a = args.p;
  if (waves > 1) {  // uniform: this wave's part
    const int each = (n_pages + waves - 1) >> ((W == 8 ? 3 : 2) - log_heads);
    v0 += mine * each;
    n_pages = max(min(each, n_pages - mine * each), 0);
  }
  if (!is_head) n_pages = 0;
  b = __builtin_amdgcn_readfirstlane(b);
  v0 = __builtin_amdgcn_readfirstlane(v0);
  n_pages = __builtin_amdgcn_readfirstlane(n_pages);
  row0 = __builtin_amdgcn_readfirstlane(row0);
  n_rows = __builtin_amdgcn_readfirstlane(n_rows);
  head = __builtin_amdgcn_readfirstlane(head);
  skip = __builtin_amdgcn_readfirstlane(skip);
  auto page_at = [&](int v) { return v < head ? v : v + skip; };
  const int shift = a.page_shift, sub_mask = (1 << shift) - 1;

  // Ids of the ring's next refills, and of those a turn later on their way: scalar loads.
  const int32_t* row = a.block_tables + (size_t)b * a.bt_stride;
  auto load_ids = [&](int i, int (&ids)[D]) {
#pragma unroll
    for (int j = 0; j < D; ++j)
      ids[j] = scalar_load(row + (min(page_at(v0 + max(min(i + j, n_pages - 1), 0)),
                                      a.max_pages - 1) >> shift));
  };
  int first_ids[D], ids[D], ids_next[D];
  load_ids(0, first_ids);
  load_ids(D, ids);

  u4 q[NB][KK];
  RegBits<NB> bits;
  int from[NB];  // first token of the row's window
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int x = row0 + 16 * nb + l16;
    const bool is = x < n_rows;
    const _Float16* qp = a.q + map.out_row(args, is ? x : row0) * HD;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const u4 x = *(const u4*)(qp + KV::q_dims(kk, g16));
      q[nb][kk] = is ? x : u4{0u, 0u, 0u, 0u};
    }
    const int qi = map.place(args, is ? x : row0).y / a.by_group;
    bits.b[nb] = draft_bits(a, b, qi, is);
    from[nb] = args.window > 0
                   ? (int)max((long long)len - a.q_len + qi + 1 - args.window, 0LL) : 0;
  }

  const unsigned tok_bytes = a.token_stride;
  const unsigned k_lane = l16 * tok_bytes + map.kvh * a.head_stride + KV::k_lane_bytes(g16);
  const unsigned v_lane = 4 * g16 * tok_bytes + map.kvh * a.head_stride + KV::v_lane_bytes(l16);
  const size_t sub_bytes = (size_t)kPageSize * tok_bytes;
  // Lanes 0-31 load the page's K scale, 32-63 its V scale.
  const char* scale_lane = KV::kScaled
                               ? (const char*)(lane < 32 ? args.scales.k : args.scales.v) +
                                     (size_t)map.kvh * args.scales.head_stride
                               : nullptr;
  struct Slot {
    typename KV::Regs kv;
    float scale;
  };
  // pid < 0: zeros, without touching memory.
  auto load_page = [&](int pid, int p, Slot& s) {
    pid = __builtin_amdgcn_readfirstlane(pid);
    const size_t off =
        pid >= 0 ? (size_t)pid * (size_t)a.page_stride + (size_t)(p & sub_mask) * sub_bytes : 0;
    const int nrec = pid >= 0 ? (int)a.page_extent : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((const char*)a.k + off), (short)0, nrec, kBufferFlags);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((const char*)a.v + off), (short)0, nrec, kBufferFlags);
    if constexpr (KV::kScaled)
      s.scale = *(const float*)(scale_lane + max(pid, 0) * args.scales.page_stride);
    KV::load(s.kv, kr, vr, k_lane, v_lane, tok_bytes);
  };
  Slot ring[D];
#pragma unroll
  for (int j = 0; j < D; ++j)
    load_page(j < n_pages ? clamp_page(first_ids[j], a.num_pages) : -1, page_at(v0 + j), ring[j]);

  WaveState<NB, HD> st;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    st.m[nb] = -INFINITY;
    st.l[nb] = 0.f;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) st.acc[mb][nb] = f4{0.f, 0.f, 0.f, 0.f};
  }
  // Masked pages: with a token from the draft block on (never a shared page: `len`), or
  // before the last row's window and past the first tokens.
  const int mask_from = len - a.q_len;
  const int all_from = args.window > 0 ? (int)max((long long)len - args.window, 0LL) : 0;

  auto mask = [&](f4 (&s)[NB], int t0) {  // scores of the page at token t0
    const int tok0 = t0 + 4 * g16;
    mask_scores<NB>(s, bits.b, mask_from, tok0, len);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = tok0 + e;
        const unsigned in = (unsigned)(t >= from[nb]) | (unsigned)(t < args.sink);
        s[nb][e] = in ? s[nb][e] : -INFINITY;
      }
  };

  for (int i = 0; i < n_pages; i += D) {
    load_ids(i + 2 * D, ids_next);
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int ii = i + j;
      if (ii < n_pages) {
        const int p = page_at(v0 + ii);
        const int t0 = p * kPageSize;
        const bool masked = t0 + kPageSize > mask_from ||
                            (t0 < all_from && t0 + kPageSize > args.sink);  // uniform
        f4 s[NB];
        code_scores<NB, HD, E, KV>(s, ring[j].kv, q);
        if constexpr (KV::kScaled) {
          const float ks = __builtin_bit_cast(
              float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ring[j].scale), 0));
          const float vs = __builtin_bit_cast(
              float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ring[j].scale), 32));
          const bool loud = !(vs < 0x1p-64f);
          const float lv = loud ? __builtin_amdgcn_logf(vs) : -64.f;
          const float inv_vs = loud ? __builtin_amdgcn_rcpf(vs) : 0x1p64f;
          float c = a.scale_log2 * ks, add = lv;
          if (masked) {
            // After the scales, so that one of 0, infinity or NaN leaves them -inf.
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) s[nb] = s[nb] * c + lv;
            c = 1.f;
            add = 0.f;
            mask(s, t0);
            if constexpr (KV::kNan) nan_values<NB, HD, KV>(st, ring[j].kv, s);
          }
          scaled_page<NB, HD, KV>(st, ring[j].kv, s, masked, c, add, inv_vs, loud);
        } else {
          if (masked) mask(s, t0);
          plain_page<NB, HD, E, KV>(st, ring[j].kv, s, masked, a.scale_log2, a.bf16);
        }
      }
      load_page(ii + D < n_pages ? clamp_page(ids[j], a.num_pages) : -1, page_at(v0 + ii + D),
                ring[j]);
    }
#pragma unroll
    for (int j = 0; j < D; ++j) ids[j] = ids_next[j];
  }
  // An infinity on a page that is not masked is NaN by now in bf16, whose second part of P may
  // be 0 or negative, and under a probability or a change of the maximum that rounds to 0. The
  // values that are not finite are added up once more by themselves, and are what they add up
  // to.
  if constexpr (KV::kInf) {
    NanOf nan;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) nan.add(mb * NB + nb, st.acc[mb][nb]);
    if (__builtin_expect(nan.any(), 0)) {  // uniform
      f4 wild[MB][NB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) wild[mb][nb] = f4{0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < n_pages; ++i) {
        const int p = page_at(v0 + i);
        Slot slot;
        load_page(clamp_page(scalar_load(row + (min(p, a.max_pages - 1) >> shift)), a.num_pages), p,
                  slot);
        PageV<HD, 1> pv;
        KV::template expand_v<E>(slot.kv, pv.v[0]);
        f4 s[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[nb] = f4{0.f, 0.f, 0.f, 0.f};
        mask(s, p * kPageSize);
        add_wild<NB, HD, E, true>(wild, pv, s, a.bf16);
      }
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            st.acc[mb][nb][e] = wild[mb][nb][e] == 0.f ? st.acc[mb][nb][e] : wild[mb][nb][e];
    }
  }
  leave_rows<NB, HD, E>(own_args(), st, sm_stage + head_in * waves * 16 * (HD + 4), waves, mine,
                        direct, map, row0, n_rows, is_head);
  if (!crosses || at >= end) return;  // uniform over the workgroup
  }
}

// GROUPS: the first shared_wgs workgroups serve the groups, the others sequences.
template <int NB, int D, int HD, typename E, typename KV, bool GROUPS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1)))
void sqa_part_kernel(PartArgs args) {
  __shared__ float sm_stage[4 * 16 * (HD + 4)];
  const bool shared = GROUPS && (int)blockIdx.x < args.shared_wgs;
  part_share<NB, D, HD, 4, E, KV>(sm_stage, GROUPS && !shared ? blockIdx.x - args.shared_wgs
                                                                 : blockIdx.x, shared);
}

// Ring depths: about 32 KiB of a 16-bit cache or 16 of codes in flight per wave, half of
// that at 33 to 64 rows, whose accumulators take the registers.
template <int HD, typename E, typename KV, bool GROUPS>
void launch_part_hd(const PartArgs& a, int rows, dim3 grid, hipStream_t stream) {
  constexpr int D = 4 * 128 / HD;
  const dim3 block(256);
  if (rows <= 16)
    hipLaunchKernelGGL((sqa_part_kernel<1, D, HD, E, KV, GROUPS>), grid, block, 0, stream, a);
  else if (rows <= 32)
    hipLaunchKernelGGL((sqa_part_kernel<2, D, HD, E, KV, GROUPS>), grid, block, 0, stream, a);
  else if constexpr (HD != 256)
    hipLaunchKernelGGL((sqa_part_kernel<4, D / 2, HD, E, KV, GROUPS>), grid, block, 0, stream, a);
}

template <typename E, template <int> class KV, bool GROUPS>
void launch_part_as(const PartArgs& a, int rows, dim3 grid, hipStream_t stream) {
  if (a.p.head_dim == 64)
    launch_part_hd<64, E, KV<64>, GROUPS>(a, rows, grid, stream);
  else if (a.p.head_dim == 128)
    launch_part_hd<128, E, KV<128>, GROUPS>(a, rows, grid, stream);
  else
    launch_part_hd<256, E, KV<256>, GROUPS>(a, rows, grid, stream);
}

template <typename E, bool GROUPS>
void launch_part(const PartArgs& a, int rows, dim3 grid, hipStream_t stream) {
  if (a.scaled && a.kv_type == kInt8)
    launch_part_as<E, PartCodesInt8, GROUPS>(a, rows, grid, stream);
  else if (a.scaled)
    launch_part_as<E, PartCodesFp8, GROUPS>(a, rows, grid, stream);
  else if (a.kv_type == kE4M3)
    launch_part_as<E, PartFp8, GROUPS>(a, rows, grid, stream);
  else
    launch_part_as<E, PartNative, GROUPS>(a, rows, grid, stream);
}

// Workgroups that the sequences' own pages take.
inline long long own_workgroups(const PartArgs& a) {
  const long long shares = a.splits > 0 ? (long long)a.p.batch * a.splits : a.own_items;
  return shares * ((a.p.hkv + a.wg_heads - 1) / a.wg_heads);
}

}  // namespace
}  // namespace sqa

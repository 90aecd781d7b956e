// Device code of the kernels over parts of sequences: which pages a sequence's own splits
// cover, values that are not finite beside tokens a row does not see, partial rows.
#pragma once

#include "sqa_part.h"
#include "sqa_cache_device.h"

namespace sqa {
namespace {

// The kernel pages of a sequence that its own splits cover: [0, head) and [tail, head's
// pages + tail ...): n pages in all, page v of them at() of the sequence.
struct Span {
  int head, tail, n;
  int count, size;  // splits and pages per split
  bool shared;      // the pages before `tail` are a group's
  __device__ __forceinline__ int at(int v) const { return v < head ? v : v - head + tail; }
};

// Window: of the pages before row 0's window (the earliest) only those of the first `sink`
// tokens. Shared prefix: what follows it, provided that every row lies behind it; a shorter
// sequence goes over all of its pages by itself.
__device__ __forceinline__ Span span_of(const PartArgs& a, int b, int len) {
  const int pages = min((int)(((unsigned)len + kPageSize - 1) / kPageSize), a.p.max_pages);
  Span s;
  s.head = 0;
  s.tail = 0;
  s.shared = false;
  if (a.window > 0) {
    const long long from = (long long)len - a.p.q_len + 1 - a.window;
    s.head = min((int)(((unsigned)a.sink + kPageSize - 1) / kPageSize), pages);
    s.tail = from > 0 ? (int)min(from / kPageSize, (long long)pages) : 0;
    s.tail = max(s.tail, s.head);
  }
  if (a.groups != nullptr) {
    const int g = scalar_load(a.group_of + b);
    if (g >= 0) {
      const int shared = scalar_load(&a.groups[g].pages);
      s.shared = shared > 0 && (len - a.p.q_len) / kPageSize >= shared && len >= a.p.q_len;
      s.tail = s.shared ? shared : 0;
    }
  }
  s.n = s.head + max(pages - s.tail, 0);
  // Splits of equal size, none of them under kMinSplitPages while there are two.
  const int most = max(min(a.splits, s.n / kMinSplitPages), 1);
  s.size = max(ceil_quotient(s.n, most, __builtin_amdgcn_rcpf((float)most)), 1);
  s.count = ceil_quotient(s.n, s.size, __builtin_amdgcn_rcpf((float)s.size));
  return s;
}

// Values of a masked page that are not finite: in the PV product one would reach every row
// of its block, those that do not see its token too (0 * NaN). They become 0 here, and what
// they are in the sums of the rows that do see them. Rare: pages without one pay a few
// instructions, on masked pages only.
template <int NB, int HD, typename E>
__device__ __forceinline__ void wild_values(WaveState<NB, HD>& st, PageV<HD, 1>& pv,
                                            const f4 (&s)[NB], bool bf16) {
  constexpr int MB = Dims<HD>::MB, VW = Dims<HD>::VW;
  const unsigned inf = bf16 ? 0x7f80u : 0x7c00u, one = bf16 ? 0x3f80u : 0x3c00u;
  const unsigned up = (0x8000u - inf) * 0x10001u;
  unsigned any = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int w = 0; w < VW; ++w) any |= (pv.v[0][e][w] & 0x7fff7fffu) + up;
  if (!__any((any & 0x80008000u) != 0u)) return;  // uniform
  u2 rows[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    float seen[4], sum = 0.f;
    u2 none;
#pragma unroll
    for (int e = 0; e < 4; ++e) seen[e] = s[nb][e] == -INFINITY ? 0.f : 1.f;
    rows[nb] = E::round_p(seen[0], seen[1], seen[2], seen[3], sum, none);
  }
  // Sums of ones: over what is NaN or +infinity, then over what is NaN or -infinity.
#pragma unroll
  for (int sign = 0; sign < 2; ++sign) {
    unsigned mark[4][VW];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        unsigned m = 0u;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const unsigned x = pv.v[0][e][w] >> (16 * half) & 0xffffu;
          const bool other = x == (sign ? inf : inf | 0x8000u);
          m |= ((x & 0x7fffu) >= inf && !other ? one : 0u) << (16 * half);
        }
        mark[e][w] = m;
      }
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      const int j = mb >> 1;
      const u2 av = (mb & 1) == 0
                        ? u2{pack_lo(mark[0][j], mark[1][j]), pack_lo(mark[2][j], mark[3][j])}
                        : u2{pack_hi(mark[0][j], mark[1][j]), pack_hi(mark[2][j], mark[3][j])};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const f4 hits = E::mma_pv(av, rows[nb], u2{0u, 0u}, f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 4; ++e)
          st.acc[mb][nb][e] += hits[e] > 0.f ? (sign ? -INFINITY : INFINITY) : 0.f;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      const unsigned x = pv.v[0][e][w];
      const unsigned bad = (((x & 0x7fff7fffu) + up) & 0x80008000u) >> 15;
      pv.v[0][e][w] = x & ~(bad * 0xffffu);
    }
}

// Leaves one wave's rows: normalised rows of the output, or fp32 sums and (max, sum) at
// partial rows. Block nb's row slot r is real(nb, r); its partial row is first + 16 nb + r,
// its place in the output out_row(nb, r) (in rows of HD). Through LDS one block at a time,
// so that a store instruction writes whole rows (write_results() in sqa_device.h has the
// figures); partial rows are fp32 for both types of queries, as after block scales.
template <int NB, int HD, typename E, typename Real, typename OutRow>
__device__ __forceinline__ void leave_rows(const PartialArgs& a, WaveState<NB, HD>& st,
                                           float* stage, bool direct, long long first,
                                           Real&& real, OutRow&& out_row) {
  constexpr int MB = Dims<HD>::MB;
  constexpr int kStageRow = HD + 4;
  constexpr int CPR = HD / 4;  // 4-value chunks per row
  const int lane = piece_tid() & 63;
  const int g16 = lane >> 4, l16 = lane & 15;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) st.l[nb] = xor_sum(st.l[nb]);
  const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
      (void*)a.part_o, (short)0, (int)a.part_o_bytes, kBufferFlags);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    if (!real(nb, 0)) break;  // uniform
    // l = 0: the row saw no key (written as 0). A NaN l passes.
    const float inv_l = !(st.l[nb] <= 0.f) ? 1.f / st.l[nb] : 0.f;
    const float sc = direct ? a.out_scale * inv_l : 1.f;
    float* dst = stage + l16 * kStageRow + (HD / 4) * g16;
#pragma unroll
    for (int rr = 0; rr < 4; ++rr)
#pragma unroll
      for (int h = 0; h < MB / 4; ++h) {
        f4 o;
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) o[mb] = st.acc[4 * h + mb][nb][rr] * sc;
        *(f4*)(dst + MB * rr + 4 * h) = o;
      }
    // The staging rows are this wave's own: LDS keeps a wave's accesses in order, the
    // fences keep the compiler from moving them.
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    f4 v[CPR / 4];
#pragma unroll
    for (int i = 0; i < CPR / 4; ++i) {
      const int e = i * 64 + lane;  // row e / CPR (< 16), chunk e % CPR
      v[i] = *(const f4*)(stage + (e / CPR) * kStageRow + 4 * (e % CPR));
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
    for (int i = 0; i < CPR / 4; ++i) {
      const int e = i * 64 + lane;
      const int rs = e / CPR;
      if (direct) {
        if (real(nb, rs)) {
          const float o[4] = {v[i][0], v[i][1], v[i][2], v[i][3]};
          *(u2*)(a.out + out_row(nb, rs) * HD + 4 * (e % CPR)) = E::pack4(o);
        }
      } else {
        const unsigned at = (unsigned)(((first + 16 * nb + rs) * HD + 4 * (e % CPR)) * 4);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v[i]), pr,
                                               real(nb, rs) ? at : kDroppedOffset, 0, kThroughAux);
      }
    }
    if (!direct && g16 == 0 && real(nb, l16)) {
      // A NaN sum travels with a finite max, so the join counts the split.
      const float m_out = st.l[nb] == st.l[nb] ? st.m[nb] : 0.f;
      store_through(a.part_ml + (first + 16 * nb + l16) * 2,
                    __builtin_bit_cast(unsigned long long, float2{m_out, st.l[nb]}));
    }
  }
}

// The first sequence of a group whose rows all lie behind the shared pages, -1: none (then
// nobody reads the group's partials). Its table row names the pages: a padded sequence's
// need not.
__device__ __forceinline__ int leader_of(const PartArgs& a, const SharedGroup& g) {
  const int lane = threadIdx.x & 63;
  for (int i = 0; i < g.count; i += 64) {
    const int b = g.first + min(i + lane, g.count - 1);
    const int len = a.p.seq_lens[b];
    const unsigned long long hit =
        __ballot(len >= a.p.q_len && (len - a.p.q_len) / kPageSize >= g.pages);
    if (hit) return g.first + min(i + (int)__builtin_ctzll(hit), g.count - 1);
  }
  return -1;
}

// How a cache's elements go to the products. kScaled: codes with block scales.
template <int HD>
struct PartNative : KvNative<HD> {
  static constexpr bool kScaled = false;
};
template <int HD>
struct PartFp8 : KvFp8<HD> {
  static constexpr bool kScaled = false;
};
template <int HD>
struct PartCodesFp8 : CodesFp8<HD> {
  static constexpr bool kScaled = true;
};
template <int HD>
struct PartCodesInt8 : CodesInt8<HD> {
  static constexpr bool kScaled = true;
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
  if (masked) wild_values<NB, HD, E>(st, pv, s, bf16);
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

// One workgroup = four waves on their own, wave w with kv head w % wg_heads of the
// workgroup's heads and share w / wg_heads of its shares; a share is a split of a
// sequence's own pages (SHARED false) or a block of a group's rows over a split of the
// shared pages (true; NB 16 rows at most). A wave holds all rows of its share and keeps a
// ring of D pages in flight in registers; no barrier.
template <int NB, int D, int HD, typename E, typename KV, bool SHARED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1)))
void sqa_part_kernel(PartArgs args) {
  const PartialArgs& a = args.p;
  constexpr int KK = Dims<HD>::KK, MB = Dims<HD>::MB;
  __shared__ float sm_stage[4 * 16 * (HD + 4)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int g16 = lane >> 4, l16 = lane & 15;
  const int wgh = args.wg_heads;
  const int rest = (int)blockIdx.x / a.by_head_groups;
  const int kvh = ((int)blockIdx.x - rest * ((a.hkv + wgh - 1) / wgh)) * wgh + wave % wgh;
  const int share = rest * (4 / wgh) + wave / wgh;
  if (kvh >= a.hkv) return;

  // The share: its table row, the pages v0 .. v0 + n_pages of `span`, its rows.
  Span span;
  int b, len, v0, n_pages, row0 = 0, n_rows;
  long long first;  // its first partial row
  bool direct = false;
  if constexpr (SHARED) {
    if (share >= args.n_items) return;
    const SharedItem it = args.items[share];
    const SharedGroup g = args.groups[__builtin_amdgcn_readfirstlane(it.group)];
    const int split = __builtin_amdgcn_readfirstlane(it.split);
    row0 = __builtin_amdgcn_readfirstlane(it.block) * (16 * NB);
    b = __builtin_amdgcn_readfirstlane(leader_of(args, g));
    if (b < 0) return;  // uniform
    len = 0x7fffffff;
    span.head = 0;
    span.tail = 0;
    n_rows = __builtin_amdgcn_readfirstlane(g.count) * a.rows - row0;
    v0 = split * __builtin_amdgcn_readfirstlane(g.size);
    n_pages = max(min(v0 + __builtin_amdgcn_readfirstlane(g.size),
                      min(__builtin_amdgcn_readfirstlane(g.pages), a.max_pages)) - v0, 0);
    first = args.shared_at + g.base + ((long long)split * a.hkv + kvh) * g.count * a.rows + row0;
    // Rows of all sequences of the group: from the group's first query on.
    b = __builtin_amdgcn_readfirstlane(b);
  } else {
    if (share >= a.batch * args.splits) return;
    b = share / a.by_splits;
    const int split = share - b * args.splits;
    len = max(scalar_load(a.seq_lens + b), 0);
    span = span_of(args, b, len);
    direct = !span.shared && span.count <= 1;
    if (split >= max(span.count, 1)) return;  // uniform
    v0 = split * span.size;
    n_pages = max(min(v0 + span.size, span.n) - v0, 0);
    n_rows = a.rows;
    first = ((long long)share * a.hkv + kvh) * a.rows;
  }
  v0 = __builtin_amdgcn_readfirstlane(v0);
  n_pages = __builtin_amdgcn_readfirstlane(n_pages);
  const int head = __builtin_amdgcn_readfirstlane(span.head);
  const int skip = __builtin_amdgcn_readfirstlane(span.tail - span.head);
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

  auto real = [&](int nb, int r) { return 16 * nb + r < n_rows; };
  // Place of a row in query and output, in rows of HD.
  auto out_row = [&](int nb, int r) -> long long {
    const int x = row0 + 16 * nb + r;
    int i = 0, y = x;
    long long at = b;
    if constexpr (SHARED) {
      i = x / args.by_rows;
      y = x - i * a.rows;
      at = args.groups[args.items[share].group].first + i;
    }
    const int qi = y / a.by_group;
    return (at * a.q_len + qi) * a.hq + kvh * a.group + (y - qi * a.group);
  };
  u4 q[NB][KK];
  RegBits<NB> bits;
  int from[NB];  // first token of the row's window
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const bool is = real(nb, l16);
    const _Float16* qp = a.q + (is ? out_row(nb, l16) : out_row(0, 0)) * HD;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const u4 x = *(const u4*)(qp + KV::q_dims(kk, g16));
      q[nb][kk] = is ? x : u4{0u, 0u, 0u, 0u};
    }
    if constexpr (!SHARED) {
      const int qi = is ? (16 * nb + l16) / a.by_group : 0;
      bits.b[nb] = draft_bits(a, b, qi, is);
      from[nb] = args.window > 0
                     ? (int)max((long long)len - a.q_len + qi + 1 - args.window, 0LL) : 0;
    }
  }

  const unsigned tok_bytes = a.token_stride;
  const unsigned k_lane = l16 * tok_bytes + kvh * a.head_stride + KV::k_lane_bytes(g16);
  const unsigned v_lane = 4 * g16 * tok_bytes + kvh * a.head_stride + KV::v_lane_bytes(l16);
  const size_t sub_bytes = (size_t)kPageSize * tok_bytes;
  // Lanes 0-31 load the page's K scale, 32-63 its V scale.
  const char* scale_lane = KV::kScaled
                               ? (const char*)(lane < 32 ? args.scales.k : args.scales.v) +
                                     (size_t)kvh * args.scales.head_stride
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
  // Masked pages: with a token from the draft block on, or before the last row's window and
  // past the first tokens.
  const int mask_from = len - a.q_len;
  const int all_from = SHARED || args.window <= 0
                           ? 0 : (int)max((long long)len - args.window, 0LL);

  for (int i = 0; i < n_pages; i += D) {
    load_ids(i + 2 * D, ids_next);
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int ii = i + j;
      if (ii < n_pages) {
        const int p = page_at(v0 + ii);
        const int t0 = p * kPageSize;
        const bool masked = !SHARED && (t0 + kPageSize > mask_from ||
                                        (t0 < all_from && t0 + kPageSize > args.sink));
        f4 s[NB];
        code_scores<NB, HD, E, KV>(s, ring[j].kv, q);
        auto mask = [&] {
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
            if constexpr (!SHARED) {
              // After the scales, so that one of 0, infinity or NaN leaves them -inf.
#pragma unroll
              for (int nb = 0; nb < NB; ++nb) s[nb] = s[nb] * c + lv;
              c = 1.f;
              add = 0.f;
              mask();
              if constexpr (KV::kNan) nan_values<NB, HD, KV>(st, ring[j].kv, s);
            }
          }
          scaled_page<NB, HD, KV>(st, ring[j].kv, s, masked, c, add, inv_vs, loud);
        } else {
          if (masked) {
            if constexpr (!SHARED) mask();
          }
          plain_page<NB, HD, E, KV>(st, ring[j].kv, s, masked, a.scale_log2, a.bf16);
        }
      }
      load_page(ii + D < n_pages ? clamp_page(ids[j], a.num_pages) : -1, page_at(v0 + ii + D),
                ring[j]);
    }
#pragma unroll
    for (int j = 0; j < D; ++j) ids[j] = ids_next[j];
  }
  leave_rows<NB, HD, E>(a, st, sm_stage + wave * 16 * (HD + 4), direct, first, real, out_row);
}

// Ring depths: about 32 KiB of a 16-bit cache or 16 of codes in flight per wave, half of
// that at 33 to 64 rows, whose accumulators take the registers.
template <int HD, typename E, typename KV, bool SHARED>
void launch_part_hd(const PartArgs& a, int rows, dim3 grid, hipStream_t stream) {
  constexpr int D = 4 * 128 / HD;
  const dim3 block(256);
  if (rows <= 16)
    hipLaunchKernelGGL((sqa_part_kernel<1, D, HD, E, KV, SHARED>), grid, block, 0, stream, a);
  else if (rows <= 32)
    hipLaunchKernelGGL((sqa_part_kernel<2, D, HD, E, KV, SHARED>), grid, block, 0, stream, a);
  else if constexpr (HD != 256)
    hipLaunchKernelGGL((sqa_part_kernel<4, D / 2, HD, E, KV, SHARED>), grid, block, 0, stream, a);
}

template <typename E, template <int> class KV, bool SHARED>
void launch_part_as(const PartArgs& a, int rows, dim3 grid, hipStream_t stream) {
  if (a.p.head_dim == 64)
    launch_part_hd<64, E, KV<64>, SHARED>(a, rows, grid, stream);
  else if (a.p.head_dim == 128)
    launch_part_hd<128, E, KV<128>, SHARED>(a, rows, grid, stream);
  else
    launch_part_hd<256, E, KV<256>, SHARED>(a, rows, grid, stream);
}

template <typename E, bool SHARED>
void launch_part(const PartArgs& a, int rows, dim3 grid, hipStream_t stream) {
  if (a.scaled && a.kv_type == kInt8)
    launch_part_as<E, PartCodesInt8, SHARED>(a, rows, grid, stream);
  else if (a.scaled)
    launch_part_as<E, PartCodesFp8, SHARED>(a, rows, grid, stream);
  else if (a.kv_type == kE4M3)
    launch_part_as<E, PartFp8, SHARED>(a, rows, grid, stream);
  else
    launch_part_as<E, PartNative, SHARED>(a, rows, grid, stream);
}

dim3 part_grid(const PartArgs& a, long long shares) {
  const int head_groups = (a.p.hkv + a.wg_heads - 1) / a.wg_heads;
  const int per_wg = 4 / a.wg_heads;
  return dim3((unsigned)((shares + per_wg - 1) / per_wg * head_groups));
}

}  // namespace
}  // namespace sqa

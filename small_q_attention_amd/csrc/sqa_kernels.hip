// gfx950 kernels for paged small-q (speculative-decoding "MTP") attention.
//
// Semantics (reference: /root/reference/src/small_q_attention/reference.py:46-72,
// csrc/small_q_attention_ext.cu:37-54): query head h reads kv head h / group;
// draft row qi of sequence b sees tokens t < seq_lens[b] - q_len + qi + 1;
// token t is slot t % 16 of page block_tables[b, t / 16]; scale head_dim^-1/2;
// fp32 softmax; fp16 output.
//
// Work decomposition. One workgroup owns one work item (sequence b, split: a
// range of its pages) for 4 kv heads, one wave per kv head. A wave holds every
// query row that reads its kv head: rows = q_len * group, row
// r = qi * group + g <-> query head kvh * group + g, so each K/V byte is loaded
// from HBM once and used by all rows straight from registers. The four waves
// walk the same pages in step, so a page's four 256-byte head slices per token
// are requested together (1 KiB contiguous runs).
//
// Per 16-token page a wave issues 4 K and 4 V 16-byte-per-lane buffer loads
// (1 KiB each).
//   S^T[token][row] = K . Q^T : v_mfma_f32_16x16x32_f16, A = K (lane l: token
//     l%16, 8 consecutive dims), B = Q^T (lane l: row l%16, same dims). The head
//     dimension is contracted in the order d = 32*kk + 8*(l/16) + e, which is
//     the same for A and B, so it needs no data movement.
//   O^T[d][row] += V^T . P^T : v_mfma_f32_16x16x16_f16. The S^T accumulator
//     (lane l: tokens 4*(l/16)+0..3 of row l%16) is exactly the B operand, so
//     P never leaves its registers. Lane l loads V rows 4*(l/16)+0..3, dims
//     8*(l%16)+0..7 (four full 256-byte rows per instruction) and regroups
//     them with one byte permute per half pair: output block mb covers dims
//     d = 8*m + mb, m = 0..15.
// Rows beyond q_len*group (q_len*group not a multiple of 16) carry some row's Q
// (zeros in the 8-wave kernel) and are never stored. The figures above are for head dim 128; the kernels are
// also built for 64 and 256 (HD), where the per-lane counts scale with HD
// (Dims<HD>) and a ring slot holds a page of HD-wide rows, and at head dim 64
// a wave takes two kv heads (HPW = 2; a workgroup then serves 8 kv heads):
// with up to 8 rows per kv head in one block (rows 0-7 and 8-15), with up to
// 16 or 32 in one or two blocks each (NB = 2 or 4). The element
// traits swap in the bf16 MFMAs (PV then as one 16x16x32 over P's high and low
// parts) and e4m3 K/V widened in registers; where the registers allow, the
// page loop runs the next page's QK products under this page's softmax.
#include "sqa_device.h"

namespace sqa {
namespace {

// One workgroup = one (sequence b, split) x WW waves; wave w serves the HPW kv
// heads from (head_group * WW + w) * HPW with all of their rows (NB blocks of
// 16; with HPW = 2 either one block, rows 0-7 of the first head and 8-15 of
// the second, or one block per head); WPE = waves per SIMD the register
// budget allows. All waves walk the
// same pages in the same order, so the heads' 256-byte slices of each page are
// requested together and HBM sees 1 KiB (4 heads) or 2 KiB (8 heads) runs; the
// head groups of a page range are dispatch neighbours. Each wave keeps its own
// softmax state and writes its own partials (or, with a single split, the
// output). Every K/V byte is read by one wave only, so the loads are
// non-temporal.
// The two kinds of plan are instantiations of their own (BAL: balanced), here and in
// the merge kernel: a call of a few pages runs almost every instruction for the
// first time, and the way to its first load led around the other plan's code (the
// GPU's part of a call, back to back, one kernel for both -> each its own: one
// sequence of 1K keys, q_len 2, 10.2 -> 9.3 us, where the whole call is bounded by the
// host's part, 12.4; of 8K, q_len 4, 13.85 -> 13.2, q_len 8 17.7 -> 16.7; of 4K, q_len
// 16, in the 8-wave kernel, 18.7 -> 17.3; long calls +-0.3%).
// The page ring runs through the pieces of an item: the next piece's first pages
// are requested in this one's last turn and its Q and mask words as soon as this
// one begins, so a sequence end costs the epilogue (about 1 us) and not a drained
// ring, a second barrier and three round trips (8.7 us at 16 ragged sequences of
// 2K-32K tokens). Whole calls, before -> after: 64 sequences of up to 512 keys at
// q_len 2 32.2 -> 27.5 us, 128 of up to 330 40.8 -> 34.3; 32 of up to 1K at q_len 8
// 36.4 -> 33.5; head dim 64, 4 of 2K, 18.7 -> 16.7 (there each thread also loaded
// nine page ids for every piece, now one for the item). Long uniform batches, whose
// items end with their sequences, are unchanged. What bounds it: HBM, and for few
// pages per item the start-up.
template <int NB, int D, int WW, int WPE, int HD, typename E, typename KV, int HPW, bool BAL,
          bool RB = false>
__global__ __launch_bounds__(WW * 64) __attribute__((amdgpu_waves_per_eu(WPE)))
void sqa_partial_kernel(PartialArgs a) {
  constexpr int KK = Dims<HD>::KK, MB = Dims<HD>::MB;
  // The arguments on the way to the first page ids, asked for together (one round
  // trip): left to itself the compiler loads them where they are first used, six
  // dependent trips through the scalar cache.
  asm volatile("" ::"s"(a.block_tables), "s"(a.seq_lens), "s"(a.batch), "s"(a.hkv),
               "s"(a.num_splits), "s"(a.pages_per_split), "s"(a.bt_stride), "s"(a.max_pages),
               "s"(a.page_shift), "s"(a.spec_pages), "s"(a.spec_pps), "s"(a.hg_items[0]),
               "s"(a.by_head_groups.mul), "s"(a.by_head_groups.shift), "s"(a.by_splits.mul),
               "s"(a.by_splits.shift));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // blockIdx.x = item * head_groups + head_group, or with items per head group
  // (hg_items) as head_group_items() deals them.
  const int head_groups = (a.hkv + WW * HPW - 1) / (WW * HPW);
  const bool hg_split = BAL && a.hg_items[0] > 0;
  const HeadGroupItems hgi =
      head_group_items(a.hg_items, a.batch, a.spec_pps, a.hg_spec_pps1, blockIdx.x);
  const int whole = (int)blockIdx.x / a.by_head_groups;
  const int hgrp = hg_split ? hgi.group : (int)blockIdx.x - whole * head_groups;
  const int item = hg_split ? hgi.item : whole;
  const PlanView view = hg_split ? plan_view(a, hgi) : plan_view(a);
  const int slot_heads = hg_split ? WW : a.hkv;  // partial slot layout (write_results)
  const int head0 = hg_split ? hgrp * WW : 0;
  const int slot_base = hg_split ? hgi.slot_base : 0;
  const int kvh = (hgrp * WW + wave) * HPW;  // the wave's first kv head
  // Waves past the last kv head (hkv not a multiple of WW * HPW) idle but stay
  // for the barrier.
  const bool active = kvh < a.hkv;
  const WaveRows<NB, HPW> map{kvh, a.rows, a.hkv};

  constexpr bool balanced = BAL;  // the plan; its code only
  const bool single = !balanced && a.num_splits == 1;  // no merge kernel follows

  // The page loop of each of the three forms below (see there).
  constexpr bool kPipelined = NB >= 2 && D >= 3 && NB * HD <= 256;
  constexpr bool kPairSteps = __is_same(E, ElemF16) && KV::kBytes == 1 && HD == 128 &&
                              NB == 4 && HPW == 1 && D % 2 == 0;
  static_assert(!RB || (!BAL && KV::kBytes == 2 && HD <= 128 && D >= kRingPages),
                "whole-ring steps: fixed plans over 16-bit K/V");
  constexpr bool kQRegs =
      ((NB == 4 && KV::kBytes == 1) || HD == 256) && HPW == 1 && !kPipelined;

  // LDS, all of it a wave's own but the page ids: the Q fragments of the wave's
  // rows, [buffer][nb][kk][lane] (the B-operand layout), and their draft-mask
  // words, twice (the piece at hand and the next one; once where the loop holds
  // Q in registers); the item's page ids (below); the results on their way out.
  constexpr int kQBufs = kQRegs || kPairSteps ? 1 : 2;
  constexpr int kQLds = NB * KK * 64;                    // u4 per wave and buffer
  constexpr int kBitsLds = NB * 32 < 64 ? 64 : NB * 32;  // dwords per wave and buffer
  // Ids of the item's pages in walking order, each piece padded with -1 to whole
  // turns of the ring: at most kMaxSplitPages pages in kMaxBalancedBatch pieces.
  constexpr int kIds = kMaxSplitPages + kMaxBalancedBatch * (D - 1) + 2 * D + 2;
  __shared__ u4 sm_q[WW * kQBufs * kQLds];
  __shared__ unsigned sm_bits[WW * 2 * kBitsLds];
  __shared__ float sm_stage[WW * 16 * (HD + 4)];
  __shared__ int sm_ids[kIds];

  // The first piece of the item and the ids of its first D pages, requested.
  ItemWalk walk;
  int first_id[D];
  if (!first_piece<D, false, BAL>(a, view, item, walk, first_id)) return;  // uniform
  ItemRange it = walk.it;
  const size_t first_slot = (size_t)it.slot0 + it.split;
  if (it.p_begin >= it.p_end && !single) {  // fixed plan only
    if (active) write_empty_split<NB>(a, map, first_slot, it.n_valid == 1 ? -1.f : 0.f);
    return;  // uniform
  }
  const int tid = piece_tid();
  const int lane = tid & 63;
  const int g16 = lane >> 4;
  const int l16 = lane & 15;
  const int shift = a.page_shift;
  const int sub_mask = (1 << shift) - 1;
  auto padded = [](int n) { return (n + D - 1) / D * D; };

  // Q fragments and mask words of a piece's rows on their way into buffer `buf`
  // (padding rows take some row's, unused).
  u4* my_q = sm_q + wave * kQBufs * kQLds;
  unsigned* my_bits = sm_bits + wave * 2 * kBitsLds;
  auto fetch_rows = [&](int b, int buf) {
    if (!active) return;  // uniform
    const int t = piece_tid() & 63;
    const int tg = t >> 4, tl = t & 15;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = map.row(nb, tl);
      const bool real = map.real(nb, tl);
      const int qi = real ? r / a.by_group : 0;
      const int gg = real ? r - qi * a.group : 0;
      const int hh = (real ? map.head(nb, tl) : map.kvh) * a.group + gg;
      const _Float16* qp = a.q + ((size_t)(b * a.q_len + qi) * a.hq + hh) * HD;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        copy16_to_lds(qp + KV::q_dims(kk, tg),
                      (unsigned)(size_t)(my_q + ((buf % kQBufs) * NB + nb) * KK * 64 + kk * 64));
    }
    if (a.draft_mask != nullptr) {  // uniform
#pragma unroll
      for (int i = 0; i < kBitsLds / 64; ++i) {
        // Lane t fills dword 64 i + t: block nb, word w, row slot r.
        const int nb = min(2 * i + (t >> 5), NB - 1), w = (t >> 4) & 1;
        const int qi = map.real(nb, tl) ? map.row(nb, tl) / a.by_group : 0;
        copy4_to_lds(a.draft_mask + (size_t)(b * a.q_len + qi) * a.mask_words +
                         (a.mask_words > 1 ? w : 0),
                     (unsigned)(size_t)(my_bits + buf * kBitsLds + 64 * i));
      }
    }
  };

  // Ids of the item's pages, entry tid of each run of WW * 64: the address in the
  // block table, found piece by piece, or -1 (padding). Long items (more than one
  // run, so hundreds of pages) fill all but the first run here; the first run's
  // loads go out with Q and the first pages below.
  const int32_t* ids_base =
      balanced ? a.block_tables : a.block_tables + (size_t)it.b * a.bt_stride;
  int n_flat = 0;
  auto id_at = [&](int e) {
    walk.it = it;
    int at = -1;
    n_flat = 0;
    do {  // uniform
      const int n = walk.it.p_end - walk.it.p_begin;
      const int rel = e - n_flat;
      if (rel >= 0 && rel < n)
        at = (balanced ? walk.it.b * a.bt_stride : 0) + ((walk.it.p_begin + rel) >> shift);
      n_flat += padded(n);
    } while (balanced && piece_at(a, walk, item, walk.it.g_end));
    return at;
  };
  const int at0 = id_at(tid);
  for (int e = WW * 64; e < n_flat; e += WW * 64) {  // uniform
    const int at = id_at(e + tid);
    const int x = ids_base[max(at, 0)];
    if (e + tid < kIds) sm_ids[e + tid] = at >= 0 ? clamp_page(x, a.num_pages) : -1;
  }
  const int id0 = ids_base[max(at0, 0)];
  fetch_rows(it.b, 0);

  // K/V pages are read with buffer loads: the resource (4 SGPRs) is rebuilt per
  // page at the page's base address and bounded to the page, and the lane
  // offsets below stay in one VGPR each for the whole loop.
  const int kvh_c = active ? kvh : 0;
  const unsigned tok_bytes = a.token_stride;
  const unsigned k_lane = l16 * tok_bytes + kvh_c * a.head_stride + KV::k_lane_bytes(g16);
  const unsigned v_lane = 4 * g16 * tok_bytes + kvh_c * a.head_stride + KV::v_lane_bytes(l16);
  // Offset of the wave's second head (the first head again if it does not exist).
  const unsigned head1 = HPW == 2 && kvh_c + 1 < a.hkv ? a.head_stride : 0u;
  // pid < 0 gives a zero-length resource: the loads return zeros without
  // touching memory, so every slot refill below is unconditional and the
  // compiler's wait counts stay exact (one page retires per step). K/V are
  // streamed once, so the loads are non-temporal.
  // Kernel page p of the sequence is sub-page p & sub_mask of cache page
  // block_tables[b][p >> shift].
  const size_t sub_bytes = (size_t)kPageSize * tok_bytes;
  auto load_page = [&](int pid, int p, typename KV::Regs (&pg)[HPW]) {
    // The page is the same for the whole wave: its resource lives in SGPRs.
    pid = __builtin_amdgcn_readfirstlane(pid);
    const size_t off =
        pid >= 0 ? (size_t)pid * (size_t)a.page_stride + (size_t)(p & sub_mask) * sub_bytes : 0;
    const int nrec = pid >= 0 ? (int)a.page_extent : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((const char*)a.k + off), (short)0, nrec, kBufferFlags);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((const char*)a.v + off), (short)0, nrec, kBufferFlags);
    KV::load(pg[0], kr, vr, k_lane, v_lane, tok_bytes);
    if constexpr (HPW == 2) KV::load(pg[HPW - 1], kr, vr, k_lane + head1, v_lane + head1, tok_bytes);
  };
  // Ring of D pages in flight: page i is processed from slot i % D, which is
  // then refilled with page i + D, past a piece's (padded) end with the next
  // piece's first pages: the ring runs through the piece boundaries of an item.
  typename KV::Regs ring[D][HPW];
#pragma unroll
  for (int j = 0; j < D; ++j) {
    load_page(active && j < it.p_end - it.p_begin ? clamp_page(first_id[j], a.num_pages) : -1,
              it.p_begin + j, ring[j]);
  }
  sm_ids[tid] = at0 >= 0 ? clamp_page(id0, a.num_pages) : -1;
  __syncthreads();  // the ids are in LDS: the item's only barrier
  if (!active) return;  // uniform over the wave: no barrier follows
  auto page_id = [&](int i) -> int {
    const int x = sm_ids[i];
    return i < n_flat ? x : -1;
  };
  const bool upper = l16 >= 8;
  static_assert(WW * 64 <= kIds, "the first run of ids fits the table");

  // Each piece of the work item (one, except where a balanced item spans the end
  // of a sequence): its page range of one sequence, ids from table entry f on.
  int f = 0;
  for (int buf = 0;; buf ^= 1) {
  const int len = it.len;
  const int p_begin = it.p_begin;
  const int n_pages = it.p_end - it.p_begin;
  const int n_padded = padded(max(n_pages, 0));
  // A sequence with at most one split is finished here; otherwise this
  // workgroup leaves a partial for the merge kernel.
  const bool direct = it.n_valid <= 1;
  const size_t slot = (size_t)it.slot0 + it.split;
  // The piece after this one: its first pages enter the ring during this one's
  // last turn, its Q fragments now (with one buffer: once this piece's are in
  // registers).
  walk.it = it;
  const bool more = balanced && piece_at(a, walk, item, it.g_end);
  const int next_begin = walk.it.p_begin;
  if (kQBufs == 2 && more) fetch_rows(walk.it.b, buf ^ 1);
  // This piece's Q and mask words are in LDS: D pages were requested after them, each
  // in kLoads instructions per head (tests/test_kernel_code_cpu.py counts them).
  wait_vmcnt_fence<D * HPW * KV::kLoads>();
  const u4* q_lds = my_q + (buf % kQBufs) * kQLds;
  const StagedBits<NB, HPW, kPairSteps> bits{my_bits + buf * kBitsLds, a.draft_mask != nullptr,
                                             a.mask_words > 1, a.by_group, l16, map};
  // Pages holding a token >= mask_from (draft block or past the end) are masked.
  const int mask_from = len - a.q_len;

  WaveState<NB, HD> st;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    st.m[nb] = -INFINITY;
    st.l[nb] = 0.f;
    st.thr[nb] = -INFINITY;
    st.nmu[nb] = -0.f;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) st.acc[mb][nb] = f4{0.f, 0.f, 0.f, 0.f};
  }
  u4 qf[kQRegs || kPairSteps ? NB : 1][KK];
  if constexpr (kQRegs || kPairSteps) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) qf[nb][kk] = q_lds[(nb * KK + kk) * 64 + lane];
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      fetch_rows(walk.it.b, buf ^ 1);
    }
  }

  // With two or four row blocks whose accumulators take at most 64 VGPRs
  // (NB * HD <= 256) the page loop is software-pipelined: the scores of page
  // i + 1 are issued before page i's mask, softmax and PV products, so their
  // MFMAs run under the softmax (16 x 32K keys, head dim 64: q16 177.7 -> 173.8
  // us, e4m3 q8 / q16 117.2 / 168.5 -> 111.6 / 154.2 us; head dim 128 q8 317.5
  // -> 316.1 us; bit-identical results). Page i + 1 must then be resident one
  // step earlier and its scores held alongside: with 128 accumulator VGPRs
  // (head dim 128 at 64 rows) the extra registers spill (e4m3 q16 261 -> 269
  // us), with a ring of 2 the wait is longer (head dim 256: 662 -> 916 us),
  // and at one block there is little softmax to hide (e4m3 head dim 64 q4:
  // -1.5%).
  // fp16 queries over an e4m3 cache at 64 rows and head dim 128 take the
  // pages two at a time (pair_finish).
  // Splits that fit the ring in one softmax step (below) in instantiations of their
  // own, RB, for fixed plans of so few pages per split: 16-bit K/V, whose ring
  // registers the MFMAs read as they are. Balanced items of so few pages take the
  // loop: the step's refill of the ring for the next piece waited for its loads (4
  // sequences of 1000 keys under a wide table, q_len 2 / 4 / 8: 14.9 / 15.0 / 18.0 us
  // per call with the step, 13.3 / 13.6 / 15.9 without), and the bits would follow the
  // pages a caller expects.
  int next_pid = page_id(f + D);
  if constexpr (kPairSteps) {
    // The Q fragments stay in registers for the whole loop (16 x 4 dwords; the
    // ring, scores and accumulators take the 256 arch VGPRs, so they live in
    // AGPRs, which the MFMAs read directly). Left to itself the compiler
    // copied every fragment to a second set of AGPRs before each pair (104
    // v_accvgpr_mov per 4 pages); the empty asm below states that the values
    // sit in AGPRs at that point, and the copies are gone (cfg3 shape q16:
    // 217.8 -> 209.6 us).
    for (int i = 0; i < n_pages; i += D) {
      const int p_ahead = i + D < n_padded ? p_begin + i + D : next_begin;
#pragma unroll
      for (int j = 0; j < D; j += 2) {
        const int ii = i + j;
        if (ii < n_pages) {
          const int p = p_begin + ii;
          const bool masked = (p + 2) * kPageSize > mask_from;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) asm volatile("" : "+a"(qf[nb][kk]));
          f4 s0[NB], s1[NB];
          // One page's scores after the other: one widened K page live at a time
          // (interleaving the two pages' MFMA chains kept both live and spilled
          // registers to AGPRs; cfg3 shape q16 202.9 -> 200.5 us, ragged 114.0 ->
          // 110.3 us).
          {
            const PageK<HD, 1> k0 = widen_k<E, KV, HD, 1>(ring[j]);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              s0[nb] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int kk = 0; kk < KK; ++kk) s0[nb] = E::mma_qk(k0.k[0][kk], qf[nb][kk], s0[nb]);
            }
          }
          {
            const PageK<HD, 1> k1 = widen_k<E, KV, HD, 1>(ring[j + 1]);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              s1[nb] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int kk = 0; kk < KK; ++kk) s1[nb] = E::mma_qk(k1.k[0][kk], qf[nb][kk], s1[nb]);
            }
          }
          pair_finish<NB>(st, s0, s1, ring[j][0], ring[j + 1][0], ii + 1 < n_pages, bits,
                          mask_from, p * kPageSize, len, masked, a.scale_log2);
        }
        const int pid0 = next_pid;
        const int pid1 = page_id(f + ii + D + 1);
        next_pid = page_id(f + ii + D + 2);
        load_page(pid0, p_ahead + j, ring[j]);
        load_page(pid1, p_ahead + j + 1, ring[j + 1]);
      }
    }
  } else if constexpr (RB) {  // the whole split is in the ring
    // Short splits (one sequence of 8K keys in 4-page splits, every split of a
    // 1K-key sequence): the ring's pages arrive together, so they are taken in
    // one softmax step, all scores first, one running-max update, then the PV
    // products, instead of D dependent page steps (the MFMAs of all pages
    // issue back to back; one sequence of 8K keys, whole calls: q_len 2 14.1
    // -> 13.7 us, q_len 4 14.8 -> 14.2 us). Zero pages past the split take no
    // part.
    f4 sb[D][NB];
    PageV<HD, HPW> pvb[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      page_scores<NB, HD, E, KV, HPW>(sb[j], widen_k<E, KV, HD, HPW>(ring[j]), q_lds, lane, upper);
      pvb[j] = widen_v<E, KV, HD, HPW>(ring[j]);
    }
    float lm[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) lm[nb] = -INFINITY;
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int p = p_begin + j;
      if (j >= n_pages) {  // uniform
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) sb[j][nb] = f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      } else if ((p + 1) * kPageSize > mask_from) {  // uniform
        unsigned long long dbits[NB];
        bits.get(dbits);
        mask_page<NB, HD, HPW>(sb[j], pvb[j], dbits, mask_from, p * kPageSize + 4 * g16, len);
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) lm[nb] = fmaxf(lm[nb], max4(sb[j][nb]) * a.scale_log2);
    }
    raise_max<NB, HD>(st, lm);
#pragma unroll
    for (int j = 0; j < D; ++j)
      if (j < n_pages) page_pv<NB, HD, E, KV, HPW>(st, sb[j], pvb[j], upper, a.scale_log2);
  } else {
  f4 s_cur[NB];
  if constexpr (kPipelined)
    page_scores<NB, HD, E, KV, HPW>(s_cur, widen_k<E, KV, HD, HPW>(ring[0]), q_lds, lane, upper);
  // 64 rows over e4m3 outside the page pairs (bf16 queries), and head dim 256:
  // the Q fragments held in AGPRs for the loop, pinned there as in the pair
  // loop (the compiler had copied them between AGPR sets every page; cfg3
  // shape: bf16 / e4m3 q16 283.7 -> 271.0 us, head dim 256 q8 680.5 -> 668.7
  // us, e4m3 324.2 -> 322.2 us).
  for (int i = 0; i < n_pages; i += D) {
    const int p_ahead = i + D < n_padded ? p_begin + i + D : next_begin;
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int ii = i + j;
      if (ii < n_pages) {
        const int p = p_begin + ii;
        const bool masked = (p + 1) * kPageSize > mask_from;
        if constexpr (kPipelined) {
          // Slot (j + 1) % D holds page ii + 1 (a zero page past the split).
          f4 s_next[NB];
          page_scores<NB, HD, E, KV, HPW>(s_next, widen_k<E, KV, HD, HPW>(ring[(j + 1) % D]),
                                          q_lds, lane, upper);
          PageV<HD, HPW> pv = widen_v<E, KV, HD, HPW>(ring[j]);
          page_finish<NB, HD, E, KV, HPW>(st, s_cur, pv, upper, bits, mask_from,
                                          p * kPageSize + 4 * g16, len, masked, a.scale_log2);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) s_cur[nb] = s_next[nb];
        } else {
          // K and V widened together, then the scores (the order that schedules
          // best where no pipelining is done).
          const PageK<HD, HPW> kf = widen_k<E, KV, HD, HPW>(ring[j]);
          PageV<HD, HPW> pv = widen_v<E, KV, HD, HPW>(ring[j]);
          if constexpr (kQRegs) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
              for (int kk = 0; kk < KK; ++kk) asm volatile("" : "+a"(qf[nb][kk]));
              s_cur[nb] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int kk = 0; kk < KK; ++kk)
                s_cur[nb] = E::mma_qk(kf.k[0][kk], qf[nb][kk], s_cur[nb]);
            }
          } else {
            page_scores<NB, HD, E, KV, HPW>(s_cur, kf, q_lds, lane, upper);
          }
          page_finish<NB, HD, E, KV, HPW>(st, s_cur, pv, upper, bits, mask_from,
                                          p * kPageSize + 4 * g16, len, masked, a.scale_log2);
        }
      }
      const int pid = next_pid;
      next_pid = page_id(f + ii + D + 1);
      load_page(pid, p_ahead + j, ring[j]);
    }
  }
  }
  write_results<NB, HD, E>(a, st, sm_stage + wave * 16 * (HD + 4), map, direct,
                           !single && !balanced, it.b, slot + slot_base, slot_heads, head0);
  if (!more) break;  // uniform
  f += n_padded;
  it = walk.it;
  }
}

// The rows of one wave of the 8-wave kernel: rows base .. base + 31 of kv head
// kvh (two 16-row blocks).
struct HalfRows {
  int kvh, rows, hkv, base;
  __device__ __forceinline__ int head(int, int) const { return kvh; }
  __device__ __forceinline__ int row(int nb, int r) const { return base + 16 * nb + r; }
  __device__ __forceinline__ bool real(int nb, int r) const {
    return kvh < hkv && row(nb, r) < rows;
  }
};

// s_waitcnt vmcnt(n) with the other counters left alone (gfx9 encoding: vmcnt in
// bits 3:0 and 15:14, expcnt 6:4, lgkmcnt 11:8).
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt holds 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// One 16-byte non-temporal buffer load per lane straight into LDS (gfx950
// buffer_load_dwordx4 ... lds): lane l's 16 bytes land at LDS byte address
// lds + 16 l. Written as inline asm on purpose: the compiler's own wait-count
// pass, seeing such a load, waits for all vector memory (vmcnt(0)) before every
// later LDS read that might alias it, which would drain a ring of these loads at
// each step; the callers place their vmcnt waits themselves and issue no other
// vector-memory loads meanwhile. m0 (the LDS base of the load) is saved and
// restored around it, with the wait state (s_nop) that a load into LDS needs after a
// write of m0.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, unsigned voffset,
                                            unsigned lds) {
  unsigned saved;
  asm volatile(
      "s_mov_b32 %[saved], m0\n\t"
      "s_mov_b32 m0, %[lds]\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %[off], %[rsrc], 0 offen nt lds\n\t"
      "s_mov_b32 m0, %[saved]"
      : [saved] "=&s"(saved)
      : [lds] "s"(lds), [off] "v"(voffset), [rsrc] "s"(rsrc)
      : "memory");
}

// LDS layout of one head's page slice (16 tokens x HD elements of the cache's
// type) for the 8-wave kernel, and the reads that turn it into the register
// form KV::load gives the main kernel (KV::Regs), so the math is shared.
// 16-bit caches: 16 chunks of 16 bytes per token; chunk c of token t sits at
// position 16 t + (c ^ t), so the 16 tokens an MFMA operand read takes at one
// chunk fall in 16 different bank groups.
template <typename KV>
struct LdsSlice;

template <>
struct LdsSlice<KvNative<128>> {
  static constexpr int kChunks = 16;  // 16-byte chunks per token row (256 bytes)
  __device__ __forceinline__ static int pos(int t, int c) { return 16 * t + (c ^ t); }
  __device__ __forceinline__ static int token_of(int p) { return p >> 4; }
  __device__ __forceinline__ static int chunk_of(int p) { return (p & 15) ^ (p >> 4); }
  // K fragment kk of lane (g, l16): token l16, dims 32 kk + 8 g (chunk 4 kk + g);
  // V: tokens 4 g + e, dims 8 l16 .. + 7 (chunk l16).
  __device__ __forceinline__ static void read(KvNative<128>::Regs& r, const char* ks,
                                              const char* vs, int g, int l16) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) r.k[kk] = *(const u4*)(ks + 16 * pos(l16, 4 * kk + g));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const u4 x = *(const u4*)(vs + 16 * pos(4 * g + e, l16));
#pragma unroll
      for (int w = 0; w < 4; ++w) r.v[e][w] = x[w];
    }
  }
};

// 33..64 query rows per kv head (q_len 16 at GQA 4) at head dim 128. Eight
// waves per workgroup: two per kv head, each with 32 of the head's rows in two
// 16-row blocks (the 32-row math), so no wave holds the 128 accumulator
// registers of 64 rows, and two waves share each SIMD, one's MFMAs under the
// other's softmax. The two waves of a head read each page once between them:
// the workgroup's K and V of 4 heads (32 KiB a page of 16-bit K and V) arrive
// in a ring of D LDS slots by direct buffer loads
// (load_to_lds: 1 KiB of a head's page slice per wave and load, in the layout of
// LdsSlice), so the bytes in flight take no registers. Per page: wait for this
// thread's loads of the page (manual vmcnt: nothing else in the loop touches
// vector memory), one barrier (the page is in LDS, and every wave has read the
// previous page's slot, which it did before that page's math), read the wave's K
// and V into registers, refill the previous page's slot with the page D - 1
// ahead, then the math: D - 1 pages stay in flight. One barrier a page rather
// than two (read, barrier, refill this page's slot with D in flight) measured
// 0.3% faster for fp16 and 3.8% for bf16 at KV 32K x 16 sequences. Pages past the
// split load through a zero-length resource (zeros, no memory traffic), as in
// sqa_partial_kernel.
template <int D, typename E, typename KV, bool BAL>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2)))
void sqa_partial_lds_kernel(PartialArgs a) {
  constexpr int HD = 128, NB = 2, KK = Dims<HD>::KK, MB = Dims<HD>::MB;
  using L = LdsSlice<KV>;
  constexpr int kHeadSlice = 16 * L::kChunks * 16;  // one head's K (or V) of a page
  constexpr int kSlot = 2 * 4 * kHeadSlice;         // K and V of 4 heads
  constexpr int kLoads = kSlot / (512 * 16);        // loads per thread and page
  constexpr int kThreads = 512;
  static_assert(HD * KV::kBytes == 16 * L::kChunks, "a token row is kChunks 16-byte chunks");
  // As in sqa_partial_kernel: one round trip for the arguments.
  asm volatile("" ::"s"(a.block_tables), "s"(a.seq_lens), "s"(a.batch), "s"(a.hkv),
               "s"(a.num_splits), "s"(a.pages_per_split), "s"(a.bt_stride), "s"(a.max_pages),
               "s"(a.page_shift), "s"(a.spec_pages), "s"(a.spec_pps), "s"(a.pair_items),
               "s"(a.by_head_groups.mul), "s"(a.by_head_groups.shift), "s"(a.by_splits.mul),
               "s"(a.by_splits.shift));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // blockIdx.x = item * head_groups + head_group; with paired items (two head
  // groups), 4k + 2 head_group + (item & 1) for item 2k + (item & 1), so both
  // workgroups of an item run on XCDs of the item's parity. wave = half * 4 +
  // head slot.
  const int head_groups = (a.hkv + 3) / 4;
  const bool pairs = BAL && a.pair_items != 0;
  const int whole = (int)blockIdx.x / a.by_head_groups;
  const int hgrp = pairs ? (blockIdx.x & 3) >> 1 : blockIdx.x - whole * head_groups;
  const int item = pairs ? (blockIdx.x >> 2) * 2 + (blockIdx.x & 1) : whole;
  const int hs = wave & 3;
  const int kvh = hgrp * 4 + hs;
  const HalfRows map{kvh, a.rows, a.hkv, 32 * (wave >> 2)};
  // Waves without rows (a head past the last, or no rows past 32) still load
  // and meet the barriers; they skip the math.
  const bool active = kvh < a.hkv && map.base < a.rows;

  constexpr bool balanced = BAL;
  const bool single = !balanced && a.num_splits == 1;
  static_assert(D + 1 <= kIdPad, "page-id table padding must cover the ring's look-ahead");
  constexpr int kIdSlots = (kMaxSplitPages + kIdPad + kThreads - 1) / kThreads;
  // The ring and, after a piece's page loop, the waves' output staging.
  __shared__ __attribute__((aligned(16))) char sm_ring[D * kSlot];
  __shared__ int sm_ids[kIdSlots * kThreads];
  // Load i of a thread fills 1 KiB piece ci = 8 i + wave of a slot: K (first
  // half of the pieces) or V, head slot (ci / parts) % 4, part ci % parts of the
  // head's slice; lane l fills position 64 part + l, i.e. chunk
  // L::chunk_of(position) of token L::token_of(position).
  constexpr int kParts = kHeadSlice / 1024;  // 1 KiB pieces per head slice
  const unsigned tok_bytes = a.token_stride;
  unsigned voff[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int ci = 8 * i + wave;
    const int pos = 64 * (ci % kParts) + (threadIdx.x & 63);
    voff[i] = L::token_of(pos) * tok_bytes + (hgrp * 4 + (ci / kParts) % 4) * a.head_stride +
              16 * L::chunk_of(pos);
  }

  // Paired items: the page loop's time (100 MHz counter) and pages, for the
  // merge kernel's choice of the next call's item sizes under adaptive pairs
  // (zero if the item has no piece).
  float loop_ticks = 0.f;
  int loop_pages = 0;
  const bool paired_call =
      for_each_piece<D, BAL>(a, plan_view(a), item, [&](const ItemRange& it, const int (&first_id)[D]) {
  const int tid = piece_tid();
  const int lane = tid & 63;
  const int g16 = lane >> 4;
  const int l16 = lane & 15;
  const int b = max(it.b, 0);
  const int len = it.len;
  const int p_begin = it.p_begin;
  const int p_end = it.p_end;
  const int32_t* bt_row = a.block_tables + (size_t)b * a.bt_stride;
  const int shift = a.page_shift;
  const int sub_mask = (1 << shift) - 1;
  if (it.b < 0) return;  // uniform
  const bool direct = it.n_valid <= 1;
  const size_t slot = (size_t)it.slot0 + it.split;
  if (p_begin >= p_end && !single) {  // fixed plan only
    write_empty_split<NB>(a, map, slot, it.n_valid == 1 ? -1.f : 0.f);
    return;  // uniform
  }
  const int n_split = p_end > p_begin ? p_end - p_begin : 0;

  // Q fragments (kept in registers), draft bits, then the split's page ids.
  u4 qreg[NB][KK];
  RegBits<NB> bits;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = map.row(nb, l16);
    const bool real = map.real(nb, l16);
    const int qi = real ? r / a.by_group : 0;
    const int gg = real ? r - qi * a.group : 0;
    const int hh = real ? kvh * a.group + gg : 0;
    const _Float16* qp = a.q + ((size_t)(b * a.q_len + qi) * a.hq + hh) * HD;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const u4 x = *(const u4*)(qp + KV::q_dims(kk, g16));
      qreg[nb][kk] = real ? x : u4{0u, 0u, 0u, 0u};
    }
    bits.b[nb] = draft_bits(a, b, qi, real);
  }
  int idreg[kIdSlots];
  const int last_id = n_split > 0 ? n_split - 1 : 0;
#pragma unroll
  for (int k = 0; k < kIdSlots; ++k) {
    const int i = tid + k * kThreads;
    const int x = bt_row[(p_begin + min(i, last_id)) >> shift];
    idreg[k] = i < n_split ? x : -1;
  }

  const size_t sub_bytes = (size_t)kPageSize * tok_bytes;
  auto issue_page = [&](int pid, int p, int j) {
    // The page is the same for the whole workgroup: its resource lives in SGPRs.
    pid = __builtin_amdgcn_readfirstlane(pid);
    const size_t off =
        pid >= 0 ? (size_t)pid * (size_t)a.page_stride + (size_t)(p & sub_mask) * sub_bytes : 0;
    const int nrec = pid >= 0 ? (int)a.page_extent : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((const char*)a.k + off), (short)0, nrec, kBufferFlags);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((const char*)a.v + off), (short)0, nrec, kBufferFlags);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_to_lds(i < kLoads / 2 ? kr : vr, voff[i],
                  (unsigned)(size_t)(sm_ring + j * kSlot + (8 * i + wave) * 1024));
  };
#pragma unroll
  for (int j = 0; j < D - 1; ++j)
    issue_page(j < n_split ? clamp_page(first_id[j], a.num_pages) : -1, p_begin + j, j);
#pragma unroll
  for (int k = 0; k < kIdSlots; ++k) {
    const int i = tid + k * kThreads;
    sm_ids[i] = idreg[k] >= 0 ? clamp_page(idreg[k], a.num_pages) : -1;
  }
  const int mask_from = len - a.q_len;

  WaveState<NB, HD> st;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    st.m[nb] = -INFINITY;
    st.l[nb] = 0.f;
    st.thr[nb] = -INFINITY;
    st.nmu[nb] = -0.f;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) st.acc[mb][nb] = f4{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();  // sm_ids written

  const unsigned long long t_loop = it.paired ? __builtin_amdgcn_s_memrealtime() : 0;
  int next_pid = sm_ids[D - 1];
  for (int i = 0; i < n_split; i += D) {
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int ii = i + j;
      if (ii < n_split) {  // uniform over the workgroup
        wait_vmcnt<kLoads * (D - 2)>();  // this thread's loads of page ii
        __syncthreads();  // page ii is in slot j; every wave is done with page ii - 1
        const char* ks = sm_ring + j * kSlot + hs * kHeadSlice;
        typename KV::Regs raw[1];
        L::read(raw[0], ks, ks + 4 * kHeadSlice, g16, l16);
        const int pid = next_pid;
        next_pid = sm_ids[ii + D];
        issue_page(pid, p_begin + ii + D - 1, (j + D - 1) % D);
        if (active) {
          const int p = p_begin + ii;
          const bool masked = (p + 1) * kPageSize > mask_from;
          const PageK<HD, 1> kf = widen_k<E, KV, HD, 1>(raw);
          PageV<HD, 1> pv = widen_v<E, KV, HD, 1>(raw);
          f4 sc[NB];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            sc[nb] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) sc[nb] = E::mma_qk(kf.k[0][kk], qreg[nb][kk], sc[nb]);
          }
          page_finish<NB, HD, E, KV, 1>(st, sc, pv, false, bits, mask_from,
                                        p * kPageSize + 4 * g16, len, masked, a.scale_log2);
        }
      }
    }
  }
  if (it.paired) {
    loop_ticks = (float)(__builtin_amdgcn_s_memrealtime() - t_loop);
    loop_pages = n_split;
  }
  // Loads past the piece still write (zeros) into the ring: drain them before
  // the ring becomes the output staging.
  wait_vmcnt<0>();
  __syncthreads();
  if (active)
    write_results<NB, HD, E>(a, st, (float*)sm_ring + wave * 16 * (HD + 4), map, direct,
                             !single && !balanced, b, slot, a.hkv, 0);
  });
  // An adaptive paired call (the same answer in every workgroup) leaves a record
  // from every workgroup. Whenever adaptive pairing was asked for, workgroup 0
  // stamps the call (or clears the stamp when the lengths made it fall back):
  // the merge kernel reads the records only under a stamp of this call.
  if (BAL && a.pair_items == kPairsAdaptive && threadIdx.x == 0) {
    if (paired_call)
      *(int2*)(a.tune + 4 + 2 * blockIdx.x) =
          int2{__float_as_int(loop_ticks), loop_pages | (item & 1) << 30 | 1 << 31};
    if (blockIdx.x == 0) a.tune[2] = paired_call ? __uint_as_float(kTuneStamp) : 0.f;
  }
}

// Log-sum-exp merge of split partials (reference: csrc/small_q_attention_ext.cu:339-366):
// M = max_s m_s; O = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M); splits
// with l_s <= 0 are skipped and a row with no visible key is written as 0.
// fp16 partials hold acc_s / l_s (so acc_s = l_s times the stored row).
//
// One pass, every load of a round in flight at once: TPR threads serve one
// output row; each thread owns the 16 bytes of a partial row at dims DPT c ..
// DPT c + DPT - 1 (DPT = 8 fp16 or 4 fp32 values) and the splits g, g + SG, ...
// of its split group g, U splits per round (one round wherever the row's
// splits allow: the round trip to the partials, not their bytes, sets the
// time). Each group keeps a running max and rescales its sums when the max
// grows (as the online softmax does), so no pass over the maxima precedes the
// sums; the groups then meet by shuffles within a wave and in LDS across the
// row's waves.
// A (first slot, count) entry held to the slots that exist, whatever the table
// holds (the partial kernel writes it within them).
__device__ __forceinline__ SeqSplits in_range(SeqSplits t, int num_splits) {
  t.first = min(max(t.first, 0), num_splits - 1);
  t.count = min(max(t.count, 0), num_splits - t.first);
  return t;
}

// Paired items: the next call's delta from this call's page-loop times (one
// workgroup of 256 threads). Even items took P + d pages, odd ones P - d; with
// per-page times t_e and t_o the two end together at delta = (t_o - t_e) /
// (t_o + t_e), whatever this call's delta was. The new value moves halfway
// there (one call's times are noisy), within +-kPairDeltaMax. Only after a
// call that ran paired (its stamp in tune[2]); the stamp is cleared with the
// records, so a later call that did not pair (a length that differs) changes
// nothing.
__device__ __noinline__ void update_pair_delta(float* tune, int records) {
  __shared__ float sums[4][4];
  const int t = threadIdx.x;
  if (__float_as_uint(tune[2]) != kTuneStamp) return;  // uniform over the workgroup
  float te = 0.f, pe = 0.f, to = 0.f, po = 0.f;
  for (int i = t; i < records; i += 256) {
    const int2 r = *(const int2*)(tune + 4 + 2 * i);
    if (r.y < 0) {  // recorded by this call's partial kernel
      const float pages = (float)(r.y & 0x3fffffff);
      const float ticks = __int_as_float(r.x);
      if ((r.y >> 30) & 1) {
        to += ticks;
        po += pages;
      } else {
        te += ticks;
        pe += pages;
      }
    }
  }
  for (int o = 32; o >= 1; o >>= 1) {
    te += __shfl_xor(te, o);
    pe += __shfl_xor(pe, o);
    to += __shfl_xor(to, o);
    po += __shfl_xor(po, o);
  }
  if ((t & 63) == 0) {
    sums[t >> 6][0] = te;
    sums[t >> 6][1] = pe;
    sums[t >> 6][2] = to;
    sums[t >> 6][3] = po;
  }
  __syncthreads();
  if (t == 0) {
    te = sums[0][0] + sums[1][0] + sums[2][0] + sums[3][0];
    pe = sums[0][1] + sums[1][1] + sums[2][1] + sums[3][1];
    to = sums[0][2] + sums[1][2] + sums[2][2] + sums[3][2];
    po = sums[0][3] + sums[1][3] + sums[2][3] + sums[3][3];
    if (pe > 0.f && po > 0.f && te > 0.f && to > 0.f) {
      const float ue = te / pe, uo = to / po;
      const float target = (uo - ue) / (uo + ue);
      float old = __float_as_uint(tune[0]) == kTuneMagic ? tune[1] : 0.f;
      old = old == old ? fminf(fmaxf(old, -kPairDeltaMax), kPairDeltaMax) : 0.f;
      tune[1] = fminf(fmaxf(0.5f * (old + target), -kPairDeltaMax), kPairDeltaMax);
      tune[0] = __uint_as_float(kTuneMagic);
    }
  }
  // Records and stamp are marked as read: a later call that writes none changes
  // nothing.
  for (int i = t; i < records; i += 256) tune[4 + 2 * i + 1] = 0.f;
  if (t == 0) tune[2] = 0.f;
}

template <int N>
struct Count {
  static constexpr int value = N;
};

template <int TPR, int HD, typename E, int U, bool BAL>
__global__ __launch_bounds__(256) void sqa_merge_kernel(MergeArgs a) {
  // Each thread owns DPT dims of the row, 16 bytes of every partial row (fp16
  // partials: 8 dims; fp32: 4), and the splits g, g + SG, ... of its split
  // group g; a row's TPR threads cover SG = TPR / CH splits per load
  // instruction and U SG splits per round.
  constexpr int DPT = E::kHalfPartials ? 8 : 4;
  constexpr int CH = HD / DPT;      // threads per partial row
  constexpr int SG = TPR / CH;      // split groups of a row
  constexpr int WPR = TPR / 64;     // waves of a row (0: several rows per wave)
  constexpr int RPW = 256 / TPR;    // rows per workgroup
  static_assert(SG >= 1 && TPR % CH == 0 && 256 % TPR == 0, "a row's threads must cover its dims");
  static_assert(SG == 1 || WPR >= 1, "split groups meet within whole waves");
  // The arguments in one round trip, as in sqa_partial_kernel.
  asm volatile("" ::"s"(a.part_o), "s"(a.part_ml), "s"(a.seq_splits), "s"(a.batch), "s"(a.q_len),
               "s"(a.hq), "s"(a.hkv), "s"(a.group), "s"(a.rows), "s"(a.pages_per_split),
               "s"(a.num_splits), "s"(a.spec_pages), "s"(a.spec_pps), "s"(a.hg_items[0]),
               "s"(a.by_hq.mul), "s"(a.by_hq.shift), "s"(a.by_seq_rows.mul),
               "s"(a.by_seq_rows.shift), "s"(a.by_group.mul), "s"(a.by_group.shift),
               "s"(a.by_spec_pps.mul), "s"(a.by_spec_pps.shift), "s"(a.tune), "s"(a.out),
               "s"(a.out_scale));
  const int t = threadIdx.x;
  const int tr = t % TPR;
  const int c = tr % CH;
  const int g = tr / CH;
  // Where a row's threads are whole waves everything about the row is uniform.
  // Several rows per wave are dealt out over the grid, so that the rows of one long
  // sequence do not meet in a few workgroups.
  const int row =
      WPR >= 1 ? blockIdx.x * RPW + __builtin_amdgcn_readfirstlane(t / TPR)
               : (t / TPR) * gridDim.x + blockIdx.x;
  const int total = a.batch * a.q_len * a.hq;
  const bool live = row < total;  // uniform per row
  if (BAL && a.tune != nullptr && blockIdx.x == 0) update_pair_delta(a.tune, a.tune_records);
  const int rowc = live ? row : 0;
  const int b = rowc / a.by_seq_rows;
  const int row_of_seq = rowc - b * a.q_len * a.hq;
  const int qi = row_of_seq / a.by_hq;
  const int h = row_of_seq - qi * a.hq;
  const int kvh = h / a.by_group;
  const int r = qi * a.group + (h - kvh * a.group);

  // Where the row's splits are. Fixed plan: all num_splits slots of the
  // sequence, no length needed (splits past its pages hold l = 0, and l = -1
  // in split 0 says the partial kernel already wrote the row). Balanced plan:
  // the (first slot, count) table the partial kernel wrote; when every
  // sequence was expected to span spec_pages pages, the layout of that case
  // (sequence b's pages from b * spec_pages on, items of spec_pps pages) is
  // assumed while the table is read, and the row is merged again from the
  // table if the two differ.
  constexpr bool balanced = BAL;
  const bool expect = balanced && a.spec_pages > 0;
  // With items per head group (hg_items) the row's head group has its own
  // region of slots (four kv heads each), table, slot count and item size.
  const bool hg_split = BAL && a.hg_items[0] > 0;
  const int grp = kvh >> 2;
  const int num_splits = hg_split ? a.hg_items[grp] + a.batch : a.num_splits;
  const SeqSplits* seq_splits = a.seq_splits + (hg_split ? grp * a.batch : 0);
  const FastDiv by_spec_pps = hg_split && grp ? a.by_spec_pps1 : a.by_spec_pps;
  // items between consecutive splits of this row, and the row's item in split 0
  const size_t stride = (size_t)(hg_split ? 4 : a.hkv) * a.rows;
  const size_t row_item =
      hg_split ? ((size_t)(grp ? a.hg_items[0] + a.batch : 0) * 4 + (kvh & 3)) * a.rows + r
               : (size_t)kvh * a.rows + r;
  int n_valid, slot0;
  SeqSplits table = {0, 0};
  if (expect) {
    const int start = b * a.spec_pages;
    const int i0 = start / by_spec_pps;
    n_valid = (start + a.spec_pages - 1) / by_spec_pps - i0 + 1;
    slot0 = i0 + b;
  } else if (balanced) {
    table = in_range(seq_splits[b], num_splits);
    n_valid = table.count;
    slot0 = table.first;
  } else {
    n_valid = a.num_splits;
    slot0 = b * a.num_splits;
  }
  if (!live) n_valid = 0;

  float mt = -INFINITY, den = 0.f;
  float acc[DPT];
  // Rounds after the first, for rows of more splits than the launch expects, take
  // kTail splits per thread while many are left: one sequence of 2K keys among 127
  // of 20, q_len 8, has 100 splits a row where two are expected (36.6 -> 28.5 us
  // per call with the rows below dealt over the workgroups; 8 per round 30.7).
  constexpr int kTail = WPR == 0 ? 16 : U;
  constexpr int kMost = kTail > U ? kTail : U;
  u4 o[kMost];
  float m[kMost], l[kMost];
  // One round: splits sb + u * SG (u < N) of the slots [s0, s0 + nv). Loads are
  // unconditional, from an in-bounds slot (past the last split: split 0 of the
  // row again, weight 0), so rounds need no branch around their loads.
  auto load_round = [&](auto n_of, int s0, int nv, int sb) {
    constexpr int N = decltype(n_of)::value;
    const float* ml = a.part_ml + ((size_t)s0 * stride + row_item) * 2;
    const size_t o0 = ((size_t)s0 * stride + row_item) * HD + DPT * c;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int sp = sb + u * SG;
      const size_t it = (size_t)(sp < nv ? sp : 0) * stride;
      if constexpr (E::kHalfPartials)
        o[u] = *(const u4*)((const _Float16*)a.part_o + o0 + it * HD);
      else
        o[u] = *(const u4*)(a.part_o + o0 + it * HD);
      const float2 p = *(const float2*)(ml + it * 2);  // (max, sum) in one load
      m[u] = p.x;
      l[u] = sp < nv ? p.y : 0.f;
    }
  };
  auto add_round = [&](auto n_of) {
    constexpr int N = decltype(n_of)::value;
    float cm = -INFINITY;
#pragma unroll
    for (int u = 0; u < N; ++u) cm = !(l[u] <= 0.f) ? fmaxf(cm, m[u]) : cm;
    const float nm = fmaxf(mt, cm);
    if (nm != -INFINITY) {
      const float sc = mt == -INFINITY ? 0.f : fast_exp2(mt - nm);
      den *= sc;
#pragma unroll
      for (int i = 0; i < DPT; ++i) acc[i] *= sc;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        // Splits without keys (l <= 0) never touch the sums: their partial sums
        // were never written and may hold anything. A NaN sum (the split saw a
        // NaN) is used, so the row comes out NaN.
        const bool use = !(l[u] <= 0.f);
        const float w = use ? fast_exp2(m[u] - nm) : 0.f;
        den += w * l[u];
        // Normalised partials weigh in with their sum.
        const float wo = E::kHalfPartials ? w * l[u] : w;
        float x[DPT];
        if constexpr (E::kHalfPartials) {
          const h8 v = __builtin_bit_cast(h8, o[u]);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
        } else {
          const f4 v = __builtin_bit_cast(f4, o[u]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = v[i];
        }
#pragma unroll
        for (int i = 0; i < DPT; ++i) acc[i] = use ? fmaf(wo, x[i], acc[i]) : acc[i];
      }
      mt = nm;
    }
  };
  // The first round is issued before anything else is waited for (the
  // expected layout's table read rides along with it); later rounds, rare, loop.
  auto merge_splits = [&](int s0, int nv) {
    mt = -INFINITY;
    den = 0.f;
#pragma unroll
    for (int i = 0; i < DPT; ++i) acc[i] = 0.f;
    load_round(Count<U>{}, s0, nv, g);
    if (expect) table = in_range(seq_splits[b], num_splits);
    const float first_l = l[0];  // split g (split 0 for group 0)
    add_round(Count<U>{});
    for (int sb = g + U * SG; sb < nv;) {
      if (kTail > U && nv - sb > 8) {
        load_round(Count<kTail>{}, s0, nv, sb);
        add_round(Count<kTail>{});
        sb += kTail * SG;
      } else {
        load_round(Count<U>{}, s0, nv, sb);
        add_round(Count<U>{});
        sb += U * SG;
      }
    }
    return first_l;
  };
  float first_l = merge_splits(slot0, n_valid);
  if (expect && live && (table.first != slot0 || table.count != n_valid)) {
    n_valid = table.count;
    slot0 = table.first;
    first_l = merge_splits(slot0, n_valid);
  }
  // A sequence with one split was written by the partial kernel: the balanced
  // plan says so by its count, a fixed plan by l = -1 in split 0, which group 0
  // (the one that stores) reads first. A sequence with no splits (no keys at
  // all) is written here as 0.
  const bool done = balanced ? n_valid == 1 : (g == 0 && first_l < 0.f);
  const bool skip = !live || done;

  // Combine the SG groups of the row: within a wave by shuffles (lanes c,
  // c + CH, ...), then the row's waves through LDS.
  auto combine = [&](float mo, float dn, const float (&ao)[DPT]) {
    const float nm = fmaxf(mt, mo);
    if (nm == -INFINITY) return;
    const float sa = mt == -INFINITY ? 0.f : fast_exp2(mt - nm);
    const float so = mo == -INFINITY ? 0.f : fast_exp2(mo - nm);
    den = den * sa + dn * so;
#pragma unroll
    for (int i = 0; i < DPT; ++i) acc[i] = acc[i] * sa + ao[i] * so;
    mt = nm;
  };
  static_assert(CH >= 8, "split groups of a wave meet over 8, 16 and 32 lanes");
  if constexpr (SG > 1 && CH <= 8) {
    // Lanes l and l ^ 8 of a row of 16: a rotation by 8.
    auto other = [](float x) {
      return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
          0, __builtin_bit_cast(int, x), 0x128, 0xf, 0xf, false));  // row_ror:8
    };
    const float mo = other(mt), dn = other(den);
    float ao[DPT];
#pragma unroll
    for (int i = 0; i < DPT; ++i) ao[i] = other(acc[i]);
    combine(mo, dn, ao);
  }
  auto meet = [&](auto pair_of) {
    const LanePair m2 = pair_of(mt), d2 = pair_of(den);
    float ao[DPT];
    mt = m2.lo;
    den = d2.lo;
#pragma unroll
    for (int i = 0; i < DPT; ++i) {
      const LanePair a2 = pair_of(acc[i]);
      acc[i] = a2.lo;
      ao[i] = a2.hi;
    }
    combine(m2.hi, d2.hi, ao);
  };
  if constexpr (SG > 1 && CH <= 16) meet([](float x) { return lane_pair<16>(x); });
  if constexpr (SG > 1 && CH <= 32) meet([](float x) { return lane_pair<32>(x); });
  if constexpr (WPR > 1) {
    static_assert(RPW == 1, "the LDS combine serves one row per workgroup");
    __shared__ float sm_acc[WPR][CH][DPT + 1];
    __shared__ float sm_m[WPR][CH], sm_d[WPR][CH];
    if (!live || (balanced && n_valid == 1)) return;  // uniform over the workgroup (one row)
    const int wave = t >> 6;
    if ((t & 63) < CH) {
#pragma unroll
      for (int i = 0; i < DPT; ++i) sm_acc[wave][c][i] = acc[i];
      sm_m[wave][c] = mt;
      sm_d[wave][c] = den;
    }
    __syncthreads();
    if (t >= CH) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      float ao[DPT];
#pragma unroll
      for (int i = 0; i < DPT; ++i) ao[i] = sm_acc[w][c][i];
      combine(sm_m[w][c], sm_d[w][c], ao);
    }
  }
  if (skip || g != 0) return;
  const float inv = !(den <= 0.f) ? a.out_scale / den : 0.f;  // 0: no key; NaN stays NaN
  if constexpr (DPT == 8) {
    // Two 8-byte stores: the output need only be 8-byte aligned.
    const float lo[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    const float hi[4] = {acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv};
    u2* op = (u2*)(a.out + (size_t)row * HD + 8 * c);
    op[0] = E::pack4(lo);
    op[1] = E::pack4(hi);
  } else {
    const float out[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    *(u2*)(a.out + (size_t)row * HD + 4 * c) = E::pack4(out);
  }
}

// Ring depth: the pages in flight per wave hold about 32 KiB of 16-bit K and
// V: 4 pages at head dim 128 (3 at 64 rows, where the registers run out), 8 at
// head dim 64 (4 at 64 rows: bf16 q16 201.5 -> 194.5 us, fp16 174.5 -> 173.9)
// and 2 at 256, which holds at most 32 rows (its accumulators double). e4m3
// caches keep the same page counts although their pages hold half the bytes,
// and at 64 rows 3 at head dim 64 and, at head dim 128, 2 under bf16 queries
// or 4 under fp16 ones (two page pairs): the widened K and V fragments take
// the registers a deeper ring would need.
// Measured at 16 sequences of 32K keys, partial kernel, e4m3 ring at twice
// these depths -> these: head dim 128 q2 / q8 170.7 / 181.4 -> 169.7 / 174.2
// us, q16 278 (6 pages) -> 261 (3) -> 251 us (2); head dim 256 q8 342.7 ->
// 325.1 us; head dim 64 q4 / q8 / q16 104.2 / 119.8 / 185 -> 100.7 / 116.6 /
// 169 us (2 pages at 64 rows there lose the pipelined loop: 154 -> 165 us).
template <int HD, typename E, typename KV, bool BAL>
void launch_partial_hd(const PartialArgs& a, const LaunchShape& sh, dim3 grid, dim3 block,
                       hipStream_t stream) {
  constexpr int D4 = 4 * 128 / HD, D2 = 2 * 128 / HD;
  static_assert(HD != 128 || D4 == kRingPages, "the host's ring-batch test assumes this ring");
  // e4m3 at head dim 128: 2 pages, or 4 under fp16 queries, whose pair steps
  // (pair_finish) need a second pair in flight while one is computed.
  constexpr int D3 = KV::kBytes == 1 ? (HD == 128 ? (__is_same(E, ElemF16) ? 4 : 2) : 3)
                                     : (HD == 64 ? 4 : 3 * 128 / HD);
  if (sh.hpw == 2) {
    // Two heads per wave: half the pages in flight, each twice the bytes.
    if constexpr (HD == 64) {
      if (sh.row_blocks == 1)
        hipLaunchKernelGGL((sqa_partial_kernel<1, D2, 4, 1, HD, E, KV, 2, BAL>), grid, block, 0,
                           stream, a);
      else if (sh.row_blocks == 2)
        hipLaunchKernelGGL((sqa_partial_kernel<2, D2, 4, 1, HD, E, KV, 2, BAL>), grid, block, 0,
                           stream, a);
      else
        hipLaunchKernelGGL((sqa_partial_kernel<4, D2, 4, 1, HD, E, KV, 2, BAL>), grid, block, 0,
                           stream, a);
    }
  } else if (sh.row_blocks == 1) {
    if constexpr (HD == 128 && KV::kBytes == 2 && !BAL) {
      if (a.ring_batch) {
        hipLaunchKernelGGL((sqa_partial_kernel<1, D4, 4, 1, HD, E, KV, 1, BAL, true>), grid, block,
                           0, stream, a);
        return;
      }
    }
    hipLaunchKernelGGL((sqa_partial_kernel<1, D4, 4, 1, HD, E, KV, 1, BAL>), grid, block, 0, stream,
                       a);
  } else if (sh.row_blocks == 2) {
    if constexpr (HD == 128 && KV::kBytes == 2 && !BAL) {
      if (a.ring_batch) {
        hipLaunchKernelGGL((sqa_partial_kernel<2, D4, 4, 1, HD, E, KV, 1, BAL, true>), grid, block,
                           0, stream, a);
        return;
      }
    }
    hipLaunchKernelGGL((sqa_partial_kernel<2, D4, 4, 1, HD, E, KV, 1, BAL>), grid, block, 0, stream,
                       a);
  } else if constexpr (HD == 128 && KV::kBytes == 2) {
    // 33..64 rows of 16-bit K and V: two waves per kv head sharing an LDS ring
    // of 128 KiB (4 pages). e4m3 caches take the one-wave-per-head kernel below:
    // it widens each page once per head where two waves would both widen it
    // (cfg3 shape q16: 256.3 -> 246.6 us; B4 KV 8K 34.8 -> 33.6 us).
    hipLaunchKernelGGL((sqa_partial_lds_kernel<4, E, KV, BAL>), grid, dim3(512), 0, stream, a);
  } else if constexpr (HD != 256) {
    hipLaunchKernelGGL((sqa_partial_kernel<4, D3, 4, 1, HD, E, KV, 1, BAL>), grid, block, 0, stream,
                       a);
  }
}

template <typename E, template <int> class KV, bool BAL>
void launch_partial_as(const PartialArgs& a, const LaunchShape& sh, dim3 grid, dim3 block,
                       hipStream_t stream) {
  if (a.head_dim == 64)
    launch_partial_hd<64, E, KV<64>, BAL>(a, sh, grid, block, stream);
  else if (a.head_dim == 256)
    launch_partial_hd<256, E, KV<256>, BAL>(a, sh, grid, block, stream);
  else
    launch_partial_hd<128, E, KV<128>, BAL>(a, sh, grid, block, stream);
}

template <int HD, typename E, int TPR, bool BAL>
void launch_merge_u(const MergeArgs& a, int u, hipStream_t stream) {
  constexpr int kRows = 256 / TPR;  // per workgroup
  const dim3 grid((unsigned)((a.batch * a.q_len * a.hq + kRows - 1) / kRows));
  if (u <= 2)
    hipLaunchKernelGGL((sqa_merge_kernel<TPR, HD, E, 2, BAL>), grid, dim3(256), 0, stream, a);
  else if (u <= 4)
    hipLaunchKernelGGL((sqa_merge_kernel<TPR, HD, E, 4, BAL>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((sqa_merge_kernel<TPR, HD, E, 8, BAL>), grid, dim3(256), 0, stream, a);
}

template <int HD, typename E, bool BAL>
void launch_merge_hd(const MergeArgs& a, int per_row, int cus, hipStream_t stream) {
  constexpr int kChunks = HD / (E::kHalfPartials ? 8 : 4);  // threads a partial row takes
  const int threads =
      merge_row_threads((long long)a.batch * a.q_len * a.hq, per_row, kChunks, cus);
  const int at_once = threads / kChunks;  // splits per load instruction
  const int u = (per_row + at_once - 1) / at_once;
  if (threads == 256)
    launch_merge_u<HD, E, 256, BAL>(a, u, stream);
  else if (threads == 64)
    launch_merge_u<HD, E, 64, BAL>(a, u, stream);
  else
    launch_merge_u<HD, E, kChunks, BAL>(a, u, stream);
}

template <typename E, bool BAL>
void launch_merge_as(const MergeArgs& a, int per_row, int cus, hipStream_t stream) {
  if (a.head_dim == 64)
    launch_merge_hd<64, E, BAL>(a, per_row, cus, stream);
  else if (a.head_dim == 256)
    launch_merge_hd<256, E, BAL>(a, per_row, cus, stream);
  else
    launch_merge_hd<128, E, BAL>(a, per_row, cus, stream);
}

template <bool BAL>
void launch_partial_plan(const PartialArgs& a, const LaunchShape& sh, dim3 grid, dim3 block,
                         hipStream_t stream) {
  if (a.bf16) {
    if (a.kv_fp8)
      launch_partial_as<ElemBF16, KvFp8, BAL>(a, sh, grid, block, stream);
    else
      launch_partial_as<ElemBF16, KvNative, BAL>(a, sh, grid, block, stream);
  } else {
    if (a.kv_fp8)
      launch_partial_as<ElemF16, KvFp8, BAL>(a, sh, grid, block, stream);
    else
      launch_partial_as<ElemF16, KvNative, BAL>(a, sh, grid, block, stream);
  }
}

template <bool BAL>
void launch_merge_plan(const MergeArgs& a, int per_row, int cus, hipStream_t stream) {
  if (BAL && a.bf16 == 2)
    launch_merge_as<ElemF16Wide, true>(a, per_row, cus, stream);
  else if (a.bf16)
    launch_merge_as<ElemBF16, BAL>(a, per_row, cus, stream);
  else
    launch_merge_as<ElemF16, BAL>(a, per_row, cus, stream);
}

}  // namespace

hipError_t launch_partial(const PartialArgs& a, hipStream_t stream) {
  const LaunchShape sh = launch_shape(a.rows, a.hkv, a.head_dim);
  const int head_groups = (a.hkv + sh.heads - 1) / sh.heads;
  // Work items: fixed plan, one per slot; balanced, num_splits - batch (a
  // sequence's share of the spare slots comes from the item it ends in).
  const long long items = is_balanced(a.pages_per_split)
                              ? (long long)(a.num_splits - a.batch)
                              : (long long)a.batch * a.num_splits;
  const dim3 grid((unsigned)(items * head_groups));
  const dim3 block(sh.waves() * 64);
  if (is_balanced(a.pages_per_split))
    launch_partial_plan<true>(a, sh, grid, block, stream);
  else
    launch_partial_plan<false>(a, sh, grid, block, stream);
  return hipGetLastError();
}

hipError_t launch_merge(const MergeArgs& a, int cus, hipStream_t stream) {
  // Splits per sequence, for the choice of merge variant: a fixed plan's
  // num_splits; the balanced plan's count per sequence is known only on the
  // device: the batch average, items / batch. It depends on the slot count
  // alone, so the plain balanced plan and the one with an expected page count
  // merge with the same variant (and give the same bits).
  // With items per head group, the larger group's count (a row of the other
  // group then loads a few more splits than it has, as splits past a row's
  // last do).
  const int items = a.hg_items[0] > 0 ? max(a.hg_items[0], a.hg_items[1]) : a.num_splits - a.batch;
  const int per_row = is_balanced(a.pages_per_split) ? (items + a.batch - 1) / a.batch
                                                     : a.num_splits;
  if (is_balanced(a.pages_per_split))
    launch_merge_plan<true>(a, per_row, cus, stream);
  else
    launch_merge_plan<false>(a, per_row, cus, stream);
  return hipGetLastError();
}

}  // namespace sqa

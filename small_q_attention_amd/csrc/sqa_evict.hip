// gfx950 kernels that thin out a paged cache: the attention weight every cached token
// receives, added up over calls, and the eviction of the lighter tokens.
//
//   weight[b][h][t] += sum over the rows (i, g) of kv head h of
//                      exp(scale * q(i, g) . k(t) - lse(i, g)),
// where the call's own draft tokens start at 0. Two kernels: the first reads K once and
// leaves, for each row and work item, the maximum and the sum of exponentials; the second
// joins them to the rows' log-sum-exp and adds the weights up. Between them the scores
// either go through memory in fp32 (rows * 8 bytes a token and head, written and read) or
// K is read and multiplied again, whichever moves fewer bytes.
#include "sqa_cache.h"
#include "sqa_cache_device.h"

namespace sqa {
namespace {

// K of a 16-token page in registers: 16-byte loads, token l % 16 of a lane.
template <int HD>
struct KeysNative {
  static constexpr int KK = Dims<HD>::KK, kLoads = KK, kBytes = 2;
  static __device__ __forceinline__ int q_dims(int kk, int g) { return 32 * kk + 8 * g; }
  struct Regs {
    u4 k[KK];
  };
  template <typename E>
  static __device__ __forceinline__ void expand(const Regs& r, u4 (&k)[KK]) {
#pragma unroll
    for (int i = 0; i < KK; ++i) k[i] = r.k[i];
  }
};
template <int HD>
struct KeysFp8 {
  static constexpr int KK = Dims<HD>::KK, kLoads = KK / 2, kBytes = 1;
  static __device__ __forceinline__ int q_dims(int kk, int g) { return KvFp8<HD>::q_dims(kk, g); }
  struct Regs {
    u4 k[KK / 2];
  };
  template <typename E>
  static __device__ __forceinline__ void expand(const Regs& r, u4 (&k)[KK]) {
#pragma unroll
    for (int i = 0; i < KK / 2; ++i) {
      k[2 * i] = E::widen_fp8(u2{r.k[i][0], r.k[i][1]});
      k[2 * i + 1] = E::widen_fp8(u2{r.k[i][2], r.k[i][3]});
    }
  }
};
template <int HD>
struct KeysInt8 : KeysFp8<HD> {
  using Regs = typename KeysFp8<HD>::Regs;
  static constexpr int KK = Dims<HD>::KK;
  template <typename E>
  static __device__ __forceinline__ void expand(const Regs& r, u4 (&k)[KK]) {
#pragma unroll
    for (int i = 0; i < KK; ++i)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const unsigned x = r.k[i / 2][2 * (i & 1) + w];
        auto byte = [&](int n) { return (float)(signed char)(x >> (8 * n)); };
        k[i][2 * w] = E::pack2(byte(0), byte(1));
        k[i][2 * w + 1] = E::pack2(byte(2), byte(3));
      }
  }
};

__device__ __forceinline__ float row16_sum(float x) {
  // Sum over the 16 lanes of a row, in all of them.
  auto ror = [](float v, auto n) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
        0, __builtin_bit_cast(int, v), 0x120 + decltype(n)::value, 0xf, 0xf, false));
  };
  x += ror(x, std::integral_constant<int, 8>{});
  x += ror(x, std::integral_constant<int, 4>{});
  x += ror(x, std::integral_constant<int, 2>{});
  x += ror(x, std::integral_constant<int, 1>{});
  return x;
}

// The log-sum-exp (log2 units) of a row from its sequence's items: lanes over items. A
// row that saw nothing: +inf, which makes every weight 0.
__device__ __forceinline__ float join_stats(const float2* st, int count) {
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, l = 0.f;
  for (int i = lane; i < count; i += 64) {
    const float2 x = st[i];
    const float nm = fmaxf(m, x.x);
    // A NaN sum must stay: its maximum travels as a finite number.
    const float a = m == -INFINITY ? 0.f : fast_exp2(m - nm);
    const float b = x.x == -INFINITY ? 0.f : fast_exp2(x.x - nm);
    l = (m == -INFINITY ? 0.f : l * a) + (x.x == -INFINITY ? 0.f : x.y * b);
    m = nm;
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const float m2 = __shfl_xor(m, o), l2 = __shfl_xor(l, o);
    const float nm = fmaxf(m, m2);
    l = (m == -INFINITY ? 0.f : l * fast_exp2(m - nm)) +
        (m2 == -INFINITY ? 0.f : l2 * fast_exp2(m2 - nm));
    m = nm;
  }
  return l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// What a wave works on: a work item of one kv head.
struct WaveItem {
  Split it;
  int kvh;
};
__device__ __forceinline__ bool wave_item(const WeighArgs& args, WaveItem& w) {
  const PartialArgs& a = args.p;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wgh = args.wg_heads;
  const int head_groups = (a.hkv + wgh - 1) / wgh;
  w.kvh = (blockIdx.x % head_groups) * wgh + wave % wgh;
  const int item = (blockIdx.x / head_groups) * (4 / wgh) + wave / wgh;
  if (w.kvh >= a.hkv) return false;
  w.it.b = w.it.len = w.it.p_begin = w.it.p_end = w.it.slot = w.it.first = 0;
  w.it.count = 1;
  if (!find_split(a, args.items, item, nullptr, w.it)) return false;
  w.it.b = __builtin_amdgcn_readfirstlane(w.it.b);
  w.it.len = __builtin_amdgcn_readfirstlane(w.it.len);
  w.it.p_begin = __builtin_amdgcn_readfirstlane(w.it.p_begin);
  w.it.p_end = __builtin_amdgcn_readfirstlane(w.it.p_end);
  w.it.first = __builtin_amdgcn_readfirstlane(w.it.first);
  w.it.count = __builtin_amdgcn_readfirstlane(w.it.count);
  return w.it.p_end > w.it.p_begin;
}

// The scores of an item's pages, page by page: pass 1 (SUM false) keeps each row's
// maximum and sum and, with STORE, leaves the scores in memory; pass 2 (SUM true) adds up
// the weights from the rows' log-sum-exp. As the attention kernel, a wave on its own with
// a ring of D pages of K in flight.
template <int NB, int D, int HD, typename E, typename KEYS, bool SUM, bool STORE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void sqa_weigh_kernel(WeighArgs args) {
  const PartialArgs& a = args.p;
  constexpr int KK = Dims<HD>::KK;
  static_assert(64 % D == 0 && D % 4 == 0, "ring turns within 64 ids, weights four pages at a time");
  WaveItem w;
  if (!wave_item(args, w)) return;  // uniform
  const int lane = threadIdx.x & 63;
  const int g16 = lane >> 4, l16 = lane & 15;
  const int b = w.it.b, len = w.it.len, p_begin = w.it.p_begin, kvh = w.kvh;
  const int n_pages = w.it.p_end - p_begin;
  const int shift = a.page_shift, sub_mask = (1 << shift) - 1;

  const int32_t* row = a.block_tables + (size_t)b * a.bt_stride;
  auto load_ids = [&](int c) {
    const long long p = (long long)p_begin + 64 * c + lane;
    return row[min(p, (long long)a.max_pages - 1) >> shift];
  };
  int ids = load_ids(0), ids_next = load_ids(1);

  const WaveRows<NB, 1> map{kvh, a.rows, a.hkv};
  u4 q[NB][KK];
  RegBits<NB> bits;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = map.row(nb, l16);
    const bool real = map.real(nb, l16);
    const int qi = real ? r / a.by_group : 0;
    const int hh = kvh * a.group + (real ? r - qi * a.group : 0);
    const _Float16* qp = a.q + ((size_t)(b * a.q_len + qi) * a.hq + hh) * HD;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const u4 x = *(const u4*)(qp + KEYS::q_dims(kk, g16));
      q[nb][kk] = real ? x : u4{0u, 0u, 0u, 0u};
    }
    bits.b[nb] = draft_bits(a, b, qi, real);
  }
  float lse[NB];
  if constexpr (SUM) {
    // Lane l takes the log-sum-exp of row 16 nb + l % 16.
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      lse[nb] = INFINITY;
      for (int r = 0; r < 16 && 16 * nb + r < a.rows; ++r) {  // uniform
        const float x = join_stats(
            args.stats + (size_t)(kvh * a.rows + 16 * nb + r) * args.items + w.it.first,
            w.it.count);
        lse[nb] = l16 == r ? x : lse[nb];
      }
    }
  }

  const unsigned tok_bytes = a.token_stride;
  const unsigned k_lane = l16 * tok_bytes + kvh * a.head_stride + 16 * g16;
  const size_t sub_bytes = (size_t)kPageSize * tok_bytes;
  const char* scale_at = (const char*)args.k_scale + (size_t)kvh * args.scale_head;
  struct Slot {
    typename KEYS::Regs k;
    float scale;
  };
  auto load_page = [&](int pid, int p, Slot& s) {
    pid = __builtin_amdgcn_readfirstlane(pid);
    const size_t off =
        pid >= 0 ? (size_t)pid * (size_t)a.page_stride + (size_t)(p & sub_mask) * sub_bytes : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((const char*)a.k + off), (short)0, pid >= 0 ? (int)a.page_extent : 0, kBufferFlags);
    s.scale = 1.f;
    if (args.k_scale) s.scale = *(const float*)(scale_at + max(pid, 0) * args.scale_page);
#pragma unroll
    for (int i = 0; i < KEYS::kLoads; ++i)
      s.k.k[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_lane + 64 * i, 0,
                                                       SUM || STORE ? kStreamAux : 0);
  };
  auto page_id = [&](int i) {
    return clamp_page(__builtin_amdgcn_readlane(ids, i & 63), a.num_pages);
  };
  Slot ring[D];
#pragma unroll
  for (int j = 0; j < D; ++j) load_page(j < n_pages ? page_id(j) : -1, p_begin + j, ring[j]);

  const int mask_from = len - a.q_len;
  float m[NB], l[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb] = -INFINITY;
    l[nb] = 0.f;
  }
  float* wrow = args.weights + b * args.w_batch + kvh * args.w_head;
  f4* out = (f4*)args.scores +
            ((size_t)(b * a.hkv + kvh) * a.max_pages + p_begin) * a.rows * 4;

  for (int i = 0; i < n_pages; i += D) {
    if (((i + D) & 63) == 0) {
      ids = ids_next;
      ids_next = load_ids((i + D) / 64 + 1);
    }
    float mine = 0.f, old = 0.f;
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int ii = i + j;
      const int p = p_begin + ii;
      // Weights of pages ii - ii % 4 .. + 3: lane (g, 4 e4 + e) holds token 4 g + e of page
      // e4 of the four.
      const int wt = (p - (j & 3)) * kPageSize + 16 * (l16 >> 2) + 4 * g16 + (l16 & 3);
      if constexpr (SUM) {
        if ((j & 3) == 0) {
          mine = 0.f;
          old = 0.f;
          if (ii + (l16 >> 2) < n_pages && wt < min(mask_from, args.width)) old = wrow[wt];
        }
      }
      if (ii < n_pages) {
        const float c =
            a.scale_log2 * __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(
                                                         __builtin_bit_cast(int, ring[j].scale)));
        u4 k[KK];
        KEYS::template expand<E>(ring[j].k, k);
        f4 s[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          s[nb] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) s[nb] = E::mma_qk(k[kk], q[nb][kk], s[nb]);
          s[nb] *= c;
        }
        if ((p + 1) * kPageSize > mask_from)  // uniform
          mask_scores<NB>(s, bits.b, mask_from, p * kPageSize + 4 * g16, len);
        if constexpr (SUM) {
          f4 t = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              t[e] += s[nb][e] == -INFINITY ? 0.f : fast_exp2(s[nb][e] - lse[nb]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = row16_sum(t[e]);
            mine = l16 == 4 * (j & 3) + e ? x : mine;
          }
        } else {
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const float mn = fmaxf(m[nb], max4(s[nb]));
            const float mu = mn == -INFINITY ? 0.f : mn;
            l[nb] = l[nb] * fast_exp2(m[nb] - mu) +
                    ((fast_exp2(s[nb][0] - mu) + fast_exp2(s[nb][1] - mu)) +
                     (fast_exp2(s[nb][2] - mu) + fast_exp2(s[nb][3] - mu)));
            m[nb] = mn;
            if constexpr (STORE)
              if (map.real(nb, l16)) out[((size_t)ii * a.rows + map.row(nb, l16)) * 4 + g16] = s[nb];
          }
        }
      }
      if constexpr (SUM) {
        if ((j & 3) == 3) {
          if (ii - 3 + (l16 >> 2) < n_pages && wt < min(len, args.width))
            wrow[wt] = wt < mask_from ? old + mine : mine;
        }
      }
      load_page(ii + D < n_pages ? page_id(ii + D) : -1, p + D, ring[j]);
    }
  }
  if constexpr (!SUM) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float top = xor_max(m[nb]);
      const float part = m[nb] == -INFINITY ? (l[nb] == l[nb] ? 0.f : l[nb])
                                            : l[nb] * fast_exp2(m[nb] - top);
      const float sum = xor_sum(part);
      if (g16 == 0 && map.real(nb, l16))
        // A NaN sum travels with a finite maximum, so that the join counts it.
        args.stats[(size_t)(kvh * a.rows + map.row(nb, l16)) * args.items + w.it.slot] =
            float2{sum == sum ? top : 0.f, sum};
    }
  }
}

// The second pass from the stored scores: a lane per token, 64 tokens at a time.
template <int U>
__global__ __launch_bounds__(256) void sqa_weigh_join_kernel(WeighArgs args) {
  const PartialArgs& a = args.p;
  WaveItem w;
  if (!wave_item(args, w)) return;  // uniform
  const int lane = threadIdx.x & 63;
  const int rows = a.rows, kvh = w.kvh;
  const int mask_from = w.it.len - a.q_len;
  const int t_end = min(min(w.it.p_end * kPageSize, w.it.len), args.width);
  const float2* stats = args.stats + (size_t)kvh * rows * args.items + w.it.first;
  const float* scores =
      args.scores + (size_t)(w.it.b * a.hkv + kvh) * a.max_pages * rows * kPageSize;
  float* wrow = args.weights + w.it.b * args.w_batch + kvh * args.w_head;
  // Lane r holds row r's log-sum-exp.
  float lse = INFINITY;
  for (int r = 0; r < rows; ++r) {
    const float x = join_stats(stats + (size_t)r * args.items, w.it.count);
    lse = lane == r ? x : lse;
  }
  for (int t0 = w.it.p_begin * kPageSize; t0 < t_end; t0 += 64 * U) {
    float sum[U], old[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + 64 * u + lane;
      sum[u] = 0.f;
      old[u] = t < min(mask_from, t_end) ? wrow[t] : 0.f;
    }
    for (int r = 0; r < rows; ++r) {
      const float lr = __builtin_bit_cast(
          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, lse), r));
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = min(t0 + 64 * u + lane, t_end - 1);
        x[u] = scores[((size_t)(t >> 4) * rows + r) * kPageSize + (t & 15)];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) sum[u] += x[u] == -INFINITY ? 0.f : fast_exp2(x[u] - lr);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + 64 * u + lane;
      if (t < t_end) wrow[t] = t < mask_from ? old[u] + sum[u] : sum[u];
    }
  }
}

// ---------------------------------------------------------------------------------
// Eviction.
// ---------------------------------------------------------------------------------

// Larger weights give larger keys; -0 and 0 the same one, NaN the least of all.
__device__ __forceinline__ unsigned weight_key(float w) {
  if (w != w) return 0u;
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.f);  // -0 + 0 = 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;

// Which tokens of one sequence and kv head stay. The smallest key that stays is found by
// a radix selection over the weights between the sink and the recent tokens (11, 11 and
// 10 bits, histograms in LDS); tokens above it stay, and of those that equal it the first.
// Each wave then counts its own run of tokens, and after one exchange writes its kept
// tokens in order. All counts are integers: the same weights give the same tokens.
__global__ __launch_bounds__(kSelectThreads) void sqa_select_kernel(EvictArgs a) {
  __shared__ int hist[2048];
  __shared__ int wave_tot[kSelectWaves], wave_sure[kSelectWaves], wave_tie[kSelectWaves];
  __shared__ int picked, above;
  const int b = blockIdx.x / a.hkv, h = blockIdx.x % a.hkv;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* w = a.weights + b * a.w_batch + h * a.w_head;
  float* nw = a.new_weights + b * a.nw_batch + h * a.nw_head;
  int32_t* kept = a.kept + (size_t)(b * a.hkv + h) * a.budget;
  const long long room = (long long)a.bt_stride * a.page_size;
  const int n = (int)min((long long)min(max(a.seq_lens[b], 0), a.width), room);
  const int m = min(n, a.budget);
  if (h == 0 && tid == 0) a.new_lens[b] = m;
  if (n <= a.budget) {
    for (int j = tid; j < a.budget; j += kSelectThreads) kept[j] = j < n ? j : -1;
    for (int j = tid; j < a.new_width; j += kSelectThreads) nw[j] = j < n ? w[j] : 0.f;
    return;
  }
  const int lo = a.sink, hi = n - a.recent;
  const int free = a.budget - a.sink - a.recent;
  unsigned threshold = 0xffffffffu;  // no key: keys of finite weights and infinities lie below
  int ties = 0;                      // how many of the tokens at the threshold stay
  if (free > 0) {
    int want = free;
    unsigned prefix = 0, mask = 0;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      const unsigned digits = pass == 2 ? 0x3ffu : 0x7ffu;
      for (int i = tid; i < 2048; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      for (int t = lo + tid; t < hi; t += kSelectThreads) {
        const unsigned k = weight_key(w[t]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digits], 1);
      }
      __syncthreads();
      // Bins from the top: thread i takes bins 2047 - 2 i and 2046 - 2 i.
      const int c0 = hist[2047 - 2 * tid], c1 = hist[2046 - 2 * tid];
      const int incl = wave_inclusive_scan_int(c0 + c1);
      if (lane == 63) wave_tot[wave] = incl;
      __syncthreads();
      int before = incl - c0 - c1;
      for (int i = 0; i < wave; ++i) before += wave_tot[i];
      if (before < want && want <= before + c0 + c1) {  // one thread
        const bool first = want <= before + c0;
        picked = first ? 2047 - 2 * tid : 2046 - 2 * tid;
        above = first ? before : before + c0;
      }
      __syncthreads();
      prefix |= (unsigned)picked << shift;
      mask |= digits << shift;
      want -= above;
    }
    threshold = prefix;
    ties = want;
  }
  // Runs of whole waves' widths, one per wave.
  const int run = ((n + kSelectThreads - 1) / kSelectThreads) * 64;
  const int begin = min(wave * run, n), end = min(begin + run, n);
  auto look = [&](int t, bool& sure, bool& tie) {
    const bool in = t < end;
    const bool always = in && (t < lo || t >= hi);
    const unsigned k = in && !always ? weight_key(w[t]) : 0u;
    sure = always || (in && free > 0 && k > threshold);
    tie = in && !always && free > 0 && k == threshold;
  };
  int sures = 0, tied = 0;
  for (int t = begin; t < end; t += 64) {
    bool sure, tie;
    look(t + lane, sure, tie);
    sures += __popcll(__ballot(sure));
    tied += __popcll(__ballot(tie));
  }
  if (lane == 0) {
    wave_sure[wave] = sures;
    wave_tie[wave] = tied;
  }
  __syncthreads();
  int at = 0, seen = 0;  // kept tokens and ties before this wave's
  for (int i = 0; i < wave; ++i) {
    at += wave_sure[i];
    seen += wave_tie[i];
  }
  at += min(seen, ties);
  const unsigned long long below = lane ? ~0ull >> (64 - lane) : 0ull;
  for (int t = begin; t < end; t += 64) {
    bool sure, tie;
    look(t + lane, sure, tie);
    const unsigned long long tie_mask = __ballot(tie);
    const bool keep = sure || (tie && seen + __popcll(tie_mask & below) < ties);
    const unsigned long long keep_mask = __ballot(keep);
    if (keep) kept[at + __popcll(keep_mask & below)] = t + lane;
    at += __popcll(keep_mask);
    seen += __popcll(tie_mask);
  }
  __syncthreads();
  // The weights move along, 1024 at a time: new_weights may be the old ones, and a token
  // never moves to a later position.
  for (int j0 = 0; j0 < a.new_width; j0 += kSelectThreads) {
    const int j = j0 + tid;
    const float x = j < m ? w[kept[j]] : 0.f;
    __syncthreads();
    if (j < a.new_width) nw[j] = x;
    __syncthreads();
  }
}

// The kept tokens of 16 new slots of one kv head, K or V, moved to their new page. 16
// bytes a lane. Scaled caches: the new block's scale is the largest of the scales its
// tokens come from, and codes from blocks of other scales are rounded again.
template <int ROW, bool SCALED, bool INT8>
__global__ __launch_bounds__(256) void sqa_move_kernel(EvictArgs a) {
  constexpr int LPT = ROW / 16;   // lanes per token (ROW: bytes of a token and head)
  constexpr int TPI = 64 / LPT;   // tokens per instruction
  constexpr int NI = 16 / TPI;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int head_groups = (a.hkv + 3) / 4;
  const int h = (blockIdx.x % head_groups) * 4 + wave;
  const int tiles = (a.budget + 15) / 16;
  const int rest = blockIdx.x / head_groups;
  const int b = rest / tiles, j0 = rest % tiles * 16;
  const int which = blockIdx.y;
  const int m = a.new_lens[b];
  if (h >= a.hkv || j0 >= m) return;
  const int page = a.page_size;
  const int np = j0 / page;
  if (np >= a.new_stride) return;
  const int to = a.new_tables[(size_t)b * a.new_stride + np];
  if (to < 0 || to >= a.new_pages) return;  // uniform: a page that is not there
  const int32_t* kept = a.kept + (size_t)(b * a.hkv + h) * a.budget;
  const int32_t* table = a.block_tables + (size_t)b * a.bt_stride;
  // Lane l: where new token j0 + l % 16 comes from.
  const int jt = min(j0 + (lane & 15), m - 1);
  const int from = max(kept[jt], 0);
  const int fp = clamp_page(table[from / page], a.num_pages);
  const long long off = (long long)fp * a.src_page + (long long)(from % page) * a.src_token;
  float old = 1.f, scale = 1.f;
  if constexpr (SCALED) {
    const char* sc = (const char*)(which ? a.src_scales.v : a.src_scales.k) +
                     (size_t)h * a.src_scales.head_stride;
    old = *(const float*)(sc + fp * a.src_scales.page_stride);
    scale = 0.f;
    const int first = np * page;
    for (int j = first + lane; j < min(first + page, m); j += 64) {
      const int p = clamp_page(table[max(kept[j], 0) / page], a.num_pages);
      scale = fmaxf(scale, *(const float*)(sc + p * a.src_scales.page_stride));
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) scale = fmaxf(scale, __shfl_xor(scale, o));
    if (j0 == first && lane == 0)
      *(float*)((char*)(which ? a.dst_scales.v : a.dst_scales.k) +
                (size_t)h * a.dst_scales.head_stride + to * a.dst_scales.page_stride) = scale;
  }
  const char* src = a.src[which] + (size_t)h * a.src_head + 16 * (lane % LPT);
  char* dst = a.dst[which] + (size_t)h * a.dst_head + (size_t)to * a.dst_page +
              (size_t)(j0 % page) * a.dst_token + 16 * (lane % LPT);
  u4 x[NI];
  float so[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int t = i * TPI + lane / LPT;
    const long long o = (long long)__shfl((int)(off >> 32), t) << 32 |
                        (unsigned)__shfl((int)off, t);
    x[i] = *(const u4*)(src + o);
    so[i] = SCALED ? __shfl(old, t) : 1.f;
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int t = i * TPI + lane / LPT;
    if constexpr (SCALED) {
      if (so[i] != scale) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            y[e] = scale > 0.f ? decode<INT8>(x[i][w], e) * so[i] / scale : 0.f;
          x[i][w] = encode4<INT8>(y);
        }
      }
    }
    if (j0 + t < m) *(u4*)(dst + (size_t)t * a.dst_token) = x[i];
  }
}

template <int HD, typename E, template <int> class KEYS, int NB>
void launch_weigh_rows(const WeighArgs& a, dim3 grid, hipStream_t stream) {
  constexpr int D = HD == 256 ? 4 : 8;
  const dim3 block(256);
  if constexpr (weights_stored(16 * (NB - 1) + 1, HD, KEYS<HD>::kBytes)) {
    if (a.scores) {
      hipLaunchKernelGGL((sqa_weigh_kernel<NB, D, HD, E, KEYS<HD>, false, true>), grid, block, 0,
                         stream, a);
      hipLaunchKernelGGL((sqa_weigh_join_kernel<4>), grid, block, 0, stream, a);
      return;
    }
  }
  {
    hipLaunchKernelGGL((sqa_weigh_kernel<NB, D, HD, E, KEYS<HD>, false, false>), grid, block, 0,
                       stream, a);
    hipLaunchKernelGGL((sqa_weigh_kernel<NB, D, HD, E, KEYS<HD>, true, false>), grid, block, 0,
                       stream, a);
  }
}

template <typename E, template <int> class KEYS>
void launch_weigh_as(const WeighArgs& a, dim3 grid, hipStream_t stream) {
  const int rows = a.p.rows;
  if (a.p.head_dim == 64) {
    if (rows <= 16)
      launch_weigh_rows<64, E, KEYS, 1>(a, grid, stream);
    else if (rows <= 32)
      launch_weigh_rows<64, E, KEYS, 2>(a, grid, stream);
    else
      launch_weigh_rows<64, E, KEYS, 4>(a, grid, stream);
  } else if (a.p.head_dim == 128) {
    if (rows <= 16)
      launch_weigh_rows<128, E, KEYS, 1>(a, grid, stream);
    else if (rows <= 32)
      launch_weigh_rows<128, E, KEYS, 2>(a, grid, stream);
    else
      launch_weigh_rows<128, E, KEYS, 4>(a, grid, stream);
  } else {
    if (rows <= 16)
      launch_weigh_rows<256, E, KEYS, 1>(a, grid, stream);
    else
      launch_weigh_rows<256, E, KEYS, 2>(a, grid, stream);
  }
}

template <int ROW>
void launch_move(const EvictArgs& a, dim3 grid, hipStream_t stream) {
  if (!a.scaled)
    hipLaunchKernelGGL((sqa_move_kernel<ROW, false, false>), grid, dim3(256), 0, stream, a);
  else if constexpr (ROW <= 256) {
    if (a.kv_type == kInt8)
      hipLaunchKernelGGL((sqa_move_kernel<ROW, true, true>), grid, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((sqa_move_kernel<ROW, true, false>), grid, dim3(256), 0, stream, a);
  }
}

}  // namespace

hipError_t launch_weigh(const WeighArgs& a, hipStream_t stream) {
  const int head_groups = (a.p.hkv + a.wg_heads - 1) / a.wg_heads;
  const int per_wg = 4 / a.wg_heads;
  const dim3 grid((unsigned)((a.items + per_wg - 1) / per_wg * head_groups));
  if (a.p.bf16) {
    if (a.kv_type == kInt8)
      launch_weigh_as<ElemBF16, KeysInt8>(a, grid, stream);
    else if (a.kv_type == kE4M3)
      launch_weigh_as<ElemBF16, KeysFp8>(a, grid, stream);
    else
      launch_weigh_as<ElemBF16, KeysNative>(a, grid, stream);
  } else {
    if (a.kv_type == kInt8)
      launch_weigh_as<ElemF16, KeysInt8>(a, grid, stream);
    else if (a.kv_type == kE4M3)
      launch_weigh_as<ElemF16, KeysFp8>(a, grid, stream);
    else
      launch_weigh_as<ElemF16, KeysNative>(a, grid, stream);
  }
  return hipGetLastError();
}

hipError_t launch_evict(const EvictArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(sqa_select_kernel, dim3((unsigned)(a.batch * a.hkv)), dim3(kSelectThreads), 0,
                     stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int tiles = (a.budget + 15) / 16;
  const dim3 grid((unsigned)((long long)a.batch * tiles * ((a.hkv + 3) / 4)), 2);
  const int row = a.head_dim * (a.kv_type >= kE4M3 ? 1 : 2);
  if (row == 64)
    launch_move<64>(a, grid, stream);
  else if (row == 128)
    launch_move<128>(a, grid, stream);
  else if (row == 256)
    launch_move<256>(a, grid, stream);
  else
    launch_move<512>(a, grid, stream);
  return hipGetLastError();
}

}  // namespace sqa

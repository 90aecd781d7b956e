// gfx950 kernels that thin out a paged cache: the attention weight every cached token
// receives, added up over calls, and the eviction of the lighter tokens.
//
//   weight[b][h][t] += sum over the rows (i, g) of kv head h of
//                      exp(scale * q(i, g) . k(t) - lse(i, g)),
// where the call's own draft tokens start at 0. Two kernels: the first reads K once and
// leaves, for each row and work item, the maximum and the sum of exponentials; the second
// joins them to the rows' log-sum-exp and adds the weights up. Between them the scores
// either go through memory in fp32 or K is read and multiplied again (weights_stored()).
//
// What bounds them: 16 sequences of 32K keys, one token each, 16-bit K (1.07 GB): the first
// kernel 231 us, of which the 67 MB of scores it writes take about 50 (182 us without),
// 4.9 TB/s in all; the second 23 us. Many rows: instructions (64 rows, 8 sequences of up to
// 12K keys, e4m3: 20 and 25 us), of which about 6 us each are the way to the first page.
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

// (max, sum) of two sets of a row's scores joined. A set that saw nothing has maximum
// -inf; a NaN sum travels with a finite maximum and stays.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  const float l = (a.x == -INFINITY ? 0.f : a.y * fast_exp2(a.x - m)) +
                  (b.x == -INFINITY ? 0.f : b.y * fast_exp2(b.x - m));
  return float2{m, l};
}

// The log-sum-exp (log2 units) of a sequence's rows from its items' [item][row] records
// `stride` apart: row r in lane r (and, for fewer than 64 rows, in lanes further on). A
// row that saw nothing: +inf, which makes every weight 0. Lanes lie over rows first, then
// over items, so the records of an item come in one line and few exchanges follow, and a
// lane asks for kAtOnce of them at a time (64 rows, 8 sequences of up to 12K keys, the
// kernel: one row after the other 72 us, four records at a time 31, sixteen 25).
constexpr int kAtOnce = 16;
__device__ __forceinline__ float rows_lse(const float2* st, int stride, int rows, int count) {
  const int lane = threadIdx.x & 63;
  int span = 1;
  while (span < rows) span *= 2;
  const int r = min(lane & (span - 1), rows - 1), parts = 64 / span;
  float2 x = {-INFINITY, 0.f};
  for (int i = lane / span; i < count; i += kAtOnce * parts) {
    float2 y[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) y[u] = st[(size_t)min(i + u * parts, count - 1) * stride + r];
    // One maximum for the round, then the sums.
    float m = x.x;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) m = i + u * parts < count ? fmaxf(m, y[u].x) : m;
    float l = x.x == -INFINITY ? 0.f : x.y * fast_exp2(x.x - m);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      if (i + u * parts < count && y[u].x != -INFINITY) l += y[u].y * fast_exp2(y[u].x - m);
    x = float2{m, l};
  }
  for (int o = span; o < 64; o *= 2)
    x = join(x, float2{__shfl_xor(x.x, o), __shfl_xor(x.y, o)});
  return x.y == 0.f ? INFINITY : x.x + __builtin_amdgcn_logf(x.y);
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
  static_assert(D % 4 == 0, "weights are added up four pages at a time");
  WaveItem w;
  if (!wave_item(args, w)) return;  // uniform
  const int lane = threadIdx.x & 63;
  const int g16 = lane >> 4, l16 = lane & 15;
  const int b = w.it.b, len = w.it.len, p_begin = w.it.p_begin, kvh = w.kvh;
  const int n_pages = w.it.p_end - p_begin;
  const int shift = a.page_shift, sub_mask = (1 << shift) - 1;

  // Ids of the ring's next refills, and of those a turn later on their way: scalar loads,
  // so that no wait for an id is a wait for the pages behind it (a vector load of the next
  // 64 ids drained the ring where it was taken over).
  const int32_t* row = a.block_tables + (size_t)b * a.bt_stride;
  auto load_ids = [&](int i, int (&ids)[D]) {
#pragma unroll
    for (int j = 0; j < D; ++j)
      ids[j] = scalar_load(row + (min(p_begin + max(min(i + j, n_pages - 1), 0), a.max_pages - 1) >>
                                  shift));
  };
  int first_ids[D], ids[D], ids_next[D];
  load_ids(0, first_ids);
  load_ids(D, ids);

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
    const float x = rows_lse(args.stats + ((size_t)w.it.first * a.hkv + kvh) * a.rows,
                             a.hkv * a.rows, a.rows, w.it.count);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float mine = __shfl(x, 16 * nb + l16);
      lse[nb] = map.real(nb, l16) ? mine : INFINITY;
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
    // The first pass reads K through the caches: non-temporal, its reads and the scores it
    // writes got in each other's way (16 x 32K keys, four rows: 245 -> 229 us, the second
    // kernel 20 -> 23).
#pragma unroll
    for (int i = 0; i < KEYS::kLoads; ++i)
      s.k.k[i] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_lane + 64 * i, 0,
                                                       SUM ? kStreamAux : 0);
  };
  Slot ring[D];
#pragma unroll
  for (int j = 0; j < D; ++j) load_page(j < n_pages ? clamp_page(first_ids[j], a.num_pages) : -1, p_begin + j, ring[j]);

  const int mask_from = len - a.q_len;
  float m[NB], l[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb] = -INFINITY;
    l[nb] = 0.f;
  }
  float* wrow = args.weights + b * args.w_batch + kvh * args.w_head;
  // Scores leave through a resource bounded to the item's pages, rows that are not there
  // sent past its end, so that no branch stands around a store.
  const unsigned head_scores = a.rows * kPageSize * 4u, page_scores = a.hkv * head_scores;  // bytes
  const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
      (void*)((char*)args.scores + ((size_t)b * a.max_pages + p_begin) * page_scores),
      (short)0, STORE ? (int)(n_pages * page_scores) : 0, kBufferFlags);
  unsigned out_lane[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
    out_lane[nb] = map.real(nb, l16) ? kvh * head_scores + 64u * map.row(nb, l16) + 16u * g16
                                     : kDroppedOffset;

  for (int i = 0; i < n_pages; i += D) {
    load_ids(i + 2 * D, ids_next);
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
        float c =
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
        }
        const bool masked = (p + 1) * kPageSize > mask_from;  // uniform
        if (masked) {
          // After the scale, so that a scale of 0, infinity or NaN leaves them -inf.
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) s[nb] *= c;
          c = 1.f;
          mask_scores<NB>(s, bits.b, mask_from, p * kPageSize + 4 * g16, len);
        }
        if constexpr (SUM) {
          f4 t = f4{0.f, 0.f, 0.f, 0.f};
          if (masked) {  // uniform
            // A token a row does not see gets nothing from it, NaN neither.
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                t[e] += s[nb][e] == -INFINITY ? 0.f : fast_exp2(s[nb][e] - lse[nb]);
          } else {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int e = 0; e < 4; ++e) t[e] += fast_exp2(fmaf(s[nb][e], c, -lse[nb]));
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = row16_sum(t[e]);
            mine = l16 == 4 * (j & 3) + e ? x : mine;
          }
        } else {
          if constexpr (STORE) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              s[nb] *= c;
              __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, s[nb]), out,
                                                     out_lane[nb], ii * page_scores, 0);
            }
            c = 1.f;
          }
          // The running maximum of a lane's scores may trail them by kMaxLag, as in the
          // attention kernels.
          float lm[NB];
          bool grow = false;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            lm[nb] = max4(s[nb]) * c;
            grow |= lm[nb] > m[nb] + kMaxLag;
          }
          if (__any(grow)) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              const float mn = fmaxf(m[nb], lm[nb]);
              l[nb] *= fast_exp2(m[nb] - (mn == -INFINITY ? 0.f : mn));
              m[nb] = mn;
            }
          }
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const float mu = m[nb] == -INFINITY ? 0.f : m[nb];
            l[nb] += (fast_exp2(fmaf(s[nb][0], c, -mu)) + fast_exp2(fmaf(s[nb][1], c, -mu))) +
                     (fast_exp2(fmaf(s[nb][2], c, -mu)) + fast_exp2(fmaf(s[nb][3], c, -mu)));
          }
        }
      }
      if constexpr (SUM) {
        if ((j & 3) == 3) {
          if (ii - 3 + (l16 >> 2) < n_pages && wt < min(len, args.width))
            wrow[wt] = wt < mask_from ? old + mine : mine;
        }
      }
      load_page(ii + D < n_pages ? clamp_page(ids[j], a.num_pages) : -1, p + D, ring[j]);
    }
#pragma unroll
    for (int j = 0; j < D; ++j) ids[j] = ids_next[j];
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
        args.stats[((size_t)w.it.slot * a.hkv + kvh) * a.rows + map.row(nb, l16)] =
            float2{sum == sum ? top : 0.f, sum};
    }
  }
}

// The second pass from the stored scores: a lane takes four consecutive tokens, a wave
// 256 at a time. The scores of four rows are requested before any is used (one row after
// the other a round waited for memory once per row: 16 x 32K keys, four rows, 25 us, 20
// so).
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
__global__ __launch_bounds__(256) void sqa_weigh_join_kernel(WeighArgs args) {
  const PartialArgs& a = args.p;
  WaveItem w;
  if (!wave_item(args, w)) return;  // uniform
  const int lane = threadIdx.x & 63;
  const int rows = a.rows, kvh = w.kvh;
  const int mask_from = w.it.len - a.q_len;
  const int t_end = min(min(w.it.p_end * kPageSize, w.it.len), args.width);
  const size_t page_scores = (size_t)a.hkv * rows * kPageSize;
  const float* scores = args.scores + (size_t)w.it.b * a.max_pages * page_scores +
                        (size_t)kvh * rows * kPageSize;
  float* wrow = args.weights + w.it.b * args.w_batch + kvh * args.w_head;
  // Lane r holds row r's log-sum-exp.
  const float lse = rows_lse(args.stats + ((size_t)w.it.first * a.hkv + kvh) * rows, a.hkv * rows,
                             rows, w.it.count);
  for (int t0 = w.it.p_begin * kPageSize; t0 < t_end; t0 += 256) {
    const int t = t0 + 4 * lane;
    const bool whole = t + 4 <= t_end;
    f4 old = f4{0.f, 0.f, 0.f, 0.f}, sum = old;
    if (whole) {
      old = *(const f4u*)(wrow + t);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (t + e < t_end) old[e] = wrow[t + e];
    }
    // Past the item's end: its last page again, unused.
    const float* at = scores + (size_t)(min(t, t_end - 1) >> 4) * page_scores + (t & 12);
    for (int r0 = 0; r0 < rows; r0 += 4) {
      f4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = *(const f4*)(at + min(r0 + i, rows - 1) * kPageSize);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (r0 + i >= rows) break;  // uniform
        const float lr = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, lse), r0 + i));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum[e] += x[i][e] == -INFINITY ? 0.f : fast_exp2(x[i][e] - lr);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += t + e < mask_from ? old[e] : 0.f;
    if (whole) {
      *(f4u*)(wrow + t) = sum;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (t + e < t_end) wrow[t + e] = sum[e];
    }
  }
}

// ---------------------------------------------------------------------------------
// Eviction.
// ---------------------------------------------------------------------------------

// Larger weights give larger keys; -0 and 0 the same one, NaN the least of all. Keys of
// weights lie in [kNanKey, kAlways); 0 is no token, kAlways one that stays in any case.
constexpr unsigned kNanKey = 1u, kAlways = 0xffffffffu;
__device__ __forceinline__ unsigned weight_key(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.f);  // -0 + 0 = 0
  const unsigned k = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return w != w ? kNanKey : k;
}
constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;

// What bounds eviction: 32 sequences of up to 4K keys, half of each kept, 16-bit (0.53 GB):
// the selection 10 us, the moves 108 us, 4.9 TB/s, a large copy's rate. 16 of up to 32K, 4K
// of each kept, e4m3: selection 25 us (a workgroup of one compute unit per sequence and
// head, 126 registers a thread; 35 with the weights' keys made again each time, 59 from
// memory), moves 60.

struct SelectShared {
  int hist[2048];
  int wave_tot[kSelectWaves], wave_sure[kSelectWaves], wave_tie[kSelectWaves];
  int picked, above;
};

// Which tokens of one sequence and kv head stay. The smallest key that stays is found by
// a radix selection over the weights between the sink and the recent tokens (11, 11 and
// 10 bits, histograms in LDS); tokens above it stay, and of those that equal it the first.
// Each wave then counts its own run of tokens, and after one exchange writes its kept
// tokens in order. All counts are integers: the same weights give the same tokens.
// R > 0: a thread holds its R tokens' weights and keys in registers through all of it (up to
// 1024 R tokens, none past the weights' width); R = 0 reads the weights again each time, and
// tokens past their width weigh 0 (the test of the width in the registers' form, too: 16
// ragged contexts of up to 32K, e4m3, a call 98 us for 85.5).
template <int R>
__device__ __forceinline__ void select_tokens(const EvictArgs& a, SelectShared& sm, int n,
                                              const float* w, float* nw, int32_t* kept) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m = a.budget, weighed = R > 0 ? n : min(n, a.width);
  // A wave's run: `steps` times 64 consecutive tokens.
  const int steps = (n + kSelectThreads - 1) / kSelectThreads;
  const int begin = wave * steps * 64;
  const int lo = a.sink, hi = n - a.recent;
  auto weight_at = [&](int t) {
    const float x = w[min(t, weighed - 1)];
    return R > 0 || t < weighed ? x : 0.f;
  };
  auto key_at = [&](int t, float x) {
    const unsigned k = t >= lo && t < hi ? weight_key(x) : kAlways;
    return t < n ? k : 0u;
  };
  constexpr int kHeld = R > 0 ? R : 1;
  float held_w[kHeld];
  unsigned held[kHeld];
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) held_w[i] = i < steps ? weight_at(begin + 64 * i + lane) : 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) held[i] = key_at(begin + 64 * i + lane, held_w[i]);
  }
  // each(f): f(token, key, weight) for the thread's tokens of the run in order.
  auto each = [&](auto f) {
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (i < steps) f(begin + 64 * i + lane, held[i], held_w[i]);  // uniform
    } else {
      for (int i = 0; i < steps; ++i) {
        const int t = begin + 64 * i + lane;
        const float x = weight_at(t);
        f(t, key_at(t, x), x);
      }
    }
  };
  const int free = a.budget - a.sink - a.recent;
  unsigned threshold = kAlways - 1;  // above the keys of all weights
  int ties = 0;                      // how many of the tokens at the threshold stay
  if (free > 0) {
    int want = free;
    unsigned prefix = 0, mask = 0;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      const unsigned digits = pass == 2 ? 0x3ffu : 0x7ffu;
      for (int i = tid; i < 2048; i += kSelectThreads) sm.hist[i] = 0;
      __syncthreads();
      each([&](int, unsigned k, float) {
        if (k - 1u < kAlways - 1u && (k & mask) == prefix)
          atomicAdd(&sm.hist[(k >> shift) & digits], 1);
      });
      __syncthreads();
      // Bins from the top: thread i takes bins 2047 - 2 i and 2046 - 2 i.
      const int c0 = sm.hist[2047 - 2 * tid], c1 = sm.hist[2046 - 2 * tid];
      const int incl = wave_inclusive_scan_int(c0 + c1);
      if (lane == 63) sm.wave_tot[wave] = incl;
      __syncthreads();
      int before = incl - c0 - c1;
#pragma unroll
      for (int i = 0; i < kSelectWaves; ++i) before += i < wave ? sm.wave_tot[i] : 0;
      if (before < want && want <= before + c0 + c1) {  // one thread
        const bool first = want <= before + c0;
        sm.picked = first ? 2047 - 2 * tid : 2046 - 2 * tid;
        sm.above = first ? before : before + c0;
      }
      __syncthreads();
      prefix |= (unsigned)sm.picked << shift;
      mask |= digits << shift;
      want -= sm.above;
    }
    threshold = prefix;
    ties = want;
  }
  int sures = 0, tied = 0;
  each([&](int, unsigned k, float) {
    sures += __popcll(__ballot(k > threshold));
    tied += __popcll(__ballot(k == threshold));
  });
  if (lane == 0) {
    sm.wave_sure[wave] = sures;
    sm.wave_tie[wave] = tied;
  }
  __syncthreads();
  int at = 0, seen = 0;  // kept tokens and ties before this wave's
#pragma unroll
  for (int i = 0; i < kSelectWaves; ++i) {
    at += i < wave ? sm.wave_sure[i] : 0;
    seen += i < wave ? sm.wave_tie[i] : 0;
  }
  at = __builtin_amdgcn_readfirstlane(at + min(seen, ties));
  seen = __builtin_amdgcn_readfirstlane(seen);
  auto below = [](unsigned long long mask) {  // its bits under the lane's
    return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32),
                                          __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
  };
  each([&](int t, unsigned k, float x) {
    bool keep = k > threshold;
    const unsigned long long tie_mask = __ballot(k == threshold);
    if (tie_mask && seen < ties) keep |= k == threshold && seen + below(tie_mask) < ties;  // uniform
    const unsigned long long keep_mask = __ballot(keep);
    if (keep) {
      const int to = at + below(keep_mask);
      kept[to] = t;
      if constexpr (R > 0) nw[to] = x;  // every weight has been read: nw may be w
    }
    at += __popcll(keep_mask);
    seen += __popcll(tie_mask);
  });
  if constexpr (R > 0) {
    for (int j = m + tid; j < a.new_width; j += kSelectThreads) nw[j] = 0.f;
  } else {
    __syncthreads();
    // The weights move along, 1024 at a time: new_weights may be the old ones, and a token
    // never moves to a later position.
    for (int j0 = 0; j0 < a.new_width; j0 += kSelectThreads) {
      const int j = j0 + tid;
      const int t = j < m ? kept[j] : weighed;
      const float x = t < weighed ? w[t] : 0.f;
      __syncthreads();
      if (j < a.new_width) nw[j] = x;
      __syncthreads();
    }
  }
}

template <int R>
__global__ __launch_bounds__(kSelectThreads) void sqa_select_kernel(EvictArgs a) {
  __shared__ SelectShared sm;
  const int b = blockIdx.x / a.hkv, h = blockIdx.x % a.hkv;
  const int tid = threadIdx.x;
  const float* w = a.weights + b * a.w_batch + h * a.w_head;
  float* nw = a.new_weights + b * a.nw_batch + h * a.nw_head;
  int32_t* kept = a.kept + (size_t)(b * a.hkv + h) * a.budget;
  const long long room = (long long)a.bt_stride * a.page_size;
  const int n = (int)min((long long)max(a.seq_lens[b], 0), room);
  if (h == 0 && tid == 0) a.new_lens[b] = min(n, a.budget);
  if (n <= a.budget) {
    const int weighed = min(n, a.width);
    for (int j = tid; j < a.budget; j += kSelectThreads) kept[j] = j < n ? j : -1;
    for (int j = tid; j < a.new_width; j += kSelectThreads) nw[j] = j < weighed ? w[j] : 0.f;
  } else if (n <= min(R * kSelectThreads, a.width)) {
    select_tokens<R>(a, sm, n, w, nw, kept);
  } else {
    select_tokens<0>(a, sm, n, w, nw, kept);
  }
}

// The kept tokens of 64 new slots of one kv head, K or V, moved to their new pages: a lane
// looks one token's places up, then the wave moves the rows, 16 bytes a lane, all loads
// before the first store. Scaled caches: the new block's scale is the largest of the
// scales its tokens come from, and codes from blocks of other scales are rounded again.
template <int ROW, bool SCALED, bool INT8>
__global__ __launch_bounds__(256) void sqa_move_kernel(EvictArgs a) {
  constexpr int LPT = ROW / 16;   // lanes per token (ROW: bytes of a token and head)
  constexpr int TPI = 64 / LPT;   // tokens per instruction
  constexpr int NI = 64 / TPI;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int head_groups = (a.hkv + 3) / 4;
  const int h = (blockIdx.x % head_groups) * 4 + wave;
  const int tiles = (a.budget + 63) / 64;
  const int rest = blockIdx.x / head_groups;
  const int b = rest / tiles, j0 = rest % tiles * 64;
  const int which = blockIdx.y;
  const int m = a.new_lens[b];
  if (h >= a.hkv || j0 >= m) return;
  const int page = a.page_size;
  const int32_t* kept = a.kept + (size_t)(b * a.hkv + h) * a.budget;
  const int32_t* table = a.block_tables + (size_t)b * a.bt_stride;
  // Lane l: new token j0 + l (past the last one: it again), where from and where to.
  const int j = min(j0 + lane, m - 1);
  const int from = max(kept[j], 0);
  const int np = j / page;
  const int to = np < a.new_stride ? a.new_tables[(size_t)b * a.new_stride + np] : -1;
  // A page that is not there is not written.
  const bool there = j0 + lane < m && to >= 0 && to < a.new_pages;
  const int fp = clamp_page(table[from / page], a.num_pages);
  const long long src_at = (long long)fp * a.src_page + (long long)(from % page) * a.src_token;
  const long long dst_at =
      there ? (long long)to * a.dst_page + (long long)(j % page) * a.dst_token : -1;
  float old = 1.f, scale = 1.f;
  if constexpr (SCALED) {
    const char* sc = (const char*)(which ? a.src_scales.v : a.src_scales.k) +
                     (size_t)h * a.src_scales.head_stride;
    old = *(const float*)(sc + fp * a.src_scales.page_stride);
    scale = old;
    if (page > 64) {  // the page's other tokens
      for (int i = np * page + lane; i < min(np * page + page, m); i += 64) {
        const int p = clamp_page(table[max(kept[i], 0) / page], a.num_pages);
        scale = fmaxf(scale, *(const float*)(sc + p * a.src_scales.page_stride));
      }
    }
    for (int o = 1; o < min(page, 64); o *= 2) scale = fmaxf(scale, __shfl_xor(scale, o));
    if (there && j % page == 0)
      *(float*)((char*)(which ? a.dst_scales.v : a.dst_scales.k) +
                (size_t)h * a.dst_scales.head_stride + to * a.dst_scales.page_stride) = scale;
  }
  const char* src = a.src[which] + (size_t)h * a.src_head + 16 * (lane % LPT);
  char* dst = a.dst[which] + (size_t)h * a.dst_head + 16 * (lane % LPT);
  auto of_token = [&](long long x, int t) {
    return (long long)__shfl((int)(x >> 32), t) << 32 | (unsigned)__shfl((int)x, t);
  };
  u4 x[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) x[i] = *(const u4*)(src + of_token(src_at, i * TPI + lane / LPT));
  const Quotient by = quotient(scale);
  const bool fast = __all(by.fast);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int t = i * TPI + lane / LPT;
    if constexpr (SCALED) {
      const float so = __shfl(old, t);
      const Quotient q = {__shfl(scale, t), __shfl(by.r, t), true};
      if (so != q.s) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = decode<INT8>(x[i][w], e) * so;
            y[e] = fast ? divide_fast(v, q) : (q.s > 0.f ? v / q.s : 0.f);
          }
          x[i][w] = encode4<INT8>(y);
        }
      }
    }
    const long long o = of_token(dst_at, t);
    if (o >= 0) *(u4*)(dst + o) = x[i];
  }
}

template <int HD, typename E, template <int> class KEYS, int NB>
void launch_weigh_rows(const WeighArgs& a, dim3 grid, hipStream_t stream) {
  constexpr int D = 4;
  const dim3 block(256);
  if constexpr (weights_stored(16 * (NB - 1) + 1, HD, KEYS<HD>::kBytes)) {
    if (a.scores) {
      hipLaunchKernelGGL((sqa_weigh_kernel<NB, D, HD, E, KEYS<HD>, false, true>), grid, block, 0,
                         stream, a);
      hipLaunchKernelGGL(sqa_weigh_join_kernel, grid, block, 0, stream, a);
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
  const dim3 each((unsigned)(a.batch * a.hkv)), threads(kSelectThreads);
  // The registers that the longest sequence with weights of its own needs; one that is
  // longer than its weights are wide takes the form without.
  const long long most = std::min((long long)a.width, (long long)a.bt_stride * a.page_size);
  if (most <= 4 * kSelectThreads)
    hipLaunchKernelGGL((sqa_select_kernel<4>), each, threads, 0, stream, a);
  else if (most <= 16 * kSelectThreads)
    hipLaunchKernelGGL((sqa_select_kernel<16>), each, threads, 0, stream, a);
  else if (most <= 32 * kSelectThreads)
    hipLaunchKernelGGL((sqa_select_kernel<32>), each, threads, 0, stream, a);
  else
    hipLaunchKernelGGL((sqa_select_kernel<0>), each, threads, 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int tiles = (a.budget + 63) / 64;
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

// gfx950 kernels for caches held in 8 bits with a scale for each page and kv head:
// the quantising append and small-q attention.
//
// A code c of page p and head h stands for c * s, s = scale[p][h]. With x the tokens of
// the block, s = max|x| / M (M = 448 for e4m3, 127 for int8) and c = x / s rounded to
// nearest even. Attention folds the scales into the softmax and the probabilities:
//   score(row, t)  = (scale * k_scale[page of t]) * (q . k_code[t])
//   out(row)       = sum_t (p(row, t) * v_scale[page of t]) v_code[t] / sum_t p(row, t)
// so the codes go to the MFMAs as they are (both types widen exactly to 16 bits) and a
// page costs two scalars.
//
// What bounds attention: HBM up to 32 rows, instructions at 64. 16 x 32K keys, e4m3, 1.08
// GB, whole calls beside those of e4m3 with one scale per tensor, same box: q_len 1 175 and
// 166 us, q_len 4 177 and 168, q_len 8 180 and 176 (6.0 TB/s), q_len 16 250 and 209. Batches
// whose sequences do not divide the work items leave some of the chip idle (find_split()).
// Append: 2 x 16K tokens, 0.2 GB, 43 us, 4.7 TB/s, near a large copy's 5.1.
#include "sqa_cache.h"
#include "sqa_cache_device.h"

namespace sqa {
namespace {

// ---------------------------------------------------------------------------------
// Attention.
// ---------------------------------------------------------------------------------

// One workgroup = four waves on their own: wave w serves kv head w % wg_heads of the
// workgroup's heads and work item w / wg_heads of its items, with all query rows of the
// head (NB blocks of 16). A wave keeps a ring of D pages of codes and their two scales in
// flight in registers. No barrier: waves of a workgroup meet only in the memory system,
// where the heads' slices of a token row are neighbours.
//
// The V scale of a page enters the exponent: P = 2^(c s + log2 v_scale - m), with m the
// running maximum of exactly that, is what the page's codes weigh in the sums O, so one
// fp16 rounding of P is relative to its part of the result (2^-11 of it, and 2^-25 of the
// row's largest part where it is tiny beside that), however the blocks' scales differ; two
// bf16 parts of p * v_scale cost 28 operations a page more at 32 rows (16 x 32K keys,
// whole calls: q_len 8 201 -> 178 us, q_len 16 293 -> 245). What that rounding costs: fp16
// outputs are 2.32e-4 of their size from the 64-bit result at 16 x 32K keys, q_len 8, and
// 2.06e-4 with P in 32 bits; bf16 outputs do not change. The row sum gets P / v_scale in
// fp32, unrounded: a quiet block's tokens weigh as much in it as a loud one's. Pages of a
// scale under 2^-64, 0 among them, count as of that scale in the maximum and the row sums
// and add nothing to O (a scale further down would push their P out of fp32's range).
template <int NB, int D, int HD, typename E, typename KV>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1)))
void sqa_scaled_attention_kernel(ScaledArgs args) {
  const PartialArgs& a = args.p;
  constexpr int KK = Dims<HD>::KK, MB = Dims<HD>::MB;
  __shared__ float sm_stage[4 * 16 * (HD + 4)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int g16 = lane >> 4, l16 = lane & 15;
  const int wgh = args.wg_heads;
  const int head_groups = (a.hkv + wgh - 1) / wgh;
  const int kvh = (blockIdx.x % head_groups) * wgh + wave % wgh;
  const int item = (blockIdx.x / head_groups) * (4 / wgh) + wave / wgh;
  const WaveRows<NB, 1> map{kvh, a.rows, a.hkv};
  if (kvh >= a.hkv) return;

  Split it;
  it.b = it.len = it.p_begin = it.p_end = it.slot = 0;
  it.count = 1;
  const bool writer = blockIdx.x == 0 && wave == 0;
  if (!find_split(a, args.items, item, writer ? a.seq_splits : nullptr, it)) return;  // uniform
  const int b = __builtin_amdgcn_readfirstlane(it.b);
  const int len = __builtin_amdgcn_readfirstlane(it.len);
  const int p_begin = __builtin_amdgcn_readfirstlane(it.p_begin);
  const int n_pages = max(__builtin_amdgcn_readfirstlane(it.p_end) - p_begin, 0);
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
      const u4 x = *(const u4*)(qp + KV::q_dims(kk, g16));
      q[nb][kk] = real ? x : u4{0u, 0u, 0u, 0u};
    }
    bits.b[nb] = draft_bits(a, b, qi, real);
  }

  const unsigned tok_bytes = a.token_stride;
  const unsigned k_lane = l16 * tok_bytes + kvh * a.head_stride + KV::k_lane_bytes(g16);
  const unsigned v_lane = 4 * g16 * tok_bytes + kvh * a.head_stride + KV::v_lane_bytes(l16);
  const size_t sub_bytes = (size_t)kPageSize * tok_bytes;
  // Lanes 0-31 load the page's K scale, 32-63 its V scale: one instruction, one register.
  const char* scale_lane =
      (const char*)(lane < 32 ? args.scales.k : args.scales.v) +
      (size_t)kvh * args.scales.head_stride;
  struct Slot {
    typename KV::Regs kv;
    float scale;
  };
  // pid < 0: zeros, without touching memory (and some page's scales).
  auto load_page = [&](int pid, int p, Slot& s) {
    pid = __builtin_amdgcn_readfirstlane(pid);
    const size_t off =
        pid >= 0 ? (size_t)pid * (size_t)a.page_stride + (size_t)(p & sub_mask) * sub_bytes : 0;
    const int nrec = pid >= 0 ? (int)a.page_extent : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((const char*)a.k + off), (short)0, nrec, kBufferFlags);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
        (void*)((const char*)a.v + off), (short)0, nrec, kBufferFlags);
    s.scale = *(const float*)(scale_lane + max(pid, 0) * args.scales.page_stride);
    KV::load(s.kv, kr, vr, k_lane, v_lane, tok_bytes);
  };
  Slot ring[D];
#pragma unroll
  for (int j = 0; j < D; ++j) load_page(j < n_pages ? clamp_page(first_ids[j], a.num_pages) : -1, p_begin + j, ring[j]);

  WaveState<NB, HD> st;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    st.m[nb] = -INFINITY;
    st.l[nb] = 0.f;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) st.acc[mb][nb] = f4{0.f, 0.f, 0.f, 0.f};
  }
  const int mask_from = len - a.q_len;  // pages with a token from here on are masked

  for (int i = 0; i < n_pages; i += D) {
    load_ids(i + 2 * D, ids_next);
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int ii = i + j;
      if (ii < n_pages) {
        const int p = p_begin + ii;
        const float ks = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ring[j].scale), 0));
        const float vs = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ring[j].scale), 32));
        const bool loud = !(vs < 0x1p-64f);
        const float lv = loud ? __builtin_amdgcn_logf(vs) : -64.f;
        const float inv_vs = loud ? __builtin_amdgcn_rcpf(vs) : 0x1p64f;
        float c = a.scale_log2 * ks, add = lv;
        f4 s[NB];
        code_scores<NB, HD, E, KV>(s, ring[j].kv, q);
        const bool masked = (p + 1) * kPageSize > mask_from;  // uniform
        if (masked) {
          // After the scales, so that one of 0, infinity or NaN leaves them -inf.
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) s[nb] = s[nb] * c + lv;
          c = 1.f;
          add = 0.f;
          const int tok0 = p * kPageSize + 4 * g16;
          mask_scores<NB>(s, bits.b, mask_from, tok0, len);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (tok0 + e >= len)
#pragma unroll
              for (int w = 0; w < Dims<HD>::VW / 2; ++w) ring[j].kv.v[e][w] = 0u;
          if constexpr (KV::kNan) nan_values<NB, HD, KV>(st, ring[j].kv, s);
        }
        float lm[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) lm[nb] = fmaf(max4(s[nb]), c, add);
        raise_max<NB, HD>(st, lm);
        u2 ph[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float off = add - (st.m[nb] == -INFINITY ? 0.f : st.m[nb]);
          float pr[4], rounded = 0.f;
          u2 none;
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
          const u2 none = {0u, 0u};
          u2 av[MB];
          KV::operand_v(ring[j].kv, av);
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              st.acc[mb][nb] = ElemF16::mma_pv(av[mb], ph[nb], none, st.acc[mb][nb]);
        }
      }
      load_page(ii + D < n_pages ? clamp_page(ids[j], a.num_pages) : -1, p_begin + ii + D, ring[j]);
    }
#pragma unroll
    for (int j = 0; j < D; ++j) ids[j] = ids_next[j];
  }
  write_results<NB, HD, PartialRows<E>>(a, st, sm_stage + wave * 16 * (HD + 4), map, it.count <= 1, false, b,
                           (size_t)it.slot, a.hkv, 0);
}

// ---------------------------------------------------------------------------------
// Append.
// ---------------------------------------------------------------------------------

template <bool BF16>
__device__ __forceinline__ float from_half(unsigned bits) {
  if constexpr (BF16)
    return __builtin_bit_cast(float, bits << 16);
  else
    return (float)__builtin_bit_cast(_Float16, (unsigned short)bits);
}

// The token as it is stored: infinities count as the type's largest finite value.
template <bool BF16>
__device__ __forceinline__ float finite(float x) {
  const float top = BF16 ? 3.3895313892515355e38f : 65504.f;
  return x != x ? x : fminf(fmaxf(x, -top), top);
}

// One block: a cache page's tokens of one kv head, K or V. Its waves (page / 16, at most
// four) take TPW runs of 16 tokens each and meet for the block's largest magnitude; the
// workgroup's other waves take other heads. The new tokens are read once and held in
// registers from the maximum to the codes. A block that keeps earlier tokens of its
// sequence (the first one, if the new tokens start inside a page) keeps their scale as a
// lower bound; where it grows, their codes are rounded again in the new one. Slots past
// the last new token stay as they are.
template <int HD, int TPW, bool BF16, bool INT8>
__global__ __launch_bounds__(256) void sqa_append_kernel(AppendArgs a) {
  constexpr int LPT = HD / 8;       // lanes per token, 8 dims each
  constexpr int TPI = 64 / LPT;     // tokens per instruction
  constexpr int NI = 16 / TPI;      // instructions per run of 16 tokens
  __shared__ float sm_top[4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int runs = a.page_size / 16;
  const int wpb = runs < 4 ? runs : 4;  // waves per block
  const int heads = 4 / wpb;            // heads per workgroup
  const int head_groups = (a.hkv + heads - 1) / heads;
  const int which = blockIdx.y;
  const int h = (blockIdx.x % head_groups) * heads + wave / wpb;
  const int rest = blockIdx.x / head_groups;
  const int b = rest / a.touched, at = rest % a.touched;
  const int len = max(a.seq_lens[b], 0);
  int fresh = a.new_lens ? a.new_lens[b] : a.q_len;
  fresh = min(max(fresh, 0), min(a.q_len, len));
  const int first = len - fresh;             // position of the first new token
  const int pg = first / a.page_size + at;   // page within the sequence
  const int base = pg * a.page_size;
  if (fresh == 0 || base >= len || pg >= a.bt_stride) return;  // uniform over the workgroup
  const int pid = a.block_tables[(size_t)b * a.bt_stride + pg];
  if (pid < 0 || pid >= a.num_pages) return;  // uniform: a page that is not there is not written
  const bool active = h < a.hkv;
  const int lo = max(first - base, 0), hi = min(len - base, a.page_size);
  const int token = lane / LPT, dim = 8 * (lane % LPT);

  char* codes = (char*)a.cache[which] + (size_t)pid * a.page_stride + (size_t)h * a.head_stride;
  const char* src = (const char*)a.src[which] + (long long)b * a.src_batch[which] +
                    (long long)h * a.src_head[which];
  float* scale_at = (float*)((char*)(which ? a.scales.v : a.scales.k) +
                             (size_t)pid * a.scales.page_stride + (size_t)h * a.scales.head_stride);
  u4 x[TPW][NI];
  const float old = active ? *scale_at : 0.f;
#pragma unroll
  for (int t = 0; t < TPW; ++t) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int slot = 16 * ((wave % wpb) * TPW + t) + i * TPI + token;
      x[t][i] = u4{0u, 0u, 0u, 0u};
      if (active && slot >= lo && slot < hi)
        x[t][i] = *(const u4*)(src + (long long)(base + slot - first) * a.src_token[which] +
                               2 * dim);
    }
  }
  // The largest magnitude as the largest bit pattern; at the infinity's and past it
  // (rare) the values are looked at again.
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  constexpr unsigned kInfinity = BF16 ? 0x7f80u : 0x7c00u;
  us2 most = {0, 0};
#pragma unroll
  for (int t = 0; t < TPW; ++t)
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w)
        most = __builtin_elementwise_max(most,
                                         __builtin_bit_cast(us2, x[t][i][w] & 0x7fff7fffu));
  const unsigned bits = max((unsigned)most[0], (unsigned)most[1]);
  float top = from_half<BF16>(bits);
  const bool wild = __any(bits >= kInfinity);  // uniform
  if (wild) {
    top = 0.f;
#pragma unroll
    for (int t = 0; t < TPW; ++t)
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          // fmaxf passes over NaN.
          top = fmaxf(top, fabsf(finite<BF16>(from_half<BF16>(x[t][i][w] & 0xffffu))));
          top = fmaxf(top, fabsf(finite<BF16>(from_half<BF16>(x[t][i][w] >> 16))));
        }
  }
#pragma unroll
  for (int o = 1; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
  if (wpb > 1) {  // uniform
    if (lane == 0) sm_top[wave] = top;
    __syncthreads();
    for (int i = 0; i < wpb; ++i) top = fmaxf(top, sm_top[wave / wpb * wpb + i]);
  }
  if (!active) return;
  float scale = top / code_max(INT8 ? kInt8 : kE4M3);
  if (lo > 0) scale = fmaxf(scale, old);
  if (wave % wpb == 0 && lane == 0) *scale_at = scale;
  const bool again = lo > 0 && scale != old;  // uniform over the block
  const Quotient by = quotient(scale);
  const bool plain = __all(by.fast) && !wild;  // uniform
  auto store = [&](auto divide, auto value) {
#pragma unroll
    for (int t = 0; t < TPW; ++t) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int slot = 16 * ((wave % wpb) * TPW + t) + i * TPI + token;
        u2* to = (u2*)(codes + (size_t)slot * a.token_stride + dim);
        float y[2][4];
        if (slot >= lo && slot < hi) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const unsigned w = x[t][i][e / 2];
            y[e / 4][e % 4] = divide(value(from_half<BF16>(e & 1 ? w >> 16 : w & 0xffffu)));
          }
          *to = u2{encode4<INT8>(y[0]), encode4<INT8>(y[1])};
        } else if (again && slot < lo) {
          const u2 w = *to;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e / 4][e % 4] = divide(decode<INT8>(w[e / 4], e % 4) * old);
          *to = u2{encode4<INT8>(y[0]), encode4<INT8>(y[1])};
        }
      }
    }
  };
  if (plain)
    store([&](float v) { return divide_fast(v, by); }, [](float v) { return v; });
  else
    store([&](float v) { return scale > 0.f ? v / scale : 0.f; },
          [](float v) { return finite<BF16>(v); });
}

template <int HD, bool BF16, bool INT8>
void launch_append_hd(const AppendArgs& a, dim3 grid, hipStream_t stream) {
  if (a.page_size <= 64)
    hipLaunchKernelGGL((sqa_append_kernel<HD, 1, BF16, INT8>), grid, dim3(256), 0, stream, a);
  else if (a.page_size == 128)
    hipLaunchKernelGGL((sqa_append_kernel<HD, 2, BF16, INT8>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((sqa_append_kernel<HD, 4, BF16, INT8>), grid, dim3(256), 0, stream, a);
}

template <bool BF16, bool INT8>
void launch_append_as(const AppendArgs& a, dim3 grid, hipStream_t stream) {
  if (a.head_dim == 64)
    launch_append_hd<64, BF16, INT8>(a, grid, stream);
  else if (a.head_dim == 128)
    launch_append_hd<128, BF16, INT8>(a, grid, stream);
  else
    launch_append_hd<256, BF16, INT8>(a, grid, stream);
}

// Ring depths: as many pages in flight as hold about 16 KiB of codes per wave; half of
// that at 33 to 64 rows, whose accumulators take the registers. Whole calls, 16 x 32K keys,
// e4m3, us, with half as many pages / these / twice as many: head dim 128 (4 pages) q_len 1
// 181 / 175 / 177, q_len 8 200 / 181 / 183, q_len 16 (2 pages) 370 / 254 / 255; head dim
// 256 (2) q_len 1 334 / 319 / 321, q_len 8 490 / 330 / 331; head dim 64 (8) q_len 1 109 /
// 113 / -, q_len 4 105 / 107 / 109 (12 pages), q_len 8 125 / 125 / -, with int8 150 / 147 /
// -, q_len 16 (4) 183 / 175 / 176.
template <int HD, typename E, typename KV>
void launch_scaled_hd(const ScaledArgs& a, dim3 grid, hipStream_t stream) {
  constexpr int D = 4 * 128 / HD;
  const dim3 block(256);
  if (a.p.rows <= 16)
    hipLaunchKernelGGL((sqa_scaled_attention_kernel<1, D, HD, E, KV>), grid, block, 0,
                       stream, a);
  else if (a.p.rows <= 32)
    hipLaunchKernelGGL((sqa_scaled_attention_kernel<2, D, HD, E, KV>), grid, block, 0,
                       stream, a);
  else if constexpr (HD != 256)
    hipLaunchKernelGGL((sqa_scaled_attention_kernel<4, D / 2, HD, E, KV>), grid, block, 0,
                       stream, a);
}

template <typename E, template <int> class KV>
void launch_scaled_as(const ScaledArgs& a, dim3 grid, hipStream_t stream) {
  if (a.p.head_dim == 64)
    launch_scaled_hd<64, E, KV<64>>(a, grid, stream);
  else if (a.p.head_dim == 128)
    launch_scaled_hd<128, E, KV<128>>(a, grid, stream);
  else
    launch_scaled_hd<256, E, KV<256>>(a, grid, stream);
}

}  // namespace

hipError_t launch_scaled(const ScaledArgs& a, hipStream_t stream) {
  const int head_groups = (a.p.hkv + a.wg_heads - 1) / a.wg_heads;
  const int per_wg = 4 / a.wg_heads;
  const int items = a.items > a.p.batch ? a.items : a.p.batch;
  const dim3 grid((unsigned)((items + per_wg - 1) / per_wg * head_groups));
  if (a.p.bf16) {
    if (a.int8)
      launch_scaled_as<ElemBF16, CodesInt8>(a, grid, stream);
    else
      launch_scaled_as<ElemBF16, CodesFp8>(a, grid, stream);
  } else {
    if (a.int8)
      launch_scaled_as<ElemF16, CodesInt8>(a, grid, stream);
    else
      launch_scaled_as<ElemF16, CodesFp8>(a, grid, stream);
  }
  return hipGetLastError();
}

hipError_t launch_append(const AppendArgs& a, hipStream_t stream) {
  const int runs = a.page_size / 16;
  const int heads = 4 / (runs < 4 ? runs : 4);
  const int head_groups = (a.hkv + heads - 1) / heads;
  const dim3 grid((unsigned)((long long)a.batch * a.touched * head_groups), 2);
  if (a.bf16) {
    if (a.int8)
      launch_append_as<true, true>(a, grid, stream);
    else
      launch_append_as<true, false>(a, grid, stream);
  } else {
    if (a.int8)
      launch_append_as<false, true>(a, grid, stream);
    else
      launch_append_as<false, false>(a, grid, stream);
  }
  return hipGetLastError();
}

}  // namespace sqa

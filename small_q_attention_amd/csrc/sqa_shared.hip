// gfx950 kernels of attention over the pages that a group of sequences shares: the rows of
// all of them, count * Q * (Hq / Hkv) of a kv head, against one K and V, so that a page is
// read once for the group and not once for each sequence.
#include "sqa_part.h"
#include "sqa_part_device.h"

namespace sqa {

namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));

// Products over 16 k: operands of 8 elements per lane (lane l: m or n = l % 32, k = 8 (l / 32)
// + 0 .. 7), results in 16 registers (r: m = 8 (r / 4) + 4 (l / 32) + r % 4, n = l % 32).
template <typename E>
__device__ __forceinline__ f16v mma32(u4 a, u4 b, f16v c) {
  if constexpr (E::kHalfPartials)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a),
                                                  __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a),
                                                   __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

constexpr int kTilePages = 4;                      // 64 keys
constexpr int kTileKeys = kTilePages * kPageSize;

// A tile of 64 rows (tokens) of HD 16-bit elements in LDS. The 16-byte chunks of a row are
// permuted by the row, so that neither eight rows' reads of one chunk (K) nor four rows'
// reads of 64 neighbouring bytes (V, transposed) meet in a bank.
template <int HD>
struct Tile {
  static constexpr int kRow = 2 * HD;  // bytes
  static constexpr int kBytes = kTileKeys * kRow;
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (HD == 64)
      return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
    else
      return (row & 3) << 2 | ((row >> 2) & 3);
  }
  static __device__ __forceinline__ int at(int row, int chunk) {
    return row * kRow + ((chunk ^ swizzle(row)) << 4);
  }
};

// How a page travels from memory to LDS: 16-byte loads, 16-bit elements kept, codes widened
// (exactly) as they are stored.
template <int HD, int BYTES>
struct PageLoads {
  static constexpr int kLanes = HD * BYTES / 16;     // lanes per token
  static constexpr int kTokens = 64 / kLanes;        // tokens per load
  static constexpr int kLoads = kPageSize / kTokens;
  u4 x[kLoads];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned lane_at, unsigned tok) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      x[i] = __builtin_amdgcn_raw_buffer_load_b128(r, lane_at, i * kTokens * tok, 0);
  }
};

struct StoreNative {
  static constexpr int kBytes = 2;
  static constexpr bool kScaled = false;
  template <typename E>
  static __device__ __forceinline__ void widen(u4 x, u4 (&to)[1]) { to[0] = x; }
};
struct StoreFp8 {
  static constexpr int kBytes = 1;
  static constexpr bool kScaled = false;
  template <typename E>
  static __device__ __forceinline__ void widen(u4 x, u4 (&to)[2]) {
    to[0] = E::widen_fp8(u2{x[0], x[1]});
    to[1] = E::widen_fp8(u2{x[2], x[3]});
  }
};
struct StoreCodesFp8 : StoreFp8 {
  static constexpr bool kScaled = true;
};
struct StoreCodesInt8 {
  static constexpr int kBytes = 1;
  static constexpr bool kScaled = true;
  template <typename E>
  static __device__ __forceinline__ void widen(u4 x, u4 (&to)[2]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      auto byte = [&](int e) { return (float)(signed char)(x[i] >> (8 * e)); };
      to[i / 2][2 * (i & 1)] = E::pack2(byte(0), byte(1));
      to[i / 2][2 * (i & 1) + 1] = E::pack2(byte(2), byte(3));
    }
  }
};

// One workgroup: a block of 128 NBW of a group's rows of one kv head, 32 NBW to a wave, over
// one split of the shared pages, 64 keys at a time. Each wave brings one of a tile's four
// pages to LDS, two buffers in turn; all waves read all of it.
//
// S^T = K Q^T leaves a lane with half of the keys of its row, so that maxima and sums stay
// in the lane but for one exchange between two lanes; O^T = V^T P^T takes P from those
// registers as they are: the product's k order is the order the registers hold the keys in,
// and V comes transposed from LDS in the same order.
template <int HD, int NBW, typename E, typename KV>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1)))
void sqa_shared_kernel(PartArgs args) {
  using EV = std::conditional_t<KV::kScaled, ElemF16, E>;  // type of P and V
  using T = Tile<HD>;
  using Loads = PageLoads<HD, KV::kBytes>;
  constexpr int KS = HD / 16;    // k steps of the scores
  constexpr int MB = HD / 32;    // blocks of 32 output dims
  constexpr int kStageRow = HD + 4;
  constexpr int kStage = 4 * 32 * kStageRow * 4;
  constexpr int kLds = 4 * T::kBytes > kStage ? 4 * T::kBytes : kStage;
  __shared__ __attribute__((aligned(16))) char lds[kLds];
  __shared__ float lds_scale[2][2][kTilePages];  // of a tile's pages: buffer, K and V, page
  const PartialArgs& a = args.p;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int l32 = lane & 31, h = lane >> 5;
  const int share = (int)blockIdx.x / a.by_head_groups;  // heads
  const int kvh = blockIdx.x - share * a.hkv;
  const SharedItem it = args.items[share];
  const SharedGroup g = args.groups[it.group];
  const int b = __builtin_amdgcn_readfirstlane(leader_of(args, g));
  if (b < 0) return;  // uniform over the workgroup
  const int first_page = it.split * g.size;
  const int n_pages = max(min(first_page + g.size, min(g.pages, a.max_pages)) - first_page, 0);
  const int tiles = (n_pages + kTilePages - 1) / kTilePages;
  const int row0 = it.block * (128 * NBW) + wave * (32 * NBW);  // of the group's rows
  const int n_rows = g.count * a.rows;

  // This wave's page of a tile, from memory to registers.
  const int shift = a.page_shift, sub_mask = (1 << shift) - 1;
  const int32_t* table = a.block_tables + (size_t)b * a.bt_stride;
  const unsigned tok = a.token_stride;
  const size_t sub_bytes = (size_t)kPageSize * tok;
  const int ltok = lane / Loads::kLanes, lchunk = lane % Loads::kLanes;
  const unsigned lane_at = ltok * tok + kvh * a.head_stride + 16 * lchunk;
  auto id_of = [&](int tile) {
    const int p = min(first_page + max(min(tile * kTilePages + wave, n_pages - 1), 0),
                      a.max_pages - 1);
    return scalar_load(table + (p >> shift));
  };
  Loads kreg, vreg;
  float scale_reg = 0.f;
  auto fetch = [&](int tile, int id) {
    const int i = tile * kTilePages + wave;
    const int pid = i < n_pages ? clamp_page(id, a.num_pages) : -1;
    const size_t off = pid >= 0 ? (size_t)pid * (size_t)a.page_stride +
                                      (size_t)((first_page + i) & sub_mask) * sub_bytes : 0;
    const int nrec = pid >= 0 ? (int)a.page_extent : 0;
    kreg.load(__builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.k + off), (short)0, nrec,
                                                kBufferFlags), lane_at, tok);
    vreg.load(__builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.v + off), (short)0, nrec,
                                                kBufferFlags), lane_at, tok);
    if constexpr (KV::kScaled)  // lanes 0-31 the page's K scale, 32-63 its V scale
      scale_reg = *(const float*)((const char*)(h == 0 ? args.scales.k : args.scales.v) +
                                  max(pid, 0) * args.scales.page_stride +
                                  (size_t)kvh * args.scales.head_stride);
  };
  auto put = [&](int buffer) {
    char* to = lds + buffer * 2 * T::kBytes;
    constexpr int N = 2 / KV::kBytes;  // LDS chunks per loaded chunk
#pragma unroll
    for (int i = 0; i < Loads::kLoads; ++i) {
      const int row = wave * kPageSize + i * Loads::kTokens + ltok;
      u4 x[N], y[N];
      KV::template widen<E>(kreg.x[i], x);
      KV::template widen<EV>(vreg.x[i], y);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        *(u4*)(to + T::at(row, N * lchunk + n)) = x[n];
        *(u4*)(to + T::kBytes + T::at(row, N * lchunk + n)) = y[n];
      }
    }
    if constexpr (KV::kScaled)
      if (l32 == 0) lds_scale[buffer][h][wave] = scale_reg;
  };

  // Rows of the queries as the scores' B operand.
  auto out_row = [&](int x) -> long long {
    const int i = x / args.by_rows;
    const int y = x - i * a.rows;
    const int qi = y / a.by_group;
    return ((long long)(g.first + i) * a.q_len + qi) * a.hq + kvh * a.group + (y - qi * a.group);
  };
  int id_next = id_of(0);
  fetch(0, id_next);
  id_next = id_of(1);
  u4 q[NBW][KS];
#pragma unroll
  for (int nb = 0; nb < NBW; ++nb) {
    const int x = row0 + 32 * nb + l32;
    const _Float16* qp = a.q + out_row(min(x, n_rows - 1)) * HD + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[nb][ks] = *(const u4*)(qp + 16 * ks);
      if (x >= n_rows) q[nb][ks] = u4{0u, 0u, 0u, 0u};
    }
  }
  f16v acc[MB][NBW];
  float m[NBW], l[NBW];
#pragma unroll
  for (int nb = 0; nb < NBW; ++nb) {
    m[nb] = -INFINITY;
    l[nb] = 0.f;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[mb][nb][r] = 0.f;
  }
  // Where the lane reads its operands in a tile.
  int k_at[KS], v_at[MB][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) k_at[ks] = T::at(l32, 2 * ks + h);
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int l16 = lane & 15, pair = (lane >> 4) & 1;
      v_at[mb][half] = T::at(8 * half + 4 * h + l16 / 4, 4 * mb + 2 * pair + (l16 % 4) / 2) +
                       8 * (l16 % 2) + T::kBytes;
    }

  put(0);
  __syncthreads();
  const float c = a.scale_log2;
  for (int t = 0; t < tiles; ++t) {
    const char* tile = lds + (t & 1) * 2 * T::kBytes;
    if (t + 1 < tiles) {  // uniform
      fetch(t + 1, id_next);
      id_next = id_of(t + 2);
    }
    f16v s[2][NBW];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int nb = 0; nb < NBW; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][nb][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u4 k = *(const u4*)(tile + k_at[ks] + kb * 32 * T::kRow);
#pragma unroll
        for (int nb = 0; nb < NBW; ++nb) s[kb][nb] = mma32<E>(k, q[nb][ks], s[kb][nb]);
      }
    }
    // Codes: scores and, in the exponent, the V scale (as in sqa_scaled_attention_kernel).
    float cs = c;
    float inv_vs[kTilePages];
    bool loud[kTilePages];
    if constexpr (KV::kScaled) {
      cs = 1.f;
#pragma unroll
      for (int pg = 0; pg < kTilePages; ++pg) {
        auto uniform = [](float x) {
          return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
        };
        const float ks = c * uniform(lds_scale[t & 1][0][pg]);
        const float vs = uniform(lds_scale[t & 1][1][pg]);
        loud[pg] = !(vs < 0x1p-64f);
        const float lv = loud[pg] ? __builtin_amdgcn_logf(vs) : -64.f;
        inv_vs[pg] = loud[pg] ? __builtin_amdgcn_rcpf(vs) : 0x1p64f;
#pragma unroll
        for (int nb = 0; nb < NBW; ++nb)
#pragma unroll
          for (int r = 8 * (pg % 2); r < 8 * (pg % 2) + 8; ++r)
            s[pg / 2][nb][r] = fmaf(s[pg / 2][nb][r], ks, lv);
      }
    }
    const int left = n_pages - t * kTilePages;  // pages of the tile and after it
    if (left < kTilePages) {                    // uniform: the last tile of a split
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int nb = 0; nb < NBW; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[kb][nb][r] = 2 * kb + r / 8 < left ? s[kb][nb][r] : -INFINITY;
    }
    float lm[NBW];
    bool grow = false;
#pragma unroll
    for (int nb = 0; nb < NBW; ++nb) {
      float x = max3_raw(s[0][nb][0], s[0][nb][1], s[0][nb][2]);
#pragma unroll
      for (int r = 3; r < 31; r += 2)
        x = max3_raw(x, s[r / 16][nb][r % 16], s[(r + 1) / 16][nb][(r + 1) % 16]);
      x = max3_raw(x, s[1][nb][15], s[1][nb][15]);
      lm[nb] = x * cs;
      grow |= lm[nb] > m[nb] + kMaxLag;
    }
    if (__any(grow)) {
#pragma unroll
      for (int nb = 0; nb < NBW; ++nb) {
        const LanePair both = lane_pair<32>(lm[nb]);
        const float mn = fmaxf(m[nb], fmaxf(both.lo, both.hi));
        const float alpha = fast_exp2(m[nb] - (mn == -INFINITY ? 0.f : mn));
        m[nb] = mn;
        l[nb] *= alpha;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) acc[mb][nb] *= alpha;
      }
    }
    u4 p[2][2][NBW];  // of 16 keys each
#pragma unroll
    for (int nb = 0; nb < NBW; ++nb) {
      const float mu = m[nb] == -INFINITY ? 0.f : m[nb];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          float e[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) e[r] = fast_exp2(fmaf(s[kb][nb][8 * st + r], cs, -mu));
          if constexpr (KV::kScaled) {
            const int pg = 2 * kb + st;
            l[nb] = fmaf(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])),
                         inv_vs[pg], l[nb]);
            const u4 w = EV::pack8(e);
            p[kb][st][nb] = loud[pg] ? w : u4{0u, 0u, 0u, 0u};
          } else if constexpr (EV::kHalfPartials) {
            const h2 ones = {(_Float16)1.0f, (_Float16)1.0f};
            u4 w;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const h2 x = {(_Float16)e[2 * r], (_Float16)e[2 * r + 1]};
              l[nb] = __builtin_amdgcn_fdot2(x, ones, l[nb], false);
              w[r] = __builtin_bit_cast(unsigned, x);
            }
            p[kb][st][nb] = w;
          } else {
            l[nb] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
            p[kb][st][nb] = EV::pack8(e);
          }
        }
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          u4 v;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int at = v_at[mb][half] + (32 * kb + 16 * st) * T::kRow;
            const u2 x = __builtin_bit_cast(
                u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s4v*)(tile + at)));
            v[2 * half] = x[0];
            v[2 * half + 1] = x[1];
          }
#pragma unroll
          for (int nb = 0; nb < NBW; ++nb) acc[mb][nb] = mma32<EV>(v, p[kb][st][nb], acc[mb][nb]);
        }
    if (t + 1 < tiles) put((t + 1) & 1);
    __syncthreads();
  }

  // Partial rows, a block of 32 at a time through LDS.
  const long long first = args.shared_at + g.base + ((long long)it.split * a.hkv + kvh) * n_rows;
  float* stage = (float*)lds + wave * 32 * kStageRow;
  const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
      (void*)a.part_o, (short)0, (int)a.part_o_bytes, kBufferFlags);
#pragma unroll
  for (int nb = 0; nb < NBW; ++nb) {
    const int x0 = row0 + 32 * nb;
    if (x0 >= n_rows) break;  // uniform
    const LanePair both = lane_pair<32>(l[nb]);
    const float sum = both.lo + both.hi;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = acc[mb][nb][4 * i + r];
        *(f4*)(stage + l32 * kStageRow + 32 * mb + 8 * i + 4 * h) = o;
      }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    constexpr int CPR = HD / 4;
#pragma unroll
    for (int i = 0; i < CPR / 2; ++i) {
      const int e = i * 64 + lane;  // row e / CPR (< 32), chunk e % CPR
      const int rs = e / CPR;
      const f4 v = *(const f4*)(stage + rs * kStageRow + 4 * (e % CPR));
      const unsigned at = (unsigned)(((first + x0 + rs) * HD + 4 * (e % CPR)) * 4);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), pr,
                                             x0 + rs < n_rows ? at : kDroppedOffset, 0,
                                             kThroughAux);
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    if (h == 0 && x0 + l32 < n_rows) {
      // A NaN sum travels with a finite max, so the join counts the split.
      const float m_out = sum == sum ? m[nb] : 0.f;
      store_through(a.part_ml + (first + x0 + l32) * 2,
                    __builtin_bit_cast(unsigned long long, float2{m_out, sum}));
    }
  }
}

template <int HD, typename E, typename KV>
void launch_tile_hd(const PartArgs& a, dim3 grid, hipStream_t stream) {
  if constexpr (HD != 256)
    if (a.block_rows == 256) {
      hipLaunchKernelGGL((sqa_shared_kernel<HD, 2, E, KV>), grid, dim3(256), 0, stream, a);
      return;
    }
  hipLaunchKernelGGL((sqa_shared_kernel<HD, 1, E, KV>), grid, dim3(256), 0, stream, a);
}

template <typename E, typename KV>
void launch_tile_as(const PartArgs& a, dim3 grid, hipStream_t stream) {
  if (a.p.head_dim == 64)
    launch_tile_hd<64, E, KV>(a, grid, stream);
  else if (a.p.head_dim == 128)
    launch_tile_hd<128, E, KV>(a, grid, stream);
  else
    launch_tile_hd<256, E, KV>(a, grid, stream);
}

template <typename E>
void launch_tile(const PartArgs& a, dim3 grid, hipStream_t stream) {
  if (a.scaled && a.kv_type == kInt8)
    launch_tile_as<E, StoreCodesInt8>(a, grid, stream);
  else if (a.scaled)
    launch_tile_as<E, StoreCodesFp8>(a, grid, stream);
  else if (a.kv_type == kE4M3)
    launch_tile_as<E, StoreFp8>(a, grid, stream);
  else
    launch_tile_as<E, StoreNative>(a, grid, stream);
}

}  // namespace

hipError_t launch_shared(const PartArgs& a, hipStream_t stream) {
  if (a.block_rows > 64) {
    PartArgs t = a;
    t.p.by_head_groups = fast_div(a.p.hkv);
    const dim3 grid((unsigned)((long long)a.n_items * a.p.hkv));
    if (a.p.bf16)
      launch_tile<ElemBF16>(t, grid, stream);
    else
      launch_tile<ElemF16>(t, grid, stream);
    return hipGetLastError();
  }
  const dim3 grid = part_grid(a, a.n_items);
  if (a.p.bf16)
    launch_part<ElemBF16, true>(a, a.block_rows, grid, stream);
  else
    launch_part<ElemF16, true>(a, a.block_rows, grid, stream);
  return hipGetLastError();
}

}  // namespace sqa

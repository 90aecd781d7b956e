// Attention over the pages that a group of sequences shares, where its rows are more than
// one wave holds: the rows of all of them, count * Q * (Hq / Hkv) of a kv head, against one K
// and V, so that a page is read once for a block of rows and not once for each sequence.
#pragma once

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

// How tokens travel from memory to LDS: 16-byte loads (8 where a wave's tokens are fewer than
// fill them), 16-bit elements kept, codes widened (exactly) as they are stored.
template <int HD, int BYTES, int TOKENS>
struct PageLoads {
  static constexpr int kWidth = TOKENS * HD * BYTES < 64 * 16 ? 8 : 16;  // bytes of a load
  static constexpr int kLanes = HD * BYTES / kWidth;                     // lanes per token
  static constexpr int kTokens = 64 / kLanes;                            // tokens per load
  static constexpr int kLoads = TOKENS / kTokens;
  static constexpr int kChunks = kWidth / BYTES / 8;                     // of LDS, per load
  static_assert(kLoads >= 1, "a wave brings at least one load's tokens");
  u4 x[kLoads];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned lane_at, unsigned tok) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if constexpr (kWidth == 16) {
        x[i] = __builtin_amdgcn_raw_buffer_load_b128(r, lane_at, i * kTokens * tok, 0);
      } else {
        const u2 y = __builtin_amdgcn_raw_buffer_load_b64(r, lane_at, i * kTokens * tok, 0);
        x[i] = u4{y[0], y[1], 0u, 0u};
      }
    }
  }
};

// kInf: elements may be infinite.
struct StoreNative {
  static constexpr int kBytes = 2;
  static constexpr bool kScaled = false, kInf = true;
  template <typename E>
  static __device__ __forceinline__ void widen(u4 x, u4 (&to)[1]) { to[0] = x; }
};
struct StoreFp8 {
  static constexpr int kBytes = 1;
  static constexpr bool kScaled = false, kInf = false;
  template <typename E>
  static __device__ __forceinline__ void widen(u4 x, u4 (&to)[2]) {
    to[0] = E::widen_fp8(u2{x[0], x[1]});
    to[1] = E::widen_fp8(u2{x[2], x[3]});
  }
};
struct StoreCodesFp8 : StoreFp8 {
  static constexpr bool kScaled = true, kInf = false;
};
struct StoreCodesInt8 {
  static constexpr int kBytes = 1;
  static constexpr bool kScaled = true, kInf = false;
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

// One workgroup: a block of 32 W of a group's rows of one kv head, 32 to a wave, over one
// split of the shared pages, 64 keys at a time. Each wave brings a part of a tile's four
// pages to LDS, two or three buffers in turn; all waves read all of it.
//
// S^T = K Q^T leaves a lane with half of the keys of its row, so that maxima and sums stay
// in the lane but for one exchange between two lanes; O^T = V^T P^T takes P from those
// registers as they are: the product's k order is the order the registers hold the keys in,
// and V comes transposed from LDS in the same order.
//
// The products bound it: a call of 64 sequences over 32K tokens, q_len 8, 8 kv heads, head dim
// 128, with next to no tokens of their own, takes 302 to 326 us in fp16 and 288 to 308 in bf16,
// the join among it: 840 to 950 TFLOP/s, where a large product of the library's reaches 1160
// and 1210. The device lowers its clock under them (on zeros: a quarter less time), so what is
// left to gain is in instructions saved, not in waits. 32 rows to a wave: with 64, and one wave
// to a SIMD, half the reads from LDS and the same time (338 and 340 us). Eight waves to a
// block of 256 rows rather than two workgroups of four beside each other: every tile is
// brought for twice the rows (96 sequences over two prefixes, bf16: 204 and 212 us).
template <int HD, int W, typename E, typename KV>
struct TileShare {
  // The type of P and V: every 8-bit code is an fp16 number.
  using EV = std::conditional_t<KV::kBytes == 1, ElemF16, E>;
  using T = Tile<HD>;
  static constexpr int kTokens = kTileKeys / W;  // of a tile that a wave brings
  using Loads = PageLoads<HD, KV::kBytes, kTokens>;
  static constexpr int KS = HD / 16;  // k steps of the scores
  static constexpr int MB = HD / 32;  // blocks of 32 output dims
  static constexpr int kStageRow = HD + 4;
  static constexpr int kStage = W * 32 * kStageRow * 4;
  // Tiles in LDS. With three, a wave that has a tile's first half behind it may bring the next
  // one but one over what no wave can still be reading: one barrier a tile. Two (where three
  // do not fit, or would keep a second workgroup away) take one more.
  static constexpr int kBuffers = W == 8 ? 3 : 2;
  static constexpr int kBuffer = 2 * T::kBytes;  // K, then V
  static constexpr int kLds = kBuffers * kBuffer > kStage ? kBuffers * kBuffer : kStage;

  static __device__ __forceinline__ void run(const PartArgs& args, char* lds,
                                             float (&lds_scale)[3][2][kTilePages], int block) {
  const PartialArgs& a = args.p;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int l32 = lane & 31, h = lane >> 5;
  const int share = block / args.by_shared_heads;
  const int kvh = block - share * a.hkv;
  const SharedItem it = item_of(args, share);
  const int b = it.group.pages > 0 ? __builtin_amdgcn_readfirstlane(leader_of(args, it.group)) : -1;
  if (b < 0 || it.split >= args.most_splits) return;  // uniform over the workgroup
  const int first_page = __builtin_amdgcn_readfirstlane(it.begin);
  const int n_pages = __builtin_amdgcn_readfirstlane(it.n);
  const int tiles = (n_pages + kTilePages - 1) / kTilePages;
  const int row0 = __builtin_amdgcn_readfirstlane(it.block) * (32 * W) + wave * 32;
  const int n_rows = __builtin_amdgcn_readfirstlane(it.group.count) * a.rows;
  const int first = __builtin_amdgcn_readfirstlane(it.group.first);
  const RowMap map = shared_map(args, first, __builtin_amdgcn_readfirstlane(it.split),
                                __builtin_amdgcn_readfirstlane(it.group.pages), kvh);

  // This wave's page of a tile, from memory to registers.
  const int shift = a.page_shift, sub_mask = (1 << shift) - 1;
  const int32_t* table = a.block_tables + (size_t)b * a.bt_stride;
  const unsigned tok = a.token_stride;
  const size_t sub_bytes = (size_t)kPageSize * tok;
  const int ltok = lane / Loads::kLanes, lchunk = lane % Loads::kLanes;
  const unsigned lane_at = ltok * tok + kvh * a.head_stride + Loads::kWidth * lchunk;
  const int my_page = wave * kTokens / kPageSize, my_slot = wave * kTokens % kPageSize;
  auto id_of = [&](int tile) {
    const int p = min(first_page + max(min(tile * kTilePages + my_page, n_pages - 1), 0),
                      a.max_pages - 1);
    return scalar_load(table + (p >> shift));
  };
  Loads kreg, vreg;
  float scale_reg = 0.f;
  auto fetch = [&](int tile, int id) {
    const int i = tile * kTilePages + my_page;
    const int pid = i < n_pages ? clamp_page(id, a.num_pages) : -1;
    const size_t off = pid >= 0 ? (size_t)pid * (size_t)a.page_stride +
                                      (size_t)((first_page + i) & sub_mask) * sub_bytes : 0;
    const int nrec = pid >= 0 ? (int)a.page_extent : 0;
    const unsigned at = lane_at + my_slot * tok;
    kreg.load(__builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.k + off), (short)0, nrec,
                                                kBufferFlags), at, tok);
    vreg.load(__builtin_amdgcn_make_buffer_rsrc((void*)((const char*)a.v + off), (short)0, nrec,
                                                kBufferFlags), at, tok);
    if constexpr (KV::kScaled)  // lanes 0-31 the page's K scale, 32-63 its V scale
      scale_reg = *(const float*)((const char*)(h == 0 ? args.scales.k : args.scales.v) +
                                  max(pid, 0) * args.scales.page_stride +
                                  (size_t)kvh * args.scales.head_stride);
  };
  auto put = [&](int buffer) {
    char* to = lds + buffer * kBuffer;
    constexpr int N = Loads::kChunks;
#pragma unroll
    for (int i = 0; i < Loads::kLoads; ++i) {
      const int row = wave * kTokens + i * Loads::kTokens + ltok;
      u4 x[2 / KV::kBytes], y[2 / KV::kBytes];
      KV::template widen<E>(kreg.x[i], x);
      KV::template widen<EV>(vreg.x[i], y);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        *(u4*)(to + T::at(row, N * lchunk + n)) = x[n];
        *(u4*)(to + T::kBytes + T::at(row, N * lchunk + n)) = y[n];
      }
    }
    if constexpr (KV::kScaled)
      if (l32 == 0) lds_scale[buffer][h][my_page] = scale_reg;
  };

  // Rows of the queries as the scores' B operand.
  int id_next = id_of(0);
  fetch(0, id_next);
  id_next = id_of(1);
  u4 q[KS];
  {
    const int x = row0 + l32;
    const _Float16* qp = a.q + map.out_row(args, min(x, n_rows - 1)) * HD + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      q[ks] = *(const u4*)(qp + 16 * ks);
      if (x >= n_rows) q[ks] = u4{0u, 0u, 0u, 0u};
    }
  }
  f16v acc[MB];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[mb][r] = 0.f;
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

  const float c = a.scale_log2;
  // The two pages of a step: exponents are s mul + add - m. With codes mul holds the K scale,
  // add log2 of the V scale, inv 1 / V scale for the row sum (see
  // sqa_scaled_attention_kernel); pages past the split's end get add -infinity.
  struct Pages {
    float mul[2], add[2], inv[2];
    bool loud[2];
  };
  auto pages_of = [&](int t, int buffer, int kb) {
    Pages x;
    const int left = n_pages - t * kTilePages - 2 * kb;  // pages from these two on
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) {
      x.mul[pg] = c;
      x.add[pg] = 0.f;
      if constexpr (KV::kScaled) {
        auto uniform = [](float y) {
          return __builtin_bit_cast(
              float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, y)));
        };
        const float vs = uniform(lds_scale[buffer][1][2 * kb + pg]);
        x.mul[pg] = c * uniform(lds_scale[buffer][0][2 * kb + pg]);
        x.loud[pg] = !(vs < 0x1p-64f);
        x.add[pg] = x.loud[pg] ? __builtin_amdgcn_logf(vs) : -64.f;
        x.inv[pg] = x.loud[pg] ? __builtin_amdgcn_rcpf(vs) : 0x1p64f;
      }
      if (pg >= left) {  // zeros in LDS, and some page's scales
        x.add[pg] = -INFINITY;
        if constexpr (KV::kScaled) {
          x.mul[pg] = x.inv[pg] = 0.f;
          x.loud[pg] = false;
        }
      }
    }
    return x;
  };
  auto read_k = [&](int kb, int ks) { return *(const u4*)(lds + kb * 32 * T::kRow + k_at[ks]); };
  // Dims 32 mb .. + 31 of 16 keys, transposed.
  auto read_v = [&](int kb, int i) {
    const int st = i / MB, mb = i % MB;
    u4 v;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int at = v_at[mb][half] + (32 * kb + 16 * st) * T::kRow;
      const u2 x = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                              (__attribute__((address_space(3))) s4v*)(lds + at)));
      v[2 * half] = x[0];
      v[2 * half + 1] = x[1];
    }
    return v;
  };
  // The running maximum, raised where some lane is too far ahead of its own (`top`: the
  // largest score of each page in the lane).
  auto raise = [&](const float (&top)[2], const Pages& pages) {
    const float lm = __builtin_elementwise_maximum(fmaf(top[0], pages.mul[0], pages.add[0]),
                                                   fmaf(top[1], pages.mul[1], pages.add[1]));
    if (__any(lm > m + kMaxLag)) {
      const LanePair both = lane_pair<32>(lm);
      const float mn = fmaxf(m, fmaxf(both.lo, both.hi));
      const float alpha = fast_exp2(m - (mn == -INFINITY ? 0.f : mn));
      m = mn;
      l *= alpha;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) acc[mb] *= alpha;
    }
  };
  auto score = [&](u4 k, int ks, f16v& s) {
    if (ks == 0)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
    s = mma32<E>(k, q[ks], s);
  };
  auto fold_top = [&](const f16v& s, int i, float (&top)[2]) {  // i of 8
    float& x = top[i / 4];
    x = i % 4 == 0 ? __builtin_elementwise_maximum(s[2 * i], s[2 * i + 1])
                   : max3_raw(x, s[2 * i], s[2 * i + 1]);
  };
  // 32 keys a step: P = 2^(s - m) of the scores `now`, added up into l, and their product with
  // V (half v_kb of the tile at v_at), while the scores `next` of other keys (half k_kb of the
  // tile at k_at) come about. The matrix cores and the vector units run beside each other where
  // a wave gives both something to do, so the next scores' products stand among this step's
  // exponentials, the maxima of the next among the products with V, and reads from LDS kAhead
  // pieces before their use; the compiler, left alone, puts one after the other (64 sequences
  // over 32K tokens, q_len 8: 345 us so, 338 in this order).
  // P is rounded once to the type of the products, over bf16 caches too (2^-8 of a probability,
  // as the output's own rounding; sums stay in 32 bits): a second product for what is rounded
  // off, as pages in waves have it, would cost half of the products again, and these bound the
  // kernel.
  constexpr int kAhead = 3;
  auto step = [&](const f16v& now, const Pages& pages, int v_kb, f16v& next,
                  const Pages& next_pages, int k_kb) {
    u4 k[KS], v[2 * MB], p[2];
    float off[2];
#pragma unroll
    for (int pg = 0; pg < 2; ++pg) off[pg] = pages.add[pg] - (m == -INFINITY ? 0.f : m);
#pragma unroll
    for (int ks = 0; ks < kAhead; ++ks) k[ks] = read_k(k_kb, ks);
    __builtin_amdgcn_sched_barrier(0);
    auto weigh = [&](int w) {  // pair w of 8: registers 2 w and 2 w + 1
      const int st = w / 4;
      const float x = fast_exp2(fmaf(now[2 * w], pages.mul[st], off[st]));
      const float y = fast_exp2(fmaf(now[2 * w + 1], pages.mul[st], off[st]));
      unsigned packed = EV::pack2(x, y);
      // The row sum is that of the rounded ones (but with V scales, which lie between the two),
      // so that the weights of a row add up to one.
      if constexpr (KV::kScaled) {
        l = fmaf(x + y, pages.inv[st], l);
        packed = pages.loud[st] ? packed : 0u;
      } else if constexpr (EV::kHalfPartials) {
        const h2 ones = {(_Float16)1.0f, (_Float16)1.0f};
        l = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, packed), ones, l, false);
      } else {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        const b2 ones = {(__bf16)1.0f, (__bf16)1.0f};
        l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, packed), ones, l, false);
      }
      p[st][w % 4] = packed;
    };
    // Five of a row's eight pairs among the scores' products, three among the first half of
    // those with V, which take the pairs before.
    constexpr int kEarly = 5;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + kAhead < KS)
        k[ks + kAhead] = read_k(k_kb, ks + kAhead);
      else
        v[ks + kAhead - KS] = read_v(v_kb, ks + kAhead - KS);
      score(k[ks], ks, next);
#pragma unroll
      for (int w = 0; w < kEarly; ++w)
        if (w * KS / kEarly == ks) weigh(w);
      __builtin_amdgcn_sched_barrier(0);
    }
    float top[2];
#pragma unroll
    for (int i = 0; i < 2 * MB; ++i) {
      if (i + kAhead < 2 * MB) v[i + kAhead] = read_v(v_kb, i + kAhead);
      acc[i % MB] = mma32<EV>(v[i], p[i / MB], acc[i % MB]);
      if (i < MB) {
#pragma unroll
        for (int w = kEarly; w < 8; ++w)
          if ((w - kEarly) * MB / (8 - kEarly) == i) weigh(w);
      } else {
#pragma unroll
        for (int w = 0; w < 8; ++w)
          if (w * MB / 8 == i - MB) fold_top(next, w, top);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    raise(top, next_pages);
  };

  // A tile's second step takes the next tile's first scores, so tile t + 1 comes to LDS
  // half-way through tile t.
  put(0);
  __syncthreads();
  if (tiles > 1) fetch(1, id_next);
  id_next = id_of(2);
  f16v s0, s1;
  float top[2];
  Pages pages = pages_of(0, 0, 0);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) score(read_k(0, ks), ks, s0);
#pragma unroll
  for (int w = 0; w < 8; ++w) fold_top(s0, w, top);
  raise(top, pages);
  int buffer = 0;
  for (int t = 0; t < tiles; ++t) {
    const int following = buffer == kBuffers - 1 ? 0 : buffer + 1;
    const int onward = (following - buffer) * kBuffer;
    const Pages second = pages_of(t, buffer, 1);
    step(s0, pages, 0, s1, second, 1);
    if (t + 1 < tiles) put(following);
    __syncthreads();
    if (t + 2 < tiles) {  // uniform
      fetch(t + 2, id_next);
      id_next = id_of(t + 3);
    }
    // Past the last tile the scores are of what the buffer holds, and nobody's.
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k_at[ks] += onward;
    pages = pages_of(t + 1, following, 0);
    step(s1, second, 1, s0, pages, 0);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int half = 0; half < 2; ++half) v_at[mb][half] += onward;
    buffer = following;
    if constexpr (kBuffers == 2) __syncthreads();
  }
  __syncthreads();  // before the tiles' place is taken

  float* stage = (float*)lds + wave * 32 * kStageRow;
  // An infinity is NaN by now under a probability, or a change of the maximum, that rounds to
  // 0. All rows see all tokens, so what is not finite is added up once more, by dims.
  if constexpr (KV::kInf) {
    NanOf nan;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        nan.add(i, f4{acc[mb][4 * i], acc[mb][4 * i + 1], acc[mb][4 * i + 2], acc[mb][4 * i + 3]});
    if (__builtin_expect(nan.any(), 0)) {  // uniform
      constexpr int N = HD / 64;  // dims of a lane
      float wild[N];
#pragma unroll
      for (int n = 0; n < N; ++n) wild[n] = 0.f;
      for (int i = 0; i < n_pages; ++i) {
        const int p = first_page + i;
        const int id = clamp_page(scalar_load(table + (min(p, a.max_pages - 1) >> shift)),
                                  a.num_pages);
        const unsigned short* v =
            (const unsigned short*)((const char*)a.v + (size_t)id * (size_t)a.page_stride +
                                    (size_t)(p & sub_mask) * sub_bytes + kvh * a.head_stride) +
            N * lane;
        for (int t = 0; t < kPageSize; ++t, v += tok / 2)
#pragma unroll
          for (int n = 0; n < N; ++n) {
            const float x = E::kHalfPartials ? (float)__builtin_bit_cast(_Float16, v[n])
                                             : __builtin_bit_cast(float, (unsigned)v[n] << 16);
            wild[n] += fabsf(x) < INFINITY ? 0.f : x;
          }
      }
#pragma unroll
      for (int n = 0; n < N; ++n) stage[N * lane + n] = wild[n];
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float w = stage[32 * mb + 8 * (r / 4) + 4 * h + r % 4];
          acc[mb][r] = w == 0.f ? acc[mb][r] : w;
        }
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    }
  }

  // Partial rows through LDS.
  const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
      (void*)a.part_o, (short)0, (int)a.part_o_bytes, kBufferFlags);
  const LanePair both = lane_pair<32>(l);
  const float sum = both.lo + both.hi;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = acc[mb][4 * i + r];
      *(f4*)(stage + l32 * kStageRow + 32 * mb + 8 * i + 4 * h) = o;
    }
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  const bool mine = row0 + l32 < n_rows;
  const int to = mine ? (int)map.part_row(args, row0 + l32) : -1;  // there are less than 2^31
  constexpr int CPR = HD / 4;
  auto leave = [&](int i) {
    const int e = i * 64 + lane;  // row e / CPR (< 32), chunk e % CPR
    const int rs = e / CPR;
    const f4 v = *(const f4*)(stage + rs * kStageRow + 4 * (e % CPR));
    const int at = __shfl(to, rs);
    store_partial<HD>(args, pr, v, at, e % CPR, at >= 0);
  };
  if (__builtin_expect(args.far_rows, 0)) {  // uniform
#pragma unroll 1
    for (int i = 0; i < CPR / 2; ++i) leave(i);
  } else {
#pragma unroll
    for (int i = 0; i < CPR / 2; ++i) leave(i);
  }
  if (h == 0 && mine) {
    // A NaN sum travels with a finite max, so the join counts the split.
    const float m_out = sum == sum ? m : 0.f;
    store_through(a.part_ml + (long long)to * 2,
                  __builtin_bit_cast(unsigned long long, float2{m_out, sum}));
  }
  }
};

// How the sequences' own splits read the same cache.
template <int HD, typename KV>
struct OwnCache;
template <int HD>
struct OwnCache<HD, StoreNative> { using Type = PartNative<HD>; };
template <int HD>
struct OwnCache<HD, StoreFp8> { using Type = PartFp8<HD>; };
template <int HD>
struct OwnCache<HD, StoreCodesFp8> { using Type = PartCodesFp8<HD>; };
template <int HD>
struct OwnCache<HD, StoreCodesInt8> { using Type = PartCodesInt8<HD>; };

// One launch for both: the first shared_wgs workgroups serve the groups, the others what
// follows in every sequence (NB blocks of 16 rows). The one waits for the matrix cores, the
// other for memory.
template <int HD, int W, int NB, typename E, typename KV>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(W / 4)))
void sqa_tiles_kernel(PartArgs args) {
  using Share = TileShare<HD, W, E, KV>;
  constexpr int kOwn = W * 16 * (HD + 4) * 4;
  __shared__ __attribute__((aligned(16))) char lds[Share::kLds > kOwn ? Share::kLds : kOwn];
  __shared__ float lds_scale[3][2][kTilePages];  // of a tile's pages: buffer, K and V, page
  if ((int)blockIdx.x < args.shared_wgs)
    Share::run(own_args(), lds, lds_scale, blockIdx.x);
  else
    part_share<NB, (NB > 2 || W > 4 ? 2 : 4) * 128 / HD, HD, W, E, typename OwnCache<HD, KV>::Type>(
        (float*)lds, blockIdx.x - args.shared_wgs, false);
}

// Eight waves have 256 registers each, too few for 64 rows of a sequence beside the page ring.
template <int HD, typename E, typename KV>
void launch_tiles_hd(const PartArgs& a, dim3 grid, hipStream_t stream) {
  if constexpr (HD != 256) {
    if (a.block_rows == 256) {
      hipLaunchKernelGGL((sqa_tiles_kernel<HD, 8, 2, E, KV>), grid, dim3(512), 0, stream, a);
      return;
    }
    if (a.p.rows > 32) {
      hipLaunchKernelGGL((sqa_tiles_kernel<HD, 4, 4, E, KV>), grid, dim3(256), 0, stream, a);
      return;
    }
  }
  hipLaunchKernelGGL((sqa_tiles_kernel<HD, 4, 2, E, KV>), grid, dim3(256), 0, stream, a);
}

template <typename E, typename KV>
void launch_tiles_as(const PartArgs& a, dim3 grid, hipStream_t stream) {
  if (a.p.head_dim == 64)
    launch_tiles_hd<64, E, KV>(a, grid, stream);
  else if (a.p.head_dim == 128)
    launch_tiles_hd<128, E, KV>(a, grid, stream);
  else
    launch_tiles_hd<256, E, KV>(a, grid, stream);
}

template <typename E>
hipError_t launch_tiles_of(const PartArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(a.shared_wgs + own_workgroups(a)));
  if (a.scaled && a.kv_type == kInt8)
    launch_tiles_as<E, StoreCodesInt8>(a, grid, stream);
  else if (a.scaled)
    launch_tiles_as<E, StoreCodesFp8>(a, grid, stream);
  else if (a.kv_type == kE4M3)
    launch_tiles_as<E, StoreFp8>(a, grid, stream);
  else
    launch_tiles_as<E, StoreNative>(a, grid, stream);
  return hipGetLastError();
}

}  // namespace
}  // namespace sqa

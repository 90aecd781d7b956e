// Internal interface between the C ABI (sqa_cache_capi.hip) and the kernels around the
// paged cache: the quantising append and attention over 8-bit caches with block scales
// (sqa_scaled.hip), attention weights and eviction (sqa_evict.hip).
#pragma once

#include "sqa_internal.h"

namespace sqa {

// Element types of caches and tokens, as the public header numbers them.
enum { kF16 = 0, kBF16 = 1, kE4M3 = 2, kInt8 = 3 };

// The largest magnitude a code stands for, in units of its block's scale.
__host__ __device__ inline float code_max(int kv_type) { return kv_type == kInt8 ? 127.f : 448.f; }

// Scales of an 8-bit cache: one float for each cache page and kv head, for K and for V.
struct BlockScales {
  float* k;
  float* v;
  long long page_stride;  // bytes between consecutive pages
  unsigned head_stride;   // bytes between consecutive kv heads
};

// Attention over an 8-bit cache with block scales. Of `p` the fields that name buffers,
// shapes, strides and scales; the plan is the kernel's own (sqa_scaled.hip): `items`
// work items, partial slot i for item i, p.seq_splits written by the kernel.
struct ScaledArgs {
  PartialArgs p;
  BlockScales scales;
  int items;
  int int8;      // codes: 0 e4m3, 1 int8
  int wg_heads;  // kv heads a workgroup serves (1, 2 or 4); its other waves take more items
};
hipError_t launch_scaled(const ScaledArgs& a, hipStream_t stream);

struct AppendArgs {
  const void* src[2];               // K and V of the new tokens, [B, Q, Hkv, D]
  long long src_batch[2], src_token[2], src_head[2];  // strides in bytes
  void* cache[2];                   // K and V codes
  BlockScales scales;
  const int32_t* block_tables;
  const int32_t* seq_lens;
  const int32_t* new_lens;          // NULL: q_len new tokens everywhere
  long long num_pages, page_stride; // strides in bytes (codes)
  long long token_stride, head_stride;
  int batch, q_len, hkv, head_dim, page_size, bt_stride;
  int touched;                      // most pages the new tokens of a sequence lie on
  int bf16, int8;
};
hipError_t launch_append(const AppendArgs& a, hipStream_t stream);

// Whether the scores of a call travel from its first to its second kernel through memory,
// 4 bytes per row and token written and read again, or K is read and multiplied a second
// time. Writes among the reads cost more than their bytes: the two meet where the scores
// are a quarter of K. Whole calls, stored / computed again, head dim 128: 16 x 32K keys,
// 16-bit K, 4 rows 254 / 388 us, 8 278 / 383, 16 329 / 381, 24 392 / 383, 32 436 / 384;
// e4m3 4 rows 150 / 203, 8 173 / 201, 12 202 / 201, 16 224 / 204. 4 x 8K, 16-bit: 4 rows
// 23 / 29, 8 25 / 29, 12 30 / 29, 16 31 / 29; e4m3: 4 rows 18 / 19, 8 21 / 19. Head dim 64,
// 16 x 32K: 16-bit 4 rows 147 / 197, 8 170 / 197, 16 221 / 198, e4m3 4 rows 97 / 120, 8 122 /
// 120; 4 x 8K: 16-bit 8 rows 21 / 19, 16 27 / 19, e4m3 4 rows 17 / 18. Head dim 256, 16 x
// 32K: 16-bit 8 rows 461 / 708, 16 523 / 708, 32 624 / 711, e4m3 16 rows 332 / 389, 32 440 /
// 393; 4 x 8K: 16-bit 32 rows 62 / 57, e4m3 16 rows 34 / 31.
__host__ __device__ constexpr bool weights_stored(long long rows, int head_dim, int kv_bytes) {
  return 16 * rows <= (long long)head_dim * kv_bytes;
}

// Attention weights added up. Of `p` the fields of the query side, of K and of the tables.
struct WeighArgs {
  PartialArgs p;
  const float* k_scale;        // NULL: 1
  long long scale_page;        // strides in bytes
  unsigned scale_head;
  int items;                   // work items of the cut
  int wg_heads;
  int kv_type;                 // kF16, kBF16, kE4M3 or kInt8
  float* weights;              // [B, Hkv, width]
  long long w_batch, w_head;   // strides in floats
  int width;
  float2* stats;               // [items][Hkv][rows]: (max in log2 units, sum)
  float* scores;               // [B][pages][Hkv][rows][16] in log2 units, or NULL: the second
                               // kernel computes them again
};
hipError_t launch_weigh(const WeighArgs& a, hipStream_t stream);

struct EvictArgs {
  const float* weights;        // [B, Hkv, width]
  long long w_batch, w_head;   // strides in floats
  int width;
  float* new_weights;          // [B, Hkv, new_width]; may be `weights`
  long long nw_batch, nw_head;
  int new_width;
  int32_t* kept;               // [B, Hkv, budget]
  const int32_t* seq_lens;
  int32_t* new_lens;
  int budget, sink, recent;
  const char* src[2];          // K and V
  char* dst[2];
  long long src_page, src_token, src_head, dst_page, dst_token, dst_head;  // bytes
  BlockScales src_scales, dst_scales;
  const int32_t* block_tables;
  const int32_t* new_tables;
  int bt_stride, new_stride;
  long long num_pages, new_pages;
  int batch, hkv, head_dim, page_size;
  int kv_type, scaled;
};
hipError_t launch_evict(const EvictArgs& a, hipStream_t stream);

}  // namespace sqa

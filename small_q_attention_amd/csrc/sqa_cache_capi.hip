// C ABI of the operators around the paged cache (declared in include/sqa.h): validates
// arguments and launches the kernels of sqa_scaled.hip and sqa_evict.hip on the caller's
// stream. Allocates nothing.
#include "sqa.h"
#include "sqa_cache.h"

#include <math.h>
#include <string.h>

#include <algorithm>

namespace {

using sqa::fail;
using sqa::hip_fail;

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

int page_shift_of(int page_size) {
  for (int sh = 0; sh <= sqa::kMaxPageShift; ++sh)
    if (page_size == (sqa::kPageSize << sh)) return sh;
  return -1;
}

bool is_codes(int kv_dtype) { return kv_dtype == SQA_DTYPE_FP8_E4M3 || kv_dtype == SQA_DTYPE_INT8; }

// Shapes every operator over a paged cache shares.
int check_cache(int batch, int num_kv_heads, int head_dim, int page_size, int64_t num_pages,
                int max_pages) {
  if (batch <= 0 || num_kv_heads <= 0)
    return fail(SQA_ERR_INVALID, "batch and head counts must be positive");
  if (num_pages <= 0 || max_pages <= 0)
    return fail(SQA_ERR_INVALID, "empty KV cache is not supported");
  if (num_pages > 0x7fffffffLL) return fail(SQA_ERR_INVALID, "page ids are 32 bits");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(SQA_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256 (got %d)", head_dim);
  if (page_shift_of(page_size) < 0)
    return fail(SQA_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256 (got %d)",
                page_size);
  const long long kernel_pages = (long long)max_pages << page_shift_of(page_size);
  if (kernel_pages >= (1LL << 26))
    return fail(SQA_ERR_INVALID, "block-table rows must be under 2^30 tokens");
  if ((long long)batch * kernel_pages >= (1LL << 30))
    return fail(SQA_ERR_INVALID, "batch * pages per row must be under 2^30");
  return SQA_OK;
}

// Strides of one pool in elements of `bytes`, and the reach of a 16-token page.
int check_strides(const sqa_kv_cache& kv, int bytes, int num_kv_heads, int head_dim,
                  long long* extent) {
  const int64_t ps = kv.page_stride, ts = kv.token_stride, hs = kv.head_stride;
  if (ps < 0 || ts < 0 || hs < 0 || ps % 8 || ts % 8 || hs % 8)
    return fail(SQA_ERR_INVALID, "cache strides must be non-negative multiples of 8 elements");
  if (((uintptr_t)kv.k | (uintptr_t)kv.v) % 16)
    return fail(SQA_ERR_INVALID, "cache base pointers must be 16-byte aligned");
  constexpr int64_t kFar = (int64_t)1 << 40;
  if (ps > kFar || ts > 0x7fffffffLL || hs > 0x7fffffffLL)
    return fail(SQA_ERR_INVALID, "cache strides are too large");
  *extent = bytes * ((long long)(sqa::kPageSize - 1) * ts + (long long)(num_kv_heads - 1) * hs +
                     head_dim);
  if (*extent > 0x7fffffffLL)
    return fail(SQA_ERR_INVALID, "one page of the cache spans more than 2 GiB");
  return SQA_OK;
}

int check_scales(const sqa_block_scales& s, bool value) {
  if (!s.k || (value && !s.v)) return fail(SQA_ERR_INVALID, "null scale pointer");
  if (((uintptr_t)s.k | (uintptr_t)s.v) % 4)
    return fail(SQA_ERR_INVALID, "scales must be 4-byte aligned");
  if (s.page_stride < 0 || s.head_stride < 0 || s.page_stride > ((int64_t)1 << 40) ||
      s.head_stride > 0x1fffffffLL)
    return fail(SQA_ERR_INVALID, "scale strides must be non-negative and within 32 bits");
  return SQA_OK;
}

sqa::BlockScales scales_of(const sqa_block_scales& s) {
  return {(float*)s.k, (float*)s.v, 4 * (long long)s.page_stride, (unsigned)(4 * s.head_stride)};
}

// kv heads a workgroup of the attention kernel serves, and the items that fill the chip
// once: one workgroup of four waves per compute unit.
int wg_heads(int num_kv_heads) { return num_kv_heads >= 3 ? 4 : num_kv_heads; }

long long scaled_items(int cus, int num_kv_heads) {
  const int wgh = wg_heads(num_kv_heads);
  return ceil_div(cus, ceil_div(num_kv_heads, wgh)) * (4 / wgh);
}

}  // namespace

extern "C" {

int sqa_plan_scaled(int device, int batch, int num_kv_heads, int max_seq_len, int max_pages,
                    int* num_splits) {
  if (!num_splits) return fail(SQA_ERR_INVALID, "null output pointer");
  if (batch <= 0 || num_kv_heads <= 0 || max_pages <= 0)
    return fail(SQA_ERR_INVALID, "batch, heads and max_pages must be positive");
  const int cus = sqa_device_cu_count(device);
  if (cus <= 0) return SQA_ERR_HIP;
  long long pages = max_pages;
  if (max_seq_len > 0) pages = std::min(pages, ceil_div(max_seq_len, sqa::kPageSize));
  const long long most = batch * ceil_div(pages, sqa::kMinSplitPages);
  const long long items = std::max((long long)batch, std::min(scaled_items(cus, num_kv_heads), most));
  if (items * num_kv_heads > 0x7fffffffLL) return fail(SQA_ERR_INVALID, "grid too large");
  *num_splits = (int)items;
  return SQA_OK;
}

int sqa_paged_attention_scaled(const sqa_attention_args* args, const sqa_block_scales* scales) {
  if (!args || !scales) return fail(SQA_ERR_INVALID, "null argument struct");
  if (args->struct_size != sizeof(sqa_attention_args))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                args->struct_size, sizeof(sqa_attention_args));
  const sqa_attention_args& a = *args;
  if (!a.query || !a.kv.k || !a.kv.v || !a.block_tables || !a.seq_lens || !a.output)
    return fail(SQA_ERR_INVALID, "null tensor pointer");
  if (int rc = check_cache(a.batch, a.num_kv_heads, a.head_dim, a.page_size, a.kv.num_pages,
                           a.max_pages))
    return rc;
  if (a.q_len <= 0 || a.num_query_heads <= 0 || a.num_query_heads % a.num_kv_heads)
    return fail(SQA_ERR_INVALID,
                "q_len and num_query_heads must be positive, heads divisible by num_kv_heads");
  const int group = a.num_query_heads / a.num_kv_heads;
  const long long rows = (long long)a.q_len * group;
  const int max_rows = a.head_dim == 256 ? sqa::kMaxRowsHd256 : sqa::kMaxRows;
  if (rows > max_rows)
    return fail(SQA_ERR_UNSUPPORTED, "q_len * group = %lld exceeds %d at head_dim %d", rows,
                max_rows, a.head_dim);
  if (a.dtype != SQA_DTYPE_F16 && a.dtype != SQA_DTYPE_BF16)
    return fail(SQA_ERR_UNSUPPORTED, "dtype must be SQA_DTYPE_F16 or SQA_DTYPE_BF16 (got %d)",
                a.dtype);
  if (!is_codes(a.kv_dtype))
    return fail(SQA_ERR_UNSUPPORTED,
                "kv_dtype must be SQA_DTYPE_FP8_E4M3 or SQA_DTYPE_INT8 (got %d)", a.kv_dtype);
  long long extent = 0;
  if (int rc = check_strides(a.kv, 1, a.num_kv_heads, a.head_dim, &extent)) return rc;
  if (int rc = check_scales(*scales, true)) return rc;
  if ((uintptr_t)a.query % 16 || (uintptr_t)a.output % 8)
    return fail(SQA_ERR_INVALID, "query must be 16-byte and output 8-byte aligned");
  if (((uintptr_t)a.block_tables | (uintptr_t)a.seq_lens | (uintptr_t)a.draft_mask) % 4)
    return fail(SQA_ERR_INVALID, "block_tables, seq_lens and draft_mask must be 4-byte aligned");
  if (a.draft_mask && (a.mask_words < (a.q_len + 31) / 32 || a.mask_words > 2))
    return fail(SQA_ERR_INVALID, "draft_mask needs %d..2 words per row, got %d",
                (a.q_len + 31) / 32, a.mask_words);
  if (!(a.scale > 0.f) || !isfinite(a.scale) || !isfinite(a.out_scale))
    return fail(SQA_ERR_INVALID, "scale must be positive and finite, out_scale finite");
  if (a.flags) return fail(SQA_ERR_INVALID, "unknown flags %#x", (unsigned)a.flags);
  if (a.pages_per_split != 0)
    return fail(SQA_ERR_INVALID, "pages_per_split must be 0: the device cuts the pages");
  if (a.num_splits < a.batch)
    return fail(SQA_ERR_INVALID, "num_splits must be at least the batch (%d), got %d", a.batch,
                a.num_splits);
  if ((long long)a.num_splits * a.num_kv_heads > 0x7fffffffLL)
    return fail(SQA_ERR_INVALID, "grid too large");
  const size_t need = sqa_workspace_bytes(a.batch, a.q_len, a.num_query_heads, a.num_kv_heads,
                                          a.head_dim, a.num_splits, 0);
  if (!a.workspace || a.workspace_bytes < need)
    return fail(SQA_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                a.workspace ? a.workspace_bytes : (size_t)0);
  if ((uintptr_t)a.workspace % 16)
    return fail(SQA_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  const unsigned long long items = (unsigned long long)a.num_splits * a.num_kv_heads * rows;
  const unsigned long long part_bytes = items * a.head_dim * (a.dtype == SQA_DTYPE_F16 ? 2 : 4);
  if (part_bytes > sqa::kMaxPartialBytes)
    return fail(SQA_ERR_INVALID, "the plan's partials (%llu bytes) exceed %llu bytes", part_bytes,
                sqa::kMaxPartialBytes);

  sqa::ScaledArgs s;
  memset(&s, 0, sizeof(s));
  sqa::PartialArgs& p = s.p;
  p.q = (const _Float16*)a.query;
  p.k = (const _Float16*)a.kv.k;
  p.v = (const _Float16*)a.kv.v;
  p.block_tables = a.block_tables;
  p.seq_lens = a.seq_lens;
  p.draft_mask = a.draft_mask;
  p.mask_words = a.draft_mask ? a.mask_words : 0;
  p.out = (_Float16*)a.output;
  p.part_o = (float*)a.workspace;
  p.part_ml = (float*)a.workspace + items * a.head_dim;
  p.seq_splits = (sqa::SeqSplits*)(p.part_ml + items * 2);
  p.part_o_bytes = (unsigned)part_bytes;
  p.num_pages = a.kv.num_pages;
  p.page_stride = a.kv.page_stride;
  p.token_stride = (unsigned)a.kv.token_stride;
  p.head_stride = (unsigned)a.kv.head_stride;
  p.page_extent = (unsigned)extent;
  p.batch = a.batch;
  p.q_len = a.q_len;
  p.hq = a.num_query_heads;
  p.hkv = a.num_kv_heads;
  p.group = group;
  p.rows = (int)rows;
  p.head_dim = a.head_dim;
  p.bt_stride = a.max_pages;
  p.page_shift = page_shift_of(a.page_size);
  p.max_pages = a.max_pages << p.page_shift;
  p.num_splits = a.num_splits;
  p.by_group = sqa::fast_div(group);
  p.scale_log2 = (float)(1.4426950408889634 * (double)a.scale);
  p.out_scale = a.out_scale;
  p.bf16 = a.dtype == SQA_DTYPE_BF16;
  s.scales = scales_of(*scales);
  s.items = a.num_splits;
  s.int8 = a.kv_dtype == SQA_DTYPE_INT8;
  s.wg_heads = wg_heads(a.num_kv_heads);

  hipStream_t stream = (hipStream_t)a.stream;
  hipEvent_t* ev = (hipEvent_t*)a.timing_events;
  hipError_t e;
  if (ev && (e = hipEventRecord(ev[0], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  if ((e = sqa::launch_scaled(s, stream)) != hipSuccess)
    return hip_fail(e, "scaled attention kernel launch");
  if (ev && (e = hipEventRecord(ev[1], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  // Rows of at most kMinSplitPages pages are never split.
  if (p.max_pages > sqa::kMinSplitPages) {
    int device = -1;
    const int cus = hipGetDevice(&device) == hipSuccess ? sqa_device_cu_count(device) : 0;
    sqa::MergeArgs m;
    memset(&m, 0, sizeof(m));
    m.part_o = p.part_o;
    m.part_ml = p.part_ml;
    m.seq_splits = p.seq_splits;
    m.seq_lens = a.seq_lens;
    m.out = p.out;
    m.batch = a.batch;
    m.q_len = a.q_len;
    m.hq = a.num_query_heads;
    m.hkv = a.num_kv_heads;
    m.group = group;
    m.rows = (int)rows;
    m.head_dim = a.head_dim;
    m.max_pages = p.max_pages;
    m.num_splits = a.num_splits + a.batch;  // the merge's rule counts items past the batch's slots
    m.by_hq = sqa::fast_div(a.num_query_heads);
    m.by_seq_rows = sqa::fast_div(a.q_len * a.num_query_heads);
    m.by_group = p.by_group;
    m.by_spec_pps = m.by_spec_pps1 = sqa::fast_div(1);
    m.out_scale = a.out_scale;
    m.bf16 = p.bf16;
    if ((e = sqa::launch_merge(m, cus, stream)) != hipSuccess)
      return hip_fail(e, "merge kernel launch");
  }
  if (ev && (e = hipEventRecord(ev[2], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  return SQA_OK;
}

int sqa_append_scaled(const sqa_append_args* args) {
  if (!args) return fail(SQA_ERR_INVALID, "null argument struct");
  if (args->struct_size != sizeof(sqa_append_args))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                args->struct_size, sizeof(sqa_append_args));
  const sqa_append_args& a = *args;
  if (!a.key || !a.value || !a.kv.k || !a.kv.v || !a.block_tables || !a.seq_lens)
    return fail(SQA_ERR_INVALID, "null tensor pointer");
  if (int rc = check_cache(a.batch, a.num_kv_heads, a.head_dim, a.page_size, a.kv.num_pages,
                           a.max_pages))
    return rc;
  if (a.q_len <= 0) return fail(SQA_ERR_INVALID, "q_len must be positive");
  if (a.dtype != SQA_DTYPE_F16 && a.dtype != SQA_DTYPE_BF16)
    return fail(SQA_ERR_UNSUPPORTED, "dtype must be SQA_DTYPE_F16 or SQA_DTYPE_BF16 (got %d)",
                a.dtype);
  if (!is_codes(a.kv_dtype))
    return fail(SQA_ERR_UNSUPPORTED,
                "kv_dtype must be SQA_DTYPE_FP8_E4M3 or SQA_DTYPE_INT8 (got %d)", a.kv_dtype);
  long long extent = 0;
  if (int rc = check_strides(a.kv, 1, a.num_kv_heads, a.head_dim, &extent)) return rc;
  if (int rc = check_scales(a.scales, true)) return rc;
  if (((uintptr_t)a.key | (uintptr_t)a.value) % 16)
    return fail(SQA_ERR_INVALID, "key and value must be 16-byte aligned");
  if (((uintptr_t)a.block_tables | (uintptr_t)a.seq_lens | (uintptr_t)a.new_lens) % 4)
    return fail(SQA_ERR_INVALID, "block_tables, seq_lens and new_lens must be 4-byte aligned");
  const int64_t strides[6] = {a.key_strides[0],   a.key_strides[1],   a.key_strides[2],
                              a.value_strides[0], a.value_strides[1], a.value_strides[2]};
  for (int64_t st : strides)
    if (st < 0 || st % 8 || st > ((int64_t)1 << 40))
      return fail(SQA_ERR_INVALID,
                  "key and value strides must be non-negative multiples of 8 elements");
  sqa::AppendArgs k;
  memset(&k, 0, sizeof(k));
  k.src[0] = a.key;
  k.src[1] = a.value;
  for (int i = 0; i < 2; ++i) {
    k.src_batch[i] = 2 * strides[3 * i];
    k.src_token[i] = 2 * strides[3 * i + 1];
    k.src_head[i] = 2 * strides[3 * i + 2];
  }
  k.cache[0] = (void*)a.kv.k;
  k.cache[1] = (void*)a.kv.v;
  k.scales = scales_of(a.scales);
  k.block_tables = a.block_tables;
  k.seq_lens = a.seq_lens;
  k.new_lens = a.new_lens;
  k.num_pages = a.kv.num_pages;
  k.page_stride = a.kv.page_stride;
  k.token_stride = a.kv.token_stride;
  k.head_stride = a.kv.head_stride;
  k.batch = a.batch;
  k.q_len = a.q_len;
  k.hkv = a.num_kv_heads;
  k.head_dim = a.head_dim;
  k.page_size = a.page_size;
  k.bt_stride = a.max_pages;
  // q_len tokens from the last slot of a page on.
  k.touched = (int)std::min((long long)a.max_pages, ceil_div(a.q_len - 1LL, a.page_size) + 1);
  k.bf16 = a.dtype == SQA_DTYPE_BF16;
  k.int8 = a.kv_dtype == SQA_DTYPE_INT8;
  if ((long long)a.batch * k.touched * a.num_kv_heads > 0x7fffffffLL)
    return fail(SQA_ERR_INVALID, "grid too large");
  hipError_t e = sqa::launch_append(k, (hipStream_t)a.stream);
  return e == hipSuccess ? SQA_OK : hip_fail(e, "append kernel launch");
}

}  // extern "C"

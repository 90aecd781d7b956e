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

// Plan of sqa_attention_weights: work items and the parts of its workspace.
struct WeighPlan {
  long long rows, pages, items;
  size_t stats, scores;  // bytes
};

// Scores past this are computed twice instead (a wide table under a large batch).
constexpr size_t kMostScores = (size_t)1 << 30;

int weigh_plan(int device, int batch, int q_len, int num_query_heads, int num_kv_heads,
               int head_dim, int max_seq_len, int max_pages, int kv_dtype, WeighPlan* plan) {
  if (batch <= 0 || q_len <= 0 || num_kv_heads <= 0 || num_query_heads <= 0 || max_pages <= 0)
    return fail(SQA_ERR_INVALID, "batch, q_len, heads and max_pages must be positive");
  const int cus = sqa_device_cu_count(device);
  if (cus <= 0) return SQA_ERR_HIP;
  plan->rows = (long long)q_len * (num_query_heads / num_kv_heads);
  plan->pages = max_pages;
  if (max_seq_len > 0) plan->pages = std::min(plan->pages, ceil_div(max_seq_len, sqa::kPageSize));
  plan->scores = (size_t)batch * num_kv_heads * plan->pages * sqa::kPageSize * plan->rows * 4;
  if (!sqa::weights_stored(plan->rows, head_dim, is_codes(kv_dtype) ? 1 : 2) ||
      plan->scores > kMostScores)
    plan->scores = 0;
  // Two workgroups per compute unit; four where the second kernel only adds the stored
  // scores up, a wait for memory after the other (16 x 32K keys, four rows: its share of
  // the call 27.4 us with two, 22.3 with four; but with K read again, 64 rows, 8
  // sequences of up to 12K keys, 32 us with two and 60 with four).
  const long long most = batch * ceil_div(plan->pages, sqa::kMinSplitPages);
  plan->items = std::max((long long)batch, std::min((plan->scores ? 4 : 2) *
                                                        scaled_items(cus, num_kv_heads), most));
  plan->stats = (size_t)plan->items * num_kv_heads * plan->rows * sizeof(float2);
  return SQA_OK;
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
  const unsigned long long part_bytes = items * a.head_dim * 4;
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
  p.by_splits = sqa::fast_div(a.num_splits);
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
    m.bf16 = p.bf16 ? 1 : 2;  // fp32 partial rows for both
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
  if (a.kv.k == a.kv.v || a.scales.k == a.scales.v)
    return fail(SQA_ERR_INVALID, "keys and values are written: each needs its own cache and scales");
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

size_t sqa_weights_workspace_bytes(int device, int batch, int q_len, int num_query_heads,
                                   int num_kv_heads, int head_dim, int max_seq_len, int max_pages,
                                   int kv_dtype) {
  WeighPlan plan;
  if (weigh_plan(device, batch, q_len, num_query_heads, num_kv_heads, head_dim, max_seq_len,
                 max_pages, kv_dtype, &plan))
    return 0;
  return plan.stats + plan.scores;
}

int sqa_attention_weights(const sqa_weights_args* args) {
  if (!args) return fail(SQA_ERR_INVALID, "null argument struct");
  if (args->struct_size != sizeof(sqa_weights_args))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                args->struct_size, sizeof(sqa_weights_args));
  const sqa_weights_args& a = *args;
  if (!a.query || !a.kv.k || !a.block_tables || !a.seq_lens || !a.weights)
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
  if (a.kv_dtype != a.dtype && !is_codes(a.kv_dtype))
    return fail(SQA_ERR_UNSUPPORTED, "kv_dtype must be dtype or an 8-bit type (got %d)",
                a.kv_dtype);
  if (a.k_scale && !is_codes(a.kv_dtype))
    return fail(SQA_ERR_INVALID, "scales belong to 8-bit caches");
  if (a.kv_dtype == SQA_DTYPE_INT8 && !a.k_scale)
    return fail(SQA_ERR_INVALID, "int8 caches need scales");
  if (a.k_scale) {
    const sqa_block_scales sc = {a.k_scale, nullptr, a.scale_page_stride, a.scale_head_stride};
    if (int rc = check_scales(sc, false)) return rc;
  }
  const int bytes = is_codes(a.kv_dtype) ? 1 : 2;
  long long extent = 0;
  sqa_kv_cache kv = a.kv;
  kv.v = nullptr;
  if (int rc = check_strides(kv, bytes, a.num_kv_heads, a.head_dim, &extent)) return rc;
  if ((uintptr_t)a.query % 16) return fail(SQA_ERR_INVALID, "query must be 16-byte aligned");
  if (((uintptr_t)a.block_tables | (uintptr_t)a.seq_lens | (uintptr_t)a.draft_mask |
       (uintptr_t)a.weights) % 4)
    return fail(SQA_ERR_INVALID,
                "block_tables, seq_lens, draft_mask and weights must be 4-byte aligned");
  if (a.draft_mask && (a.mask_words < (a.q_len + 31) / 32 || a.mask_words > 2))
    return fail(SQA_ERR_INVALID, "draft_mask needs %d..2 words per row, got %d",
                (a.q_len + 31) / 32, a.mask_words);
  if (!(a.scale > 0.f) || !isfinite(a.scale))
    return fail(SQA_ERR_INVALID, "scale must be positive and finite");
  if (a.weights_width <= 0 || a.weights_batch_stride < 0 || a.weights_head_stride < 0)
    return fail(SQA_ERR_INVALID, "weights need a positive width and non-negative strides");
  int device = -1;
  if (hipError_t e = hipGetDevice(&device); e != hipSuccess) return hip_fail(e, "hipGetDevice");
  const int shift = page_shift_of(a.page_size);
  WeighPlan plan;
  if (int rc = weigh_plan(device, a.batch, a.q_len, a.num_query_heads, a.num_kv_heads, a.head_dim,
                          a.max_seq_len, a.max_pages << shift, a.kv_dtype, &plan))
    return rc;
  if (plan.items * a.num_kv_heads > 0x7fffffffLL) return fail(SQA_ERR_INVALID, "grid too large");
  const size_t need = plan.stats + plan.scores;
  if (!a.workspace || a.workspace_bytes < need)
    return fail(SQA_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                a.workspace ? a.workspace_bytes : (size_t)0);
  if ((uintptr_t)a.workspace % 16)
    return fail(SQA_ERR_WORKSPACE, "workspace must be 16-byte aligned");

  sqa::WeighArgs w;
  memset(&w, 0, sizeof(w));
  sqa::PartialArgs& p = w.p;
  p.q = (const _Float16*)a.query;
  p.k = (const _Float16*)a.kv.k;
  p.block_tables = a.block_tables;
  p.seq_lens = a.seq_lens;
  p.draft_mask = a.draft_mask;
  p.mask_words = a.draft_mask ? a.mask_words : 0;
  p.num_pages = a.kv.num_pages;
  p.page_stride = bytes * a.kv.page_stride;
  p.token_stride = (unsigned)(bytes * a.kv.token_stride);
  p.head_stride = (unsigned)(bytes * a.kv.head_stride);
  p.page_extent = (unsigned)extent;
  p.batch = a.batch;
  p.q_len = a.q_len;
  p.hq = a.num_query_heads;
  p.hkv = a.num_kv_heads;
  p.group = group;
  p.rows = (int)rows;
  p.head_dim = a.head_dim;
  p.bt_stride = a.max_pages;
  p.page_shift = shift;
  p.max_pages = (int)plan.pages;
  p.by_splits = sqa::fast_div((unsigned)plan.items);
  p.by_group = sqa::fast_div(group);
  p.scale_log2 = (float)(1.4426950408889634 * (double)a.scale);
  p.bf16 = a.dtype == SQA_DTYPE_BF16;
  w.k_scale = a.k_scale;
  w.scale_page = 4 * (long long)a.scale_page_stride;
  w.scale_head = (unsigned)(4 * a.scale_head_stride);
  w.items = (int)plan.items;
  w.wg_heads = wg_heads(a.num_kv_heads);
  w.kv_type = a.kv_dtype;
  w.weights = a.weights;
  w.w_batch = a.weights_batch_stride;
  w.w_head = a.weights_head_stride;
  w.width = a.weights_width;
  // The scores first: 16-byte stores.
  w.scores = plan.scores ? (float*)a.workspace : nullptr;
  w.stats = (float2*)((char*)a.workspace + plan.scores);
  hipError_t e = sqa::launch_weigh(w, (hipStream_t)a.stream);
  return e == hipSuccess ? SQA_OK : hip_fail(e, "attention weights kernel launch");
}

int sqa_evict(const sqa_evict_args* args) {
  if (!args) return fail(SQA_ERR_INVALID, "null argument struct");
  if (args->struct_size != sizeof(sqa_evict_args))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                args->struct_size, sizeof(sqa_evict_args));
  const sqa_evict_args& a = *args;
  if (!a.weights || !a.new_weights || !a.kept || !a.seq_lens || !a.new_lens || !a.kv.k ||
      !a.kv.v || !a.into.k || !a.into.v || !a.block_tables || !a.new_tables)
    return fail(SQA_ERR_INVALID, "null tensor pointer");
  if (int rc = check_cache(a.batch, a.num_kv_heads, a.head_dim, a.page_size, a.kv.num_pages,
                           a.max_pages))
    return rc;
  if (int rc = check_cache(a.batch, a.num_kv_heads, a.head_dim, a.page_size, a.into.num_pages,
                           a.new_max_pages))
    return rc;
  if (a.kv_dtype != SQA_DTYPE_F16 && a.kv_dtype != SQA_DTYPE_BF16 && !is_codes(a.kv_dtype))
    return fail(SQA_ERR_UNSUPPORTED, "unknown kv_dtype %d", a.kv_dtype);
  const int bytes = is_codes(a.kv_dtype) ? 1 : 2;
  long long extent = 0;
  for (const sqa_kv_cache* c : {&a.kv, &a.into}) {
    if (int rc = check_strides(*c, bytes, a.num_kv_heads, a.head_dim, &extent)) return rc;
    const int64_t any = c->page_stride | c->token_stride | c->head_stride;
    if (any * bytes % 16)
      return fail(SQA_ERR_INVALID, "cache strides must be multiples of 16 bytes");
  }
  const bool scaled = a.scales.k != nullptr;
  if (scaled && !is_codes(a.kv_dtype))
    return fail(SQA_ERR_INVALID, "scales belong to 8-bit caches");
  if (a.kv_dtype == SQA_DTYPE_INT8 && !scaled)
    return fail(SQA_ERR_INVALID, "int8 caches need scales");
  if (scaled) {
    if (int rc = check_scales(a.scales, true)) return rc;
    if (int rc = check_scales(a.into_scales, true)) return rc;
  }
  if (a.budget <= 0 || a.sink < 0 || a.recent < 0 || (long long)a.sink + a.recent > a.budget)
    return fail(SQA_ERR_INVALID,
                "budget must be positive and hold sink + recent tokens (got %d, %d, %d)", a.budget,
                a.sink, a.recent);
  if (a.budget > (long long)a.new_max_pages * a.page_size)
    return fail(SQA_ERR_INVALID, "new_tables rows hold %lld tokens, the budget is %d",
                (long long)a.new_max_pages * a.page_size, a.budget);
  if (a.weights_width <= 0 || a.new_weights_width < a.budget)
    return fail(SQA_ERR_INVALID, "weights must not be empty, new_weights hold the budget");
  if (a.weights_batch_stride < 0 || a.weights_head_stride < 0 || a.new_weights_batch_stride < 0 ||
      a.new_weights_head_stride < 0)
    return fail(SQA_ERR_INVALID, "strides must not be negative");
  if (((uintptr_t)a.weights | (uintptr_t)a.new_weights | (uintptr_t)a.kept |
       (uintptr_t)a.seq_lens | (uintptr_t)a.new_lens | (uintptr_t)a.block_tables |
       (uintptr_t)a.new_tables) % 4)
    return fail(SQA_ERR_INVALID, "weights, lengths and tables must be 4-byte aligned");
  const long long grid =
      (long long)a.batch * ceil_div(a.budget, sqa::kPageSize) * ceil_div(a.num_kv_heads, 4);
  if (grid > 0x7fffffffLL || (long long)a.batch * a.num_kv_heads > 0x7fffffffLL)
    return fail(SQA_ERR_INVALID, "grid too large");

  if (a.into.k == a.into.v || (scaled && a.into_scales.k == a.into_scales.v))
    return fail(SQA_ERR_INVALID, "keys and values are written: each needs its own cache and scales");
  // Workgroups of other heads may read a length after the first one has written the new one.
  const uintptr_t old_lens = (uintptr_t)a.seq_lens, new_lens = (uintptr_t)a.new_lens;
  const uintptr_t lens_bytes = sizeof(int32_t) * (uintptr_t)a.batch;
  if (old_lens < new_lens + lens_bytes && new_lens < old_lens + lens_bytes)
    return fail(SQA_ERR_INVALID, "new_lens must not overlap seq_lens");
  sqa::EvictArgs k;
  memset(&k, 0, sizeof(k));
  k.weights = a.weights;
  k.w_batch = a.weights_batch_stride;
  k.w_head = a.weights_head_stride;
  k.width = a.weights_width;
  k.new_weights = a.new_weights;
  k.nw_batch = a.new_weights_batch_stride;
  k.nw_head = a.new_weights_head_stride;
  k.new_width = a.new_weights_width;
  k.kept = a.kept;
  k.seq_lens = a.seq_lens;
  k.new_lens = a.new_lens;
  k.budget = a.budget;
  k.sink = a.sink;
  k.recent = a.recent;
  k.src[0] = (const char*)a.kv.k;
  k.src[1] = (const char*)a.kv.v;
  k.dst[0] = (char*)a.into.k;
  k.dst[1] = (char*)a.into.v;
  k.src_page = bytes * a.kv.page_stride;
  k.src_token = bytes * a.kv.token_stride;
  k.src_head = bytes * a.kv.head_stride;
  k.dst_page = bytes * a.into.page_stride;
  k.dst_token = bytes * a.into.token_stride;
  k.dst_head = bytes * a.into.head_stride;
  k.src_scales = scales_of(a.scales);
  k.dst_scales = scales_of(a.into_scales);
  k.block_tables = a.block_tables;
  k.new_tables = a.new_tables;
  k.bt_stride = a.max_pages;
  k.new_stride = a.new_max_pages;
  k.num_pages = a.kv.num_pages;
  k.new_pages = a.into.num_pages;
  k.batch = a.batch;
  k.hkv = a.num_kv_heads;
  k.head_dim = a.head_dim;
  k.page_size = a.page_size;
  k.kv_type = a.kv_dtype;
  k.scaled = scaled;
  hipError_t e = sqa::launch_evict(k, (hipStream_t)a.stream);
  return e == hipSuccess ? SQA_OK : hip_fail(e, "eviction kernel launch");
}

}  // extern "C"

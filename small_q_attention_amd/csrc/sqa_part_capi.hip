// C ABI of attention over a window and over a shared prefix (declared in include/sqa.h):
// validates arguments, plans, and launches the kernels of sqa_part.hip and sqa_shared.hip
// on the caller's stream. Allocates nothing.
#include "sqa.h"
#include "sqa_part.h"

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

// Shapes that the plans and the calls check alike.
int check_shape(int batch, int q_len, int num_query_heads, int num_kv_heads, int head_dim,
                long long* rows) {
  if (batch <= 0 || q_len <= 0 || num_kv_heads <= 0 || num_query_heads <= 0 ||
      num_query_heads % num_kv_heads)
    return fail(SQA_ERR_INVALID,
                "batch, q_len and heads must be positive, query heads divisible by kv heads");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(SQA_ERR_UNSUPPORTED, "head_dim must be 64, 128 or 256 (got %d)", head_dim);
  *rows = (long long)q_len * (num_query_heads / num_kv_heads);
  const int most = head_dim == 256 ? sqa::kMaxRowsHd256 : sqa::kMaxRows;
  if (*rows > most)
    return fail(SQA_ERR_UNSUPPORTED, "q_len * group = %lld exceeds %d at head_dim %d", *rows, most,
                head_dim);
  if ((long long)batch * q_len * num_query_heads > 0x7fffffffLL)
    return fail(SQA_ERR_INVALID, "grid too large");
  return SQA_OK;
}

// kv heads a workgroup of single waves serves.
int wg_heads(int num_kv_heads) { return num_kv_heads >= 3 ? 4 : num_kv_heads; }

// Splits of sequences that span up to `pages` pages each: workgroups of four waves, one to
// a compute unit, so that the rounds they take times (pages of a split + what a workgroup
// costs besides, in pages) is least; two splits and more also pay for the join.
long long own_splits(int cus, long long batch, int num_kv_heads, long long pages) {
  constexpr long long kStart = 6, kJoin = 8;
  const int wgh = wg_heads(num_kv_heads);
  const long long head_groups = ceil_div(num_kv_heads, wgh);
  const long long most = std::max(pages / sqa::kMinSplitPages, 1LL);
  long long best = 1, best_cost = 0;
  for (long long n = 1; n <= std::min(most, 256LL); ++n) {
    const long long rounds = ceil_div(ceil_div(batch * n, 4 / wgh) * head_groups, cus);
    const long long cost = rounds * (ceil_div(pages, n) + kStart) + (n > 1 ? kJoin : 0);
    if (n == 1 || cost < best_cost) {
      best = n;
      best_cost = cost;
    }
  }
  return best;
}

// Pages that a window leaves of a sequence of up to `pages`: the first tokens', and those
// of `window + q_len - 1` tokens that begin anywhere in a page.
long long window_pages(long long pages, long long window, long long sink, int q_len) {
  const long long first = ceil_div(sink, sqa::kPageSize);
  const long long last = ceil_div(window + q_len - 2, sqa::kPageSize) + 1;
  return std::min(pages, first + last);
}

// The checks of a call and its kernel arguments, but for the plan.
int fill(const sqa_attention_args& a, const sqa_block_scales* scales, sqa::PartArgs* out) {
  if (!a.query || !a.kv.k || !a.kv.v || !a.block_tables || !a.seq_lens || !a.output)
    return fail(SQA_ERR_INVALID, "null tensor pointer");
  long long rows = 0;
  if (int rc = check_shape(a.batch, a.q_len, a.num_query_heads, a.num_kv_heads, a.head_dim, &rows))
    return rc;
  const int shift = page_shift_of(a.page_size);
  if (shift < 0)
    return fail(SQA_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256 (got %d)",
                a.page_size);
  if (a.kv.num_pages <= 0 || a.max_pages <= 0)
    return fail(SQA_ERR_INVALID, "empty KV cache is not supported");
  if (a.kv.num_pages > 0x7fffffffLL) return fail(SQA_ERR_INVALID, "page ids are 32 bits");
  if (((long long)a.max_pages << shift) >= (1LL << 26))
    return fail(SQA_ERR_INVALID, "block-table rows must be under 2^30 tokens");
  if (a.dtype != SQA_DTYPE_F16 && a.dtype != SQA_DTYPE_BF16)
    return fail(SQA_ERR_UNSUPPORTED, "dtype must be SQA_DTYPE_F16 or SQA_DTYPE_BF16 (got %d)",
                a.dtype);
  const bool codes = a.kv_dtype == SQA_DTYPE_FP8_E4M3 || a.kv_dtype == SQA_DTYPE_INT8;
  if (a.kv_dtype != a.dtype && !codes)
    return fail(SQA_ERR_UNSUPPORTED, "kv_dtype must be dtype or an 8-bit type (got %d)",
                a.kv_dtype);
  if (scales && !codes) return fail(SQA_ERR_INVALID, "scales belong to 8-bit caches");
  if (!scales && a.kv_dtype == SQA_DTYPE_INT8)
    return fail(SQA_ERR_INVALID, "int8 caches need scales");
  if (scales) {
    if (!scales->k || !scales->v) return fail(SQA_ERR_INVALID, "null scale pointer");
    if (((uintptr_t)scales->k | (uintptr_t)scales->v) % 4)
      return fail(SQA_ERR_INVALID, "scales must be 4-byte aligned");
    if (scales->page_stride < 0 || scales->head_stride < 0 ||
        scales->page_stride > ((int64_t)1 << 40) || scales->head_stride > 0x1fffffffLL)
      return fail(SQA_ERR_INVALID, "scale strides must be non-negative and within 32 bits");
  }
  const int bytes = codes ? 1 : 2;
  const int64_t ps = a.kv.page_stride, ts = a.kv.token_stride, hs = a.kv.head_stride;
  if (ps < 0 || ts < 0 || hs < 0 || ps % 8 || ts % 8 || hs % 8)
    return fail(SQA_ERR_INVALID, "cache strides must be non-negative multiples of 8 elements");
  if (((uintptr_t)a.kv.k | (uintptr_t)a.kv.v) % 16)
    return fail(SQA_ERR_INVALID, "cache base pointers must be 16-byte aligned");
  if (ps > ((int64_t)1 << 40) || ts > 0x3fffffffLL || hs > 0x3fffffffLL)
    return fail(SQA_ERR_INVALID, "cache strides are too large");
  const long long extent = bytes * ((long long)(sqa::kPageSize - 1) * ts +
                                    (long long)(a.num_kv_heads - 1) * hs + a.head_dim);
  if (extent > 0x7fffffffLL)
    return fail(SQA_ERR_INVALID, "one page of the cache spans more than 2 GiB");
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
  if (a.num_splits <= 0) return fail(SQA_ERR_INVALID, "num_splits must be positive");

  memset(out, 0, sizeof(*out));
  sqa::PartialArgs& p = out->p;
  p.q = (const _Float16*)a.query;
  p.k = (const _Float16*)a.kv.k;
  p.v = (const _Float16*)a.kv.v;
  p.block_tables = a.block_tables;
  p.seq_lens = a.seq_lens;
  p.draft_mask = a.draft_mask;
  p.mask_words = a.draft_mask ? a.mask_words : 0;
  p.out = (_Float16*)a.output;
  p.num_pages = a.kv.num_pages;
  p.page_stride = bytes * a.kv.page_stride;
  p.token_stride = (unsigned)(bytes * a.kv.token_stride);
  p.head_stride = (unsigned)(bytes * a.kv.head_stride);
  p.page_extent = (unsigned)extent;
  p.batch = a.batch;
  p.q_len = a.q_len;
  p.hq = a.num_query_heads;
  p.hkv = a.num_kv_heads;
  p.group = a.num_query_heads / a.num_kv_heads;
  p.rows = (int)rows;
  p.head_dim = a.head_dim;
  p.bt_stride = a.max_pages;
  p.page_shift = shift;
  p.max_pages = a.max_pages << shift;
  p.num_splits = a.num_splits;
  p.scale_log2 = (float)(1.4426950408889634 * (double)a.scale);
  p.out_scale = a.out_scale;
  p.bf16 = a.dtype == SQA_DTYPE_BF16;
  if (scales)
    out->scales = {(float*)scales->k, (float*)scales->v, 4 * (long long)scales->page_stride,
                   (unsigned)(4 * scales->head_stride)};
  out->scaled = scales != nullptr;
  out->kv_type = codes ? (a.kv_dtype == SQA_DTYPE_INT8 ? sqa::kInt8 : sqa::kE4M3) : sqa::kF16;
  out->wg_heads = wg_heads(a.num_kv_heads);
  out->splits = a.num_splits;
  p.by_head_groups = sqa::fast_div((unsigned)ceil_div(a.num_kv_heads, out->wg_heads));
  p.by_splits = sqa::fast_div(a.num_splits);
  p.by_group = sqa::fast_div(p.group);
  out->by_rows = sqa::fast_div(p.rows);
  return SQA_OK;
}

// The partials' place in the workspace: `rows` rows of sums, then of (max, sum).
int place(const sqa_attention_args& a, long long rows, size_t need, sqa::PartArgs* s) {
  if (need == 0) return SQA_OK;
  if (!a.workspace || a.workspace_bytes < need)
    return fail(SQA_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                a.workspace ? a.workspace_bytes : (size_t)0);
  if ((uintptr_t)a.workspace % 16)
    return fail(SQA_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  const unsigned long long bytes = (unsigned long long)rows * a.head_dim * 4;
  if (bytes > sqa::kMaxPartialBytes)
    return fail(SQA_ERR_INVALID, "the plan's partials (%llu bytes) exceed %llu bytes", bytes,
                sqa::kMaxPartialBytes);
  s->p.part_o = (float*)a.workspace;
  s->p.part_o_bytes = (unsigned)bytes;
  s->p.part_ml = s->p.part_o + rows * a.head_dim;
  return SQA_OK;
}

// Where the parts of a plan's table are, in bytes.
struct SharedTable {
  size_t group_of, items, bytes;
};
SharedTable table_of(int num_groups, int batch, long long num_items) {
  SharedTable t;
  t.group_of = (size_t)num_groups * sizeof(sqa::SharedGroup);
  t.items = t.group_of + ((size_t)batch * 4 + 15) / 16 * 16;
  t.bytes = t.items + (size_t)num_items * sizeof(sqa::SharedItem);
  return t;
}

// Rows of a block: those of the widest group, as one wave takes them while they fit one,
// else as a workgroup does.
int rows_of_block(long long most, int head_dim) {
  if (most <= 16) return 16;
  if (most <= 32) return 32;
  if (most <= 64 && head_dim != 256) return 64;
  return most <= 128 || head_dim == 256 ? 128 : 256;
}

// Splits of `pages` pages of at most `size` each, all alike but for the last.
long long splits_of(long long pages, long long size) {
  return ceil_div(pages, ceil_div(pages, ceil_div(pages, size)));
}

// Pages of a split, so that the rounds the groups' workgroups take times (pages of a split +
// what a workgroup costs besides) is least.
struct SharedCut {
  int cus, num_kv_heads, block_rows;
  long long workgroups(long long items) const {
    if (block_rows > 64) return items * num_kv_heads;
    const int wgh = wg_heads(num_kv_heads);
    return ceil_div(items, 4 / wgh) * ceil_div(num_kv_heads, wgh);
  }
  template <typename Groups>
  long long pages(const Groups& groups, int num_groups) const {
    constexpr long long kStart = 12;
    long long longest = 1;
    for (int g = 0; g < num_groups; ++g) longest = std::max(longest, (long long)groups(g).pages);
    const auto items = [&](long long size) {
      long long n = 0;
      for (int g = 0; g < num_groups; ++g)
        n += groups(g).blocks * ceil_div(groups(g).pages, size);
      return n;
    };
    long long best = longest, best_cost = -1;
    for (int rounds = 1; rounds <= 8; ++rounds) {
      long long lo = sqa::kMinSplitPages, hi = std::max(longest, lo);  // the fewest that fit
      while (lo < hi) {
        const long long mid = (lo + hi) / 2;
        if (workgroups(items(mid)) <= (long long)rounds * cus)
          hi = mid;
        else
          lo = mid + 1;
      }
      const long long real = ceil_div(workgroups(items(lo)), cus);
      const long long cost = real * (lo + kStart);
      if (best_cost < 0 || cost < best_cost) {
        best = lo;
        best_cost = cost;
      }
    }
    return best;
  }
};

int check_plan(const sqa_shared_plan* p) {
  if (!p) return fail(SQA_ERR_INVALID, "null plan");
  if (p->struct_size != sizeof(sqa_shared_plan))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                p->struct_size, sizeof(sqa_shared_plan));
  if (p->num_groups < 0 || p->num_items < 0 || p->partial_rows < 0)
    return fail(SQA_ERR_INVALID, "not a plan of sqa_plan_shared_prefix");
  return SQA_OK;
}

bool workgroups_fit(const sqa::PartArgs& s) {
  return (long long)s.p.batch * s.splits * s.p.hkv <= 0x7fffffffLL;
}

}  // namespace

extern "C" {

int sqa_plan_windowed(int device, int batch, int q_len, int num_query_heads, int num_kv_heads,
                      int head_dim, int64_t window, int sink, int max_seq_len, int max_pages,
                      int* num_splits) {
  if (!num_splits) return fail(SQA_ERR_INVALID, "null output pointer");
  long long rows = 0;
  if (int rc = check_shape(batch, q_len, num_query_heads, num_kv_heads, head_dim, &rows)) return rc;
  if (max_pages <= 0) return fail(SQA_ERR_INVALID, "max_pages must be positive");
  if (window <= 0 || sink < 0)
    return fail(SQA_ERR_INVALID, "window must be positive and sink not negative");
  const int cus = sqa_device_cu_count(device);
  if (cus <= 0) return SQA_ERR_HIP;
  long long pages = max_pages;
  if (max_seq_len > 0) pages = std::min(pages, ceil_div(max_seq_len, sqa::kPageSize));
  pages = window_pages(pages, std::min(window, (int64_t)1 << 31), sink, q_len);
  *num_splits = (int)own_splits(cus, batch, num_kv_heads, pages);
  return SQA_OK;
}

int sqa_paged_attention_windowed(const sqa_attention_args* args, const sqa_block_scales* scales,
                                 int64_t window, int sink) {
  if (!args) return fail(SQA_ERR_INVALID, "null argument struct");
  if (args->struct_size != sizeof(sqa_attention_args))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                args->struct_size, sizeof(sqa_attention_args));
  const sqa_attention_args& a = *args;
  if (window <= 0 || sink < 0)
    return fail(SQA_ERR_INVALID, "window must be positive and sink not negative");
  sqa::PartArgs s;
  if (int rc = fill(a, scales, &s)) return rc;
  s.window = std::min(window, (int64_t)1 << 31);
  s.sink = sink;
  if (!workgroups_fit(s)) return fail(SQA_ERR_INVALID, "grid too large");
  const long long rows = (long long)a.batch * a.num_splits * a.num_kv_heads * s.p.rows;
  const size_t need = sqa_workspace_bytes(a.batch, a.q_len, a.num_query_heads, a.num_kv_heads,
                                          a.head_dim, a.num_splits, 1);
  if (int rc = place(a, rows, need, &s)) return rc;

  hipStream_t stream = (hipStream_t)a.stream;
  hipEvent_t* ev = (hipEvent_t*)a.timing_events;
  hipError_t e;
  if (ev && (e = hipEventRecord(ev[0], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  if ((e = sqa::launch_own(s, stream)) != hipSuccess)
    return hip_fail(e, "windowed attention kernel launch");
  if (ev && (e = hipEventRecord(ev[1], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  if (a.num_splits > 1 && (e = sqa::launch_join(s, stream)) != hipSuccess)
    return hip_fail(e, "join kernel launch");
  if (ev && (e = hipEventRecord(ev[2], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  return SQA_OK;
}

int sqa_plan_shared_prefix(int device, int batch, int q_len, int num_query_heads,
                           int num_kv_heads, int head_dim, int page_size, int num_groups,
                           const int32_t* groups, sqa_shared_plan* plan, void* table) {
  if (!plan) return fail(SQA_ERR_INVALID, "null output pointer");
  long long rows = 0;
  if (int rc = check_shape(batch, q_len, num_query_heads, num_kv_heads, head_dim, &rows)) return rc;
  const int shift = page_shift_of(page_size);
  if (shift < 0)
    return fail(SQA_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256 (got %d)",
                page_size);
  if (num_groups < 0 || (num_groups > 0 && !groups))
    return fail(SQA_ERR_INVALID, "null or negative groups");
  const int cus = sqa_device_cu_count(device);
  if (cus <= 0) return SQA_ERR_HIP;
  // A group of one sequence, or of no pages, shares nothing.
  long long most_rows = 0, most_pages = 0, least = 0;
  int shared = 0, end = 0, covered = 0;
  for (int i = 0; i < num_groups; ++i) {
    const int first = groups[3 * i], count = groups[3 * i + 1], pages = groups[3 * i + 2];
    if (first < end || count <= 0 || pages < 0 || count > batch - first)
      return fail(SQA_ERR_INVALID,
                  "groups are (first, count, pages) in order, apart and within the batch");
    if (((long long)pages << shift) >= (1LL << 26))
      return fail(SQA_ERR_INVALID, "block-table rows must be under 2^30 tokens");
    end = first + count;
    if (count == 1 || pages == 0) continue;
    ++shared;
    covered += count;
    most_rows = std::max(most_rows, count * rows);
    most_pages = std::max(most_pages, (long long)pages);
    least = shared == 1 ? pages : std::min(least, (long long)pages);
  }
  const int block_rows = rows_of_block(most_rows, head_dim);
  struct Group {
    long long blocks, pages;
    int first, count;
  };
  // The i-th group that shares something; groups are few beside the work they stand for.
  const auto shared_group = [&](int want) {
    for (int i = 0;; ++i) {
      if (groups[3 * i + 1] == 1 || groups[3 * i + 2] == 0 || want-- > 0) continue;
      return Group{ceil_div(groups[3 * i + 1] * rows, block_rows),
                   (long long)groups[3 * i + 2] << shift, groups[3 * i], groups[3 * i + 1]};
    }
  };
  const SharedCut cut{cus, num_kv_heads, block_rows};
  const long long size = shared ? cut.pages(shared_group, shared) : 1;
  long long items = 0, partial_rows = 0;
  for (int g = 0; g < shared; ++g) {
    const Group x = shared_group(g);
    const long long splits = splits_of(x.pages, size);
    items += x.blocks * splits;
    partial_rows += splits * num_kv_heads * x.count * rows;
  }
  if (items * num_kv_heads > 0x7fffffffLL) return fail(SQA_ERR_INVALID, "grid too large");
  const SharedTable t = table_of(shared, batch, items);
  sqa_shared_plan out;
  memset(&out, 0, sizeof(out));
  out.struct_size = sizeof(out);
  out.batch = batch;
  out.q_len = q_len;
  out.num_query_heads = num_query_heads;
  out.num_kv_heads = num_kv_heads;
  out.head_dim = head_dim;
  out.page_size = page_size;
  out.num_groups = shared;
  out.num_items = (int)items;
  out.block_rows = block_rows;
  out.most_pages = (int)most_pages;
  out.least_pages = covered == batch ? (int)least : 0;
  out.partial_rows = partial_rows;
  out.table_bytes = t.bytes;
  *plan = out;
  if (!table) return SQA_OK;
  sqa::SharedGroup* to = (sqa::SharedGroup*)table;
  int32_t* group_of = (int32_t*)((char*)table + t.group_of);
  sqa::SharedItem* item = (sqa::SharedItem*)((char*)table + t.items);
  memset(table, 0, t.items);
  for (int b = 0; b < batch; ++b) group_of[b] = -1;
  long long base = 0;
  for (int g = 0; g < shared; ++g) {
    const Group x = shared_group(g);
    const int splits = (int)splits_of(x.pages, size);
    const int each = (int)ceil_div(x.pages, splits);
    to[g] = {x.first, x.count, (int)x.pages, splits, each, (int)x.blocks, base};
    base += (long long)splits * num_kv_heads * x.count * rows;
    for (int b = x.first; b < x.first + x.count; ++b) group_of[b] = g;
    for (int j = 0; j < splits; ++j)
      for (int k = 0; k < x.blocks; ++k) *item++ = {g, k, j, 0};
  }
  return SQA_OK;
}

int sqa_plan_shared_own(int device, const sqa_shared_plan* plan, int max_seq_len, int max_pages,
                        int* num_splits) {
  if (!num_splits) return fail(SQA_ERR_INVALID, "null output pointer");
  if (int rc = check_plan(plan)) return rc;
  if (max_pages <= 0) return fail(SQA_ERR_INVALID, "max_pages must be positive");
  const int cus = sqa_device_cu_count(device);
  if (cus <= 0) return SQA_ERR_HIP;
  long long pages = max_pages;
  if (max_seq_len > 0) pages = std::min(pages, ceil_div(max_seq_len, sqa::kPageSize));
  pages -= (long long)plan->least_pages * (plan->page_size / sqa::kPageSize);
  *num_splits = (int)own_splits(cus, plan->batch, plan->num_kv_heads, std::max(pages, 1LL));
  return SQA_OK;
}

size_t sqa_shared_workspace_bytes(const sqa_shared_plan* plan, int num_splits) {
  if (check_plan(plan) || num_splits <= 0) return 0;
  if (num_splits == 1 && plan->num_groups == 0) return 0;
  const size_t rows = (size_t)plan->q_len * (plan->num_query_heads / plan->num_kv_heads);
  const size_t own = (size_t)plan->batch * num_splits * plan->num_kv_heads * rows;
  return (own + (size_t)plan->partial_rows) * ((size_t)plan->head_dim + 2) * sizeof(float);
}

int sqa_paged_attention_shared_prefix(const sqa_attention_args* args,
                                      const sqa_block_scales* scales, const sqa_shared_plan* plan,
                                      const void* table) {
  if (!args) return fail(SQA_ERR_INVALID, "null argument struct");
  if (args->struct_size != sizeof(sqa_attention_args))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                args->struct_size, sizeof(sqa_attention_args));
  if (int rc = check_plan(plan)) return rc;
  const sqa_attention_args& a = *args;
  sqa::PartArgs s;
  if (int rc = fill(a, scales, &s)) return rc;
  if (plan->batch != a.batch || plan->q_len != a.q_len ||
      plan->num_query_heads != a.num_query_heads || plan->num_kv_heads != a.num_kv_heads ||
      plan->head_dim != a.head_dim || plan->page_size != a.page_size)
    return fail(SQA_ERR_INVALID, "the plan was made for another batch, q_len, heads or page size");
  if (plan->most_pages > a.max_pages)
    return fail(SQA_ERR_INVALID, "the plan shares %d pages, block_tables rows hold %d",
                plan->most_pages, a.max_pages);
  if (plan->num_groups > 0) {
    if (!table) return fail(SQA_ERR_INVALID, "null plan table");
    if ((uintptr_t)table % 16) return fail(SQA_ERR_INVALID, "plan table must be 16-byte aligned");
    const SharedTable t = table_of(plan->num_groups, plan->batch, plan->num_items);
    s.groups = (const sqa::SharedGroup*)table;
    s.group_of = (const int32_t*)((const char*)table + t.group_of);
    s.items = (const sqa::SharedItem*)((const char*)table + t.items);
    s.n_items = plan->num_items;
    s.block_rows = plan->block_rows;
  }
  if (!workgroups_fit(s)) return fail(SQA_ERR_INVALID, "grid too large");
  s.shared_at = (long long)a.batch * a.num_splits * a.num_kv_heads * s.p.rows;
  const size_t need = sqa_shared_workspace_bytes(plan, a.num_splits);
  if (int rc = place(a, s.shared_at + plan->partial_rows, need, &s)) return rc;

  hipStream_t stream = (hipStream_t)a.stream;
  hipEvent_t* ev = (hipEvent_t*)a.timing_events;
  hipError_t e;
  if (ev && (e = hipEventRecord(ev[0], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  if (s.n_items > 0 && (e = sqa::launch_shared(s, stream)) != hipSuccess)
    return hip_fail(e, "shared prefix kernel launch");
  if ((e = sqa::launch_own(s, stream)) != hipSuccess)
    return hip_fail(e, "own part kernel launch");
  if (ev && (e = hipEventRecord(ev[1], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  if ((a.num_splits > 1 || s.n_items > 0) && (e = sqa::launch_join(s, stream)) != hipSuccess)
    return hip_fail(e, "join kernel launch");
  if (ev && (e = hipEventRecord(ev[2], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  return SQA_OK;
}

}  // extern "C"

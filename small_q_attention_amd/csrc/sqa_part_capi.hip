// C ABI of attention over a window and over a shared prefix (declared in include/sqa.h):
// validates arguments, plans, and launches the kernels of sqa_part.hip, sqa_groups.hip and
// sqa_tiles.h on the caller's stream. Allocates nothing.
#include "sqa.h"
#include "sqa_part.h"

#include <math.h>

#include <cmath>
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

// A model of a call's time, in microseconds, by which the cuts are chosen. Workgroups of
// `waves` waves, one to a compute unit: a second one there waits for the first one's loads,
// so what counts is rounds.
struct Model {
  int cus, batch, rows, num_kv_heads, head_dim, kv_bytes;

  // A page (16 tokens of one head's K and V) for each wave of a workgroup, `n` of them at
  // work: the device's 6.6 TB/s shared out, at most 34 GB/s to a unit (both measured, 16 to
  // 128 sequences of 34 to 258 pages), less where the heads read together make short runs; no
  // less than a wave's chain over a page takes, by its dims and rows, codes widened or not.
  double page(long long n, int heads, int waves) const {
    const int run = std::min(heads, num_kv_heads) * head_dim * kv_bytes;
    const double worse = run >= 1024 ? 1.0 : run >= 512 ? 1.04 : run >= 256 ? 1.2 : 1.4;
    const double bytes = 32.0 * head_dim * kv_bytes * waves * worse;
    const double work = std::max(head_dim / 128.0 * ((rows + 15) / 16), 1.0);
    return std::max({(kv_bytes == 1 ? 0.58 : 0.55) * work, bytes * std::min<long long>(n, cus) / 6.6e6,
                     bytes / 34e3});
  }
  // Partial rows written and read again, and the kernel that joins them.
  double join(double slots) const {
    return 4 + slots * num_kv_heads * rows * head_dim * 8 / 3e6;
  }
  // Keeps cuts of huge batches from a workspace of more than 4 GiB where others do with less.
  double memory(double slots) const {
    return 1e-3 * std::max(slots * num_kv_heads * rows * head_dim * 4 -
                               (double)sqa::kMaxPartialBytes, 0.0);
  }
};

// How the sequences' own pages are dealt out: `splits` equal splits of every sequence, or
// (0) `items` equal items of the whole batch; `heads` kv heads to a workgroup.
struct OwnCut {
  int splits, items, heads;
  double workgroups, longest, mean;  // times of one of them
  double slots;                      // partial slots that are written
  double places(int batch) const {   // and that there are, with a group
    return splits > 0 ? (double)batch * splits : slots;
  }
};

// Calls try(cut) for the cuts worth a look. Sequences have up to `most` pages, `mean` on
// average.
template <typename Try>
void own_cuts(const Model& m, int waves, long long most, double mean, bool may_cross,
              Try&& attempt) {
  const double start_us = 5, piece_us = 3 + m.rows / 8.0;
  for (int heads = 4; heads >= 1; heads /= 2) {
    if (heads / 2 >= m.num_kv_heads) continue;  // a smaller workgroup holds them all
    const long long head_groups = ceil_div(m.num_kv_heads, heads);
    const int share = waves / heads;  // waves that divide a share's pages
    for (int n = 1; n <= 256 && (n == 1 || n * sqa::kMinSplitPages <= most);
         n += std::max(1, n / 8)) {
      const long long wgs = m.batch * n * head_groups;
      const double pages = (double)ceil_div(ceil_div(most, n), share);
      const double at_mean = std::max(std::ceil(mean / n / share), 1.0) * m.page(wgs, heads, waves);
      // The longest, as others have ended, takes what a unit gives.
      attempt(OwnCut{n, 0, heads, (double)wgs,
                     start_us + std::max(pages * m.page(1, heads, waves), at_mean), 2 + at_mean,
                     n > 1 ? (double)m.batch * n : 0.0});
    }
    if (m.batch == 1 || !may_cross) continue;
    const double total = std::max(m.batch * mean, 1.0);
    const long long all = std::max<long long>(m.cus / head_groups, 1);
    for (long long n = all; n >= 1; n = n > 8 ? n * 7 / 8 : n - 1) {
      if (n > 1 && total / n < sqa::kMinSplitPages) continue;
      const double pages = std::max(std::ceil(total / n / share), 1.0);
      const double time = start_us + piece_us * (1 + (double)m.batch / n) +
                          pages * m.page(n * head_groups, heads, waves);
      attempt(OwnCut{0, (int)n, heads, (double)(n * head_groups), time, time,
                     (double)(n + m.batch)});
    }
  }
}

// When `first` workgroups of time t1, then those of a cut, have run on the device, each unit
// taking the next as it gets free (which in a long row of them begins beside the last).
double finish(int cus, double first, double t1, const OwnCut& c) {
  const double whole = std::floor(first / cus), rest = first - whole * cus, free = cus - rest;
  const double base = whole * t1;
  // While the last of those run:
  const double beside = rest > 0 ? std::floor(t1 / c.longest) * free : 0;
  if (c.workgroups <= beside)
    return base + std::max(t1, std::ceil(c.workgroups / free) * c.longest);
  const double rounds = (c.workgroups - beside) / cus;  // many end one by one
  return base + (rest > 0 ? t1 : 0) +
         (rounds > 2 ? rounds * c.mean + 0.5 * c.longest : std::ceil(rounds) * c.longest);
}

// The cut of sequences without a group.
OwnCut best_own(const Model& m, long long most, double mean, bool may_cross) {
  OwnCut best{};
  double best_cost = -1;
  own_cuts(m, 4, most, mean, may_cross, [&](const OwnCut& c) {
    const double cost = finish(m.cus, 0, 1, c) +
                        (c.slots > 0 ? m.join(c.slots) + m.memory(c.slots) : 0);
    if (best_cost < 0 || cost < best_cost * 0.995) {
      best = c;
      best_cost = cost;
    }
  });
  return best;
}

// Whether the pages of a batch, with what every sequence counts besides, can be numbered from
// end to end.
bool may_cross(long long batch, long long kernel_pages) {
  return batch * (kernel_pages + sqa::kSeamPages) < (1LL << 27);
}

// Pages that a window leaves of a sequence of up to `pages`: the first tokens', and those
// of `window + q_len - 1` tokens that begin anywhere in a page.
long long window_pages(long long pages, long long window, long long sink, int q_len) {
  const long long first = ceil_div(sink, sqa::kPageSize);
  const long long last = ceil_div(window + q_len - 2, sqa::kPageSize) + 1;
  return std::min(pages, first + last);
}

// The checks of a call and its kernel arguments, but for the plan.
int fill(const sqa_attention_args& a, const sqa_block_scales* scales, int wg_heads,
         sqa::PartArgs* out) {
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
  if (a.pages_per_split != 0 && a.pages_per_split != 1)
    return fail(SQA_ERR_INVALID, "pages_per_split must be 0 or 1, as the plan has it");
  if (a.num_splits <= 0 || (a.pages_per_split == 0 && a.num_splits <= a.batch))
    return fail(SQA_ERR_INVALID, "num_splits must be positive, and more than the batch where "
                                 "splits cross sequence ends");
  if (a.pages_per_split == 0 && !may_cross(a.batch, (long long)a.max_pages << shift))
    return fail(SQA_ERR_INVALID, "batch * pages per row must be under 2^27");
  if (wg_heads != 1 && wg_heads != 2 && wg_heads != 4)
    return fail(SQA_ERR_INVALID, "wg_heads must be 1, 2 or 4, got %d", wg_heads);

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
  out->splits = a.pages_per_split ? a.num_splits : 0;
  out->own_items = a.pages_per_split ? 0 : a.num_splits - a.batch;
  out->wg_heads = wg_heads;
  p.by_head_groups = sqa::fast_div((unsigned)ceil_div(a.num_kv_heads, wg_heads));
  p.by_splits = sqa::fast_div(a.num_splits);
  p.by_group = sqa::fast_div(p.group);
  out->by_rows = sqa::fast_div(p.rows);
  return SQA_OK;
}

// The queries are read until the end, by workgroups beside those that write results.
int check_apart(const sqa_attention_args& a) {
  const unsigned long long bytes =
      2ull * a.batch * a.q_len * (unsigned long long)a.num_query_heads * a.head_dim;
  const uintptr_t q = (uintptr_t)a.query, o = (uintptr_t)a.output;
  if ((q < o ? o - q : q - o) < bytes) return fail(SQA_ERR_INVALID, "output overlaps query");
  return SQA_OK;
}

// Slots of the sequences' own pages.
long long own_slots(int batch, int num_splits, int pages_per_split) {
  return pages_per_split ? (long long)batch * num_splits : num_splits;
}

// The partials' place in the workspace: `rows` rows of sums, then of (max, sum), then the
// sequences' first slots and counts.
int place(const sqa_attention_args& a, long long rows, size_t need, sqa::PartArgs* s) {
  if (need == 0) return SQA_OK;
  if (!a.workspace || a.workspace_bytes < need)
    return fail(SQA_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                a.workspace ? a.workspace_bytes : (size_t)0);
  if ((uintptr_t)a.workspace % 16)
    return fail(SQA_ERR_WORKSPACE, "workspace must be 16-byte aligned");
  if (rows > 0x7fffffffLL) return fail(SQA_ERR_INVALID, "grid too large");
  const unsigned long long bytes = (unsigned long long)rows * a.head_dim * 4;
  s->p.part_o = (float*)a.workspace;
  s->far_rows = bytes > sqa::kMaxPartialBytes;
  s->p.part_o_bytes = s->far_rows ? 0 : (unsigned)bytes;
  s->p.part_ml = s->p.part_o + rows * a.head_dim;
  s->p.seq_splits = (sqa::SeqSplits*)(s->p.part_ml + rows * 2);
  return SQA_OK;
}

// Rows of a block: those of the widest group, as one wave takes them while they fit one,
// else as a workgroup does (256 with up to 32 rows of a sequence, at head dims 64 and 128).
int rows_of_block(long long most, long long rows, int head_dim) {
  const long long n = std::max(most, rows);
  if (n <= 16) return 16;
  if (n <= 32) return 32;
  if (n <= 64 && head_dim != 256) return 64;
  return n <= 128 || head_dim == 256 || rows > 32 ? 128 : 256;
}

struct SharedGroup {
  long long count, pages;  // 16-token pages
};

// Slots for the groups' splits, in multiples of the batch: for each sequence as many as the
// longest prefix has splits, or packed where that takes fewer (and the pages of all sequences'
// prefixes can be counted in 32 bits).
int shared_places(int batch, long long longest, long long all, long long size) {
  const int even = sqa::even_splits(longest, size).count;
  if (all > 0x7fffffffLL) return even;
  return (int)std::min<long long>(even, ceil_div(sqa::packed_slots(batch, all, size), batch));
}

struct SharedCut {
  OwnCut own;
  int block_rows;
  long long size;  // most pages of a group's split
  double cost;
};

// The cut of a batch with groups, whose workgroups begin first, in blocks of block_rows. Where
// a wave holds a block's rows they take their pages like the sequences'; tiles are bound by the
// matrix cores and by what the clock is then: a page of head dim 128 takes 0.40 us for 256
// rows on a few units and 0.54 on all, 0.34 for 128 rows, where a second workgroup on a unit
// takes as much again, and one of head dim 256 0.56; all of them 12 besides.
template <typename Groups>
SharedCut shared_cut(const Model& m, int block_rows, int num_groups, const Groups& group,
                     long long own_most, double own_mean, bool crosses) {
  const bool tiles = block_rows > 64;
  const int waves = block_rows == 256 ? 8 : 4;
  const auto tile_page = [&](double n) {
    if (m.head_dim == 256) return 0.56;
    return (block_rows == 256 ? 0.40 + 0.14 * std::min(n / m.cus, 1.0) : 0.34) * m.head_dim / 128;
  };
  long long longest = 1, all = 0;
  for (int g = 0; g < num_groups; ++g) {
    longest = std::max(longest, group(g).pages);
    all += group(g).count * group(g).pages;
  }
  struct Option {
    long long size;
    double items, slots, places;
  };
  Option options[64];
  int n_options = 0;
  for (int n = 1; n <= 256 && (n == 1 || n * sqa::kMinSplitPages <= longest);
       n += std::max(1, n / 8)) {
    Option o{ceil_div(longest, n), 0, 0, 0};
    if (n_options > 0 && o.size == options[n_options - 1].size) continue;
    for (int g = 0; g < num_groups; ++g) {
      const long long splits = sqa::even_splits(group(g).pages, o.size).count;
      o.items += (double)ceil_div(group(g).count * m.rows, block_rows) * splits;
      o.slots += (double)group(g).count * splits;
    }
    o.places = shared_places(m.batch, longest, all, o.size) * (double)m.batch;
    options[n_options++] = o;
    if (n_options == 64) break;
  }
  SharedCut best{};
  own_cuts(m, waves, own_most, own_mean, crosses, [&](const OwnCut& c) {
    const double head_groups = (double)ceil_div(m.num_kv_heads, c.heads);
    // Every sequence that shares leaves partial rows.
    const double slots = c.splits > 0 ? (double)m.batch * std::max(std::min((double)c.splits,
                                            own_mean / sqa::kMinSplitPages), 1.0) : c.slots;
    for (int i = 0; i < n_options; ++i) {
      const Option& o = options[i];
      const double n1 = o.items * (tiles ? m.num_kv_heads : head_groups);
      const double t1 = tiles ? 12 + o.size * tile_page(n1)
                              : 6 + ceil_div(o.size, waves / c.heads) *
                                        m.page((long long)(n1 + c.workgroups), c.heads, waves);
      const double cost = finish(m.cus, n1, t1, c) + m.join(slots + o.slots) +
                          m.memory(c.places(m.batch) + o.places);
      if (best.cost == 0 || cost < best.cost * 0.995) best = {c, block_rows, o.size, cost};
    }
  });
  return best;
}

int check_plan(const sqa_shared_plan* p) {
  if (!p) return fail(SQA_ERR_INVALID, "null plan");
  if (p->struct_size != sizeof(sqa_shared_plan))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                p->struct_size, sizeof(sqa_shared_plan));
  if (p->batch <= 0 || p->q_len <= 0 || p->num_kv_heads <= 0 || p->num_query_heads <= 0 ||
      p->head_dim <= 0 || p->num_groups < 0 || p->num_items < 0 || p->num_splits <= 0 ||
      p->shared_splits < 0 || p->shared_size <= 0 || (p->num_items > 0 && p->num_groups == 0) ||
      (p->pages_per_split == 0 && p->num_splits <= p->batch))
    return fail(SQA_ERR_INVALID, "not a plan of sqa_plan_shared_prefix");
  return SQA_OK;
}

// Partial rows of a plan's own slots, and of all.
long long own_rows(const sqa_shared_plan& p) {
  return own_slots(p.batch, p.num_splits, p.pages_per_split) * p.q_len * p.num_query_heads;
}
long long plan_rows(const sqa_shared_plan& p) {
  return own_rows(p) + (long long)p.shared_splits * p.batch * p.q_len * p.num_query_heads;
}

int kv_bytes(int kv_dtype) {
  return kv_dtype == SQA_DTYPE_FP8_E4M3 || kv_dtype == SQA_DTYPE_INT8 ? 1 : 2;
}

bool workgroups_fit(const sqa::PartArgs& s) {
  return ((long long)s.p.batch * s.splits + s.own_items) * s.p.hkv <= 0x3fffffffLL;
}

}  // namespace

extern "C" {

int sqa_plan_windowed(int device, int batch, int q_len, int num_query_heads, int num_kv_heads,
                      int head_dim, int64_t window, int sink, int max_seq_len, int max_pages,
                      int kv_dtype, int* num_splits, int* pages_per_split, int* wg_heads) {
  if (!num_splits || !pages_per_split || !wg_heads)
    return fail(SQA_ERR_INVALID, "null output pointer");
  long long rows = 0;
  if (int rc = check_shape(batch, q_len, num_query_heads, num_kv_heads, head_dim, &rows)) return rc;
  if (max_pages <= 0) return fail(SQA_ERR_INVALID, "max_pages must be positive");
  if (window <= 0 || sink < 0)
    return fail(SQA_ERR_INVALID, "window must be positive and sink not negative");
  const int cus = sqa_device_cu_count(device);
  if (cus <= 0) return SQA_ERR_HIP;
  long long pages = max_pages;
  if (max_seq_len > 0) pages = std::min(pages, ceil_div(max_seq_len, sqa::kPageSize));
  const long long left = window_pages(pages, std::min(window, (int64_t)1 << 31), sink, q_len);
  const Model m{cus, batch, (int)rows, num_kv_heads, head_dim, kv_bytes(kv_dtype)};
  // Sequences longer than the window are all alike, shorter ones seldom.
  const OwnCut cut = best_own(m, left, left < pages ? left : 0.65 * left,
                              may_cross(batch, max_pages));
  *pages_per_split = cut.splits > 0;
  *num_splits = cut.splits > 0 ? cut.splits : cut.items + batch;
  *wg_heads = cut.heads;
  return SQA_OK;
}

int sqa_paged_attention_windowed(const sqa_attention_args* args, const sqa_block_scales* scales,
                                 int64_t window, int sink, int wg_heads) {
  if (!args) return fail(SQA_ERR_INVALID, "null argument struct");
  if (args->struct_size != sizeof(sqa_attention_args))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                args->struct_size, sizeof(sqa_attention_args));
  const sqa_attention_args& a = *args;
  if (window <= 0 || sink < 0)
    return fail(SQA_ERR_INVALID, "window must be positive and sink not negative");
  sqa::PartArgs s;
  if (int rc = fill(a, scales, wg_heads, &s)) return rc;
  s.window = std::min(window, (int64_t)1 << 31);
  s.sink = sink;
  if (!workgroups_fit(s)) return fail(SQA_ERR_INVALID, "grid too large");
  const long long rows = own_slots(a.batch, a.num_splits, a.pages_per_split) * a.num_kv_heads *
                         s.p.rows;
  const size_t need = sqa_workspace_bytes(a.batch, a.q_len, a.num_query_heads, a.num_kv_heads,
                                          a.head_dim, a.num_splits, a.pages_per_split);
  if (int rc = place(a, rows, need, &s)) return rc;
  if (int rc = check_apart(a)) return rc;

  hipStream_t stream = (hipStream_t)a.stream;
  hipEvent_t* ev = (hipEvent_t*)a.timing_events;
  hipError_t e;
  if (ev && (e = hipEventRecord(ev[0], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  if ((e = sqa::launch_own(s, stream)) != hipSuccess)
    return hip_fail(e, "windowed attention kernel launch");
  if (ev && (e = hipEventRecord(ev[1], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  if (need > 0 && (e = sqa::launch_join(s, stream)) != hipSuccess)
    return hip_fail(e, "join kernel launch");
  if (ev && (e = hipEventRecord(ev[2], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  return SQA_OK;
}

int sqa_plan_shared_prefix(int device, int batch, int q_len, int num_query_heads,
                           int num_kv_heads, int head_dim, int page_size, int kv_dtype,
                           int num_groups, const int32_t* groups, int max_seq_len, int max_pages,
                           sqa_shared_plan* plan, int32_t* table) {
  if (!plan) return fail(SQA_ERR_INVALID, "null output pointer");
  long long rows = 0;
  if (int rc = check_shape(batch, q_len, num_query_heads, num_kv_heads, head_dim, &rows)) return rc;
  const int shift = page_shift_of(page_size);
  if (shift < 0)
    return fail(SQA_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256 (got %d)",
                page_size);
  if (num_groups < 0 || (num_groups > 0 && !groups))
    return fail(SQA_ERR_INVALID, "null or negative groups");
  if (max_pages <= 0) return fail(SQA_ERR_INVALID, "max_pages must be positive");
  if (((long long)max_pages << shift) >= (1LL << 26))
    return fail(SQA_ERR_INVALID, "block-table rows must be under 2^30 tokens");
  const int cus = sqa_device_cu_count(device);
  if (cus <= 0) return SQA_ERR_HIP;
  // A group of one sequence, or of no pages, shares nothing.
  const auto group = [&](int i) {
    const bool shares = groups[3 * i + 1] > 1;
    return SharedGroup{groups[3 * i + 1], shares ? (long long)groups[3 * i + 2] << shift : 0};
  };
  long long most_rows = 0, most_pages = 0, covered = 0, longest = 0, all_shared = 0;
  int end = 0;
  for (int i = 0; i < num_groups; ++i) {
    const int first = groups[3 * i], count = groups[3 * i + 1], pages = groups[3 * i + 2];
    if (first < end || count <= 0 || pages < 0 || count > batch - first)
      return fail(SQA_ERR_INVALID,
                  "groups are (first, count, pages) in order, apart and within the batch");
    if (count > 1 && pages > max_pages)
      return fail(SQA_ERR_INVALID, "a group shares %d pages, block_tables rows hold %d", pages,
                  max_pages);
    end = first + count;
    covered += count;
    if (group(i).pages == 0) continue;
    most_rows = std::max(most_rows, count * rows);
    longest = std::max(longest, group(i).pages);
    all_shared += count * group(i).pages;
    most_pages = std::max(most_pages, (long long)pages);
  }
  // Own pages, as far as they can be guessed: what follows a prefix is as long as what the
  // longest sequence has past the longest one; a group that shares nothing has its prefix to
  // itself, and a sequence of no group anything.
  long long whole = (long long)max_pages << shift, longest_named = 0;
  if (max_seq_len > 0) whole = std::min(whole, ceil_div(max_seq_len, sqa::kPageSize));
  const auto named = [&](int i) { return std::min((long long)groups[3 * i + 2] << shift, whole); };
  for (int i = 0; i < num_groups; ++i) longest_named = std::max(longest_named, named(i));
  const long long tail = std::max(whole - longest_named, 1LL);
  long long own = covered < batch ? whole : tail;
  double own_pages = 0.65 * whole * (batch - covered);
  for (int i = 0; i < num_groups; ++i) {
    const long long alone = group(i).pages > 0 ? 0 : named(i);
    own = std::max(own, alone + tail);
    own_pages += groups[3 * i + 1] * (alone + 0.65 * tail);
  }
  const double own_mean = std::max(own_pages / batch, 1.0);
  sqa_shared_plan out;
  memset(&out, 0, sizeof(out));
  out.struct_size = sizeof(out);
  out.batch = batch;
  out.q_len = q_len;
  out.num_query_heads = num_query_heads;
  out.num_kv_heads = num_kv_heads;
  out.head_dim = head_dim;
  out.page_size = page_size;
  out.block_rows = 16;
  out.shared_size = 1;
  out.most_pages = (int)most_pages;
  const Model m{cus, batch, (int)rows, num_kv_heads, head_dim, kv_bytes(kv_dtype)};
  const bool crosses = may_cross(batch, (long long)max_pages << shift);
  OwnCut own_cut;
  if (longest == 0) {
    own_cut = best_own(m, own, own_mean, crosses);
  } else {
    out.num_groups = num_groups;
    out.block_rows = rows_of_block(most_rows, rows, head_dim);
    SharedCut cut = shared_cut(m, out.block_rows, num_groups, group, own, own_mean, crosses);
    if (out.block_rows == 256) {  // less of it empty where groups are small
      const SharedCut halves = shared_cut(m, 128, num_groups, group, own, own_mean, crosses);
      if (halves.cost < 0.97 * cut.cost) cut = halves;
    }
    out.block_rows = cut.block_rows;
    long long items = 0;
    for (int i = 0; i < num_groups; ++i) {
      const SharedGroup g = group(i);
      const int splits = sqa::even_splits(g.pages, cut.size).count;
      items += ceil_div(g.count * rows, out.block_rows) * splits;
    }
    if (items * num_kv_heads > 0x3fffffffLL) return fail(SQA_ERR_INVALID, "grid too large");
    own_cut = cut.own;
    out.num_items = (int)items;
    out.shared_size = (int)cut.size;
    out.shared_splits = shared_places(batch, longest, all_shared, cut.size);
    if ((long long)out.shared_splits * batch > 0x7fffffffLL)
      return fail(SQA_ERR_INVALID, "grid too large");
  }
  out.pages_per_split = own_cut.splits > 0;
  out.num_splits = own_cut.splits > 0 ? own_cut.splits : own_cut.items + batch;
  out.wg_heads = own_cut.heads;
  *plan = out;
  if (!table) return SQA_OK;
  for (int i = 0; i < 3 * num_groups; ++i) table[i] = groups[i];
  int32_t* of = table + 3 * num_groups;
  for (int b = 0; b < batch; ++b) {
    of[2 * b] = -1;
    of[2 * b + 1] = 0;
  }
  long long before = 0;
  for (int i = 0; i < num_groups; ++i)
    for (int b = groups[3 * i]; group(i).pages > 0 && b < groups[3 * i] + groups[3 * i + 1]; ++b) {
      of[2 * b] = (int32_t)std::min(before, 0x7fffffffLL);
      of[2 * b + 1] = groups[3 * i + 2];
      before += group(i).pages;
    }
  return SQA_OK;
}

size_t sqa_shared_workspace_bytes(const sqa_shared_plan* plan) {
  if (check_plan(plan)) return 0;
  if (plan->pages_per_split && plan->num_splits == 1 && plan->num_items == 0) return 0;
  return (size_t)plan_rows(*plan) * ((size_t)plan->head_dim + 2) * sizeof(float) +
         (plan->pages_per_split ? 0 : (size_t)plan->batch * sizeof(sqa::SeqSplits));
}

int sqa_paged_attention_shared_prefix(const sqa_attention_args* args,
                                      const sqa_block_scales* scales, const sqa_shared_plan* plan,
                                      const int32_t* table) {
  if (!args) return fail(SQA_ERR_INVALID, "null argument struct");
  if (args->struct_size != sizeof(sqa_attention_args))
    return fail(SQA_ERR_INVALID, "struct_size %zu does not match this library's %zu",
                args->struct_size, sizeof(sqa_attention_args));
  if (int rc = check_plan(plan)) return rc;
  const sqa_attention_args& a = *args;
  sqa::PartArgs s;
  if (int rc = fill(a, scales, plan->wg_heads, &s)) return rc;
  if (plan->batch != a.batch || plan->q_len != a.q_len ||
      plan->num_query_heads != a.num_query_heads || plan->num_kv_heads != a.num_kv_heads ||
      plan->head_dim != a.head_dim || plan->page_size != a.page_size ||
      plan->num_splits != a.num_splits || plan->pages_per_split != a.pages_per_split)
    return fail(SQA_ERR_INVALID, "the plan was made for another batch, q_len, heads, page size or "
                                 "number of splits");
  if (plan->most_pages > a.max_pages)
    return fail(SQA_ERR_INVALID, "the plan shares %d pages, block_tables rows hold %d",
                plan->most_pages, a.max_pages);
  const bool tiles = plan->block_rows > 64;
  if (plan->num_items > 0) {
    if (!table || (uintptr_t)table % 4)
      return fail(SQA_ERR_INVALID, "the plan's table must be given, 4-byte aligned");
    const int b = plan->block_rows;
    if ((b != 16 && b != 32 && b != 64 && b != 128 && b != 256) ||
        (a.head_dim == 256 && (b == 64 || b == 256)) || (b == 256 && s.p.rows > 32) ||
        (!tiles && b < s.p.rows) || plan->shared_splits == 0)
      return fail(SQA_ERR_INVALID, "not a plan of sqa_plan_shared_prefix");
    s.groups = table;
    s.seq_groups = table + 3 * plan->num_groups;
    s.n_groups = plan->num_groups;
    s.n_items = plan->num_items;
    s.block_rows = b;
    s.shared_size = plan->shared_size;
    if ((long long)plan->shared_splits * a.batch > 0x7fffffffLL)
      return fail(SQA_ERR_INVALID, "grid too large");
    s.shared_slots = plan->shared_splits * a.batch;
    s.most_splits = sqa::even_splits((long long)plan->most_pages << s.p.page_shift,
                                     plan->shared_size).count;
    s.packed = plan->shared_splits < s.most_splits;
    s.slot_step = s.packed ? 1 : a.batch;
    s.by_shared_size = sqa::fast_div((unsigned)plan->shared_size);
    const long long heads = tiles ? a.num_kv_heads : ceil_div(a.num_kv_heads, s.wg_heads);
    if (heads * s.n_items > 0x3fffffffLL) return fail(SQA_ERR_INVALID, "grid too large");
    s.shared_wgs = (int)(heads * s.n_items);
    s.by_shared_heads = sqa::fast_div((unsigned)heads);
  }
  if (!workgroups_fit(s)) return fail(SQA_ERR_INVALID, "grid too large");
  s.shared_at = own_rows(*plan);
  const size_t need = sqa_shared_workspace_bytes(plan);
  if (int rc = place(a, plan_rows(*plan), need, &s)) return rc;
  if (int rc = check_apart(a)) return rc;

  hipStream_t stream = (hipStream_t)a.stream;
  hipEvent_t* ev = (hipEvent_t*)a.timing_events;
  hipError_t e;
  if (ev && (e = hipEventRecord(ev[0], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  if (s.n_items == 0)
    e = sqa::launch_own(s, stream);
  else if (!tiles)
    e = sqa::launch_waves(s, stream);
  else if (s.p.bf16)
    e = sqa::launch_tiles_bf16(s, stream);
  else
    e = sqa::launch_tiles_f16(s, stream);
  if (e != hipSuccess) return hip_fail(e, "shared prefix attention kernel launch");
  if (ev && (e = hipEventRecord(ev[1], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  if (need > 0 && (e = sqa::launch_join(s, stream)) != hipSuccess)
    return hip_fail(e, "join kernel launch");
  if (ev && (e = hipEventRecord(ev[2], stream)) != hipSuccess) return hip_fail(e, "hipEventRecord");
  return SQA_OK;
}

}  // extern "C"

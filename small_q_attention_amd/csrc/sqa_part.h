// Internal interface between the C ABI (sqa_part_capi.hip) and the kernels of attention
// over a part of every sequence (sqa_part.hip: a window and the first tokens, what follows
// a shared prefix) and over the pages that a group of sequences shares (sqa_shared.hip).
#pragma once

#include "sqa_cache.h"

namespace sqa {

// Sequences first .. first + count - 1, whose first `pages` 16-token pages are the same
// ones. Their rows, count * rows of a kv head, go over those pages together, in
// `splits` splits of `size` pages. Row r of sequence first + i, split j and kv head h leaves
// its partial at row base + ((j * hkv + h) * count + i) * rows + r of the partials.
struct SharedGroup {
  int first, count;
  int pages, splits, size;
  int blocks;      // blocks of rows
  long long base;
};

// One workgroup's share, or one wave's where a group's rows fit one: a block of a group's
// rows and a split of its pages (and one kv head, or each wave one).
struct SharedItem {
  int group, block, split, unused;
};

struct PartArgs {
  // Of PartialArgs the fields that name buffers, shapes, strides and scales. part_o, part_ml:
  // fp32 sums and (max in log2 units, sum) of the partial rows; sequence b's own splits are
  // slots b * splits + s.
  PartialArgs p;
  BlockScales scales;          // of codes with block scales
  int kv_type, scaled;         // kF16 (the query's type), kE4M3 or kInt8
  int wg_heads;                // kv heads a workgroup of single waves serves
  int splits;                  // most splits of a sequence's own pages
  long long window;            // a row sees the last `window` tokens up to its own (0: all)
  int sink;                    // and the first `sink`
  const SharedGroup* groups;   // null: none
  const int32_t* group_of;     // [B], -1: none
  const SharedItem* items;
  int n_items;
  long long shared_at;         // partial row of the groups' first one
  FastDiv by_rows;             // p.rows
  int block_rows;              // rows of a block: 16, 32 or 64 (one wave's), 128 or 256
};

hipError_t launch_own(const PartArgs& a, hipStream_t stream);
hipError_t launch_shared(const PartArgs& a, hipStream_t stream);
hipError_t launch_join(const PartArgs& a, hipStream_t stream);

}  // namespace sqa

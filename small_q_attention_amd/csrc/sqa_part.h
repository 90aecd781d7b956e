// Internal interface between the C ABI (sqa_part_capi.hip) and the kernels of attention
// over a part of every sequence (a window and the first tokens; what follows a shared
// prefix) and over the pages that a group of sequences shares.
#pragma once

#include "sqa_cache.h"

namespace sqa {

// Splits of `pages` pages of at most `size`, all alike but for the last.
struct EvenSplits {
  int count, size;
};
inline EvenSplits even_splits(long long pages, long long size) {
  const long long n = (pages + size - 1) / size;
  const long long each = n > 0 ? (pages + n - 1) / n : 1;
  return {(int)((pages + each - 1) / each), (int)each};
}

// What a workgroup pays to begin a sequence, in pages: where a batch's pages are cut from end
// to end, every sequence counts so many more than it has (96 sequences of 16 to 128 pages,
// q_len 4: 103 us a call without, 98 with).
constexpr int kSeamPages = 4;

struct PartArgs {
  // Of PartialArgs the fields that name buffers, shapes, strides and scales. part_o, part_ml:
  // fp32 sums and (max in log2 units, sum) of the partial rows. A slot of kv head h and
  // sequence b is `rows` of them. Own slot s starts at row (s * hkv + h) * rows, s = b *
  // splits + j for the sequence's split j, or (splits 0) from seq_splits[b].first on; split j
  // of the sequence's group at row shared_at + ((shared_slot() + j * slot_step) * hkv + h) * rows.
  PartialArgs p;
  BlockScales scales;      // of codes with block scales
  int kv_type, scaled;     // kF16 (the query's type), kE4M3 or kInt8
  // Sequences' own pages. splits > 0: every sequence by itself, in at most that many equal
  // splits. 0: the batch's pages end to end, cut into own_items equal items, of which the
  // part in sequence b leaves slot item + b.
  int splits, own_items;
  int wg_heads;            // kv heads a workgroup of single waves serves
  long long window;        // a row sees the last `window` tokens up to its own (0: all)
  int sink;                // and the first `sink`
  // Groups: n_groups x (first, count, pages): sequences first .. first + count - 1 begin with
  // the same `pages` table entries. Their rows, count * rows of a kv head, go over those pages
  // together, in blocks of block_rows (16, 32 or 64: one wave's; 128 or 256: a workgroup's)
  // and splits of at most shared_size 16-token pages; n_items blocks x splits in all.
  const int32_t* groups;
  // [B][2]: (16-token pages that the sequences before this one share, a page counted for
  // each, -1: this one shares none; its group's pages)
  const int32_t* seq_groups;
  int n_groups, n_items, block_rows, shared_size;
  int most_splits;         // of a group
  int shared_wgs;          // workgroups that serve the groups, the first of the grid
  long long shared_at;     // partial row of the groups' first slot
  FastDiv by_rows;         // p.rows
  FastDiv by_shared_heads; // workgroups per item
  // Slots of the groups' splits, shared_slots in all: the batch's for each split, one after the
  // other (slot_step the batch), or `packed` (where prefixes are so unlike that most of those
  // would stay empty) a sequence's (slot_step 1).
  int packed, shared_slots, slot_step;
  int far_rows;            // partials past 32-bit offsets (p.part_o_bytes is not theirs)
  FastDiv by_shared_size;
};

// Slots of all groups' splits, packed: sequence b's first is b + before / size, `before` the
// pages that the sequences before it share. A sequence of p = k size + r pages (r < size) has
// at most k splits, k + 1 where r > 0, and to the next one's first slot it is at least 1 + k.
inline long long packed_slots(long long batch, long long pages, long long size) {
  return batch + pages / size;
}

hipError_t launch_own(const PartArgs& a, hipStream_t stream);
hipError_t launch_waves(const PartArgs& a, hipStream_t stream);  // groups of one wave's rows
hipError_t launch_tiles_f16(const PartArgs& a, hipStream_t stream);  // of a workgroup's
hipError_t launch_tiles_bf16(const PartArgs& a, hipStream_t stream);
hipError_t launch_join(const PartArgs& a, hipStream_t stream);

}  // namespace sqa

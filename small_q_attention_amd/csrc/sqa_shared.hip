// gfx950 kernels of attention over the pages that a group of sequences shares: the rows of
// all of them, count * Q * (Hq / Hkv) of a kv head, against one K and V, so that a page is
// read once for the group and not once for each sequence.
#include "sqa_part.h"
#include "sqa_part_device.h"

namespace sqa {

hipError_t launch_shared(const PartArgs& a, hipStream_t stream) {
  const dim3 grid = part_grid(a, a.n_items);
  if (a.p.bf16)
    launch_part<ElemBF16, true>(a, a.block_rows, grid, stream);
  else
    launch_part<ElemF16, true>(a, a.block_rows, grid, stream);
  return hipGetLastError();
}

}  // namespace sqa

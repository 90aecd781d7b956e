// gfx950 kernels of attention over shared prefixes, groups whose rows one wave holds: the
// sequences' own pages and the groups' go through the same page loop.
#include "sqa_part.h"
#include "sqa_part_device.h"

namespace sqa {

hipError_t launch_waves(const PartArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)(a.shared_wgs + own_workgroups(a)));
  if (a.p.bf16)
    launch_part<ElemBF16, true>(a, a.block_rows, grid, stream);
  else
    launch_part<ElemF16, true>(a, a.block_rows, grid, stream);
  return hipGetLastError();
}

}  // namespace sqa

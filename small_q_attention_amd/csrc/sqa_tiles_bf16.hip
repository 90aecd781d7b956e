// gfx950 kernels of attention over shared prefixes, groups of many rows, bf16 queries.
#include "sqa_tiles.h"

namespace sqa {

hipError_t launch_tiles_bf16(const PartArgs& a, hipStream_t stream) {
  return launch_tiles_of<ElemBF16>(a, stream);
}

}  // namespace sqa

// paged_attn's kernels for trees of new tokens over e4m3 rows.
#include "paged_wide.h"

namespace wz {
int paged_tree_e4m3(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  return paged_tree_launch<true>(D, a, ask, workers, stream);
}
}  // namespace wz

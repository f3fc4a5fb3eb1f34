// paged_attn's kernels for trees of new tokens over bf16 rows.
#include "paged_wide.h"

namespace wz {
int paged_tree_bf16(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  return paged_tree_launch<false>(D, a, ask, workers, stream);
}
}  // namespace wz

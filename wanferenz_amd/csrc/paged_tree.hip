// paged_attn's kernels for trees of new tokens over bf16 rows.
#include "paged_attn.h"

namespace wz {
int paged_tree_bf16(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  return paged_attn_launch<false, true>(D, a, ask, workers, stream);
}
}  // namespace wz

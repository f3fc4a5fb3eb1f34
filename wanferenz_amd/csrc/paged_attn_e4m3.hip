// paged_attn's kernels for e4m3 rows.
#include "paged_attn.h"

namespace wz {
int paged_attn_e4m3(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  return paged_attn_launch<true>(D, a, ask, workers, stream);
}
}  // namespace wz

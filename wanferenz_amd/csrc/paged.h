// What the paged cache's kernels share: the cache's geometry and the lookup of a slot.
#pragma once

#include "common.h"

namespace wz {

// A wz_paged_kv as the kernels take it.
struct PagedView {
  uint8_t* k;
  uint8_t* v;  // k where one row serves as both
  float* ks;
  float* vs;
  float* weights;
  int32_t* positions;
  int pages, heads, page, shift;  // page = 1 << shift
  int dtype;
  bool shared;
};

// Row (of [pages, heads, page]) that holds a slot, or -1 where the table has no page for it.
__device__ __forceinline__ int64_t paged_row(const PagedView& c, const int32_t* __restrict__ trow, int width, int head,
                                             int slot) {
  const int p = slot >> c.shift;
  if (slot < 0 || p >= width) return -1;
  const int id = trow[p];
  if (uint32_t(id) >= uint32_t(c.pages)) return -1;
  return (int64_t(id) * c.heads + head) * c.page + (slot & (c.page - 1));
}

// Checks the cache and the table's width; fills the view.
int paged_view(const char* what, const wz_paged_kv* cache, int64_t table_width, PagedView* view);

}  // namespace wz

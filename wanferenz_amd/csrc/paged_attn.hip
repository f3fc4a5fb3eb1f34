// paged_attn: the kernels for bf16 rows and the entry points.
#include "paged_attn.h"

namespace wz {

int paged_attn_bf16(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  return paged_attn_launch<false>(D, a, ask, workers, stream);
}

static int paged_attn_any(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  return a.c.dtype == WZ_KV_E4M3 ? paged_attn_e4m3(D, a, ask, workers, stream)
                                 : paged_attn_bf16(D, a, ask, workers, stream);
}

struct PagedAttnSizes {
  int64_t part, cut, ml, scores;  // floats
};

static PagedAttnSizes paged_attn_sizes(const wz_paged_kv* c, int64_t B, int64_t S, int64_t H, int64_t width,
                                       bool accumulate) {
  PagedAttnSizes z{};
  const int64_t R = S * (H / c->kv_heads);
  PagedAttnArgs a{};
  a.c.heads = c->kv_heads;
  a.c.shared = c->v == nullptr;
  a.c.dtype = c->dtype;
  a.S = int(S);
  a.H = int(H);
  int workers = 0;
  const int64_t rows = paged_attn_any(c->head_dim, a, true, &workers, nullptr);
  z.part = 2 * workers * paged_slot(int(rows), c->head_dim);
  z.cut = workers * int64_t(sizeof(PagedCut) / sizeof(float));
  if (accumulate) {
    z.ml = (2 * B * c->kv_heads * R + 3) / 4 * 4;
    z.scores = B * c->kv_heads * R * width * c->page_size;
  }
  return z;
}

}  // namespace wz

extern "C" int64_t wz_paged_attn_workspace_bytes(const wz_paged_kv* cache, int64_t B, int64_t S, int64_t H,
                                                 int64_t table_width, int accumulate) {
  using namespace wz;
  PagedView view;
  if (paged_view("paged_attn", cache, table_width, &view) != WZ_OK) return 0;
  if (B <= 0 || S <= 0 || S > kPagedMaxS || H <= 0 || H > 65536 || H % view.heads)
    return 0;
  const PagedAttnSizes z = paged_attn_sizes(cache, B, S, H, table_width, accumulate != 0);
  return (z.part + z.cut + z.ml + z.scores) * int64_t(sizeof(float));
}

extern "C" int wz_paged_attn(const wz_paged_kv* cache, const void* q_bf16, const int64_t* q_strides,
                             const float* attn_sink, const int32_t* table, int64_t table_width, const int32_t* lens,
                             void* o_bf16, int64_t B, int64_t S, int64_t H, float softmax_scale, int accumulate,
                             void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  using namespace wz;
  PagedAttnArgs a{};
  if (int rc = paged_view("paged_attn", cache, table_width, &a.c)) return rc;
  if (B < 0 || B > 65535 || S < 0 || S > kPagedMaxS)
    return set_error(WZ_EINVAL, "paged_attn: bad shape B=%lld (up to 65535) S=%lld (up to %d)", (long long)B,
                     (long long)S, kPagedMaxS);
  if (H <= 0 || H > 65536 || H % a.c.heads)
    return set_error(WZ_EINVAL, "paged_attn: %lld heads on %d KV heads", (long long)H, a.c.heads);
  if (accumulate && !a.c.weights)
    return set_error(WZ_EINVAL, "paged_attn: the cache is not tracked (weights and positions)");
  if (B == 0 || S == 0) return WZ_OK;
  if (!q_bf16 || !q_strides || !lens || !o_bf16 || (table_width > 0 && !table))
    return set_error(WZ_EINVAL, "paged_attn: null pointer");
  if ((reinterpret_cast<uintptr_t>(q_bf16) | reinterpret_cast<uintptr_t>(o_bf16) |
       reinterpret_cast<uintptr_t>(workspace)) & 15 || ((q_strides[0] | q_strides[1] | q_strides[2]) & 7))
    return set_error(WZ_EINVAL, "paged_attn: q rows, o and the workspace must be 16-byte aligned");
  if (accumulate && reinterpret_cast<uintptr_t>(a.c.weights) & 15)
    return set_error(WZ_EINVAL, "paged_attn: weights must be 16-byte aligned");
  const int64_t R = S * (H / a.c.heads);
  if (B * a.c.heads * R > 0x7FFFFFFFLL || B * a.c.heads > 65535 * int64_t(accumulate ? 1 : 65535))
    return set_error(WZ_EINVAL, "paged_attn: %lld sequences of %lld heads", (long long)B, (long long)H);
  if (B * a.c.heads * ((R + 15) / 16) > 0x7FFFFFFFLL / (table_width * a.c.page / kPagedTile + 8))
    return set_error(WZ_EINVAL, "paged_attn: %lld sequences of up to %lld slots", (long long)B,
                     (long long)(table_width * a.c.page));
  if (2 * R * int64_t(sizeof(float)) > 65536)
    return set_error(WZ_EINVAL, "paged_attn: %lld query rows on a KV head", (long long)R);
  const PagedAttnSizes z = paged_attn_sizes(cache, B, S, H, table_width, accumulate != 0);
  const int64_t need = (z.part + z.cut + z.ml + z.scores) * int64_t(sizeof(float));
  if (!workspace || workspace_bytes < need)
    return set_error(WZ_ESPACE, "paged_attn: workspace of %lld bytes, %lld needed",
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
  a.q = static_cast<const uint16_t*>(q_bf16);
  a.qb = q_strides[0];
  a.qs = q_strides[1];
  a.qh = q_strides[2];
  a.sink = attn_sink;
  a.table = table;
  a.lens = lens;
  a.o = static_cast<uint16_t*>(o_bf16);
  a.part = static_cast<float*>(workspace);
  a.cut = reinterpret_cast<PagedCut*>(a.part + z.part);
  a.ml = accumulate ? a.part + z.part + z.cut : nullptr;
  a.scores = accumulate ? a.ml + z.ml : nullptr;
  a.width = int(table_width);
  a.B = int(B);
  a.S = int(S);
  a.H = int(H);
  a.capacity = table_width * a.c.page;
  a.scale2 = softmax_scale * kLog2e;
  return paged_attn_any(cache->head_dim, a, false, nullptr, stream);
}

// paged_attn: the kernels for bf16 rows and the entry points.
#include "paged_attn.h"

namespace wz {

int paged_attn_bf16(int D, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  return paged_attn_launch<false, false>(D, a, ask, workers, stream);
}

static int paged_attn_any(int D, bool tree, const PagedAttnArgs& a, bool ask, int* workers, hipStream_t stream) {
  if (tree)
    return a.c.dtype == WZ_KV_E4M3 ? paged_tree_e4m3(D, a, ask, workers, stream) : paged_tree_bf16(D, a, ask, workers, stream);
  return a.c.dtype == WZ_KV_E4M3 ? paged_attn_e4m3(D, a, ask, workers, stream)
                                 : paged_attn_bf16(D, a, ask, workers, stream);
}

struct PagedAttnSizes {
  int64_t part, cut, ml, scores;  // floats
};

static PagedAttnSizes paged_attn_sizes(const wz_paged_kv* c, int64_t B, int64_t S, int64_t H, int64_t width,
                                       bool accumulate, bool tree) {
  PagedAttnSizes z{};
  const int64_t R = S * (H / c->kv_heads);
  PagedAttnArgs a{};
  a.c.heads = c->kv_heads;
  a.c.shared = c->v == nullptr;
  a.c.dtype = c->dtype;
  a.B = int(B);
  a.S = int(S);
  a.H = int(H);
  a.capacity = width * c->page_size;
  int workers = 0;
  const int64_t rows = paged_attn_any(c->head_dim, tree, a, true, &workers, nullptr);
  z.part = 2 * workers * paged_slot(int(rows), c->head_dim);
  z.cut = workers * int64_t(sizeof(PagedCut) / sizeof(float));
  if (accumulate) {
    z.ml = (2 * B * c->kv_heads * R + 3) / 4 * 4;
    z.scores = B * c->kv_heads * R * width * c->page_size;
  }
  return z;
}

static int64_t paged_attn_need(const wz_paged_kv* cache, int64_t B, int64_t S, int64_t H, int64_t width,
                               bool accumulate, bool tree) {
  PagedView view;
  if (paged_view("paged_attn", cache, width, &view) != WZ_OK) return 0;
  if (B <= 0 || S <= 0 || S > (tree ? kPagedMaxNodes : kPagedMaxS) || H <= 0 || H > 65536 || H % view.heads)
    return 0;
  const PagedAttnSizes z = paged_attn_sizes(cache, B, S, H, width, accumulate, tree);
  return (z.part + z.cut + z.ml + z.scores) * int64_t(sizeof(float));
}

// parent: of a tree's nodes, or null for new tokens in a row; count goes with it.
static int paged_attn_run(const char* what, const wz_paged_kv* cache, const void* q_bf16, const int64_t* q_strides,
                          const float* attn_sink, const int32_t* table, int64_t table_width, const int32_t* lens, bool tree,
                          const int32_t* parent, const int32_t* count, void* o_bf16, int64_t B, int64_t S, int64_t H,
                          float softmax_scale, bool accumulate, void* workspace, int64_t workspace_bytes,
                          hipStream_t stream) {
  PagedAttnArgs a{};
  if (int rc = paged_view(what, cache, table_width, &a.c)) return rc;
  const int most = tree ? kPagedMaxNodes : kPagedMaxS;
  if (B < 0 || B > 65535 || S < 0 || S > most)
    return set_error(WZ_EINVAL, "%s: bad shape B=%lld (up to 65535) S=%lld (up to %d)", what, (long long)B, (long long)S,
                     most);
  if (H <= 0 || H > 65536 || H % a.c.heads)
    return set_error(WZ_EINVAL, "%s: %lld heads on %d KV heads", what, (long long)H, a.c.heads);
  if (accumulate && !a.c.weights)
    return set_error(WZ_EINVAL, "%s: the cache is not tracked (weights and positions)", what);
  if (B == 0 || S == 0) return WZ_OK;
  if (!q_bf16 || !q_strides || !lens || !o_bf16 || (table_width > 0 && !table) || (tree && !parent))
    return set_error(WZ_EINVAL, "%s: null pointer", what);
  if ((reinterpret_cast<uintptr_t>(q_bf16) | reinterpret_cast<uintptr_t>(o_bf16) |
       reinterpret_cast<uintptr_t>(workspace)) & 15 || ((q_strides[0] | q_strides[1] | q_strides[2]) & 7))
    return set_error(WZ_EINVAL, "%s: q rows, o and the workspace must be 16-byte aligned", what);
  if (accumulate && reinterpret_cast<uintptr_t>(a.c.weights) & 15)
    return set_error(WZ_EINVAL, "%s: weights must be 16-byte aligned", what);
  const int64_t R = S * (H / a.c.heads);
  if (B * a.c.heads * R > 0x7FFFFFFFLL || B * a.c.heads > 65535 * int64_t(accumulate ? 1 : 65535))
    return set_error(WZ_EINVAL, "%s: %lld sequences of %lld heads", what, (long long)B, (long long)H);
  if (B * a.c.heads * ((R + 15) / 16) > 0x7FFFFFFFLL / (table_width * a.c.page / kPagedTile + 8))
    return set_error(WZ_EINVAL, "%s: %lld sequences of up to %lld slots", what, (long long)B,
                     (long long)(table_width * a.c.page));
  if (2 * R * int64_t(sizeof(float)) > 65536)
    return set_error(WZ_EINVAL, "%s: %lld query rows on a KV head", what, (long long)R);
  const PagedAttnSizes z = paged_attn_sizes(cache, B, S, H, table_width, accumulate, tree);
  const int64_t need = (z.part + z.cut + z.ml + z.scores) * int64_t(sizeof(float));
  if (!workspace || workspace_bytes < need)
    return set_error(WZ_ESPACE, "%s: workspace of %lld bytes, %lld needed", what,
                     (long long)(workspace ? workspace_bytes : 0), (long long)need);
  a.q = static_cast<const uint16_t*>(q_bf16);
  a.qb = q_strides[0];
  a.qs = q_strides[1];
  a.qh = q_strides[2];
  a.sink = attn_sink;
  a.table = table;
  a.lens = lens;
  a.parent = parent;
  a.count = count;
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
  return paged_attn_any(cache->head_dim, tree, a, false, nullptr, stream);
}

}  // namespace wz

extern "C" int64_t wz_paged_attn_workspace_bytes(const wz_paged_kv* cache, int64_t B, int64_t S, int64_t H,
                                                 int64_t table_width, int accumulate) {
  return wz::paged_attn_need(cache, B, S, H, table_width, accumulate != 0, false);
}

extern "C" int wz_paged_attn(const wz_paged_kv* cache, const void* q_bf16, const int64_t* q_strides,
                             const float* attn_sink, const int32_t* table, int64_t table_width, const int32_t* lens,
                             void* o_bf16, int64_t B, int64_t S, int64_t H, float softmax_scale, int accumulate,
                             void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  return wz::paged_attn_run("paged_attn", cache, q_bf16, q_strides, attn_sink, table, table_width, lens, false, nullptr,
                            nullptr, o_bf16, B, S, H, softmax_scale, accumulate != 0, workspace, workspace_bytes, stream);
}

extern "C" int64_t wz_paged_tree_attn_workspace_bytes(const wz_paged_kv* cache, int64_t B, int64_t S, int64_t H,
                                                      int64_t table_width) {
  return wz::paged_attn_need(cache, B, S, H, table_width, false, true);
}

extern "C" int wz_paged_tree_attn(const wz_paged_kv* cache, const void* q_bf16, const int64_t* q_strides,
                                  const float* attn_sink, const int32_t* table, int64_t table_width,
                                  const int32_t* lens, const int32_t* parent, const int32_t* count, void* o_bf16,
                                  int64_t B, int64_t S, int64_t H, float softmax_scale, void* workspace,
                                  int64_t workspace_bytes, hipStream_t stream) {
  return wz::paged_attn_run("paged_tree_attn", cache, q_bf16, q_strides, attn_sink, table, table_width, lens, true, parent,
                            count, o_bf16, B, S, H, softmax_scale, false, workspace, workspace_bytes, stream);
}

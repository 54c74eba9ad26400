// Attention over shared prefixes (described in paged_shared.h): pages of 16 bits, and the entry points.
#include "paged_shared.h"

using namespace qkv;

QKV_EXPORT int64_t qkv_paged_attention_shared_workspace_bytes(int64_t rows, int64_t max_rows, int64_t requests,
                                                              int64_t width, int64_t page, int64_t q_heads,
                                                              int64_t kv_heads, int64_t head_dim) {
  if (!good_sizes(rows, requests, width, page, q_heads, kv_heads, head_dim)) return -1;
  const SharedShape s = shared_shape_of(rows, max_rows, requests, width * page, kv_heads, q_heads / kv_heads);
  return good_shared(s, rows, requests, q_heads) ? shared_bytes(s, rows, kv_heads, head_dim) : -1;
}

QKV_EXPORT int qkv_paged_attention_shared(const void* query, const int64_t* q_strides, const void* k_pages,
                                          const void* v_pages, const int64_t* page_strides, const void* k_scales,
                                          const void* v_scales, const int64_t* scale_strides, int code,
                                          const int32_t* shared, int64_t pages, int64_t page, const int32_t* table,
                                          int64_t table_ld, int64_t width, int64_t requests, const int32_t* cu_rows,
                                          const int32_t* kv_lens, int64_t rows, int64_t max_rows, int64_t q_heads,
                                          int64_t kv_heads, int64_t head_dim, float scaling, float softcap,
                                          const float* slopes, const int32_t* prefix_lens, const int32_t* first_keys,
                                          void* workspace, int64_t workspace_bytes, void* out,
                                          const int64_t* out_strides, int dtype, void* stream) {
  const char* what = "qkv_paged_attention_shared";
  if (code < 0 || code > QKV_CODE_FP4)
    return fail(QKV_ERR_INVALID, "%s: code %d is not 0, fp8 (%d) or fp4 (%d)", what, code, QKV_CODE_FP8, QKV_CODE_FP4);
  const PagedCall c{query, q_strides, k_pages, v_pages, page_strides, k_scales, v_scales, scale_strides, pages, page, table,
                    table_ld, width, requests, cu_rows, kv_lens, rows, max_rows, q_heads, kv_heads, head_dim, scaling,
                    softcap, slopes, prefix_lens, first_keys, workspace, workspace_bytes, out, out_strides, dtype, stream};
  if (code == QKV_CODE_FP8) return shared_call_fp8(c, shared, what);
  if (code == QKV_CODE_FP4) return shared_call_fp4(c, shared, what);
  return shared_call<kHalfPages>(c, shared, what);
}

// Attention of the rows of a step over a paged K/V cache: single tokens, drafted tokens, chunks of prompts and whole
// prompts, of requests of different lengths in one call.
//
// Row i of request b (rows cu[b] .. cu[b+1]-1) is the token at p = kv_len_b - rows_b + i.  It sees the keys j with
// first_i <= j < max(p + 1, prefix_b), j < kv_len_b (none if p < 0), and
//   s_j = cap * tanh(scaling * q.k_j / cap) - slope_h * |p - j|   (cap 0: scaling * q.k_j),
//   out = sum_j exp(s_j) v_j / sum_j exp(s_j), zero where it sees none.
//
// Work.  The G query heads of a KV head share its K and V, so a tile holds the G heads of several tokens; a tile's
// keys are split over several workgroups where there are few tiles.  How far is decided on the GPU from the lengths
// (locate, below): no length is needed on the host.  Two kernels: `rows` for tiles of 128 (token, head) rows, whose
// 4 waves hold 32 rows each and share tiles of 64 keys in LDS, bound by the matrix cores (2048 tokens behind 63488, 32/8
// heads: 2.09 ms, 1036 TFLOP/s, 77 to 83% of a large library product's rate); `token` for requests of at most 16 or 32
// (token, head) rows, whose 4 waves walk different keys of the same rows, bound by memory (32 requests of up to 32768
// keys: 530 us, 6.14 TB/s).  Requests of 17 to 32 rows in the rows kernel leave three of its waves idle (7 drafts of 5
// tokens, 4 heads: 57 us, 47 in the token kernel).
//
// Both take the scores transposed, S^T = K Q^T, so that a lane holds scores of one row: the softmax is in-lane but
// for one lane swap, and P^T leaves the score accumulators in the layout that the matrix instruction of O^T = V^T P^T
// wants (the order of the keys within a step is free; V^T is read in the same order, by transposing LDS reads).
//
// Over codes (FMT) both convert K and V to 16 bits on their way, exactly: the token kernel in registers (K in the order in
// which a lane's 16 bytes lie, Q's channels alike), the rows kernel between memory and LDS.  32 single tokens over up to
// 32768 keys: 300 us in fp8, 5.6 TB/s; 29 over up to 32001 in fp4: 137 us; 2048 tokens behind 63488 in fp8: 2.22 to 2.36 ms by card.
#include "paged_tiles.h"

using namespace qkv;

QKV_EXPORT int64_t qkv_paged_attention_workspace_bytes(int64_t rows, int64_t max_rows, int64_t requests, int64_t width,
                                                       int64_t page, int64_t q_heads, int64_t kv_heads,
                                                       int64_t head_dim) {
  if (!good_sizes(rows, requests, width, page, q_heads, kv_heads, head_dim)) return -1;
  int64_t most = 0;   // over 16-bit pages and over codes
  for (const int64_t row_bytes : {2 * head_dim, head_dim, head_dim / 2})
    most = std::max(most, workspace_bytes(plan_of(rows, max_rows, requests, width * page, kv_heads, q_heads / kv_heads, row_bytes), head_dim));
  return most;
}

QKV_EXPORT int qkv_paged_attention(const void* query, const int64_t* q_strides, const void* k_pages,
                                   const void* v_pages, const int64_t* page_strides, int64_t pages, int64_t page,
                                   const int32_t* table, int64_t table_ld, int64_t width, int64_t requests,
                                   const int32_t* cu_rows, const int32_t* kv_lens, int64_t rows, int64_t max_rows,
                                   int64_t q_heads, int64_t kv_heads, int64_t head_dim, float scaling, float softcap,
                                   const float* slopes, const int32_t* prefix_lens, const int32_t* first_keys,
                                   void* workspace, int64_t workspace_bytes, void* out, const int64_t* out_strides,
                                   int dtype, void* stream) {
  return paged_call<kHalfPages>({query, q_strides, k_pages, v_pages, page_strides, nullptr, nullptr, nullptr, pages, page,
                                 table, table_ld, width, requests, cu_rows, kv_lens, rows, max_rows, q_heads, kv_heads,
                                 head_dim, scaling, softcap, slopes, prefix_lens, first_keys, workspace, workspace_bytes,
                                 out, out_strides, dtype, stream}, "qkv_paged_attention");
}

QKV_EXPORT int qkv_paged_attention_codes(const void* query, const int64_t* q_strides, const void* k_pages,
                                         const void* v_pages, const int64_t* page_strides, const void* k_scales,
                                         const void* v_scales, const int64_t* scale_strides, int code, int64_t pages,
                                         int64_t page, const int32_t* table, int64_t table_ld, int64_t width,
                                         int64_t requests, const int32_t* cu_rows, const int32_t* kv_lens, int64_t rows,
                                         int64_t max_rows, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                         float scaling, float softcap, const float* slopes, const int32_t* prefix_lens,
                                         const int32_t* first_keys, void* workspace, int64_t workspace_bytes, void* out,
                                         const int64_t* out_strides, int dtype, void* stream) {
  const char* what = "qkv_paged_attention_codes";
  if (code != QKV_CODE_FP8 && code != QKV_CODE_FP4)
    return fail(QKV_ERR_INVALID, "%s: code %d is not fp8 (%d) or fp4 (%d)", what, code, QKV_CODE_FP8, QKV_CODE_FP4);
  const PagedCall c{query, q_strides, k_pages, v_pages, page_strides, k_scales, v_scales, scale_strides, pages, page, table,
                    table_ld, width, requests, cu_rows, kv_lens, rows, max_rows, q_heads, kv_heads, head_dim, scaling,
                    softcap, slopes, prefix_lens, first_keys, workspace, workspace_bytes, out, out_strides, dtype, stream};
  return code == QKV_CODE_FP8 ? paged_call_fp8(c, what) : paged_call_fp4(c, what);
}

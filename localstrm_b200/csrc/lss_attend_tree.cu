// lss_attend_tree.cu — C ABI of the attention of drafted tokens: each sees the context and its own branch.
#include "lss_attend_host.cuh"

extern "C" {

int lss_attend_tree(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype, int T, int q_heads,
               int heads, int dim, const uint8_t* k_cache, const uint8_t* v_cache, const float* k_scale,
               const float* v_scale, int num_blocks, int block_size, const int32_t* table, int64_t table_stride,
               int width, const int32_t* starts, const int32_t* granted, const int32_t* lens, int B, float scale,
               void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse, void* workspace,
               size_t workspace_bytes, const int32_t* span, void* stream) {
  return attend_entry<true>(q, q_token_stride, q_head_stride, dtype, T, q_heads, heads, dim, k_cache, v_cache, k_scale, v_scale, num_blocks, block_size, table, table_stride, width, starts, granted, lens, B, scale, out, out_token_stride, out_head_stride, lse, workspace, workspace_bytes, span, stream);
}

}  // extern "C"

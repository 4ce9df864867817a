// Decode attention for requests that continue the same tokens (spd_attn_decode_shared).
#include "common.cuh"

using namespace spd;

extern "C" {

int64_t spd_attn_decode_shared_workspace_bytes(int64_t max_batch, int num_q_heads, int num_kv_heads, int head_dim) {
  (void)num_kv_heads;
  return spd_attn_decode_workspace_bytes(max_batch, num_q_heads, head_dim);
}

int spd_attn_decode_shared(void* out, const void* q, const void* k_pool, const void* v_pool, const int32_t* req_to_token,
                           const int64_t* req_pool_indices, const int64_t* seq_lens, const int32_t* group_indptr,
                           const int64_t* shared_lens, int64_t batch, int64_t num_groups, int64_t max_shared_len,
                           int num_q_heads, int num_kv_heads, int head_dim, int64_t q_stride, int64_t out_stride,
                           int64_t req_to_token_stride, float sm_scale, int dtype, void* workspace, int64_t workspace_bytes,
                           int sm_budget, spd_stream_t stream) {
  SPD_REQUIRE(num_groups >= 0 && max_shared_len >= 0 && (num_groups == 0 || (group_indptr && shared_lens)), SPD_E_BADARG,
              "spd_attn_decode_shared: bad groups");
  // every request reads its own pages
  return spd_attn_decode_paged_own(out, q, k_pool, v_pool, req_to_token, req_pool_indices, seq_lens, batch, num_q_heads,
                                   num_kv_heads, head_dim, q_stride, out_stride, req_to_token_stride, sm_scale, dtype, workspace,
                                   workspace_bytes, sm_budget, stream);
}

}  // extern "C"

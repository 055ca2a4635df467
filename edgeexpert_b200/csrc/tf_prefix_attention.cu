// tf_prefix_attention.cu -- causal attention of a ragged batch behind a shared
// prefix, over a paged cache (tf_shared_prefix_attention).
#include "tf_prefix_kernels.cuh"

using namespace tf;

extern "C" {

size_t tf_shared_prefix_attention_workspace_bytes(const tf_context* ctx, const tf_paged_kv* kv, uint32_t num_q_heads,
                                                  uint32_t T, uint32_t num_requests, uint32_t prefix_len,
                                                  uint32_t max_query) {
    if (!ctx || !kv || kv->num_kv_heads == 0 || num_q_heads == 0 || num_q_heads % kv->num_kv_heads) return 0;
    const Shape shape = shape_of_call(kv, num_q_heads, T, prefix_len, max_query, false);
    return layout_of(ctx, kv, num_q_heads, T, shape).bytes;
}

tf_status tf_shared_prefix_attention(tf_context* ctx, const void* q, uint64_t q_stride, const tf_paged_kv* kv,
                                     const void* prefix_pages, uint32_t prefix_len, const void* page_table,
                                     uint32_t max_pages, const void* seq_lens, const void* token_starts,
                                     uint32_t num_requests, uint32_t max_query, uint32_t T, uint32_t num_q_heads,
                                     float scale, uint32_t window, void* out, uint64_t out_stride, void* lse,
                                     void* workspace, size_t workspace_bytes, void* stream) {
    const AttentionCall c = {q, q_stride, prefix_pages, prefix_len, page_table, max_pages, seq_lens, token_starts,
                             num_requests, max_query, T, num_q_heads, scale, window, out, out_stride, lse, workspace,
                             workspace_bytes, nullptr, 0, nullptr};
    return attention_call<false>(ctx, kv, c, static_cast<cudaStream_t>(stream), "tf_shared_prefix_attention");
}

}  // extern "C"

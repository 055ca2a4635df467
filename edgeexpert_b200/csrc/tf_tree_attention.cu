// tf_tree_attention.cu -- attention of the nodes of drafted trees over a paged cache
// (tf_tree_attention): the kernels of the ragged batch with a node's ancestors in the
// place of the causal mask.
//   out_j = sum_p softmax_p(scale q_j . k_p) v_p  over the history's p that the window
//   leaves and the nodes p whose bit is set in j's ancestors.
// A row's nodes are its request's last positions, so only the units that reach them look
// at bits; those before are history, seen whole or from the window's first position on.
// Batches whose bound on a request's nodes is above eight rows per KV head go to
// tree_tiles_kernel (tcgen05), others to the streaming warps (200 single nodes behind up to
// 2048, 1.68 GB: 269 us, 6.3 TB/s; 64 of 1 to 4 behind up to 4096, 1.08 GB: 182 us, 5.9 TB/s).
// Measured (calls among others): 16 trees of 16 behind up to 4096 positions, 16 / 8 heads
// of 256, 275 MB: 62 to 64 us, HBM inside the jobs; 4 of 60 to 64 behind 32 to 64 thousand,
// 1.62 GB: 300 to 333 us by machine, 4.9 to 5.4 TB/s; 24 of 20 to 40 behind 4096 shared, 16 / 4 heads
// of 128: 73 to 76 us, bound by the tiles' way out of L2 and the ends of the jobs; one of 12
// behind 700: 16.7 us, latency.  Two threads a row, with half the keys each: 0 to 4 % faster
// for these 24, 3 % slower for the long histories, 5 % for one tree.
#include "tf_prefix_kernels.cuh"

using namespace tf;

extern "C" {

size_t tf_tree_attention_workspace_bytes(const tf_context* ctx, const tf_paged_kv* kv, uint32_t num_q_heads, uint32_t T,
                                         uint32_t num_requests, uint32_t prefix_len, uint32_t max_query) {
    if (!ctx || !kv || kv->num_kv_heads == 0 || num_q_heads == 0 || num_q_heads % kv->num_kv_heads) return 0;
    const Shape shape = shape_of_call(kv, num_q_heads, T, prefix_len, max_query, true);
    return layout_of(ctx, kv, num_q_heads, T, shape).bytes;
}

tf_status tf_tree_attention(tf_context* ctx, const void* q, uint64_t q_stride, const tf_paged_kv* kv,
                            const void* prefix_pages, uint32_t prefix_len, const void* page_table, uint32_t max_pages,
                            const void* seq_lens, const void* token_starts, uint32_t num_requests, const void* ancestors,
                            uint32_t words, const void* positions, uint32_t max_query, uint32_t T, uint32_t num_q_heads,
                            float scale, uint32_t window, void* out, uint64_t out_stride, void* lse, void* workspace,
                            size_t workspace_bytes, void* stream) {
    const AttentionCall c = {q, q_stride, prefix_pages, prefix_len, page_table, max_pages, seq_lens, token_starts,
                             num_requests, max_query, T, num_q_heads, scale, window, out, out_stride, lse, workspace,
                             workspace_bytes, ancestors, words, positions};
    return attention_call<true>(ctx, kv, c, static_cast<cudaStream_t>(stream), "tf_tree_attention");
}

}  // extern "C"

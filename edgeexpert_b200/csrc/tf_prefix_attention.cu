// tf_prefix_attention.cu -- causal attention of a ragged batch behind a shared
// prefix, over a paged cache (tf_shared_prefix_attention).
//
// For a query row at position p, with the keys split in any way into parts i:
//   m_i = max s, d_i = sum e^(s - m_i), o_i = sum e^(s - m_i) v   over the part's visible keys,
//   M = max m_i, D = sum d_i e^(m_i - M), out = sum o_i e^(m_i - M) / D, lse = M + log D,
// so the shared prefix can be one part and the request's own pages another.
#include <math.h>

#include "tf_paged.cuh"

using namespace tf;

namespace {

template <typename T>
struct AttnParams {
    const T* q;
    long long q_stride;
    PagedView<T> kv;
    const int* prefix_pages;
    const int* table;
    const int* seq_lens;
    const int* starts;
    T* out;
    long long out_stride;
    float* lse;
    uint32_t* err;
    int prefix_len, max_pages, B, max_query, T_tokens, nq, nkv, hd, window;
    float scale;
};

// One warp per (token, head): a running maximum and sum over the visible keys.
template <typename T>
__global__ void __launch_bounds__(128) attention_rows_kernel(AttnParams<T> p) {
    constexpr int E = kMaxPagedHeadDim / 32;
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (long long)p.T_tokens * p.nq) return;
    const int t = (int)(row / p.nq), h = (int)(row % p.nq), kvh = h / (p.nq / p.nkv);
    float q[E], o[E], m = -INFINITY, d = 0.f;
    for (int i = 0; i < E; ++i) {
        const int e = lane + 32 * i;
        q[i] = e < p.hd ? to_float(p.q[t * p.q_stride + (long long)h * p.hd + e]) * p.scale : 0.f;
        o[i] = 0.f;
    }
    int lo = 0, hi = p.B;  // the last b with starts[b] <= t
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.starts[mid] <= t)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int b = lo;
    if (b < p.B) {
        const int n = p.starts[b + 1] - p.starts[b], j = t - p.starts[b];
        const int len = (int)min((long long)max(0, p.seq_lens[b]), (long long)p.max_pages * p.kv.page_size);
        if (j >= p.max_query) {
            if (lane == 0) atomicOr(p.err, kErrBadPage);
        } else {
            const long long at = (long long)p.prefix_len + len - max(n - j, 1);
            const long long first = p.window ? max(0ll, at - p.window + 1) : 0;
            for (long long pos = first; pos <= at; ++pos) {
                const bool shared = pos < p.prefix_len;
                const int i = (int)(shared ? pos : pos - p.prefix_len);
                const int page = shared ? p.prefix_pages[i / p.kv.page_size]
                                        : p.table[(long long)b * p.max_pages + i / p.kv.page_size];
                if (page < 0 || page >= p.kv.num_pages) {
                    if (lane == 0) atomicOr(p.err, kErrBadPage);
                    continue;
                }
                const long long cell = page * p.kv.page_stride + (i % p.kv.page_size) * p.kv.pos_stride +
                                       kvh * p.kv.head_stride;
                float s = 0.f;
                for (int u = 0; u < E; ++u)
                    if (lane + 32 * u < p.hd) s = fmaf(q[u], to_float(p.kv.k[cell + lane + 32 * u]), s);
                for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
                const float mn = fmaxf(m, s);
                if (mn == -INFINITY) continue;  // a score of -infinity has no weight
                const float keep = expf(m - mn), w = expf(s - mn);
                d = d * keep + w;
                for (int u = 0; u < E; ++u)
                    if (lane + 32 * u < p.hd) o[u] = o[u] * keep + w * to_float(p.kv.v[cell + lane + 32 * u]);
                m = mn;
            }
        }
    }
    for (int u = 0; u < E; ++u)
        if (lane + 32 * u < p.hd)
            p.out[t * p.out_stride + (long long)h * p.hd + lane + 32 * u] = from_float<T>(d > 0.f ? o[u] / d : o[u]);
    if (lane == 0 && p.lse) p.lse[row] = d > 0.f ? m + logf(d) : m;
}

template <typename T>
tf_status launch(tf_context* ctx, const AttnParams<T>& p, cudaStream_t cs, const char* name) {
    const long long rows = (long long)p.T_tokens * p.nq;
    attention_rows_kernel<T><<<(unsigned)((rows + 3) / 4), 128, 0, cs>>>(p);
    return cuda_check(ctx, cudaGetLastError(), name);
}

}  // namespace

extern "C" {

size_t tf_shared_prefix_attention_workspace_bytes(const tf_context* ctx, const tf_paged_kv* kv, uint32_t num_q_heads,
                                                  uint32_t T, uint32_t num_requests, uint32_t prefix_len,
                                                  uint32_t max_query) {
    if (!ctx || !kv) return 0;
    return 16;
}

tf_status tf_shared_prefix_attention(tf_context* ctx, const void* q, uint64_t q_stride, const tf_paged_kv* kv,
                                     const void* prefix_pages, uint32_t prefix_len, const void* page_table,
                                     uint32_t max_pages, const void* seq_lens, const void* token_starts,
                                     uint32_t num_requests, uint32_t max_query, uint32_t T, uint32_t num_q_heads,
                                     float scale, uint32_t window, void* out, uint64_t out_stride, void* lse,
                                     void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "tf_shared_prefix_attention";
    tf_status s = enter(ctx, name);
    if (s) return s;
    s = check_paged_kv(ctx, kv, name);
    if (s) return s;
    if (num_q_heads == 0 || num_q_heads % kv->num_kv_heads || num_q_heads > 0xFFFFu)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: query heads must be a multiple of the KV heads", name);
    if (!(scale > 0.f) || isinf(scale)) return fail(ctx, TF_ERR_INVALID_ARG, "%s: scale must be above 0", name);
    if (num_requests == 0 || max_pages == 0 || (T && max_query == 0))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: no requests, pages or queries", name);
    if ((uint64_t)prefix_len + (uint64_t)max_pages * kv->page_size > 0x7FFFFFFFull || num_requests > 0xFFFFFFu ||
        window > 0x7FFFFFFFu || max_query > 0x7FFFFFFFu || (uint64_t)T * num_q_heads > 0x7FFFFFFFull ||
        (uint64_t)num_requests * max_pages > 0x7FFFFFFFull)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: positions, rows and table entries must be below 2^31", name);
    if (T == 0) return TF_OK;
    if (!q || !page_table || !seq_lens || !token_starts || !out || !workspace || (prefix_len && !prefix_pages))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: null pointer", name);
    const uint64_t width = (uint64_t)num_q_heads * kv->head_dim;
    if (T > 1 && (q_stride < width || out_stride < width))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: token strides below the heads' width", name);
    if (!aligned16(q) || !aligned16(out) || q_stride % 8 || out_stride % 8 || !aligned4(prefix_pages) ||
        !aligned4(page_table) || !aligned4(seq_lens) || !aligned4(token_starts) || !aligned4(lse) ||
        !aligned16(workspace))
        return fail(ctx, TF_ERR_MISALIGNED, "%s: q, out and workspace 16-byte aligned, strides multiples of 8", name);
    const size_t need =
        tf_shared_prefix_attention_workspace_bytes(ctx, kv, num_q_heads, T, num_requests, prefix_len, max_query);
    if (workspace_bytes < need)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes, need);

    auto fill = [&](auto& p) {
        using T_ = std::remove_const_t<std::remove_pointer_t<decltype(p.q)>>;
        p.q = static_cast<const T_*>(q);
        p.q_stride = (long long)q_stride;
        p.kv = paged_view<T_>(kv);
        p.prefix_pages = static_cast<const int*>(prefix_pages);
        p.table = static_cast<const int*>(page_table);
        p.seq_lens = static_cast<const int*>(seq_lens);
        p.starts = static_cast<const int*>(token_starts);
        p.out = static_cast<T_*>(out);
        p.out_stride = (long long)out_stride;
        p.lse = static_cast<float*>(lse);
        p.err = ctx->d_err;
        p.prefix_len = (int)prefix_len;
        p.max_pages = (int)max_pages;
        p.B = (int)num_requests;
        p.max_query = (int)max_query;
        p.T_tokens = (int)T;
        p.nq = (int)num_q_heads;
        p.nkv = (int)kv->num_kv_heads;
        p.hd = (int)kv->head_dim;
        p.window = (int)window;
        p.scale = scale;
    };
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    if (kv->dtype == TF_DTYPE_F16) {
        AttnParams<__half> p;
        fill(p);
        return launch(ctx, p, cs, name);
    }
    AttnParams<__nv_bfloat16> p;
    fill(p);
    return launch(ctx, p, cs, name);
}

}  // extern "C"

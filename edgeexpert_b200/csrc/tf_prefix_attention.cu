// tf_prefix_attention.cu -- causal attention of a ragged batch behind a shared
// prefix, over a paged cache (tf_shared_prefix_attention).
//
// For a query row at position p, with the keys split in any way into parts i:
//   m_i = max s, d_i = sum e^(s - m_i), o_i = sum e^(s - m_i) v   over the part's visible keys,
//   M = max m_i, D = sum d_i e^(m_i - M), out = sum o_i e^(m_i - M) / D, lse = M + log D,
// so the shared prefix can be one part and the request's own pages another.
#include <math.h>

#include "tf_prefix_stream.cuh"
#include "tf_prefix_tensor.cuh"

using namespace tf;

namespace {

constexpr int kJoinWarps = 8;

// One warp, one row, key by key: the definition.  Only for rows whose joined
// result is not finite: an infinity or NaN in a key that the row does not see,
// but a neighbour in its tile does, reaches the tile's product as 0 * inf; here
// such a key is not read.
template <typename T>
__device__ void attend_alone(const AttnParams<T>& p, int b, const Request& r, int j, int h) {
    constexpr int E = kMaxPagedHeadDim / 32;
    const int lane = threadIdx.x & 31, kvh = h / p.G, t = r.start + j;
    float q[E], o[E], m = -INFINITY, d = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int e = lane + 32 * i;
        q[i] = e < p.hd ? to_float(p.q[t * p.q_stride + (long long)h * p.hd + e]) * p.scale : 0.f;
        o[i] = 0.f;
    }
    int lo, hi;
    seen_by(p, r, j, lo, hi);
    for (int pos = lo; pos < hi; ++pos) {
        const bool shared = pos < p.prefix_len;
        const int at = shared ? pos : pos - p.prefix_len, in_page = at / p.kv.page_size;
        const int page = shared ? p.prefix_pages[in_page] : p.table[(long long)b * p.max_pages + in_page];
        if (page < 0 || page >= p.kv.num_pages) continue;
        const long long cell = page * p.kv.page_stride + (at - in_page * p.kv.page_size) * p.kv.pos_stride +
                               kvh * p.kv.head_stride;
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < E; ++u)
            if (lane + 32 * u < p.hd) s = fmaf(q[u], to_float(p.kv.k[cell + lane + 32 * u]), s);
        for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float top = fmaxf(m, s);
        if (top == -INFINITY && s == s) continue;  // a score of -infinity has no weight
        const float keep = expf(m - top), w = expf(s - top);
        d = d * (m == -INFINITY ? 0.f : keep) + w;
#pragma unroll
        for (int u = 0; u < E; ++u)
            if (lane + 32 * u < p.hd)
                o[u] = o[u] * (m == -INFINITY ? 0.f : keep) + w * to_float(p.kv.v[cell + lane + 32 * u]);
        m = top;
    }
#pragma unroll
    for (int u = 0; u < E; ++u)
        if (lane + 32 * u < p.hd)
            p.out[t * p.out_stride + (long long)h * p.hd + lane + 32 * u] = from_float<T>(d == 0.f ? 0.f : o[u] / d);
    if (lane == 0 && p.lse) p.lse[(long long)t * p.nq + h] = d == 0.f ? -INFINITY : m + logf(d);
}

// The parts of one row, numbered.
struct RowParts {
    int n[4];             // first, cont of the stream kernel; first, cont of the tensor kernel
    long long place[4];   // row of the first of them
    int step[4];          // rows from one to the next
};

// Joins the parts of every row: one CTA per token, a warp per head.
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) join_parts_kernel(const __grid_constant__ AttnParams<T> p,
                                                                     int stream_keys) {
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    // most batches have one token a request, and then b = t
    int b = min(t, p.B - 1);
    if (!(p.starts[b] <= t && t < p.starts[b + 1])) b = request_at(p, t);
    Request r;
    int j = 0;
    bool live = b < p.B;
    if (live) {
        r = request_of(p, b);
        j = t - r.start;
        if (j >= r.used) {
            live = false;
            if (threadIdx.x == 0) atomicOr(p.err, kErrBadPage);
        }
    }
    const int prefix_tiles = (p.prefix_len - p.prefix_lo + stream_keys - 1) / stream_keys;
    const int SU = p.stream.base[p.B];
    for (int h = threadIdx.x >> 5; h < p.nq; h += kJoinWarps) {
        const int kvh = h / p.G, grow = t * p.G + h % p.G;
        const long long row = (long long)t * p.nq + h;
        T* out = p.out + t * p.out_stride + (long long)h * p.hd;
        if (!live) {
            for (int e = lane; e < p.hd; e += 32) out[e] = from_float<T>(0.f);
            if (lane == 0 && p.lse) p.lse[row] = -INFINITY;
            continue;
        }
        RowParts parts = {};
        auto add_stream = [&](int which, int unit, int tiles, int in_tile) {
            const int c0 = cta_of(unit, SU, p.stream.ctas), c1 = cta_of(unit + tiles - 1, SU, p.stream.ctas);
            parts.n[which] = 1;
            parts.place[which] = row;
            if (c1 > c0) {  // only one of a row's two stream jobs can be in a given cont place, but both may have some
                parts.n[which + 1] = c1 - c0;
                parts.place[which + 1] = (long long)(c0 + 1) * p.stream.rows + in_tile;
                parts.step[which + 1] = p.stream.rows;
            }
        };
        const int lo = own_lo(p, r), tiles = (r.len - lo + stream_keys - 1) / stream_keys;
        if (tiles > 0 && !by_tensor(p, r)) {
            const int rows = r.used * p.G, own = j * p.G + h % p.G, row_tiles = (rows + p.stream.rows - 1) / p.stream.rows;
            add_stream(0, p.stream.base[b] + (kvh * row_tiles + own / p.stream.rows) * tiles, tiles, own % p.stream.rows);
        }
        if (p.prefix_by_stream && prefix_tiles > 0) {
            const int rows = max(0, min(p.starts[p.B], p.T_tokens)) * p.G, row_tiles = (rows + p.stream.rows - 1) / p.stream.rows;
            add_stream(2, (kvh * row_tiles + grow / p.stream.rows) * prefix_tiles, prefix_tiles, grow % p.stream.rows);
        }
        if (p.tensor.ctas) {
            const int tile = grow / kTcRows, units = (p.tensor.base[tile + 1] - p.tensor.base[tile]) / p.nkv;
            if (units) {
                const int TU = p.tensor.base[(int)(((long long)p.T_tokens * p.G + kTcRows - 1) / kTcRows)];
                const int unit = p.tensor.base[tile] + kvh * units;
                const int c0 = cta_of(unit, TU, p.tensor.ctas), c1 = cta_of(unit + units - 1, TU, p.tensor.ctas);
                if (c0 == c1 && by_tensor(p, r)) {  // the tensor kernel has written the result
                    const float mark = p.tensor.first_md[row].x;
                    if (mark != mark) attend_alone(p, b, r, j, h);
                    continue;
                }
                parts.n[2] = 1;
                parts.place[2] = row;
                parts.n[3] = c1 - c0;
                parts.place[3] = (long long)(c0 + 1) * kTcRows + grow % kTcRows;
                parts.step[3] = kTcRows;
            }
        }
        const float* src[4] = {p.stream.first, p.stream.cont, p.tensor.first,
                               p.prefix_by_stream ? p.stream.cont : p.tensor.cont};
        const float2* src_md[4] = {p.stream.first_md, p.stream.cont_md, p.tensor.first_md,
                                   p.prefix_by_stream ? p.stream.cont_md : p.tensor.cont_md};
        // the largest maximum, then the weighted sums
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            for (int i = lane; i < parts.n[k]; i += 32) {
                const float2 md = src_md[k][parts.place[k] + (long long)i * parts.step[k]];
                top = md.x != md.x ? md.x : fmaxf(top, md.x);
            }
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float d = 0.f;
        float4 o[kMaxPagedHeadDim / 128];
#pragma unroll
        for (int u = 0; u < kMaxPagedHeadDim / 128; ++u) o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            for (int i = 0; i < parts.n[k]; ++i) {
                const long long at = parts.place[k] + (long long)i * parts.step[k];
                const float2 md = src_md[k][at];
                if (md.x == -INFINITY && md.y == 0.f) continue;
                const float w = exp2_approx(md.x - top);
                d = fmaf(md.y, w, d);
#pragma unroll
                for (int u = 0; u < kMaxPagedHeadDim / 128; ++u) {
                    const int e = u * 128 + lane * 4;
                    if (e >= p.hd) break;
                    const float4 x = *reinterpret_cast<const float4*>(src[k] + at * p.hd + e);
                    o[u].x = fmaf(x.x, w, o[u].x);
                    o[u].y = fmaf(x.y, w, o[u].y);
                    o[u].z = fmaf(x.z, w, o[u].z);
                    o[u].w = fmaf(x.w, w, o[u].w);
                }
            }
        const float inv = d == 0.f ? 0.f : 1.f / d;
        bool fine = isfinite(d);
#pragma unroll
        for (int u = 0; u < kMaxPagedHeadDim / 128; ++u) {
            o[u].x *= inv;
            o[u].y *= inv;
            o[u].z *= inv;
            o[u].w *= inv;
            fine &= isfinite(o[u].x) && isfinite(o[u].y) && isfinite(o[u].z) && isfinite(o[u].w);
        }
        if (!__all_sync(0xffffffffu, fine)) {
            attend_alone(p, b, r, j, h);
            continue;
        }
#pragma unroll
        for (int u = 0; u < kMaxPagedHeadDim / 128; ++u) {
            const int e = u * 128 + lane * 4;
            if (e >= p.hd) break;
            *reinterpret_cast<uint2*>(out + e) = make_uint2(Pair<T>::pack(o[u].x, o[u].y), Pair<T>::pack(o[u].z, o[u].w));
        }
        if (lane == 0 && p.lse) p.lse[row] = d == 0.f ? -INFINITY : (top + log2f(d)) * kLn2;
    }
}

// ---- sizes and the workspace ---------------------------------------------------------
// Rows up to which a request (or the whole batch, for the prefix) is the stream kernel's.
constexpr int kFewRows = 32;

struct Shape {
    int hd, tensor_above, nt, stream_keys, stream_rows, stream_ctas, tensor_ctas;
    bool prefix_by_stream;
};

template <int HD, int NT>
void stream_shape(const tf_context* ctx, Shape& s) {
    using S = StreamShape<HD, NT>;
    s.hd = HD;
    s.nt = NT;
    s.stream_keys = S::kKeys;
    s.stream_rows = S::kRows;
    const size_t per_sm = (size_t)ctx->max_smem_optin / (S::kSmem + 1024);
    s.stream_ctas = ctx->num_sms * (int)std::max<size_t>(1, std::min<size_t>(S::kCtas, per_sm));
}

// Column tiles for `rows` query rows of a job: one up to eight rows, beyond
// that as many as a warp's registers hold (512 / head_dim).
Shape shape_for(const tf_context* ctx, uint32_t hd, long long rows) {
    Shape s = {};
    const bool few = rows <= 8;
    if (hd <= 64)
        few ? stream_shape<64, 1>(ctx, s) : stream_shape<64, 4>(ctx, s);
    else if (hd <= 128)
        few ? stream_shape<128, 1>(ctx, s) : stream_shape<128, 4>(ctx, s);
    else if (hd <= 256)
        few ? stream_shape<256, 1>(ctx, s) : stream_shape<256, 2>(ctx, s);
    else
        stream_shape<512, 1>(ctx, s);
    return s;
}

Shape shape_of_call(const tf_context* ctx, const tf_paged_kv* kv, uint32_t nq, uint32_t T, uint32_t prefix_len,
                    uint32_t max_query) {
    const long long G = nq / kv->num_kv_heads;
    const long long own = std::min<long long>(max_query, T) * G;
    Shape s = shape_for(ctx, kv->head_dim, own);
    const bool tensor = kv->head_dim <= 256;
    s.prefix_by_stream = !tensor || T * G <= kFewRows;
    // nothing for the tensor cores: no prefix of theirs and no request with many rows
    const bool used = tensor && ((prefix_len && !s.prefix_by_stream) || own > kFewRows);
    s.tensor_above = tensor ? kFewRows : 0x7FFFFFFF;
    s.tensor_ctas = used ? ctx->num_sms : 0;
    return s;
}

struct Layout {
    size_t first[2], first_md[2], cont[2], cont_md[2], base[2], bytes;
};

Layout layout_of(const tf_context* ctx, const tf_paged_kv* kv, uint32_t nq, uint32_t T, uint32_t B, const Shape& s) {
    Layout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    };
    const size_t rows = (size_t)T * nq, G = nq / kv->num_kv_heads;
    // either kernel's grid and tile may be smaller in a call, never larger
    const size_t cont[2] = {(size_t)ctx->num_sms * 2 * 64, (size_t)ctx->num_sms * kTcRows};
    const size_t bases[2] = {B + 1, (size_t)T * G / kTcRows + 2};
    for (int k = 0; k < 2; ++k) {
        l.base[k] = take(bases[k] * sizeof(int));
        l.first_md[k] = take(rows * sizeof(float2));
        l.cont_md[k] = take(cont[k] * sizeof(float2));
        l.first[k] = take(rows * kv->head_dim * sizeof(float));
        l.cont[k] = take(cont[k] * kv->head_dim * sizeof(float));
    }
    l.bytes = at;
    return l;
}

template <typename T, int HD, int NT>
tf_status launch_stream(tf_context* ctx, const AttnParams<T>& p, cudaStream_t cs, const char* name) {
    using S = StreamShape<HD, NT>;
    static bool configured[64] = {};  // per instantiation, per device
    const int dev = ctx->device & 63;
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(attention_few_rows_kernel<T, HD, NT>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
        if (e != cudaSuccess) return cuda_check(ctx, e, name);
        configured[dev] = true;
    }
    attention_few_rows_kernel<T, HD, NT><<<p.stream.ctas, S::kWarps * 32, S::kSmem, cs>>>(p);
    return cuda_check(ctx, cudaGetLastError(), name);
}

template <typename T, int HD>
tf_status launch_tensor(tf_context* ctx, const AttnParams<T>& p, cudaStream_t cs, const char* name) {
    using S = TensorShape<HD>;
    static bool configured[64] = {};  // per instantiation, per device
    const int dev = ctx->device & 63;
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(attention_many_rows_kernel<T, HD>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
        if (e != cudaSuccess) return cuda_check(ctx, e, name);
        configured[dev] = true;
    }
    attention_many_rows_kernel<T, HD><<<p.tensor.ctas, S::kThreads, S::kSmem, cs>>>(p);
    return cuda_check(ctx, cudaGetLastError(), name);
}

template <typename T>
tf_status launch(tf_context* ctx, const AttnParams<T>& p, const Shape& s, cudaStream_t cs, const char* name) {
    tf_status st = TF_OK;
    if (s.tensor_ctas) {
        st = s.hd == 64    ? launch_tensor<T, 64>(ctx, p, cs, name)
             : s.hd == 128 ? launch_tensor<T, 128>(ctx, p, cs, name)
                           : launch_tensor<T, 256>(ctx, p, cs, name);
        if (st) return st;
    }
    if (s.hd == 64)
        st = s.nt == 1 ? launch_stream<T, 64, 1>(ctx, p, cs, name) : launch_stream<T, 64, 4>(ctx, p, cs, name);
    else if (s.hd == 128)
        st = s.nt == 1 ? launch_stream<T, 128, 1>(ctx, p, cs, name) : launch_stream<T, 128, 4>(ctx, p, cs, name);
    else if (s.hd == 256)
        st = s.nt == 1 ? launch_stream<T, 256, 1>(ctx, p, cs, name) : launch_stream<T, 256, 2>(ctx, p, cs, name);
    else
        st = launch_stream<T, 512, 1>(ctx, p, cs, name);
    if (st) return st;
    join_parts_kernel<T><<<p.T_tokens, kJoinWarps * 32, 0, cs>>>(p, s.stream_keys);
    return cuda_check(ctx, cudaGetLastError(), name);
}

}  // namespace

extern "C" {

size_t tf_shared_prefix_attention_workspace_bytes(const tf_context* ctx, const tf_paged_kv* kv, uint32_t num_q_heads,
                                                  uint32_t T, uint32_t num_requests, uint32_t prefix_len,
                                                  uint32_t max_query) {
    if (!ctx || !kv || kv->num_kv_heads == 0 || num_q_heads == 0 || num_q_heads % kv->num_kv_heads) return 0;
    const Shape shape = shape_of_call(ctx, kv, num_q_heads, T, prefix_len, max_query);
    return layout_of(ctx, kv, num_q_heads, T, num_requests, shape).bytes;
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
    const uint64_t G = num_q_heads / kv->num_kv_heads;
    const Shape shape = shape_of_call(ctx, kv, num_q_heads, T, prefix_len, max_query);
    const uint64_t row_tiles = std::min<uint64_t>(max_query, T) * G / shape.stream_rows + num_requests;
    const uint64_t keys = (uint64_t)max_pages * kv->page_size / shape.stream_keys + 1;
    if (row_tiles * keys * kv->num_kv_heads > 0x7FFFFFFFull ||
        (T * G / shape.stream_rows + 1) * (prefix_len / shape.stream_keys + 1) * kv->num_kv_heads > 0x3FFFFFFFull)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: too many key tiles", name);
    const Layout l = layout_of(ctx, kv, num_q_heads, T, num_requests, shape);
    const size_t need = l.bytes;
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
        p.G = (int)G;
        p.window = (int)window;
        p.scale = scale;
        // no row stands before prefix_len - max_query
        p.prefix_lo = window ? (int)std::max<long long>(0, std::min<long long>(prefix_len, (long long)prefix_len -
                                                                                              max_query - window + 1))
                             : 0;
        p.prefix_by_stream = shape.prefix_by_stream;
        p.tensor_above = shape.tensor_above;
        uint8_t* w = static_cast<uint8_t*>(workspace);
        Parts* parts[2] = {&p.stream, &p.tensor};
        for (int k = 0; k < 2; ++k) {
            parts[k]->first = reinterpret_cast<float*>(w + l.first[k]);
            parts[k]->first_md = reinterpret_cast<float2*>(w + l.first_md[k]);
            parts[k]->cont = reinterpret_cast<float*>(w + l.cont[k]);
            parts[k]->cont_md = reinterpret_cast<float2*>(w + l.cont_md[k]);
            parts[k]->base = reinterpret_cast<int*>(w + l.base[k]);
        }
        p.stream.ctas = shape.stream_ctas;
        p.stream.rows = shape.stream_rows;
        p.tensor.ctas = shape.tensor_ctas;
        p.tensor.rows = kTcRows;
    };
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    if (kv->dtype == TF_DTYPE_F16) {
        AttnParams<__half> p;
        fill(p);
        return launch(ctx, p, shape, cs, name);
    }
    AttnParams<__nv_bfloat16> p;
    fill(p);
    return launch(ctx, p, shape, cs, name);
}

}  // extern "C"

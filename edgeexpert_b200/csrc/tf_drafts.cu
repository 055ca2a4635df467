// tf_drafts.cu -- the trees of drafted tokens in a ragged batch:
//   tf_draft_tree_plan   parents -> positions and ancestor bits of every node
//   tf_draft_accept      the walk down each tree along the chosen tokens; K and V of the
//                        nodes that are kept moved behind the history, in every layer
#include "tf_paged.cuh"

using namespace tf;

namespace {

// A request's nodes: tokens [start, start + n), `used` of them within max_query.
struct Tree {
    int start, n, used;
};
__device__ __forceinline__ Tree tree_of(const int* starts, int b, int T, int max_query, uint32_t* err) {
    Tree t;
    t.start = max(0, min(starts[b], T));
    t.n = max(t.start, min(starts[b + 1], T)) - t.start;
    t.used = min(t.n, max_query);
    if (t.n > t.used && threadIdx.x == 0) atomicOr(err, kErrBadTree);
    return t;
}

// ---- positions and ancestors -----------------------------------------------------
struct PlanParams {
    const int* parents;
    const int* seq_lens;
    const int* starts;
    int* positions;
    uint32_t* ancestors;
    uint32_t* err;
    int B, T, max_query, words, base;
};

// One CTA a request, one thread a node.  With up(i) a node that i's bits do not go
// beyond yet, bits(i) |= bits(up(i)), up(i) = up(up(i)) doubles the length of way
// covered, so a tree of 256 takes eight steps at most, whatever its shape; the depth
// is the number of bits.  Bound by its launch: 1.7 us for one tree of 12, 2.2 us for 301
// of up to 64, one after another in a graph.
template <int W>
__global__ void __launch_bounds__(W * 32) tree_plan_kernel(const PlanParams p) {
    __shared__ uint32_t bits[W * 32][W];
    __shared__ int up[W * 32];
    griddep_wait();
    griddep_launch_dependents();
    const int i = threadIdx.x, b = blockIdx.x;
    const Tree t = tree_of(p.starts, b, p.T, p.max_query, p.err);
    const bool node = i < t.used;
    int parent = node ? p.parents[t.start + i] : -1;
    if (parent < -1 || parent >= i) {
        if (node) atomicOr(p.err, kErrBadTree);
        parent = -1;
    }
    uint32_t mine[W];
#pragma unroll
    for (int w = 0; w < W; ++w) bits[i][w] = mine[w] = node && i / 32 == w ? 1u << (i & 31) : 0u;
    up[i] = parent;
    for (;;) {
        __syncthreads();
        uint32_t more[W];
        int next = -1;
        if (parent >= 0) {
            next = up[parent];
#pragma unroll
            for (int w = 0; w < W; ++w) more[w] = bits[parent][w];
        }
        if (!__syncthreads_or(parent >= 0)) break;
        if (parent >= 0) {
#pragma unroll
            for (int w = 0; w < W; ++w) bits[i][w] = mine[w] |= more[w];
            up[i] = parent = next;
        }
    }
    const int history = max(0, max(0, p.seq_lens[b]) - t.n);
    for (int j = i; j < t.n; j += W * 32) {
        const bool known = j == i && node;
        int depth = -1;
#pragma unroll
        for (int w = 0; w < W; ++w) depth += __popc(mine[w]);
        p.positions[t.start + j] = known ? p.base + history + depth : -1;
        uint32_t* to = p.ancestors + (long long)(t.start + j) * p.words;
#pragma unroll
        for (int w = 0; w < W; ++w)
            if (w < p.words) to[w] = known ? mine[w] : 0u;
        for (int w = W; w < p.words; ++w) to[w] = 0u;
    }
    // rows of no request
    const int first = max(0, min(p.starts[0], p.T)), last = max(first, min(p.starts[p.B], p.T));
    const int none = first + p.T - last;
    for (int k = b * blockDim.x + i; k < none; k += gridDim.x * blockDim.x) {
        const int r = k < first ? k : last + k - first;
        p.positions[r] = -1;
        for (int w = 0; w < p.words; ++w) p.ancestors[(long long)r * p.words + w] = 0u;
    }
}

// ---- acceptance ------------------------------------------------------------------
constexpr int kMaxNodes = 256;
constexpr int kAcceptThreads = 256;  // a thread a node

struct AcceptParams {
    const int* token_ids;
    const int* parents;
    const int* choices;
    const int* given;
    const int* seq_lens;
    const int* starts;
    const int* table;
    int* counts;
    int* paths;
    int* tokens;
    int* targets;
    uint32_t* err;
    PagedView<uint16_t> kv;  // of the first layer, whatever its 16-bit type
    long long layer_stride;
    int layers, nkv, hd, max_pages, B, T, max_query, parts;
};

// parts CTAs a request; each walks the tree by itself (a launch for the walk alone would
// cost more), the first writes the lists, all move their share of the columns: 16 bytes
// of a head of K and V in a layer.  The kept nodes path[0] < path[1] < ... go from
// position path[k] to k of the request's own.  A thread takes its column's moves in order
// and loads a few before it stores the first: what a store overwrites (k) is the source
// of an earlier move than any that is still to be loaded (path[j] >= j > k).
// One tree of 12 in 30 layers: 2.8 us, latency; 32 of 8 to 24, 42 MB in and out of L2: 6.8 us,
// 6.2 TB/s (one after another in a graph).
__global__ void __launch_bounds__(kAcceptThreads) accept_kernel(const __grid_constant__ AcceptParams p) {
    __shared__ int s_next[kMaxNodes], s_path[kMaxNodes], s_choice[kMaxNodes], s_count, s_same;
    __shared__ long long s_from[kMaxNodes], s_to[kMaxNodes];
    griddep_wait();
    griddep_launch_dependents();
    const int i = threadIdx.x, b = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    const Tree t = tree_of(p.starts, b, p.T, p.max_query, p.err);
    const int history = max(0, p.seq_lens[b]) - t.n;
    const int given = p.given ? max(1, min(p.given[b], t.used)) : 1;
    const bool node = i < t.used;
    const int parent = node ? p.parents[t.start + i] : -1;
    const int token = node ? p.token_ids[t.start + i] : 0;
    s_choice[i] = node ? p.choices[t.start + i] : 0;
    s_next[i] = kMaxNodes;
    s_path[i] = i;  // (the given ones' place)
    __syncthreads();
    if (node && i >= given) {
        if (parent < -1 || parent >= i)
            atomicOr(p.err, kErrBadTree);
        else if (parent >= given - 1 && token == s_choice[parent] && token >= 0)
            atomicMin(&s_next[parent], i);
    }
    __syncthreads();
    if (i == 0) {
        int count = 0, same = 0;  // of the leading nodes that stay where they are
        if (t.used) {
            count = given;
            for (int at = s_next[given - 1]; at < kMaxNodes; at = s_next[at]) s_path[count++] = at;
            for (same = given; same < count && s_path[same] == same;) ++same;
        }
        s_count = count;
        s_same = same;
    }
    __syncthreads();
    const int count = s_count, same = s_same;
    if (part == 0) {
        for (int k = i; k < p.max_query; k += kAcceptThreads) {
            const long long at = (long long)b * p.max_query + k;
            p.paths[at] = k < count ? s_path[k] : -1;
            p.tokens[at] = k < count - given + 1 && count ? s_choice[s_path[k + given - 1]] : -1;
        }
        if (i == 0) {
            p.counts[b] = count;
            p.targets[b] = count ? history + count : -1;
        }
    }
    if (p.layers && same + i < count) {
        const int ps = p.kv.page_size;
        auto cell = [&](int pos) {
            if (pos < 0 || pos >= (long long)p.max_pages * ps) return -1ll;
            const int page = p.table[(long long)b * p.max_pages + pos / ps];
            if (page < 0 || page >= p.kv.num_pages) return -1ll;
            return page * p.kv.page_stride + pos % ps * p.kv.pos_stride;
        };
        const long long from = cell(history + s_path[same + i]), to = cell(history + same + i);
        const bool ok = from >= 0 && to >= 0;
        if (!ok) atomicOr(p.err, kErrBadPage);
        s_from[i] = ok ? from : 0;
        s_to[i] = ok ? to : -1;
    }
    __syncthreads();
    const int moves = p.layers ? count - same : 0;
    if (moves <= 0) return;
    const int chunks = p.hd / 8, per_layer = p.nkv * chunks;
    const long long columns = (long long)p.layers * per_layer;
    for (long long c = (long long)part * kAcceptThreads + i; c < columns; c += (long long)p.parts * kAcceptThreads) {
        const int layer = (int)(c / per_layer), in = (int)(c - (long long)layer * per_layer), head = in / chunks;
        const long long at = layer * p.layer_stride + head * p.kv.head_stride + (in - head * chunks) * 8;
        uint16_t* const k = p.kv.k + at;
        uint16_t* const v = p.kv.v + at;
        constexpr int kFly = 4;
        for (int m0 = 0; m0 < moves; m0 += kFly) {
            uint4 x[kFly], y[kFly];
#pragma unroll
            for (int m = 0; m < kFly; ++m)
                if (m0 + m < moves) {
                    x[m] = *reinterpret_cast<const uint4*>(k + s_from[m0 + m]);
                    y[m] = *reinterpret_cast<const uint4*>(v + s_from[m0 + m]);
                }
#pragma unroll
            for (int m = 0; m < kFly; ++m)
                if (m0 + m < moves && s_to[m0 + m] >= 0) {
                    *reinterpret_cast<uint4*>(k + s_to[m0 + m]) = x[m];
                    *reinterpret_cast<uint4*>(v + s_to[m0 + m]) = y[m];
                }
        }
    }
}

}  // namespace

extern "C" {

tf_status tf_draft_tree_plan(tf_context* ctx, const void* parents, const void* seq_lens, const void* token_starts,
                             uint32_t num_requests, uint32_t max_query, uint32_t T, uint32_t position_base,
                             void* positions, void* ancestors, uint32_t words, void* stream) {
    const char* name = "tf_draft_tree_plan";
    tf_status s = enter(ctx, name);
    if (s) return s;
    if (num_requests == 0 || max_query == 0)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: no requests or nodes", name);
    if (max_query > (uint32_t)kMaxNodes || num_requests > 0xFFFFFFu || T > 0x7FFFFFu || position_base > 0x7FFFFFFFu)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: trees of up to %d nodes, 2^24 requests, 2^23 tokens", name, kMaxNodes);
    if (words > 0xFFFFu || words * 32 < max_query)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: %u words hold no bits of %u nodes", name, words, max_query);
    if (T == 0) return TF_OK;
    const void* all[] = {parents, seq_lens, token_starts, positions, ancestors};
    for (const void* ptr : all) {
        if (!ptr) return fail(ctx, TF_ERR_INVALID_ARG, "%s: null pointer", name);
        if (!aligned4(ptr)) return fail(ctx, TF_ERR_MISALIGNED, "%s: pointers must be 4-byte aligned", name);
    }
    PlanParams p;
    p.parents = static_cast<const int*>(parents);
    p.seq_lens = static_cast<const int*>(seq_lens);
    p.starts = static_cast<const int*>(token_starts);
    p.positions = static_cast<int*>(positions);
    p.ancestors = static_cast<uint32_t*>(ancestors);
    p.err = ctx->d_err;
    p.B = (int)num_requests;
    p.T = (int)T;
    p.max_query = (int)max_query;
    p.words = (int)words;
    p.base = (int)position_base;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    const unsigned B = num_requests;
    cudaError_t e;
    if (max_query <= 32)
        e = launch_overlapped(tree_plan_kernel<1>, B, 32, 0, cs, p);
    else if (max_query <= 64)
        e = launch_overlapped(tree_plan_kernel<2>, B, 64, 0, cs, p);
    else if (max_query <= 128)
        e = launch_overlapped(tree_plan_kernel<4>, B, 128, 0, cs, p);
    else
        e = launch_overlapped(tree_plan_kernel<8>, B, 256, 0, cs, p);
    return cuda_check(ctx, e, name);
}

tf_status tf_draft_accept(tf_context* ctx, const void* token_ids, const void* parents, const void* choices,
                          const void* given, const void* seq_lens, const void* token_starts, uint32_t num_requests,
                          uint32_t max_query, uint32_t T, void* counts, void* paths, void* tokens, void* targets,
                          const tf_paged_kv* kv, uint64_t layer_stride, uint32_t num_layers, const void* page_table,
                          uint32_t max_pages, void* stream) {
    const char* name = "tf_draft_accept";
    tf_status s = enter(ctx, name);
    if (s) return s;
    if (num_requests == 0 || max_query == 0)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: no requests or nodes", name);
    if (max_query > (uint32_t)kMaxNodes || num_requests > 0xFFFFFFu || T > 0x7FFFFFu || num_layers > 0xFFFFu)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: trees of up to %d nodes, 2^24 requests, 2^23 tokens, 2^16 layers",
                    name, kMaxNodes);
    AcceptParams p = {};
    if (num_layers) {
        s = check_paged_kv(ctx, kv, name);
        if (s) return s;
        if (!page_table || max_pages == 0)
            return fail(ctx, TF_ERR_INVALID_ARG, "%s: no page table", name);
        if (layer_stride % 8 || !aligned4(page_table))
            return fail(ctx, TF_ERR_MISALIGNED, "%s: layer stride a multiple of 8, page table 4-byte aligned", name);
        if (num_layers > 1 && layer_stride < kv->head_dim)
            return fail(ctx, TF_ERR_INVALID_ARG, "%s: layer stride below head_dim", name);
        if ((uint64_t)num_requests * max_pages > 0x7FFFFFFFull || (uint64_t)max_pages * kv->page_size > 0x7FFFFFFFull)
            return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: positions and table entries must be below 2^31", name);
        p.kv = paged_view<uint16_t>(kv);
        p.nkv = (int)kv->num_kv_heads;
        p.hd = (int)kv->head_dim;
        p.table = static_cast<const int*>(page_table);
        p.max_pages = (int)max_pages;
        p.layers = (int)num_layers;
        p.layer_stride = (long long)layer_stride;
    }
    const void* all[] = {seq_lens, token_starts, counts, paths, tokens, targets};
    for (const void* ptr : all) {
        if (!ptr) return fail(ctx, TF_ERR_INVALID_ARG, "%s: null pointer", name);
        if (!aligned4(ptr)) return fail(ctx, TF_ERR_MISALIGNED, "%s: pointers must be 4-byte aligned", name);
    }
    if (T && (!token_ids || !parents || !choices)) return fail(ctx, TF_ERR_INVALID_ARG, "%s: null pointer", name);
    if (!aligned4(token_ids) || !aligned4(parents) || !aligned4(choices) || !aligned4(given))
        return fail(ctx, TF_ERR_MISALIGNED, "%s: pointers must be 4-byte aligned", name);
    p.token_ids = static_cast<const int*>(token_ids);
    p.parents = static_cast<const int*>(parents);
    p.choices = static_cast<const int*>(choices);
    p.given = static_cast<const int*>(given);
    p.seq_lens = static_cast<const int*>(seq_lens);
    p.starts = static_cast<const int*>(token_starts);
    p.counts = static_cast<int*>(counts);
    p.paths = static_cast<int*>(paths);
    p.tokens = static_cast<int*>(tokens);
    p.targets = static_cast<int*>(targets);
    p.err = ctx->d_err;
    p.B = (int)num_requests;
    p.T = (int)T;
    p.max_query = (int)max_query;
    // a column a thread, in as many CTAs as are resident at once
    const long long columns = (long long)p.layers * p.nkv * (p.hd / 8);
    const long long fit = std::max<long long>(1, 8ll * ctx->num_sms / num_requests);
    p.parts = (int)std::max<long long>(1, std::min(fit, (columns + kAcceptThreads - 1) / kAcceptThreads));
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    return cuda_check(ctx, launch_overlapped(accept_kernel, num_requests * (unsigned)p.parts, kAcceptThreads, 0, cs, p), name);
}

}  // extern "C"

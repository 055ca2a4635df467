// tf_logit_rules.cu -- penalties for repeated tokens, biases and grammar masks on the
// logits of a ragged batch, and the token that is best under them (tf_logit_rules_apply).
//
// For a row of request b, with c = how often a token was said (in the output and on the
// row's way through its drafted tree) and `known` = said or in the prompt:
//   z = logit;  known: z = z > 0 ? z / repetition : z * repetition;
//   z -= frequency * c;  c > 0: z -= presence;  z += bias;  not allowed: -infinity.
// Each step is rounded to fp32 by itself (no contraction), so what a user computes with
// the same steps has the same bits.
#include "tf_paged.cuh"

using namespace tf;

namespace {

constexpr int kThreads = 256;
constexpr int kRowGroup = 8;  // rows of a request that share a CTA's tables
constexpr uint32_t kInPrompt = 0x80000000u, kDrafted = 0x40000000u, kCount = 0x3FFFFFFFu;
constexpr int kMaxNodes = 256;

struct RulesParams {
    const void* logits;
    void* out;
    long long logits_stride, out_stride;
    const int* starts;
    const int* history;
    long long history_stride;
    const int* history_lens;
    const int* prompt_lens;
    const float* repetition;
    const float* presence;
    const float* frequency;
    const int* bias_starts;
    const int* bias_tokens;
    const float* bias_values;
    const uint32_t* allowed;
    long long allowed_stride;
    const int* allowed_rows;
    const int* token_ids;
    const uint32_t* ancestors;
    int* tokens;
    unsigned long long* best;  // [T][chunks]
    uint32_t* err;
    int V, T, B, max_query, max_history, bias_count, allowed_count, words, chunk, chunks;
};

// Larger for a larger value, then for a lower token; 0: nothing above -infinity.
__device__ __forceinline__ unsigned long long best_key(float z, int token) {
    uint32_t u = __float_as_uint(z);
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    return z > -INFINITY ? (unsigned long long)u << 32 | (0xFFFFFFFFu - (uint32_t)token) : 0ull;
}

template <typename T>
struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    T e[N];
};
__device__ __forceinline__ float to_float(float v) { return v; }

// What is said of the chunk's tokens.
struct Tables {
    uint32_t* said;   // count, kInPrompt, kDrafted
    int* bias;        // 1 + the entry that counts, 0: none
    uint32_t* known;  // a bit for every token that has either
    int* drafted;     // the request's nodes
};

template <typename T>
struct RowRules {
    const RulesParams& p;
    const Tables& t;
    int c0, nodes;
    float rep, pres, freq;
    const uint32_t* way;  // ancestor bits of the row

    __device__ __forceinline__ float apply(float z, int e) const {
        const uint32_t word = t.said[e - c0];
        int count = (int)(word & kCount);
        if (word & kDrafted)
            for (int w = 0; w * 32 < nodes; ++w)
                for (uint32_t m = way[w]; m; m &= m - 1) {
                    const int i = w * 32 + __ffs(m) - 1;
                    if (i < nodes) count += t.drafted[i] == e;
                }
        if (count || (word & kInPrompt)) z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
        z = __fsub_rn(z, __fmul_rn(freq, (float)count));
        if (count) z = __fsub_rn(z, pres);
        if (p.bias_count) {
            const int entry = t.bias[e - c0];
            if (entry) z = __fadd_rn(z, p.bias_values[entry - 1]);
        }
        return z;
    }
};

__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T>
__global__ void __launch_bounds__(kThreads) logit_rules_kernel(const __grid_constant__ RulesParams p) {
    extern __shared__ uint32_t smem[];
    __shared__ unsigned long long s_best[kRowGroup][kThreads / 32];
    __shared__ int s_drafted[kMaxNodes];
    griddep_wait();
    griddep_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c0 = blockIdx.x * p.chunk, c1 = min(p.V, c0 + p.chunk), b = blockIdx.y;
    const int start = max(0, min(p.starts[b], p.T)), n = max(start, min(p.starts[b + 1], p.T)) - start;
    const int used = min(n, p.max_query), r0 = blockIdx.z * kRowGroup, r1 = min(used, r0 + kRowGroup);
    if (n > used && blockIdx.x == 0 && r0 == 0 && tid == 0) atomicOr(p.err, kErrBadTree);
    if (r0 >= r1) return;

    // ---- what is said of this chunk's tokens ------------------------------------------
    Tables t;
    t.said = smem;
    t.known = smem + p.chunk;
    t.bias = reinterpret_cast<int*>(t.known + p.chunk / 32);
    t.drafted = s_drafted;
    for (int i = tid; i < p.chunk; i += kThreads) {
        t.said[i] = 0u;
        if (p.bias_count) t.bias[i] = 0;
    }
    const int nodes = p.token_ids ? min(used, p.words * 32) : 0;
    __syncthreads();
    // The token's place in the chunk; false where it is in another, or in none.  (Unsigned: ids may be
    // anything, and a difference that overflows an int may pass both comparisons with its bounds.)
    const uint32_t here = (uint32_t)(c1 - c0);
    auto place = [&](int token, uint32_t& e) { return (e = (uint32_t)token - (uint32_t)c0) < here; };
    uint32_t e;
    const int len = p.history ? max(0, min(p.history_lens[b], p.max_history)) : 0;
    const int prompt = p.history && p.prompt_lens ? p.prompt_lens[b] : 0;
    const int* said = p.history + b * p.history_stride;
    for (int i = tid; i < len; i += kThreads) {
        if (!place(said[i], e)) continue;
        if (i < prompt)
            atomicOr(&t.said[e], kInPrompt);
        else
            atomicAdd(&t.said[e], 1u);
    }
    if (p.bias_count) {
        const int b0 = max(0, min(p.bias_starts[b], p.bias_count)), b1 = min(p.bias_starts[b + 1], p.bias_count);
        for (int i = b0 + tid; i < b1; i += kThreads) {
            if (place(p.bias_tokens[i], e)) atomicMax(&t.bias[e], i + 1);  // the last entry of a token counts
        }
    }
    for (int i = tid; i < nodes; i += kThreads) {
        const int token = p.token_ids[start + i];
        s_drafted[i] = token;
        if (place(token, e)) atomicOr(&t.said[e], kDrafted);
    }
    __syncthreads();
    for (int w = warp; w < p.chunk / 32; w += kThreads / 32) {
        const uint32_t any = __ballot_sync(0xffffffffu, t.said[w * 32 + lane] != 0u || (p.bias_count && t.bias[w * 32 + lane]));
        if (lane == 0) t.known[w] = any;
    }
    __syncthreads();

    // ---- rows ----------------------------------------------------------------------------
    RowRules<T> rules{p, t, c0, nodes, p.repetition ? p.repetition[b] : 1.f, p.presence ? p.presence[b] : 0.f,
                      p.frequency ? p.frequency[b] : 0.f, nullptr};
    for (int r = r0; r < r1; ++r) {
        const int row = start + r;
        const T* in = static_cast<const T*>(p.logits) + row * p.logits_stride;
        T* out = static_cast<T*>(p.out) + row * p.out_stride;
        rules.way = p.ancestors + (long long)row * p.words;
        const uint32_t* allowed = nullptr;
        if (p.allowed) {
            const int at = p.allowed_rows ? p.allowed_rows[row] : row;
            if (at >= p.allowed_count) {
                if (tid == 0) atomicOr(p.err, kErrBadTree);
            } else if (at >= 0) {
                allowed = p.allowed + at * p.allowed_stride;
            }
        }
        unsigned long long best = 0ull;
        for (int e = c0 + tid; e < c1; e += kThreads) {
            float z = to_float(in[e]);
            if (t.known[(e - c0) >> 5] >> (e & 31) & 1u) z = rules.apply(z, e);
            if (allowed && !(allowed[e >> 5] >> (e & 31) & 1u)) z = -INFINITY;
            store(out + e, z);
            const unsigned long long k = best_key(z, e);
            best = k > best ? k : best;
        }
        for (int o = 16; o; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        if (lane == 0) s_best[r - r0][warp] = best;
    }
    if (!p.tokens) return;
    __syncthreads();
    if (tid < r1 - r0) {
        unsigned long long best = 0ull;
        for (int w = 0; w < kThreads / 32; ++w) best = max(best, s_best[tid][w]);
        p.best[(long long)(start + r0 + tid) * p.chunks + blockIdx.x] = best;
    }
}

// A warp a row: the best of its chunks.
__global__ void __launch_bounds__(kThreads) best_token_kernel(const __grid_constant__ RulesParams p) {
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, b = blockIdx.x;
    const int start = max(0, min(p.starts[b], p.T)), n = max(start, min(p.starts[b + 1], p.T)) - start;
    for (int r = threadIdx.x >> 5; r < min(n, p.max_query); r += kThreads / 32) {
        unsigned long long best = 0ull;
        for (int c = lane; c < p.chunks; c += 32) best = max(best, p.best[(long long)(start + r) * p.chunks + c]);
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) p.tokens[start + r] = best ? (int)(0xFFFFFFFFu - (uint32_t)best) : -1;
    }
}

constexpr int kChunk = 4096;
inline int chunks_of(uint32_t V) { return (int)(((uint64_t)V + kChunk - 1) / kChunk); }

template <typename T>
cudaError_t launch(const RulesParams& p, cudaStream_t cs) {
    const size_t smem = p.chunk * 4 + p.chunk / 8 + (p.bias_count ? p.chunk * 4 : 0);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.chunks, (unsigned)p.B, (unsigned)((p.max_query + kRowGroup - 1) / kRowGroup));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = cs;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dependent_launches() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, logit_rules_kernel<T>, p);
}

}  // namespace

extern "C" {

size_t tf_logit_rules_workspace_bytes(uint32_t T, uint32_t V) {
    return std::max<size_t>(16, (size_t)T * chunks_of(V) * sizeof(unsigned long long));
}

tf_status tf_logit_rules_apply(tf_context* ctx, const void* logits, uint64_t logits_stride, void* out,
                               uint64_t out_stride, tf_dtype dtype, uint32_t V, uint32_t T, const void* token_starts,
                               uint32_t num_requests, uint32_t max_query, const tf_logit_rules* rules, void* tokens,
                               void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "tf_logit_rules_apply";
    tf_status s = enter(ctx, name);
    if (s) return s;
    if (!rules) return fail(ctx, TF_ERR_INVALID_ARG, "%s: no rules", name);
    if (dtype != TF_DTYPE_F16 && dtype != TF_DTYPE_BF16 && dtype != TF_DTYPE_F32)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: unknown dtype", name);
    if (num_requests == 0 || V == 0 || (T && max_query == 0))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: no requests, tokens or rows", name);
    max_query = std::min(max_query, T);
    if (V > 0x7FFFF000u || T > 0x7FFFFFu || num_requests > 0xFFFFu || max_query > 0xFFFFu * kRowGroup)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: fewer than 2^31 tokens, 2^23 rows, 2^16 requests", name);
    if (T == 0) return TF_OK;
    if (!logits || !out || !token_starts) return fail(ctx, TF_ERR_INVALID_ARG, "%s: null pointer", name);
    if (T > 1 && (logits_stride < V || out_stride < V))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: row strides below the vocabulary", name);
    const tf_logit_rules& r = *rules;
    if (r.history && (!r.history_lens || (num_requests > 1 && r.history_stride < r.max_history) || r.max_history > 0x3FFFFFFFu))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: a history has lengths, and rows of at least max_history", name);
    if (r.bias_count && (!r.bias_starts || !r.bias_tokens || !r.bias_values || r.bias_count > 0x7FFFFFFEu))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: biases have starts, tokens and values", name);
    if (r.allowed && (r.allowed_count > 0x7FFFFFFFu || (r.allowed_count > 1 && r.allowed_stride < ((uint64_t)V + 31) / 32)))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: rows of allowed tokens have a bit for each", name);
    if (r.allowed && !r.allowed_rows && r.allowed_count < T)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: a row of allowed tokens for every row", name);
    if (!r.token_ids != !r.ancestors)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: drafted tokens and their ancestors go together", name);
    if (r.token_ids && (max_query > (uint32_t)kMaxNodes || r.words > 0xFFFFu || r.words * 32 < max_query))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: trees of up to %d nodes, a bit for each", name, kMaxNodes);
    const size_t size = dtype == TF_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % size || reinterpret_cast<uintptr_t>(out) % size)
        return fail(ctx, TF_ERR_MISALIGNED, "%s: logits and out aligned to their elements", name);
    const void* all[] = {token_starts, r.history, r.history_lens, r.prompt_lens, r.repetition, r.presence, r.frequency,
                         r.bias_starts, r.bias_tokens, r.bias_values, r.allowed, r.allowed_rows, r.token_ids,
                         r.ancestors, tokens};
    for (const void* ptr : all)
        if (!aligned4(ptr)) return fail(ctx, TF_ERR_MISALIGNED, "%s: pointers must be 4-byte aligned", name);
    const size_t need = tf_logit_rules_workspace_bytes(T, V);
    if (tokens && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8 || workspace_bytes < need))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: workspace of %zu bytes, %zu needed, 8-byte aligned", name,
                    workspace_bytes, need);
    RulesParams p = {};
    p.logits = logits;
    p.out = out;
    p.logits_stride = (long long)logits_stride;
    p.out_stride = (long long)out_stride;
    p.starts = static_cast<const int*>(token_starts);
    p.history = static_cast<const int*>(r.history);
    p.history_stride = (long long)r.history_stride;
    p.history_lens = static_cast<const int*>(r.history_lens);
    p.prompt_lens = static_cast<const int*>(r.prompt_lens);
    p.repetition = static_cast<const float*>(r.repetition);
    p.presence = static_cast<const float*>(r.presence);
    p.frequency = static_cast<const float*>(r.frequency);
    p.bias_starts = static_cast<const int*>(r.bias_starts);
    p.bias_tokens = static_cast<const int*>(r.bias_tokens);
    p.bias_values = static_cast<const float*>(r.bias_values);
    p.allowed = static_cast<const uint32_t*>(r.allowed);
    p.allowed_stride = (long long)r.allowed_stride;
    p.allowed_rows = static_cast<const int*>(r.allowed_rows);
    p.token_ids = static_cast<const int*>(r.token_ids);
    p.ancestors = static_cast<const uint32_t*>(r.ancestors);
    p.tokens = static_cast<int*>(tokens);
    p.best = static_cast<unsigned long long*>(workspace);
    p.err = ctx->d_err;
    p.V = (int)V;
    p.T = (int)T;
    p.B = (int)num_requests;
    p.max_query = (int)max_query;
    p.max_history = (int)r.max_history;
    p.bias_count = (int)r.bias_count;
    p.allowed_count = (int)r.allowed_count;
    p.words = (int)r.words;
    p.chunk = kChunk;
    p.chunks = chunks_of(V);
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    cudaError_t e = dtype == TF_DTYPE_F32   ? launch<float>(p, cs)
                    : dtype == TF_DTYPE_F16 ? launch<__half>(p, cs)
                                            : launch<__nv_bfloat16>(p, cs);
    if (e == cudaSuccess && tokens) e = launch_overlapped(best_token_kernel, num_requests, kThreads, 0, cs, p);
    return cuda_check(ctx, e, name);
}

}  // extern "C"

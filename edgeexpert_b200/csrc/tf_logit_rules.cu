// tf_logit_rules.cu -- penalties for repeated tokens, biases and grammar masks on the
// logits of a ragged batch, and the token that is best under them (tf_logit_rules_apply).
//
// For a row of request b, with c = how often a token was said (in the output and on the
// row's way through its drafted tree) and `known` = said or in the prompt:
//   z = logit;  known: z = z > 0 ? z / repetition : z * repetition;
//   z -= frequency * c;  c > 0: z -= presence;  z += bias;  not allowed: -infinity.
// Each step is rounded to fp32 by itself (no contraction), so what a user computes with
// the same steps has the same bits.
//
//   gather_kernel       per request: the tokens that anything is said of, in their order,
//                       as entries (how often, in the prompt, bias)
//   logit_rules_kernel  the rows, once in and once out: a chunk waits in shared memory, gets
//                       the values of its few entries there, and is masked and compared; the
//                       row's last chunk to be done writes its token
#include "tf_paged.cuh"

using namespace tf;

namespace {

constexpr int kGatherThreads = 1024;
constexpr uint32_t kInPrompt = 0x80000000u, kDrafted = 0x40000000u, kCount = 0x3FFFFFFFu;
constexpr int kMaxNodes = 256;
constexpr uint32_t kMaxVocab = 3u << 17;  // 393216, whose bits and ranks fit shared memory
constexpr int kGatherSmem = 220 * 1024;   // of the first kernel, at most

// What the first kernel leaves for the second (in the workspace).
struct Gathered {
    int* request;      // [T]: a row's request, -1: none
    int* begin;        // [B][chunks + 1]: the first entry of a chunk's tokens
    long long* base;   // [B]: a request's first entry
    uint4* entries;    // token, count and flags, bias; in the order of the tokens
    // of the second kernel, 0 at its start:
    unsigned long long* best;  // [T]: the best of a row's chunks
    uint32_t* done;            // [T]: how many there are
};

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
    Gathered g;
    uint32_t* err;
    int V, T, B, max_query, max_history, bias_count, allowed_count, words, vocab_words, chunk, chunks;
    int window;  // entries that a request's CTA counts at once
};

// ---- what is said of a request's tokens --------------------------------------------------

// f(token) for the tokens of a list, by all threads: 16 bytes a load between what lies before and
// behind their boundaries.
template <typename F>
__device__ __forceinline__ void for_tokens(const int* list, int len, F f) {
    if (len <= 0) return;
    const int tid = threadIdx.x;
    const int lead = min(len, (int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(list) & 15u)) / 4u) % 4);
    const int quads = (len - lead) / 4;
    constexpr int kRead = 4;
#pragma unroll 1
    for (int i0 = tid; i0 < quads; i0 += kRead * kGatherThreads) {
        int4 x[kRead];
#pragma unroll
        for (int u = 0; u < kRead; ++u)
            x[u] = i0 + u * kGatherThreads < quads
                       ? *reinterpret_cast<const int4*>(list + lead + (i0 + u * kGatherThreads) * 4)
                       : make_int4(-1, -1, -1, -1);
#pragma unroll
        for (int u = 0; u < kRead; ++u) {
            f(x[u].x);
            f(x[u].y);
            f(x[u].z);
            f(x[u].w);
        }
    }
    if (tid < len - quads * 4) f(list[tid < lead ? tid : quads * 4 + tid]);
}

// One CTA a request.  Bits of the tokens that occur, their ranks by a scan, then the counts of a
// window of ranks at a time (one, unless a request has said more different tokens than fit).
// Bound by latency: a round of loads for the lists a pass, a few barriers.
__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const __grid_constant__ RulesParams p) {
    extern __shared__ __align__(16) uint32_t smem[];
    __shared__ int s_sums[32];
    const int words = p.vocab_words;  // a multiple of 4 * kGatherThreads
    uint32_t* const known = smem;
    uint32_t* const asked = known + words;   // those in the prompt
    uint32_t* const before = asked + words;  // known tokens before a word's
    uint32_t* const said = before + words;
    uint32_t* const token_of = said + p.window;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x;
    for (int i = tid; i < words / 2; i += kGatherThreads) reinterpret_cast<uint4*>(known)[i] = make_uint4(0u, 0u, 0u, 0u);
    griddep_wait();
    griddep_launch_dependents();  // after the wait: the next kernel may read the logits at once
    const int s0 = p.starts[b], s1 = p.starts[b + 1];
    const int lens = p.history ? p.history_lens[b] : 0, prompts = p.prompt_lens ? p.prompt_lens[b] : 0;
    const int bias0 = p.bias_count ? p.bias_starts[b] : 0, bias1 = p.bias_count ? p.bias_starts[b + 1] : 0;
    const int start = max(0, min(s0, p.T)), n = max(start, min(s1, p.T)) - start, used = min(n, p.max_query);
    if (n > used && tid == 0) atomicOr(p.err, kErrBadTree);
    for (int j = tid; j < n; j += kGatherThreads) {
        p.g.request[start + j] = j < used ? b : -1;
        p.g.best[start + j] = 0ull;
        p.g.done[start + j] = 0u;
    }
    if (b == 0) {
        const int end = max(start, min(p.starts[p.B], p.T));
        for (int t = tid; t < start + p.T - end; t += kGatherThreads) p.g.request[t < start ? t : end + t - start] = -1;
    }
    if (used == 0) return;
    const int nodes = p.token_ids ? min(used, p.words * 32) : 0;
    const int len = max(0, min(lens, p.max_history)), prompt = max(0, min(prompts, len));
    const int b0 = max(0, min(bias0, p.bias_count)), b1 = max(b0, min(bias1, p.bias_count));
    const int* const history = p.history + b * p.history_stride;
    // a request has no more entries than its lists have tokens
    const long long base = (long long)b * p.max_history + b0 + start;
    if (tid == 0) p.g.base[b] = base;
    __syncthreads();

    // (Unsigned: ids may be anything.  A bit that is set already is not set again: a few tokens are most
    // of a text, and atomics on one word take turns.)
    auto mark = [&](uint32_t* bits, int token) {
        const uint32_t e = (uint32_t)token, bit = 1u << (e & 31);
        if (e < (uint32_t)p.V && !(bits[e >> 5] & bit)) atomicOr(&bits[e >> 5], bit);
    };
    for_tokens(history, prompt, [&](int token) { mark(asked, token); });
    for_tokens(history + prompt, len - prompt, [&](int token) { mark(known, token); });
    for (int i = b0 + tid; i < b1; i += kGatherThreads) mark(known, p.bias_tokens[i]);
    for (int i = tid; i < nodes; i += kGatherThreads) mark(known, p.token_ids[start + i]);
    __syncthreads();

    // ranks: thread i has the words [i * per, (i + 1) * per)
    const int per = words / kGatherThreads;
    int mine = 0;
    for (int w = tid * per; w < (tid + 1) * per; w += 4) {
        uint4 x = *reinterpret_cast<const uint4*>(known + w);
        const uint4 y = *reinterpret_cast<const uint4*>(asked + w);
        x = make_uint4(x.x | y.x, x.y | y.y, x.z | y.z, x.w | y.w);
        *reinterpret_cast<uint4*>(known + w) = x;
        const int n0 = __popc(x.x), n1 = n0 + __popc(x.y), n2 = n1 + __popc(x.z);
        *reinterpret_cast<uint4*>(before + w) = make_uint4(mine, mine + n0, mine + n1, mine + n2);
        mine += n2 + __popc(x.w);
    }
    int sum = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += u;
    }
    if (lane == 31) s_sums[warp] = sum;
    __syncthreads();
    int all = s_sums[lane];  // (a warp for every lane)
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, all, o);
        if (lane >= o) all += u;
    }
    const int listed = __shfl_sync(0xffffffffu, all, 31);
    const int first = (warp ? __shfl_sync(0xffffffffu, all, warp - 1) : 0) + sum - mine;
    for (int w = tid * per; first && w < (tid + 1) * per; w += 4) {
        uint4 x = *reinterpret_cast<const uint4*>(before + w);
        x = make_uint4(x.x + first, x.y + first, x.z + first, x.w + first);
        *reinterpret_cast<uint4*>(before + w) = x;
    }
    for (int k = tid; k < min(p.window, listed); k += kGatherThreads) said[k] = 0u;
    __syncthreads();
    for (int c = tid; c <= p.chunks; c += kGatherThreads)
        p.g.begin[(long long)b * (p.chunks + 1) + c] = c < p.chunks ? (int)before[c * (p.chunk / 32)] : listed;

    for (int k0 = 0; k0 < listed; k0 += p.window) {
        const int ranks = min(p.window, listed - k0);
        // f(k) for a token that is the window's k-th
        auto with_rank = [&](int token, auto f) {
            const uint32_t e = (uint32_t)token;
            if (e >= (uint32_t)p.V) return;
            const uint32_t k = before[e >> 5] + __popc(known[e >> 5] & ((1u << (e & 31)) - 1u)) - (uint32_t)k0;
            if (k < (uint32_t)ranks) f(k);
        };
        auto name = [&](int token) {
            with_rank(token, [&](uint32_t k) { token_of[k] = (uint32_t)token; });  // (the same whoever writes it)
        };
        for_tokens(history, prompt, name);
        for_tokens(history + prompt, len - prompt, [&](int token) {
            with_rank(token, [&](uint32_t k) {
                token_of[k] = (uint32_t)token;
                atomicAdd(&said[k], 1u);
            });
        });
        for (int i = b0 + tid; i < b1; i += kGatherThreads) name(p.bias_tokens[i]);
        for (int i = tid; i < nodes; i += kGatherThreads) {
            const int token = p.token_ids[start + i];
            with_rank(token, [&](uint32_t k) {
                token_of[k] = (uint32_t)token;
                atomicOr(&said[k], kDrafted);
            });
        }
        __syncthreads();
        for (int k = tid; k < ranks; k += kGatherThreads) {
            const uint32_t e = token_of[k];
            const bool in_prompt = asked[e >> 5] >> (e & 31) & 1u;
            p.g.entries[base + k0 + k] = make_uint4(e, said[k] | (in_prompt ? kInPrompt : 0u), 0u, 0u);
            said[k] = 0u;
        }
        __syncthreads();
        if (b0 < b1) {  // a token's last bias counts
            for (int i = b0 + tid; i < b1; i += kGatherThreads)
                with_rank(p.bias_tokens[i], [&](uint32_t k) { atomicMax(&said[k], (uint32_t)(i + 1)); });
            __syncthreads();
            for (int i = b0 + tid; i < b1; i += kGatherThreads)
                with_rank(p.bias_tokens[i], [&](uint32_t k) {
                    if (said[k] == (uint32_t)(i + 1))
                        reinterpret_cast<float*>(p.g.entries + base + k0 + k)[2] = p.bias_values[i];
                });
            __syncthreads();
            for (int k = tid; k < p.window; k += kGatherThreads) said[k] = 0u;
            __syncthreads();
        }
    }
}

// ---- the rows ---------------------------------------------------------------------------

// Larger for a larger value, -0 and +0 alike.  NaN is not asked for.
__device__ __forceinline__ uint32_t ordered(float z) {
    const uint32_t u = __float_as_uint(__fadd_rn(z, 0.f));
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// The larger is the better: a larger value, of equals the lower token.
__device__ __forceinline__ unsigned long long key_of(float z, int token) {
    return (unsigned long long)ordered(z) << 32 | (0xFFFFFFFFu - (uint32_t)token);
}

__device__ __forceinline__ float to_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T rounded(float v) {
    return from_float<T>(v);
}
template <>
__device__ __forceinline__ float rounded<float>(float v) {
    return v;
}
// 16 bytes of logits, whatever their type.
template <typename T>
struct alignas(16) Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    T e[N];
};

constexpr int kRowThreads = 128;
constexpr int kFly = 8;     // granules of 16 bytes that a thread has of a chunk
constexpr int kStages = 3;  // chunks of a CTA in shared memory
template <typename T>
constexpr int kChunk = kFly * kRowThreads * Vec<T>::N;  // 4096 or 8192 tokens
constexpr int kGranules = kFly * kRowThreads + 1;       // of a chunk that does not begin on 16 bytes

__device__ __forceinline__ float largest(const Vec<float>& x) {  // (NaN is passed over)
    return fmaxf(fmaxf(x.e[0], x.e[1]), fmaxf(x.e[2], x.e[3]));
}
__device__ __forceinline__ float largest(const Vec<__half>& x) {
    const __half2* h = reinterpret_cast<const __half2*>(x.e);
    const __half2 y = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(y), __high2float(y));
}
__device__ __forceinline__ float largest(const Vec<__nv_bfloat16>& x) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(x.e);
    const __nv_bfloat162 y = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(y), __high2float(y));
}

// A chunk of a row in shared memory: the row's granules of 16 bytes, `off` tokens of the first
// lying before the chunk, and the mask's words.
template <typename T>
struct alignas(16) Stage {
    T x[kGranules * Vec<T>::N];
    uint32_t mask[kChunk<T> / 32];
};

// Where a chunk is.
template <typename T>
struct Place {
    static constexpr int N = Vec<T>::N;
    int row, chunk;
    const T* in;  // its first token
    int off, len;
    const uint32_t* mask;  // its first word, or null
    bool no_mask;          // the row's does not exist

    __device__ __forceinline__ void at_row(const RulesParams& p) {
        in = static_cast<const T*>(p.logits) + row * p.logits_stride + chunk * kChunk<T>;
        off = (int)((reinterpret_cast<uintptr_t>(in) & 15u) / sizeof(T));
        len = min(kChunk<T>, p.V - chunk * kChunk<T>);
        const int m = !p.allowed ? -1 : (p.allowed_rows ? p.allowed_rows[row] : row);
        no_mask = m >= p.allowed_count && p.allowed;
        mask = m < 0 || no_mask ? nullptr : p.allowed + m * p.allowed_stride + chunk * (kChunk<T> / 32);
    }
    __device__ __forceinline__ void advance(const RulesParams& p) {
        if (++chunk == p.chunks) {
            chunk = 0;
            if (++row < p.T) at_row(p);
        } else {
            in += kChunk<T>;
            len = min(kChunk<T>, p.V - chunk * kChunk<T>);
            if (mask) mask += kChunk<T> / 32;
        }
    }
    // Whole granules are copied: of the last one what belongs to the row; the first one's tokens before
    // the chunk are the row's own or those of the row before, except where there is none.
    __device__ __forceinline__ void load(Stage<T>& to) const {
        const int tid = threadIdx.x;
        const uint32_t dst = smem_u32(to.x) + tid * 16;
        const T* const src = in - off + tid * N;
        if (off == 0 && len == kChunk<T>) {
#pragma unroll
            for (int u = 0; u < kFly; ++u)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + u * kRowThreads * 16),
                             "l"(src + u * kRowThreads * N)
                             : "memory");
        } else {
            const bool none_before = off && row == 0 && chunk == 0;
#pragma unroll 1
            for (int g = tid; g * N < off + len; g += kRowThreads) {
                const int bytes = min(16, (off + len - g * N) * (int)sizeof(T));
                if (g || !none_before)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to.x + g * N)),
                                 "l"(in - off + g * N), "r"(bytes)
                                 : "memory");
            }
            if (none_before && tid < min(N - off, len)) to.x[off + tid] = in[tid];
        }
        if (mask) {
#pragma unroll
            for (int w = tid; w < kChunk<T> / 32; w += kRowThreads)
                if (w * 32 < len)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to.mask + w)), "l"(mask + w)
                                 : "memory");
        }
    }
};

// The chunks of all rows, one after the other, are dealt evenly to the CTAs, which have the next
// kStages - 1 of them on their way.  Bound by memory: the logits in and out.  A row's entries are
// applied to the chunk in shared memory, those of the next chunk loaded meanwhile.  The largest
// value is looked for by granules, its place in the granule once a chunk.  Logits of 16 bits: an
// entry's value is compared before it is rounded, and its place is left out of the comparison of
// the others (a bit a token in `known`, two lists in turn).
// A CTA a chunk, whose dependent loads (request, entries, mask) lay between its logits and its end,
// left the memory at 0.55 of its rate; this one with 256 threads and four granules each took 1.4
// times as long, by its instructions (133 a warp and granule).
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 4) logit_rules_kernel(const __grid_constant__ RulesParams p) {
    constexpr int N = Vec<T>::N, C = kChunk<T>;
    constexpr bool kRounds = sizeof(T) == 2;
    extern __shared__ __align__(16) uint8_t row_smem[];
    __shared__ unsigned long long s_best[2];
    __shared__ uint32_t s_known[2][kRounds ? kGranules * N / 32 + 1 : 1];
    const int tid = threadIdx.x, lane = tid & 31;
    const long long all = (long long)p.T * p.chunks;
    const int i0 = (int)(all * blockIdx.x / gridDim.x), i1 = (int)(all * (blockIdx.x + 1) / gridDim.x);
    Stage<T>* const stages = reinterpret_cast<Stage<T>*>(row_smem);
    Place<T> at;
    at.row = i0 / p.chunks;
    at.chunk = i0 - at.row * p.chunks;
    at.at_row(p);
    Place<T> ahead = at;
    int to = 0;
    auto load_ahead = [&](int i) {
        if (i < i1) {
            ahead.load(stages[to]);
            if (i + 1 < i1) ahead.advance(p);
            to = to == kStages - 1 ? 0 : to + 1;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) load_ahead(i0 + k);
    if (tid < 2) s_best[tid] = 0ull;
    if constexpr (kRounds)
        for (int w = tid; w < 2 * (int)(sizeof(s_known[0]) / 4); w += kRowThreads) (&s_known[0][0])[w] = 0u;
    griddep_wait();
    griddep_launch_dependents();

    // the entries of a chunk of request b; `first`: this thread's first one
    struct Range {
        int k0, k1;
    };
    auto range_of = [&](int b, int chunk) {
        Range r{0, 0};
        if (b >= 0) {
            const int* begin = p.g.begin + (long long)b * (p.chunks + 1) + chunk;
            r.k0 = begin[0];
            r.k1 = begin[1];
        }
        return r;
    };
    int b = p.g.request[at.row];
    float rep = 1.f, pres = 0.f, freq = 0.f;
    const uint4* entries = nullptr;
    auto look_up_request = [&]() {
        if (b < 0) return;
        entries = p.g.entries + p.g.base[b];
        if (p.repetition) rep = p.repetition[b];
        if (p.presence) pres = p.presence[b];
        if (p.frequency) freq = p.frequency[b];
    };
    look_up_request();
    Range now = range_of(b, at.chunk);
    uint4 first = make_uint4(0u, 0u, 0u, 0u);
    if (now.k0 + tid < now.k1) first = entries[now.k0 + tid];

    int last_i = i0, last_row = 0, last_b = -1;  // of the chunk before
    // One thread: the best of the chunks that are done, and, when a row is left, what it has of it to the
    // row's; whoever brings a row's last chunk has all the others before it.
    unsigned long long row_best = 0ull;
    int row_chunks = 0;
    auto take = [&](int next_row) {  // after chunk last_i, of row last_row
        if (last_b >= 0) {
            row_best = max(row_best, s_best[last_i & 1]);
            ++row_chunks;
        }
        s_best[last_i & 1] = 0ull;
        if (next_row == last_row || row_chunks == 0) return;
        if (row_best) atomicMax(&p.g.best[last_row], row_best);
        __threadfence();
        if (atomicAdd(&p.g.done[last_row], (uint32_t)row_chunks) + row_chunks == (uint32_t)p.chunks) {
            __threadfence();
            const unsigned long long best = atomicMax(&p.g.best[last_row], 0ull);
            p.tokens[last_row] = best ? (int)(0xFFFFFFFFu - (uint32_t)best) : -1;
        }
        row_best = 0ull;
        row_chunks = 0;
    };
    int from = 0;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
        Stage<T>& stage = stages[from];
        from = from == kStages - 1 ? 0 : from + 1;
        const int c0 = at.chunk * C;
        const bool row_ends = at.chunk + 1 == p.chunks, more = i + 1 < i1;
        int next_b = b;
        if (row_ends && more) next_b = p.g.request[at.row + 1];
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();  // the chunk is here, and the one before has been read
        load_ahead(i + kStages - 1);
        if (i > i0 && tid == 0 && p.tokens) take(at.row);
        uint32_t* const known = s_known[i & 1];
        const bool any = now.k0 < now.k1;
        if constexpr (kRounds)
            for (int w = tid; w < (int)(sizeof(s_known[0]) / 4); w += kRowThreads) s_known[(i + 1) & 1][w] = 0u;
        unsigned long long key = 0ull;

        // ---- the entries ---------------------------------------------------------------------
        if (any) {
            // the first one is here; the others four at a time
            auto apply = [&](const uint4& entry) {
                const uint32_t e = entry.x - (uint32_t)c0, word = entry.y;
                if (e >= (uint32_t)at.len) return;  // (lists of requests that overlap)
                float z = to_float(stage.x[at.off + e]);
                int count = (int)(word & kCount);
                if (word & kDrafted) {  // the drafted tokens on the row's way
                    const int start = max(0, min(p.starts[b], p.T));
                    const int nodes = min(min(max(start, p.starts[b + 1]), p.T) - start, min(p.max_query, p.words * 32));
                    const uint32_t* way = p.ancestors + (long long)at.row * p.words;
                    for (int w = 0; w * 32 < nodes; ++w)
                        for (uint32_t m = way[w]; m; m &= m - 1) {
                            const int j = w * 32 + __ffs(m) - 1;
                            if (j < nodes) count += p.token_ids[start + j] == (int)entry.x;
                        }
                }
                if (count || (word & kInPrompt)) z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
                z = __fsub_rn(z, __fmul_rn(freq, (float)count));
                if (count) z = __fsub_rn(z, pres);
                z = __fadd_rn(z, __uint_as_float(entry.z));
                stage.x[at.off + e] = rounded<T>(z);
                if constexpr (kRounds) {
                    atomicOr(&known[(at.off + e) >> 5], 1u << ((at.off + e) & 31));
                    if (z > -INFINITY && (!at.mask || (stage.mask[e >> 5] >> (e & 31) & 1u)))
                        key = max(key, key_of(z, c0 + (int)e));
                }
            };
            if (now.k0 + tid < now.k1) apply(first);
            constexpr int kRead = 4;
#pragma unroll 1
            for (int k = now.k0 + kRowThreads + tid; k < now.k1; k += kRead * kRowThreads) {
                uint4 x[kRead];
#pragma unroll
                for (int u = 0; u < kRead; ++u)
                    if (k + u * kRowThreads < now.k1) x[u] = entries[k + u * kRowThreads];
#pragma unroll 1
                for (int u = 0; u < kRead; ++u) {
                    if (k + u * kRowThreads < now.k1) apply(x[0]);
#pragma unroll
                    for (int v = 0; v + 1 < kRead; ++v) x[v] = x[v + 1];
                }
            }
            __syncthreads();
        }
        Range then{0, 0};
        if (more) then = range_of(next_b, row_ends ? 0 : at.chunk + 1);

        // ---- the chunk ----------------------------------------------------------------------
        if (b >= 0) {
            if (at.no_mask && tid == 0) atomicOr(p.err, kErrBadTree);
            T* const out = static_cast<T*>(p.out) + at.row * p.out_stride + c0;
            const bool masked = at.mask != nullptr, whole = (reinterpret_cast<uintptr_t>(out - at.off) & 15u) == 0;
            // the tokens of granule g that are not allowed, or not the chunk's, as bits
            auto barred = [&](int g) {
                const int t0 = g * N - at.off;
                uint32_t bits = 0u;
                if (masked) {
                    if (at.off == 0) {
                        bits = ~stage.mask[t0 >> 5] >> (t0 & 31);
                    } else {
                        const int w = t0 >> 5;  // (-1 for the first granule: its bits there are not the chunk's)
                        const uint32_t a = w >= 0 ? stage.mask[w] : 0u, z = w + 1 < C / 32 ? stage.mask[w + 1] : 0u;
                        bits = ~__funnelshift_r(a, z, t0 & 31);
                    }
                }
                return bits & ((1u << N) - 1u);
            };
            // and those that are left out of the comparison
            auto said_in = [&](int g) { return kRounds && any ? known[g >> 2] >> ((g & 3) * 8) & 0xFFu : 0u; };
            auto without = [&](Vec<T>& x, uint32_t bits) {
#pragma unroll
                for (int k = 0; k < N; ++k)
                    if (bits >> k & 1u) x.e[k] = rounded<T>(-INFINITY);
            };
            float best = -INFINITY;
            int found = 0;
            auto compare = [&](Vec<T> x, int g) {
                if (kRounds && any) without(x, said_in(g));
                const float top = largest(x);
                if (top > best) {
                    best = top;
                    found = g;
                }
            };
            if (at.off == 0 && at.len == C && whole) {
                Vec<T>* const rows = reinterpret_cast<Vec<T>*>(out) + tid;
                const Vec<T>* const staged = reinterpret_cast<const Vec<T>*>(stage.x) + tid;
#pragma unroll
                for (int u = 0; u < kFly; ++u) {
                    Vec<T> x = staged[u * kRowThreads];
                    if (masked) without(x, barred(u * kRowThreads + tid));
                    rows[u * kRowThreads] = x;
                    compare(x, u * kRowThreads + tid);
                }
            } else {
#pragma unroll 4
                for (int g = tid; g * N < at.off + at.len; g += kRowThreads) {
                    const int t0 = g * N - at.off;
                    Vec<T> x = reinterpret_cast<const Vec<T>*>(stage.x)[g];
                    without(x, barred(g));
                    if (t0 >= 0 && t0 + N <= at.len) {
                        if (whole) {
                            *reinterpret_cast<Vec<T>*>(out + t0) = x;
                        } else {
#pragma unroll
                            for (int k = 0; k < N; ++k) out[t0 + k] = x.e[k];
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < N; ++k) {
                            if (t0 + k >= 0 && t0 + k < at.len)
                                out[t0 + k] = x.e[k];
                            else
                                x.e[k] = rounded<T>(-INFINITY);
                        }
                    }
                    compare(x, g);
                }
            }
            if (p.tokens) {
                if (best > -INFINITY) {  // the granule once more, for the token
                    Vec<T> x = reinterpret_cast<const Vec<T>*>(stage.x)[found];
                    without(x, barred(found) | said_in(found));
                    int k0 = 0;
#pragma unroll
                    for (int k = N - 1; k >= 0; --k)
                        if (to_float(x.e[k]) == best && found * N + k >= at.off && found * N + k < at.off + at.len) k0 = k;
                    key = max(key, key_of(best, c0 + found * N - at.off + k0));
                }
                const uint32_t top = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32));
                const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(key >> 32) == top ? (uint32_t)key : 0u);
                if (lane == 0 && top) atomicMax(&s_best[i & 1], (unsigned long long)top << 32 | low);
            }
        }
        last_i = i;
        last_row = at.row;
        last_b = b;
        if (next_b != b) {
            b = next_b;
            look_up_request();
        }
        if (then.k0 + tid < then.k1) first = entries[then.k0 + tid];
        now = then;
        if (more) at.advance(p);
    }
    __syncthreads();
    if (tid == 0 && i0 < i1 && p.tokens) take(-1);
}

// As many CTAs as are resident at once, or as there are chunks.
template <typename T>
cudaError_t launch_rows(const RulesParams& p, int device, int sms, cudaStream_t cs) {
    constexpr int kSmem = kStages * (int)sizeof(Stage<T>);
    static bool configured[64] = {};  // per instantiation, per device
    if (!configured[device & 63]) {
        const cudaError_t e =
            cudaFuncSetAttribute(logit_rules_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return e;
        configured[device & 63] = true;
    }
    const long long all = (long long)p.T * p.chunks;
    return launch_overlapped(logit_rules_kernel<T>, (unsigned)std::min<long long>(all, 4ll * sms), kRowThreads, kSmem, cs, p);
}

// Words of the vocabulary's bits, a multiple of four a thread.
inline int words_of(uint32_t V) { return (int)((V / 32 + 4 * kGatherThreads) / (4 * kGatherThreads) * (4 * kGatherThreads)); }
inline int chunks_of(uint32_t V, tf_dtype dtype) {
    const int chunk = dtype == TF_DTYPE_F32 ? kChunk<float> : kChunk<__half>;
    return (int)((V + chunk - 1) / chunk);
}

// The workspace, for any type of logits; places are 16-byte aligned.
struct RulesLayout {
    size_t request, begin, base, entries, best, done, bytes;
};
RulesLayout layout_of(uint32_t T, uint32_t V, uint32_t B, uint32_t max_history, uint32_t bias_count) {
    RulesLayout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 15) & ~(size_t)15;
        return here;
    };
    const size_t chunks = chunks_of(V, TF_DTYPE_F32);  // the type of the smallest chunks
    l.request = take((size_t)T * sizeof(int));
    l.begin = take((size_t)B * (chunks + 1) * sizeof(int));
    l.base = take((size_t)B * sizeof(long long));
    l.entries = take(((size_t)B * max_history + bias_count + T) * sizeof(uint4));
    l.best = take((size_t)T * sizeof(unsigned long long));
    l.done = take((size_t)T * sizeof(uint32_t));
    l.bytes = at;
    return l;
}

}  // namespace

extern "C" {

size_t tf_logit_rules_workspace_bytes(uint32_t T, uint32_t V, uint32_t num_requests, uint32_t max_history,
                                      uint32_t bias_count) {
    if (V == 0 || V > kMaxVocab) return 0;
    return layout_of(T, V, num_requests, max_history, bias_count).bytes;
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
    if (V > kMaxVocab || T > 0x7FFFFFu || num_requests > 0xFFFFFFu)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: up to 393216 tokens, 2^23 rows, 2^24 requests", name);
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
    const uint32_t max_history = r.history ? r.max_history : 0;
    const RulesLayout l = layout_of(T, V, num_requests, max_history, r.bias_count);
    if (!workspace || !aligned16(workspace) || workspace_bytes < l.bytes)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", name,
                    workspace_bytes, l.bytes);
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
    uint8_t* const w = static_cast<uint8_t*>(workspace);
    p.g.request = reinterpret_cast<int*>(w + l.request);
    p.g.begin = reinterpret_cast<int*>(w + l.begin);
    p.g.base = reinterpret_cast<long long*>(w + l.base);
    p.g.entries = reinterpret_cast<uint4*>(w + l.entries);
    p.g.best = reinterpret_cast<unsigned long long*>(w + l.best);
    p.g.done = reinterpret_cast<uint32_t*>(w + l.done);
    p.err = ctx->d_err;
    p.V = (int)V;
    p.T = (int)T;
    p.B = (int)num_requests;
    p.max_query = (int)max_query;
    p.max_history = (int)max_history;
    p.bias_count = (int)r.bias_count;
    p.allowed_count = (int)r.allowed_count;
    p.words = (int)r.words;
    p.vocab_words = words_of(V);
    p.chunk = dtype == TF_DTYPE_F32 ? kChunk<float> : kChunk<__half>;
    p.chunks = chunks_of(V, dtype);
    if ((uint64_t)T * p.chunks > 0x7FFFFFFFull)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: too many rows", name);
    static bool configured[64] = {};  // per device
    if (!configured[ctx->device & 63]) {
        s = cuda_check(ctx, cudaFuncSetAttribute(gather_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGatherSmem), name);
        if (s) return s;
        configured[ctx->device & 63] = true;
    }
    // as large as what a request can have said, or as fits
    const uint64_t most = (uint64_t)max_history + r.bias_count + (r.token_ids ? max_query : 0);
    p.window = (int)std::min<uint64_t>((kGatherSmem - (uint64_t)p.vocab_words * 12) / 8, (most + 1023) / 1024 * 1024);
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    cudaError_t e = launch_overlapped(gather_kernel, num_requests, kGatherThreads,
                                      (size_t)p.vocab_words * 12 + (size_t)p.window * 8, cs, p);
    if (e == cudaSuccess)
        e = dtype == TF_DTYPE_F32   ? launch_rows<float>(p, ctx->device, ctx->num_sms, cs)
            : dtype == TF_DTYPE_F16 ? launch_rows<__half>(p, ctx->device, ctx->num_sms, cs)
                                    : launch_rows<__nv_bfloat16>(p, ctx->device, ctx->num_sms, cs);
    return cuda_check(ctx, e, name);
}

}  // extern "C"

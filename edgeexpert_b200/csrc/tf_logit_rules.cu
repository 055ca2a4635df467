// tf_logit_rules.cu -- penalties for repeated tokens, biases and grammar masks on the
// logits of a ragged batch, and the token that is best under them (tf_logit_rules_apply).
//
// For a row of request b, with c = how often a token was said (in the output and on the
// row's way through its drafted tree, where its first nodes may be a prompt's) and `known` = said or in
// the prompt:
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
    int* begin;        // [B][chunks + 1]: the first entry from token chunk * p.chunk on
    long long* base;   // [B]: a request's first entry
    uint4* entries;    // token, count and flags, bias; in the order of the tokens
    uint32_t* known;   // [B][known_words]: the tokens with an entry (for logits of 16 bits)
    int* output_ids;   // [T]: the drafted tokens, -1 in the place of a prompt's (if there are prompts among
                       // them; to look at prompt_nodes again would take the rows 2 us of 120)
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
    const int* prompt_nodes;
    const int* output_ids;  // token_ids, or what is gathered of them
    int* tokens;
    Gathered g;
    uint32_t* err;
    int V, T, B, max_query, max_history, bias_count, allowed_count, words, vocab_words, chunk, chunks;
    int known_words;  // a multiple of 4; 0: not asked for
    int window;  // entries that a request's CTA counts at once
};

// ---- what is said of a request's tokens --------------------------------------------------

// A list of tokens, read by all threads of a CTA, 16 bytes a load between what lies before and behind
// their boundaries.  The first loads stay in registers: a list of up to 16384 tokens is read once.
struct List {
    static constexpr int kHeld = 4;
    const int* list;
    int len, lead, quads;
    int4 held[kHeld];
    int edge;

    __device__ __forceinline__ List(const int* list_, int len_) : list(list_), len(len_), edge(-1) {
        const int tid = threadIdx.x;
        lead = min(len, (int)((16u - (uint32_t)(reinterpret_cast<uintptr_t>(list) & 15u)) / 4u) % 4);
        quads = (len - lead) / 4;
#pragma unroll
        for (int u = 0; u < kHeld; ++u) held[u] = quad(tid + u * kGatherThreads);
        if (tid < len - quads * 4) edge = list[edge_at()];
    }
    __device__ __forceinline__ int edge_at() const {
        return (int)threadIdx.x < lead ? (int)threadIdx.x : quads * 4 + (int)threadIdx.x;
    }
    __device__ __forceinline__ int4 quad(int i) const {
        return i < quads ? *reinterpret_cast<const int4*>(list + lead + i * 4) : make_int4(-1, -1, -1, -1);
    }
    // f(token, its place)
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int tid = threadIdx.x;
        int4 x[kHeld];
#pragma unroll
        for (int u = 0; u < kHeld; ++u) x[u] = held[u];
#pragma unroll 1
        for (int i0 = tid;;) {
#pragma unroll
            for (int u = 0; u < kHeld; ++u) {
                const int at = lead + (i0 + u * kGatherThreads) * 4;
                if (i0 + u * kGatherThreads >= quads) break;
                f(x[u].x, at);
                f(x[u].y, at + 1);
                f(x[u].z, at + 2);
                f(x[u].w, at + 3);
            }
            i0 += kHeld * kGatherThreads;
            if (i0 >= quads) break;
#pragma unroll
            for (int u = 0; u < kHeld; ++u) x[u] = quad(i0 + u * kGatherThreads);
        }
        if (tid < len - quads * 4) f(edge, edge_at());
    }
};

// One CTA a request.  Bits of the tokens that occur, their ranks by a scan, then the counts of a
// window of ranks at a time (one, unless a request has said more different tokens than fit).
// With short lists bound by latency, 6 us: what is known of the request (2.4 us from the start),
// its lists, all asked for at once and kept (1), the scan (2).  With 30000 tokens bound by its
// instructions, 23 us: 5 for the bits, 7 for the counts, 5 for 13000 entries of 16 bytes.
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
    // what the threads need of the lists, all of it asked for at once
    const List history(p.history + b * p.history_stride, len);
    int bias_token = -1, drafted = -1;
    float bias_value = 0.f;
    if (b0 + tid < b1) {
        bias_token = p.bias_tokens[b0 + tid];
        bias_value = p.bias_values[b0 + tid];
    }
    if (tid < nodes) drafted = p.token_ids[start + tid];  // (up to kMaxNodes)
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
    history.each([&](int token, int at) { mark(at < prompt ? asked : known, token); });
    if (b0 + tid < b1) mark(known, bias_token);
    for (int i = b0 + kGatherThreads + tid; i < b1; i += kGatherThreads) mark(known, p.bias_tokens[i]);
    if (tid < nodes) {
        mark(known, drafted);
        if (p.prompt_nodes) {
            const bool in_prompt = tid < p.prompt_nodes[b];
            if (in_prompt) mark(asked, drafted);
            p.g.output_ids[start + tid] = in_prompt ? -1 : drafted;
        }
    }
    __syncthreads();

    // ranks: thread i has the words [i * per, (i + 1) * per)
    const int per = words / kGatherThreads;
    int mine = 0;
    for (int w = tid * per; w < (tid + 1) * per; w += 4) {
        uint4 x = *reinterpret_cast<const uint4*>(known + w);
        const uint4 y = *reinterpret_cast<const uint4*>(asked + w);
        x = make_uint4(x.x | y.x, x.y | y.y, x.z | y.z, x.w | y.w);
        *reinterpret_cast<uint4*>(known + w) = x;
        if (w < p.known_words) *reinterpret_cast<uint4*>(p.g.known + (long long)b * p.known_words + w) = x;
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
        p.g.begin[(long long)b * (p.chunks + 1) + c] = c * p.chunk < p.V ? (int)before[c * (p.chunk / 32)] : listed;

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
        history.each([&](int token, int at) {
            with_rank(token, [&](uint32_t k) {
                token_of[k] = (uint32_t)token;
                if (at >= prompt) atomicAdd(&said[k], 1u);
            });
        });
        if (b0 + tid < b1) name(bias_token);
        for (int i = b0 + kGatherThreads + tid; i < b1; i += kGatherThreads) name(p.bias_tokens[i]);
        if (tid < nodes)
            with_rank(drafted, [&](uint32_t k) {
                token_of[k] = (uint32_t)drafted;
                atomicOr(&said[k], kDrafted);
            });
        __syncthreads();
#pragma unroll 4
        for (int k = tid; k < ranks; k += kGatherThreads) {
            const uint32_t e = token_of[k];
            const bool in_prompt = asked[e >> 5] >> (e & 31) & 1u;
            p.g.entries[base + k0 + k] = make_uint4(e, said[k] | (in_prompt ? kInPrompt : 0u), 0u, 0u);
        }
        __syncthreads();
        if (b0 < b1 || k0 + p.window < listed) {
            for (int k = tid; k < ranks; k += kGatherThreads) said[k] = 0u;
            __syncthreads();
        }
        if (b0 < b1) {  // a token's last bias counts
            auto claim = [&](int token, int i) {
                with_rank(token, [&](uint32_t k) { atomicMax(&said[k], (uint32_t)(i + 1)); });
            };
            auto give = [&](int token, int i, float value) {
                with_rank(token, [&](uint32_t k) {
                    if (said[k] == (uint32_t)(i + 1)) reinterpret_cast<float*>(p.g.entries + base + k0 + k)[2] = value;
                });
            };
            if (b0 + tid < b1) claim(bias_token, b0 + tid);
            for (int i = b0 + kGatherThreads + tid; i < b1; i += kGatherThreads) claim(p.bias_tokens[i], i);
            __syncthreads();
            if (b0 + tid < b1) give(bias_token, b0 + tid, bias_value);
            for (int i = b0 + kGatherThreads + tid; i < b1; i += kGatherThreads) give(p.bias_tokens[i], i, p.bias_values[i]);
            __syncthreads();
            for (int k = tid; k0 + p.window < listed && k < p.window; k += kGatherThreads) said[k] = 0u;
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

// -infinity where a bit is set.
__device__ __forceinline__ void bar(Vec<float>& x, uint32_t bits) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (bits >> k & 1u) x.e[k] = -INFINITY;
}
// Types of 16 bits by pairs: the product puts bit k of four at the top of byte k, which prmt then
// spreads over two bytes.
template <typename T>
__device__ __forceinline__ void bar(Vec<T>& x, uint32_t bits) {
    const T lowest = from_float<T>(-INFINITY);
    const uint32_t both = *reinterpret_cast<const uint16_t*>(&lowest) * 0x10001u;
    uint32_t* const pairs = reinterpret_cast<uint32_t*>(x.e);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint32_t tops = (bits >> 4 * half & 15u) * 0x10204080u;
        uint32_t m0, m1;
        asm("prmt.b32 %0, %1, 0, 0x9988;" : "=r"(m0) : "r"(tops));
        asm("prmt.b32 %0, %1, 0, 0xBBAA;" : "=r"(m1) : "r"(tops));
        pairs[2 * half] = (pairs[2 * half] & ~m0) | (both & m0);
        pairs[2 * half + 1] = (pairs[2 * half + 1] & ~m1) | (both & m1);
    }
}

constexpr int kRowThreads = 128;
constexpr int kFly = 8;     // granules of 16 bytes that a thread has of a chunk
constexpr int kStages = 3;  // chunks of a CTA in shared memory
template <typename T>
constexpr int kChunk = kFly * kRowThreads * Vec<T>::N;  // 4096 or 8192 tokens
constexpr int kRead = 4;    // entries that a thread loads at once
// In the place of an entry that there is not.  Its distance to a chunk's first token, unsigned, is beyond
// any chunk, also where that token is up to seven before the row's own (~0 came round to those, which are
// another row's); an entry's token is not below the row's first.
constexpr uint32_t kNoToken = 0x7FFFFFFFu;

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

// A chunk of a row in shared memory: whole granules of 16 bytes, the mask's words and, of logits of 16
// bits, those of the tokens with an entry.
template <typename T>
struct alignas(16) Stage {
    static constexpr int kWords = kChunk<T> / 32 + 1;
    T x[kChunk<T>];
    uint32_t mask[kWords];
    uint32_t known[sizeof(T) == 2 ? kWords : 1];
};

// Where a chunk is.  Its bounds are the memory's: of a row that begins `off` tokens behind a boundary
// of 16 bytes, chunk c has the tokens from c * kChunk - off on.
template <typename T>
struct Place {
    static constexpr int N = Vec<T>::N;
    int row, chunk, off;
    const T* in;           // the place of its first token
    const uint32_t* mask;  // the row's word with token chunk * kChunk, or null
    bool no_mask;          // the row's does not exist

    __device__ __forceinline__ void at_row(const RulesParams& p) {
        const T* const begin = static_cast<const T*>(p.logits) + row * p.logits_stride;
        off = (int)((reinterpret_cast<uintptr_t>(begin) & 15u) / sizeof(T));
        in = begin - off + chunk * kChunk<T>;
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
            if (mask) mask += kChunk<T> / 32;
        }
    }
    __device__ __forceinline__ int token() const { return chunk * kChunk<T> - off; }
    __device__ __forceinline__ int first() const { return chunk ? 0 : off; }
    __device__ __forceinline__ int end(const RulesParams& p) const { return max(0, min(kChunk<T>, p.V - token())); }
    // Whole granules are copied: of the last one what belongs to the row; what the first one has before
    // the row's begin is of the row before, except where there is none.
    __device__ __forceinline__ void load(Stage<T>& to, const RulesParams& p) const {
        const int tid = threadIdx.x, len = end(p);
        const uint32_t dst = smem_u32(to.x) + tid * 16;
        const T* const src = in + tid * N;
        const bool none_before = off && row == 0 && chunk == 0;
        if (len == kChunk<T> && !none_before) {
#pragma unroll
            for (int u = 0; u < kFly; ++u)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + u * kRowThreads * 16),
                             "l"(src + u * kRowThreads * N)
                             : "memory");
        } else {
#pragma unroll 1
            for (int g = tid; g * N < len; g += kRowThreads) {
                const int bytes = min(16, (len - g * N) * (int)sizeof(T));
                if (g || !none_before)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to.x + g * N)),
                                 "l"(in + g * N), "r"(bytes)
                                 : "memory");
            }
            if (none_before && tid >= off && tid < min(N, len)) to.x[tid] = in[tid];
        }
        if (mask) load_words(to.mask, mask, p);
    }
    // A row of bits: the words from the one with the chunk's first token on.
    __device__ __forceinline__ void load_words(uint32_t* to, const uint32_t* from, const RulesParams& p) const {
        const int before = off ? 1 : 0, words = (p.V + 31) / 32 - chunk * (kChunk<T> / 32);
#pragma unroll 1
        for (int w = threadIdx.x; w < kChunk<T> / 32 + before; w += kRowThreads)
            if (w - before < words && (w >= before || chunk))
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to + w)), "l"(from + w - before)
                             : "memory");
    }
    __device__ __forceinline__ void load_known(Stage<T>& to, int b, const RulesParams& p) const {
        if (b >= 0 && p.known_words)
            load_words(to.known, p.g.known + (long long)b * p.known_words + chunk * (kChunk<T> / 32), p);
    }
    // The bits of granule g.
    __device__ __forceinline__ uint32_t bits_of(const uint32_t* words, int g) const {
        constexpr uint32_t kAll = (1u << N) - 1u;
        if (off == 0) return words[g * N >> 5] >> (g * N & 31) & kAll;
        const int at = 32 - off + g * N, w = at >> 5;
        return __funnelshift_r(words[w], words[min(w + 1, kChunk<T> / 32)], at & 31) & kAll;
    }
    __device__ __forceinline__ uint32_t barred(const Stage<T>& s, int g) const { return ~bits_of(s.mask, g) & ((1u << N) - 1u); }
};

// z / r, rounded as fp32 divides, without a branch (r_inverse: 1 / r in 64 bits).  z * r_inverse is off by
// 2^-52 of the quotient at the most; a step of Newton's, whose remainder is exact, leaves no error but the
// rounding to 64 bits.  That is no matter for the rounding to fp32: a quotient of two 24-bit numbers is on
// a middle between two fp32 numbers, and then 64 bits hold it (only below the smallest normal number,
// since a middle above has 25 bits), or 2^-49 of itself or more away.  Infinities have no remainder.
__device__ __forceinline__ float quotient(float z, float r, double r_inverse) {
    const double q = (double)z * r_inverse, rest = fma(-q, (double)r, (double)z), better = fma(rest, r_inverse, q);
    return (float)(better == better ? better : q);
}

// How often a token was drafted on a row's way through its request's tree of `most` nodes at the most.
__device__ __noinline__ int drafted_before(const int* starts, int rows, int most, const uint32_t* way, const int* ids,
                                           int token) {
    const int start = max(0, min(starts[0], rows)), nodes = min(min(max(start, starts[1]), rows) - start, most);
    int count = 0;
    for (int w = 0; w * 32 < nodes; ++w)
        for (uint32_t m = way[w]; m; m &= m - 1) {
            const int j = w * 32 + __ffs(m) - 1;
            if (j < nodes) count += ids[start + j] == token;
        }
    return count;
}

// The chunks of all rows, one after the other, are dealt evenly to the CTAs, which have the next
// kStages - 1 of them on their way.  Bound by memory: the logits in and out.  A row's entries are
// applied to the chunk in shared memory, four a thread together and without a branch, those of the
// next chunk loaded meanwhile.  The largest value is looked for by granules, its place in the granule
// once a chunk.  Logits of 16 bits: an entry's value is compared before it is rounded, and its place
// is left out of the comparison of the others.
// 256 rows of 262144 fp32 logits: 102 us, 5.3 TB/s; 64 rows without rules: 6.1 TB/s.
// A CTA a chunk, whose dependent loads (request, entries, mask) lay between its logits and its end,
// left the memory at 0.55 of its rate.  This one with 256 threads and four granules each took 1.4
// times as long.  A chunk with 4500 entries takes 11 us, one with few 3: entries one at a time with
// a division and a branch each made that 15.  Chunks counted from the row's first token instead of
// from a boundary of the memory: rows at odd places 37 us instead of 33 (167 of 100003, bf16).
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 4) logit_rules_kernel(const __grid_constant__ RulesParams p) {
    constexpr int N = Vec<T>::N, C = kChunk<T>;
    constexpr bool kRounds = sizeof(T) == 2;
    extern __shared__ __align__(16) uint8_t row_smem[];
    __shared__ unsigned long long s_best[2];
    const int tid = threadIdx.x, lane = tid & 31;
    const long long all = (long long)p.T * p.chunks;
    const int i0 = (int)(all * blockIdx.x / gridDim.x), i1 = (int)(all * (blockIdx.x + 1) / gridDim.x);
    Stage<T>* const stages = reinterpret_cast<Stage<T>*>(row_smem);
    Place<T> at;
    at.row = i0 / p.chunks;
    at.chunk = i0 - at.row * p.chunks;
    at.at_row(p);
    Place<T> ahead = at;
    int to = 0, ahead_b = -1;
    auto load_ahead = [&](int i, bool gathered) {
        if (i < i1) {
            ahead.load(stages[to], p);
            if (kRounds && gathered) ahead.load_known(stages[to], ahead_b, p);
            const int row = ahead.row;
            if (i + 1 < i1) ahead.advance(p);
            if (kRounds && gathered && ahead.row != row) ahead_b = p.g.request[ahead.row];
            to = to == kStages - 1 ? 0 : to + 1;
        }
    };
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) load_ahead(i0 + k, false);
    if (tid < 2) s_best[tid] = 0ull;
    griddep_wait();
    griddep_launch_dependents();
    if (kRounds) {  // what the first chunks were loaded without
        Place<T> first = at;
#pragma unroll 1
        for (int k = 0; k < kStages - 1 && i0 + k < i1; ++k) {
            first.load_known(stages[k], p.g.request[first.row], p);
            if (i0 + k + 1 < i1) first.advance(p);
        }
        ahead_b = p.g.request[ahead.row];
    }
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) asm volatile("cp.async.commit_group;" ::: "memory");

    // the entries of a chunk (and a few before it or behind)
    struct Range {
        int k0, k1;
    };
    auto range_of = [&](int b, int chunk, int off) {
        Range r{0, 0};
        if (b >= 0) {
            const int* begin = p.g.begin + (long long)b * (p.chunks + 1) + chunk;
            r.k0 = max(0, begin[0] - off);
            r.k1 = begin[1];
        }
        return r;
    };
    int b = p.g.request[at.row];
    float rep = 1.f, pres = 0.f, freq = 0.f;
    double rep_inverse = 1.0;
    long long base = 0;
    auto look_up_request = [&]() {
        if (b < 0) return;
        base = p.g.base[b];
        if (p.repetition) {
            rep = p.repetition[b];
            rep_inverse = 1.0 / (double)rep;
        }
        if (p.presence) pres = p.presence[b];
        if (p.frequency) freq = p.frequency[b];
    };
    look_up_request();
    Range now = range_of(b, at.chunk, at.off);
    uint4 x[kRead];  // the first entries of the next chunk
    auto fetch = [&](uint4 (&x)[kRead], int k, int k1) {
#pragma unroll
        for (int u = 0; u < kRead; ++u)
            x[u] = k + u * kRowThreads < k1 ? p.g.entries[base + k + u * kRowThreads] : make_uint4(kNoToken, 0u, 0u, 0u);
    };
    fetch(x, now.k0 + tid, now.k1);

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
        const int c0 = at.token(), lo = at.first(), hi = at.end(p);
        const bool row_ends = at.chunk + 1 == p.chunks, more = i + 1 < i1;
        int next_b = b;
        if (row_ends && more) next_b = p.g.request[at.row + 1];
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();  // the chunk is here, and the one before has been read
        load_ahead(i + kStages - 1, true);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (i > i0 && tid == 0 && p.tokens) take(at.row);
        const bool any = now.k0 < now.k1;
        unsigned long long key = 0ull;

        // ---- the entries ---------------------------------------------------------------------
        if (any) {
            float said_best = -INFINITY;  // (of equals the first, which is the lower token)
            int said_token = 0;
#pragma unroll 1
            for (int k = now.k0 + tid; k < now.k1; k += kRead * kRowThreads) {
                uint4 y[kRead];
                fetch(y, k + kRead * kRowThreads, now.k1);
                float z[kRead];
                uint32_t drafted = 0u;
#pragma unroll
                for (int u = 0; u < kRead; ++u) {
                    const uint32_t e = x[u].x - (uint32_t)c0;
                    z[u] = e < (uint32_t)hi ? to_float(stage.x[e]) : NAN;
                    drafted |= x[u].y & kDrafted;
                }
                if (drafted) {
#pragma unroll
                    for (int u = 0; u < kRead; ++u)
                        if ((x[u].y & kDrafted) && x[u].x - (uint32_t)c0 < (uint32_t)hi)
                            x[u].y += drafted_before(p.starts + b, p.T, min(p.max_query, p.words * 32),
                                                     p.ancestors + (long long)at.row * p.words, p.output_ids, (int)x[u].x);
                }
                float top = -INFINITY;
#pragma unroll
                for (int u = 0; u < kRead; ++u) {
                    const uint32_t e = x[u].x - (uint32_t)c0, count = x[u].y & kCount;
                    const float divided = quotient(z[u], rep, rep_inverse), times = __fmul_rn(z[u], rep);
                    float r = count || (x[u].y & kInPrompt) ? (z[u] > 0.f ? divided : times) : z[u];
                    r = __fsub_rn(r, __fmul_rn(freq, (float)count));
                    r = count ? __fsub_rn(r, pres) : r;
                    r = __fadd_rn(r, __uint_as_float(x[u].z));
                    if (e < (uint32_t)hi) stage.x[e] = rounded<T>(r);
                    z[u] = r;
                    top = fmaxf(top, r);
                }
                if (kRounds && top > said_best) {
#pragma unroll
                    for (int u = 0; u < kRead; ++u) {
                        const int e = (int)x[u].x - c0;
                        if (z[u] > said_best && (!at.mask || !(at.barred(stage, e / N) >> (e & (N - 1)) & 1u))) {
                            said_best = z[u];
                            said_token = (int)x[u].x;
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < kRead; ++u) x[u] = y[u];
            }
            if (kRounds && said_best > -INFINITY) key = key_of(said_best, said_token);
            __syncthreads();
        }
        Range then{0, 0};
        if (more) then = range_of(next_b, row_ends ? 0 : at.chunk + 1, row_ends ? 0 : at.off);

        // ---- the chunk ----------------------------------------------------------------------
        if (b >= 0) {
            if (at.no_mask && tid == 0) atomicOr(p.err, kErrBadTree);
            T* const out = static_cast<T*>(p.out) + at.row * p.out_stride + c0;
            const bool masked = at.mask != nullptr, whole = (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
            // the tokens of a granule that are left out of the comparison, as bits
            auto said_in = [&](int g) { return kRounds && any ? at.bits_of(stage.known, g) : 0u; };
            float best = -INFINITY;
            int found = 0;
            auto compare = [&](Vec<T> x, int g) {
                if (const uint32_t bits = said_in(g)) bar(x, bits);
                const float top = largest(x);
                if (top > best) {
                    best = top;
                    found = g;
                }
            };
            if (lo == 0 && hi == C && whole) {
                Vec<T>* const rows = reinterpret_cast<Vec<T>*>(out) + tid;
                const Vec<T>* const staged = reinterpret_cast<const Vec<T>*>(stage.x) + tid;
#pragma unroll
                for (int u = 0; u < kFly; ++u) {
                    Vec<T> x = staged[u * kRowThreads];
                    if (masked) bar(x, at.barred(stage, u * kRowThreads + tid));
                    rows[u * kRowThreads] = x;
                    compare(x, u * kRowThreads + tid);
                }
            } else {
#pragma unroll 4
                for (int g = tid; g * N < hi; g += kRowThreads) {
                    const int t0 = g * N;
                    Vec<T> x = reinterpret_cast<const Vec<T>*>(stage.x)[g];
                    if (masked) bar(x, at.barred(stage, g));
                    if (t0 >= lo && t0 + N <= hi) {
                        if (whole) {
                            *reinterpret_cast<Vec<T>*>(out + t0) = x;
                        } else {
#pragma unroll
                            for (int k = 0; k < N; ++k) out[t0 + k] = x.e[k];
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < N; ++k) {
                            if (t0 + k >= lo && t0 + k < hi)
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
                    bar(x, (masked ? at.barred(stage, found) : 0u) | said_in(found));
                    int k0 = 0;
#pragma unroll
                    for (int k = N - 1; k >= 0; --k)
                        if (to_float(x.e[k]) == best && found * N + k >= lo && found * N + k < hi) k0 = k;
                    key = max(key, key_of(best, c0 + found * N + k0));
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
        fetch(x, then.k0 + tid, then.k1);
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
// A row may begin anywhere in its first granule (`aligned`: on its boundary).
inline int chunks_of(uint32_t V, tf_dtype dtype, bool aligned) {
    const int chunk = dtype == TF_DTYPE_F32 ? kChunk<float> : kChunk<__half>, granule = chunk / (kFly * kRowThreads);
    return (int)((V + (aligned ? 0 : granule - 1) + chunk - 1) / chunk);
}

inline uint32_t known_words_of(uint32_t V) { return (V + 127) / 128 * 4; }

// The workspace, for any type of logits; places are 16-byte aligned.
struct RulesLayout {
    size_t request, begin, base, entries, known, output_ids, best, done, bytes;
};
RulesLayout layout_of(uint32_t T, uint32_t V, uint32_t B, uint32_t max_history, uint32_t bias_count) {
    RulesLayout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 15) & ~(size_t)15;
        return here;
    };
    const size_t chunks = chunks_of(V, TF_DTYPE_F32, false);  // the type of the smallest chunks
    l.request = take((size_t)T * sizeof(int));
    l.begin = take((size_t)B * (chunks + 1) * sizeof(int));
    l.base = take((size_t)B * sizeof(long long));
    l.entries = take(((size_t)B * max_history + bias_count + T) * sizeof(uint4));
    l.known = take((size_t)B * known_words_of(V) * sizeof(uint32_t));
    l.output_ids = take((size_t)T * sizeof(int));
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
    if (r.history && (!r.history_lens || (num_requests > 1 && r.history_stride < r.max_history) || r.max_history > kCount))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: a history has lengths, and rows of at least max_history", name);
    if (r.bias_count && (!r.bias_starts || !r.bias_tokens || !r.bias_values || r.bias_count > 0x7FFFFFFEu))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: biases have starts, tokens and values", name);
    if (r.allowed && (r.allowed_count > 0x7FFFFFFFu || (r.allowed_count > 1 && r.allowed_stride < ((uint64_t)V + 31) / 32)))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: rows of allowed tokens have a bit for each", name);
    if (r.allowed && !r.allowed_rows && r.allowed_count < T)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: a row of allowed tokens for every row", name);
    if (!r.token_ids != !r.ancestors)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: drafted tokens and their ancestors go together", name);
    if (r.prompt_nodes && !r.token_ids)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: a prompt among no drafted tokens", name);
    if (r.token_ids && (max_query > (uint32_t)kMaxNodes || r.words > 0xFFFFu || r.words * 32 < max_query))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: trees of up to %d nodes, a bit for each", name, kMaxNodes);
    const size_t size = dtype == TF_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(logits) % size || reinterpret_cast<uintptr_t>(out) % size)
        return fail(ctx, TF_ERR_MISALIGNED, "%s: logits and out aligned to their elements", name);
    const void* all[] = {token_starts, r.history, r.history_lens, r.prompt_lens, r.repetition, r.presence, r.frequency,
                         r.bias_starts, r.bias_tokens, r.bias_values, r.allowed, r.allowed_rows, r.token_ids,
                         r.ancestors, r.prompt_nodes, tokens};
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
    p.prompt_nodes = static_cast<const int*>(r.prompt_nodes);
    p.tokens = static_cast<int*>(tokens);
    uint8_t* const w = static_cast<uint8_t*>(workspace);
    p.g.request = reinterpret_cast<int*>(w + l.request);
    p.g.begin = reinterpret_cast<int*>(w + l.begin);
    p.g.base = reinterpret_cast<long long*>(w + l.base);
    p.g.entries = reinterpret_cast<uint4*>(w + l.entries);
    p.g.known = reinterpret_cast<uint32_t*>(w + l.known);
    p.g.output_ids = reinterpret_cast<int*>(w + l.output_ids);
    p.output_ids = r.prompt_nodes ? p.g.output_ids : p.token_ids;
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
    p.known_words = size == 2 ? (int)known_words_of(V) : 0;
    p.chunk = dtype == TF_DTYPE_F32 ? kChunk<float> : kChunk<__half>;
    p.chunks = chunks_of(V, dtype, aligned16(logits) && (T == 1 || logits_stride * size % 16 == 0));
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

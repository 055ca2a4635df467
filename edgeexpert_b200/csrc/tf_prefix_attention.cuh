// tf_prefix_attention.cuh -- what the kernels of tf_shared_prefix_attention and (kTree)
// tf_tree_attention share:
// parameters, which rows see which keys, how work is dealt to CTAs, and where
// the parts of a row's softmax are kept until they are joined.
#pragma once
#include "tf_paged.cuh"

namespace tf {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTcRows = 128;  // query rows of a tensor tile
constexpr int kMaxRun = 8;

// Parts of rows.  A worker (a warp for few rows, a CTA for many) goes through a
// contiguous range of units (a unit is one tile of keys of one job); the part
// it computes of a job goes to `first` (at the row's own place) when it holds
// the job's first unit, and to `cont` (at the worker's place) otherwise: at most
// one of a worker's jobs began before it.  o is not normalised; md = (m, d), m
// in units of log2.
struct Parts {
    float* first;
    float2* first_md;
    float* cont;
    float2* cont_md;
    // for every row: the worker of its job's first unit and the row's place in the job (first_of =
    // worker << shift | place), and the worker of the last: what the joining kernel adds up
    int* first_of;
    int* last_of;
    int shift;   // log2 of the rows a cont place holds
    int places;  // workers that cont has places for
};

// The pool as TMA sees it: [page][head][64-dim block][position][64 dims], 128-byte
// swizzle.  A tile of keys is kept as groups of eight keys, [group][block][8 keys]
// [128 bytes], so a box of 8 keys and all blocks is one load ("wide") where pages
// hold whole groups and head_dim whole blocks; otherwise a box is `run` keys and
// one block.  rows: boxes of one key and one block.
struct KvMaps {
    CUtensorMap k, v, v_row;
};

// kTree: a request's query tokens are the nodes of a drafted tree.  Each sees the history before
// the nodes (hi of seen_by ends there) and those of the nodes whose bit is set in its ancestors.
template <typename T, bool kTree>
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
    const uint32_t* ancestors;  // kTree: [tokens][words]
    const int* positions;       // kTree, with a window: where the nodes stand
    int words;
    uint32_t* err;
    int* prefix_first;  // the first prefix position that any row sees, for the joining kernel (calls with a window)
    int prefix_len, max_pages, B, max_query, T_tokens, nq, nkv, G, hd, window;
    int prefix_few;   // the prefix is read by the streaming warps too (the batch has few rows)
    int many_above;   // requests of more rows per KV head than this go to the tensor cores
    float scale;
    Parts few, many;
    int run_shift;   // keys of a box, as a power of two: the largest up to 8 that divides the page size
    int g_shift;     // the query heads of a KV head as a power of two, or -1
    int page_shift;  // the page size as a power of two, or -1 (a division per unit cost 150 clocks of its latency)
    int wide;  // a box has all of a head's blocks
    KvMaps maps;
};

// Row -> token of a job's rows (token * G + head in the group).
template <typename T, bool kTree>
__device__ __forceinline__ int token_of(const AttnParams<T, kTree>& p, int row) {
    return p.g_shift >= 0 ? row >> p.g_shift : row / p.G;
}

// A request of the batch.
struct Request {
    int start, n, used, len;  // first token, tokens, tokens within max_query, own positions
};

template <typename T, bool kTree>
__device__ __forceinline__ Request request_of(const AttnParams<T, kTree>& p, int b) {
    Request r;
    const int s0 = max(0, min(p.starts[b], p.T_tokens)), s1 = max(s0, min(p.starts[b + 1], p.T_tokens));
    r.start = s0;
    r.n = s1 - s0;
    r.used = min(r.n, p.max_query);
    r.len = (int)min((long long)max(0, p.seq_lens[b]), (long long)p.max_pages * p.kv.page_size);
    return r;
}

// What runs once a job or segment is kept out of line here and below: inlined
// wherever a cursor moves it made the kernel 247 KB of code, and the loops of its
// warps, which share an instruction cache, spent half their time fetching it.

// The last b with starts[b] <= t; B for tokens behind the last request, and 0 for those before
// the first one too (whose token index is negative then).
template <typename T, bool kTree>
__device__ __noinline__ int request_at(const AttnParams<T, kTree>& p, int t) {
    int lo = 0, hi = p.B;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.starts[mid] <= t)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// Token j of request r is one of those that are computed.
__device__ __forceinline__ bool is_used(const Request& r, int j) { return j >= 0 && j < r.used; }

// Keys [lo, hi) that token j of request r sees, as positions of the whole sequence.
template <typename T, bool kTree>
__device__ __forceinline__ void seen_by(const AttnParams<T, kTree>& p, const Request& r, int j, int& lo, int& hi) {
    if constexpr (kTree) {
        hi = p.prefix_len + max(0, r.len - r.n);
        lo = p.window ? max(0, max(hi, p.positions[r.start + j]) - p.window + 1) : 0;
    } else {
        const int at = p.prefix_len + r.len - (r.n - j);
        hi = at + 1;
        lo = p.window ? max(0, at - p.window + 1) : 0;
    }
}
// The first key that any token of the request sees (nodes stand behind the history).
template <typename T, bool kTree>
__device__ __forceinline__ int seen_from(const AttnParams<T, kTree>& p, const Request& r) {
    if constexpr (kTree) return p.window ? max(0, p.prefix_len + max(0, r.len - r.n) - p.window + 1) : 0;
    int lo, hi;
    seen_by(p, r, 0, lo, hi);
    return lo;
}
// kTree: whether the token with these ancestors sees a node (of its own request).
__device__ __forceinline__ bool sees_node(const uint32_t* ancestors, int words, int node) {
    return node >= 0 && node < words * 32 && (ancestors[node >> 5] >> (node & 31) & 1u);
}

// The first prefix position that any row of the batch sees, as the parts kernel keeps it: positions
// before it have no rows, and pages of them may belong to others by now.
__device__ __forceinline__ int& shared_prefix_first() {
    __shared__ int first;
    return first;
}
template <typename T, bool kTree>
__device__ __forceinline__ int prefix_first(const AttnParams<T, kTree>& p) {
    return p.window ? shared_prefix_first() : 0;
}
// Tiles of `keys` keys that hold the prefix from there on.
template <typename T, bool kTree>
__device__ __forceinline__ int prefix_tiles(const AttnParams<T, kTree>& p, int keys) {
    const int first = prefix_first(p);
    return p.prefix_len > first ? (p.prefix_len - (first & ~(kMaxRun - 1)) + keys - 1) / keys : 0;
}

// First of a request's own positions that any of its rows sees.
template <typename T, bool kTree>
__device__ __forceinline__ int own_lo(const AttnParams<T, kTree>& p, const Request& r) {
    return max(0, min(r.len, seen_from(p, r) - p.prefix_len));
}

template <typename T, bool kTree>
__device__ __forceinline__ bool is_many(const AttnParams<T, kTree>& p, const Request& r) {
    return r.used * p.G > p.many_above;
}

// Units [c*U/N, (c+1)*U/N) are worker c's.  In double: the products are below 2^53, and a
// quotient that is no whole number is further from one than its rounding (64-bit integer
// divisions, a dozen of them at a kernel's start, took microseconds).
__device__ __forceinline__ int unit_begin(int c, int U, int N) { return (int)floor((double)c * U / N); }

// Exclusive sum of v over the block (up to 32 warps); *total receives the sum.
__device__ __forceinline__ int block_scan(int v, int* red, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int incl = v;
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    __syncthreads();  // red may still be read from before
    if (lane == 31) red[warp] = incl;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < nw; ++w) {
        const int x = red[w];
        if (w < warp) before += x;
        all += x;
    }
    *total = all;
    return before + incl - v;
}

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Waits about two seconds at most (from `since` on), then reports it and returns false.
__device__ __forceinline__ bool mbar_wait_limited(uint64_t* bar, uint32_t parity, uint32_t* err, long long since) {
    while (!mbar_try_wait(bar, parity))
        if (clock64() - since > 4000000000ll) {
            atomicOr(err, kErrMbarTimeout);
            return false;
        }
    return true;
}
__device__ __forceinline__ bool mbar_wait_limited(uint64_t* bar, uint32_t parity, uint32_t* err) {
    return mbar_try_wait(bar, parity) || mbar_wait_limited(bar, parity, err, clock64());
}

// What L2 should do with a tile: keys that one job reads, once, leave first; the prefix's, and own
// keys that several row tiles read, stay.
__device__ __forceinline__ uint64_t l2_policy(bool once) {
    uint64_t first, last;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(first));
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(last));
    return once ? first : last;
}

// 5-D tiled TMA load (no multicast).
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int v, int w,
                                            uint64_t* bar, uint64_t hint) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, "
        "%3, %4, %5, %6}], [%7], %8;" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(v), "r"(w), "r"(smem_u32(bar)), "l"(hint)
        : "memory");
}

// One lane of a converged warp, known to the compiler as one.  The operands of
// TMA and tcgen05 instructions live in uniform registers: issued under
// `lane == 0` each becomes a loop over the lanes' values (46 clocks for an MMA
// of 32, 87 for a TMA load), under this they go out back to back.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// A tile of KEYS keys, by a converged warp.  Lane l has looked up the runs l, l +
// 32, ...: the page, the place in it and (bit r) which of the run's keys exist.
// Keys that do not exist arrive as zeros: a whole box from a page behind the
// pool, and for V, whose every row meets a weight (0 * NaN would not be 0), key
// by key where a run has both.
template <int KEYS>
struct TileKeys {
    static constexpr int kMost = (KEYS + 31) / 32;
    int page[kMost], in_page[kMost], have[kMost];
};

template <int HD, int KEYS, typename T, bool kTree>
__device__ __forceinline__ void load_tile_keys(const AttnParams<T, kTree>& p, bool v, uint32_t tile, int head,
                                               const TileKeys<KEYS>& k, uint64_t* bar, bool once) {
    constexpr int kBlocks = HD / 64, kMost = TileKeys<KEYS>::kMost;
    const CUtensorMap* map = v ? &p.maps.v : &p.maps.k;
    const int lane = threadIdx.x & 31, run = 1 << p.run_shift, runs = KEYS >> p.run_shift, all = (1 << run) - 1;
    const bool one = elect_one();
    const uint64_t hint = l2_policy(once);
    if (one) mbar_arrive_expect_tx(bar, KEYS * HD * 2);
    bool complete = p.wide != 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i) complete &= i * 32 + lane >= runs || k.have[i] == all;
    if (__all_sync(0xffffffffu, complete)) {
#pragma unroll 2
        for (int r = 0; r < KEYS / 8; ++r) {
            const int pg = __shfl_sync(0xffffffffu, k.page[0], r), in = __shfl_sync(0xffffffffu, k.in_page[0], r);
            if (one) tma_load_5d(tile + r * (kBlocks * 1024), map, 0, in, 0, head, pg, bar, hint);
        }
        __syncwarp();
        return;
    }
#pragma unroll
    for (int i = 0; i < kMost; ++i)
#pragma unroll 1
        for (int l = 0; l < min(32, runs - i * 32); ++l) {
            const int pg = __shfl_sync(0xffffffffu, k.page[i], l), in = __shfl_sync(0xffffffffu, k.in_page[i], l);
            const int have = __shfl_sync(0xffffffffu, k.have[i], l), first = (i * 32 + l) * run;
            const uint32_t dst = tile + (first >> 3) * (kBlocks * 1024) + (first & 7) * 128;
            const int from = have ? pg : p.kv.num_pages;
            if (!one) continue;
            if (!v || have == all || have == 0) {
                if (p.wide)
                    tma_load_5d(dst, map, 0, in, 0, head, from, bar, hint);
                else
                    for (int b = 0; b < kBlocks; ++b) tma_load_5d(dst + b * 1024, map, b * 64, in, 0, head, from, bar, hint);
            } else {
                for (int r = 0; r < run; ++r)
                    for (int b = 0; b < kBlocks; ++b)
                        tma_load_5d(dst + b * 1024 + r * 128, &p.maps.v_row, b * 64, in + r, 0, head,
                                    (have >> r) & 1 ? pg : p.kv.num_pages, bar, hint);
            }
        }
    __syncwarp();
}

// The runs of the tile of keys that begins at position `pos0` of a segment
// whose keys are [from, hi).
template <int KEYS, typename T, bool kTree>
__device__ __forceinline__ TileKeys<KEYS> look_up_keys(const AttnParams<T, kTree>& p, int seg, int pos0, int from, int hi) {
    TileKeys<KEYS> k;
    const int lane = threadIdx.x & 31, run = 1 << p.run_shift, runs = KEYS >> p.run_shift;
#pragma unroll
    for (int i = 0; i < TileKeys<KEYS>::kMost; ++i) {
        const int pos = pos0 + ((i * 32 + lane) << p.run_shift);
        const int a = max(0, from - pos), z = min(run, hi - pos);  // keys a .. z - 1 of the run exist
        k.page[i] = k.in_page[i] = k.have[i] = 0;
        if (i * 32 + lane < runs && a < z) {
            const int at = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.kv.page_size;
            k.in_page[i] = pos - at * p.kv.page_size;
            k.have[i] = (1 << z) - (1 << a);
            k.page[i] = seg < 0 ? p.prefix_pages[at] : p.table[(long long)seg * p.max_pages + at];
        }
    }
    return k;
}
// Once the page ids are there: those outside the pool are reported and not read.
template <int KEYS, typename T, bool kTree>
__device__ __forceinline__ void check_keys(const AttnParams<T, kTree>& p, TileKeys<KEYS>& k) {
#pragma unroll
    for (int i = 0; i < TileKeys<KEYS>::kMost; ++i) {
        asm volatile("" : "+r"(k.page[i]));  // not earlier: the id is waited for here
        if (k.have[i] && (k.page[i] < 0 || k.page[i] >= p.kv.num_pages)) {
            atomicOr(p.err, kErrBadPage);
            k.have[i] = 0;
        }
    }
}

}  // namespace tf

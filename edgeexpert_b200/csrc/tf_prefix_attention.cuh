// tf_prefix_attention.cuh -- what the kernels of tf_shared_prefix_attention share:
// parameters, which rows see which keys, how work is dealt to CTAs, and where
// the parts of a row's softmax are kept until they are joined.
#pragma once
#include "tf_paged.cuh"

namespace tf {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTcRows = 128;  // query rows of a tensor tile

// Parts of rows.  A CTA works through a contiguous range of units (a unit is
// one tile of keys of one job); the part it computes of a job goes to `first`
// (at the row's own place) when it holds the job's first unit, and to `cont`
// (at the CTA's place) otherwise: at most one of a CTA's jobs began before it.
// o is not normalised; md = (m, d), m in units of log2.
struct Parts {
    float* first;
    float2* first_md;
    float* cont;
    float2* cont_md;
    int* base;  // first unit of each request (stream) or row tile (tensor); [count] = all units
    int ctas;
    int rows;  // rows a cont place holds
};

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
    int prefix_len, prefix_lo, max_pages, B, max_query, T_tokens, nq, nkv, G, hd, window;
    int prefix_by_stream;  // the stream kernel also reads the prefix (few rows)
    int tensor_above;      // requests of more rows per KV head than this are the tensor kernel's
    float scale;
    Parts stream, tensor;
};

// A request of the batch.
struct Request {
    int start, n, used, len;  // first token, tokens, tokens within max_query, own positions
};

template <typename T>
__device__ __forceinline__ Request request_of(const AttnParams<T>& p, int b) {
    Request r;
    const int s0 = max(0, min(p.starts[b], p.T_tokens)), s1 = max(s0, min(p.starts[b + 1], p.T_tokens));
    r.start = s0;
    r.n = s1 - s0;
    r.used = min(r.n, p.max_query);
    r.len = (int)min((long long)max(0, p.seq_lens[b]), (long long)p.max_pages * p.kv.page_size);
    return r;
}

// The last b with starts[b] <= t; B for tokens behind the last request.
template <typename T>
__device__ __forceinline__ int request_at(const AttnParams<T>& p, int t) {
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

// Keys [lo, hi) that token j of request r sees, as positions of the whole sequence.
template <typename T>
__device__ __forceinline__ void seen_by(const AttnParams<T>& p, const Request& r, int j, int& lo, int& hi) {
    const int at = p.prefix_len + r.len - (r.n - j);
    hi = at + 1;
    lo = p.window ? max(0, at - p.window + 1) : 0;
}

// First of a request's own positions that any of its rows sees.
template <typename T>
__device__ __forceinline__ int own_lo(const AttnParams<T>& p, const Request& r) {
    int lo, hi;
    seen_by(p, r, 0, lo, hi);
    return max(0, min(r.len, lo - p.prefix_len));
}

template <typename T>
__device__ __forceinline__ bool by_tensor(const AttnParams<T>& p, const Request& r) {
    return r.used * p.G > p.tensor_above;
}

// Units [c*U/N, (c+1)*U/N) are CTA c's.
__device__ __forceinline__ int unit_begin(int c, int U, int N) { return (int)((long long)c * U / N); }
__device__ __forceinline__ int cta_of(int u, int U, int N) { return (int)((((long long)u + 1) * N - 1) / U); }

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

// 16-byte asynchronous copy; `bytes` 0 fills the destination with zeros.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace tf

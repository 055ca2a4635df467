// tf_paged.cu -- the pages of a ragged batch and what is written into them:
//   tf_kv_pages_resize   request lengths -> page tables, slots, positions
//   tf_rope_frequencies  (host) radians per position of each rotated pair
//   tf_rope_kv_write     head norms + rotation at each token's position + paged K/V write
#include <math.h>

#include "tf_paged.cuh"

using namespace tf;

namespace {

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// ---- page tables -------------------------------------------------------------
struct ResizeParams {
    const int* seq_lens;
    const int* targets;
    int* table;
    int* ring;
    const int* state;
    int* lens_out;
    int* state_out;
    int* starts;
    int* slots;
    int* positions;
    int* requests;
    int* plan;       // [0] head, [1] free count, then per request {old length, new length, first page taken, first given back}
    int* starts_at;  // the starts as resize_fill reads them
    uint32_t* err;
    int B, max_pages, N, ps, base, max_tokens;
    int most;  // positions a request's table can hold
};

constexpr int kResizeThreads = 1024;
constexpr int kFillThreads = 256;
constexpr uint32_t kSmallTokens = 1024, kSmallRequests = 256;

// (64-bit divisions would be most of a small call's time: lengths and page sizes are below 2^31)
__device__ __forceinline__ int pages_of(int n, int ps) { return (int)(((unsigned)n + (unsigned)ps - 1u) / (unsigned)ps); }
// Place head + x of a ring of N.
__device__ __forceinline__ int ring_at(int head, long long x, int N) {
    unsigned long long at = (unsigned long long)head + (unsigned long long)x;
    if (at >= (unsigned)N) at -= (unsigned)N;
    if (at >= (unsigned)N) at %= (unsigned)N;
    return (int)at;
}

// Exclusive sum over the block's threads; *total receives the whole sum.
__device__ long long block_exclusive_sum(long long v, long long* red, long long* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    long long incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    __syncthreads();  // red may still be read from the previous sum
    if (lane == 31) red[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        long long w = lane < warps ? red[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        red[lane] = w;
    }
    __syncthreads();
    *total = red[31];
    return (warp ? red[warp - 1] : 0) + incl - v;
}

struct Ask {
    int old_len, target;
    bool grow, shrink;
    int need, back;
};

__device__ __forceinline__ Ask ask_of(const ResizeParams& p, int b) {
    Ask a;
    a.old_len = max(0, min(p.seq_lens[b], p.most));
    a.target = p.targets[b];
    const bool valid = a.target >= 0 && a.target <= p.most;
    a.grow = valid && a.target > a.old_len;
    a.shrink = valid && a.target < a.old_len;
    const int d = (a.grow || a.shrink) ? pages_of(a.target, p.ps) - pages_of(a.old_len, p.ps) : 0;
    a.need = a.grow ? d : 0;
    a.back = a.shrink ? -d : 0;
    return a;
}

// Bound by latency until there are hundreds of thousands of tokens: a decode step
// of 32 requests takes 8 us on the GPU (three sums, a bisection, dependent loads),
// 1000 requests 13 us, 1.02 million admitted tokens (12.7 MB written) 15 us.
//
// Who gets what, by three sums over the requests in order: pages asked for
// and given back, tokens of those whose pages are there, and (to close the
// gap after the first request without room for its tokens) the largest token
// sum that fits.  One CTA; thread i takes the requests [i*per, (i+1)*per).
__device__ void resize_plan(const ResizeParams& p) {
    __shared__ long long red[32];
    __shared__ long long s_fit;
    __shared__ int s_taken, s_refused;
    if (threadIdx.x == 0) {
        s_fit = 0;
        s_taken = 0;
        s_refused = 0;
    }
    int head = p.state[0];
    if (head < 0 || head >= p.N) head = (head % p.N + p.N) % p.N;
    const int free_count = max(0, min(p.state[1], p.N));
    const int per = (p.B + blockDim.x - 1) / blockDim.x;
    const int b0 = min(p.B, (int)threadIdx.x * per), b1 = min(p.B, b0 + per);

    // pages asked for (below 2^31, like the table's entries) and given back, in one sum
    long long both = 0, total;
    for (int b = b0; b < b1; ++b) {
        const Ask a = ask_of(p, b);
        both += (long long)a.need + ((long long)a.back << 32);
    }
    const long long both0 = block_exclusive_sum(both, red, &total);
    const long long need0 = both0 & 0xFFFFFFFFll, back0 = both0 >> 32, back_total = total >> 32;

    long long c = need0, added = 0;
    for (int b = b0; b < b1; ++b) {
        const Ask a = ask_of(p, b);
        c += a.need;
        if (a.grow && (a.need == 0 || c <= free_count)) added += a.target - a.old_len;
    }
    const long long added0 = block_exclusive_sum(added, red, &total);

    // the sums only grow along the requests, so those that fit are a prefix
    long long d = added0, fit = 0;
    c = need0;
    for (int b = b0; b < b1; ++b) {
        const Ask a = ask_of(p, b);
        c += a.need;
        if (a.grow && (a.need == 0 || c <= free_count)) d += a.target - a.old_len;
        if (d <= p.max_tokens) fit = d;
    }
    atomicMax((unsigned long long*)&s_fit, (unsigned long long)fit);
    __syncthreads();
    fit = s_fit;

    int refused = 0, taken = 0;
    long long r = back0;
    d = added0;
    c = need0;
    for (int b = b0; b < b1; ++b) {
        const Ask a = ask_of(p, b);
        const int first_page = (int)min(c, (long long)p.N), first_back = (int)r;
        c += a.need;
        r += a.back;
        const bool paged = a.grow && (a.need == 0 || c <= free_count);
        if (paged) d += a.target - a.old_len;
        const bool granted = paged && d <= p.max_tokens;
        if (granted && a.need) taken = (int)c;
        refused += (a.target > a.old_len && !granted) ? 1 : 0;
        const int len = granted || a.shrink ? a.target : a.old_len, start = (int)min(d, fit);
        p.plan[2 + 4 * b] = a.old_len;
        p.plan[3 + 4 * b] = len;
        p.plan[4 + 4 * b] = first_page;
        p.plan[5 + 4 * b] = first_back;
        p.lens_out[b] = len;
        p.starts[b + 1] = start;
        if (p.starts_at != p.starts) p.starts_at[b + 1] = start;
    }
    if (taken) atomicMax(&s_taken, taken);
    if (refused) atomicAdd(&s_refused, refused);
    __syncthreads();  // also: every thread has read the state, which state_out may be
    if (threadIdx.x == 0) {
        p.starts[0] = 0;
        p.starts_at[0] = 0;
        p.plan[0] = head;
        p.plan[1] = free_count;
        p.state_out[0] = ring_at(head, s_taken, p.N);
        p.state_out[1] = (int)min((long long)p.N, (long long)free_count - s_taken + back_total);
        p.state_out[2] = s_refused;
        p.state_out[3] = (int)fit;
    }
}

// Pages handed out and back (a warp per request) and the tokens' slots (a
// thread per four tokens, their request found by bisection of the starts).  Pages
// taken and pages given back lie in disjoint parts of the ring, and tables are
// written only beyond the old length, so nothing here waits for anything else.
__device__ void resize_fill(const ResizeParams& p, int cta, int ctas) {
    const int head = p.plan[0], free_count = p.plan[1];
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    for (int b = cta * warps + (threadIdx.x >> 5); b < p.B; b += ctas * warps) {
        const int old_len = p.plan[2 + 4 * b], len = p.plan[3 + 4 * b];
        const int have = pages_of(old_len, p.ps), want = pages_of(len, p.ps);
        int* row = p.table + (long long)b * p.max_pages;
        for (int j = lane; j < want - have; j += 32)
            row[have + j] = p.ring[ring_at(head, (long long)p.plan[4 + 4 * b] + j, p.N)];
        for (int j = lane; j < have - want; j += 32)
            p.ring[ring_at(head, (long long)free_count + p.plan[5 + 4 * b] + j, p.N)] = row[want + j];
    }
    const int total = p.starts_at[p.B];
    const bool vec = ((reinterpret_cast<uintptr_t>(p.slots) | reinterpret_cast<uintptr_t>(p.positions) |
                       reinterpret_cast<uintptr_t>(p.requests)) & 15) == 0;
    for (long long i0 = 4 * ((long long)cta * blockDim.x + threadIdx.x); i0 < p.max_tokens;
         i0 += 4ll * ctas * blockDim.x) {
        // the last b with starts[b] <= i0 (an empty request shares its start with the next);
        // from there on the requests follow each other
        int b = 0;
        if (i0 < total) {
            int hi = p.B - 1;
            while (b < hi) {
                const int mid = (b + hi + 1) >> 1;
                if (p.starts_at[mid] <= i0)
                    b = mid;
                else
                    hi = mid - 1;
            }
        }
        int slot[4], position[4], request[4];
        int start = p.starts_at[b], end = p.starts_at[b + 1], old_len = p.plan[2 + 4 * b], first = p.plan[4 + 4 * b];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long long i = i0 + k;
            slot[k] = position[k] = request[k] = -1;
            if (i >= total) continue;
            while (i >= end) {
                ++b;
                start = end;
                end = p.starts_at[b + 1];
                old_len = p.plan[2 + 4 * b];
                first = p.plan[4 + 4 * b];
            }
            const int at = old_len + (int)(i - start);
            request[k] = b;
            position[k] = p.base + at;
            const int page_at = at / p.ps, have = pages_of(old_len, p.ps);
            // a page taken in this call is read from the ring: the table may be written by another CTA
            const int page = page_at < have ? p.table[(long long)b * p.max_pages + page_at]
                                            : p.ring[ring_at(head, (long long)first + page_at - have, p.N)];
            if (page >= 0 && page < p.N)
                slot[k] = page * p.ps + at - page_at * p.ps;
            else
                atomicOr(p.err, kErrBadPage);
        }
        if (vec && i0 + 3 < p.max_tokens) {
            *reinterpret_cast<int4*>(p.slots + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4*>(p.positions + i0) = make_int4(position[0], position[1], position[2], position[3]);
            *reinterpret_cast<int4*>(p.requests + i0) = make_int4(request[0], request[1], request[2], request[3]);
        } else {
            for (int k = 0; k < 4 && i0 + k < p.max_tokens; ++k) {
                p.slots[i0 + k] = slot[k];
                p.positions[i0 + k] = position[k];
                p.requests[i0 + k] = request[k];
            }
        }
    }
}

// Up to a thousand tokens one CTA plans and fills (a launch costs more than
// the filling: 8.7 us for 32 requests of which each grows by a token, 12.3 for 1000 with two
// kernels) and passes the plan in shared memory; beyond, the second kernel fills with the whole GPU
// and is launched while the first still plans.  The rule does not know how many pages come back: 256
// requests of 250 pages that finish together take 119 us here and would take 14 with two kernels.
__global__ void __launch_bounds__(kSmallRequests) resize_small_kernel(ResizeParams p) {
    __shared__ int plan[2 + 4 * kSmallRequests], starts[kSmallRequests + 1];
    p.plan = plan;
    p.starts_at = starts;
    griddep_wait();
    resize_plan(p);
    __syncthreads();
    resize_fill(p, 0, 1);
}
__global__ void __launch_bounds__(kResizeThreads) resize_plan_kernel(ResizeParams p) {
    griddep_launch_dependents();
    griddep_wait();
    resize_plan(p);
}
__global__ void __launch_bounds__(kFillThreads) resize_fill_kernel(ResizeParams p) {
    griddep_wait();
    resize_fill(p, blockIdx.x, gridDim.x);
}

// ---- rotary positions ----------------------------------------------------------
struct RopeParams {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    long long q_stride, k_stride, v_stride, qo_stride;
    const int* slots;
    const int* positions;
    const double* inv_freq;
    const __nv_bfloat16* q_weight;
    const __nv_bfloat16* k_weight;
    uint32_t* err;
    float factor, eps;
    int T, nq, nkv, hd, rot, interleaved, norm;
};

// cos and sin of position * f, times the attention factor.  The angle is
// formed in turns in 64 bits and reduced there, exactly; what is left is at
// most half a turn and goes to 32 bits.
__device__ __forceinline__ float2 turn_of(int position, double f, float factor) {
    const double turns = (double)position * (f * 0.15915494309189533577);
    const float part = (float)(turns - rint(turns));
    float s, c;
    sincospif(2.f * part, &s, &c);
    return make_float2(c * factor, s * factor);
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float r = a * c - b * s;
    b = a * s + b * c;
    a = r;
}

// Bandwidth-bound: every value is read once and written once.  A CTA takes
// `tokens` tokens.  A warp takes 32 / (HD / 16) heads of one at a time, a lane two
// 16-byte chunks of a head: the two halves of eight pairs (half layout), four
// pairs in each (interleaved), or what is not turned; neighbouring lanes have
// neighbouring chunks (two chunks side by side in a lane would touch every
// 32-byte sector twice).  The loads of two such items are issued first; the
// angles of the CTA's tokens are computed, once for all heads, while they are in
// flight.  8191 tokens of 32 heads of 256 (268 MB): 50 us, 5.3 TB/s; 256 tokens 10
// us, 4 of them on the GPU.  Cosines in registers instead (computed per warp) took 128 registers
// and, at 16 warps an SM, 73 us.
constexpr int kRopeTable = 2048;  // cosines and sines a CTA keeps
template <typename T, int HD>
__global__ void __launch_bounds__(256, 4) rope_vec_kernel(RopeParams p, PagedView<T> kv, int tokens) {
    constexpr int I = HD / 16, H = 32 / I;  // lanes of a head, heads of an item
    constexpr int U = 2;
    __shared__ __align__(16) float2 table[kRopeTable];
    __shared__ long long cells[16];  // of the CTA's tokens in the pool; -1: padding
    const int lane = threadIdx.x & 31, li = lane % I, sub = lane / I, warp = threadIdx.x >> 5;
    const int heads = p.nq + 2 * p.nkv, passes = (heads + H - 1) / H;
    const int t0 = blockIdx.x * tokens, items = min(tokens, p.T - t0) * passes;
    const int half = p.rot >> 1, turned = p.rot / 16;  // lanes [0, turned) turn
    int c0, c1;  // first elements of the two chunks
    if (p.interleaved) {
        c0 = li * 8;
        c1 = HD / 2 + li * 8;
    } else if (li < turned) {
        c0 = li * 8;
        c1 = half + li * 8;
    } else {
        c0 = p.rot + (li - turned) * 8;
        c1 = c0 + (HD - p.rot) / 2;
    }
    uint4 a[U], b[U];
    auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int item = base + u * 8 + warp;
            a[u] = b[u] = make_uint4(0u, 0u, 0u, 0u);
            if (item >= items) continue;
            const int local = tokens == 1 ? 0 : item / passes, t = t0 + local, h = (item - local * passes) * H + sub;
            if (h < heads) {
                const T* src = h < p.nq ? static_cast<const T*>(p.q) + t * p.q_stride + (long long)h * HD
                               : h < p.nq + p.nkv
                                   ? static_cast<const T*>(p.k) + t * p.k_stride + (long long)(h - p.nq) * HD
                                   : static_cast<const T*>(p.v) + t * p.v_stride + (long long)(h - p.nq - p.nkv) * HD;
                a[u] = __ldcs(reinterpret_cast<const uint4*>(src + c0));
                b[u] = __ldcs(reinterpret_cast<const uint4*>(src + c1));
            }
        }
    };
    griddep_wait();
    load(0);
    for (int local = warp; local < min(tokens, p.T - t0); local += 8) {
        if (lane == 0) {
            const int slot = p.slots[t0 + local];
            long long cell = -1;
            if (slot >= kv.num_pages * kv.page_size) {
                atomicOr(p.err, kErrBadPage);
            } else if (slot >= 0) {
                const int page = slot / kv.page_size;
                cell = page * kv.page_stride + (slot - page * kv.page_size) * kv.pos_stride;
            }
            cells[local] = cell;
        }
    }
    if (tokens == 1) {
        for (int i = threadIdx.x; i < half; i += 256) table[i] = turn_of(p.positions[t0], p.inv_freq[i], p.factor);
    } else {
        for (int local = warp; local < min(tokens, p.T - t0); local += 8)
            for (int i = lane; i < half; i += 32)
                table[local * half + i] = turn_of(p.positions[t0 + local], p.inv_freq[i], p.factor);
    }
    __syncthreads();
    for (int base = 0; base < items; base += U * 8) {
        if (base) load(base);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int item = base + u * 8 + warp;
            if (item >= items) break;  // the same for the whole warp
            const int local = tokens == 1 ? 0 : item / passes, t = t0 + local, h = (item - local * passes) * H + sub;
            const int which = h < p.nq ? 0 : (h < p.nq + p.nkv ? 1 : 2);
            const long long cell = cells[local];
            float x[8], y[8], sum = 0.f;
            const T* ea = reinterpret_cast<const T*>(&a[u]);
            const T* eb = reinterpret_cast<const T*>(&b[u]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = to_float(ea[i]);
                y[i] = to_float(eb[i]);
                sum = fmaf(x[i], x[i], sum);
                sum = fmaf(y[i], y[i], sum);
            }
            if (p.norm) {
#pragma unroll
                for (int o = 1; o < I; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const float inv = rsqrtf(sum / (float)HD + p.eps);
                const __nv_bfloat16* wt = which == 0 ? p.q_weight : (which == 1 ? p.k_weight : nullptr);
                uint4 w0 = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u), w1 = w0;  // ones
                if (wt) {
                    w0 = *reinterpret_cast<const uint4*>(wt + c0);
                    w1 = *reinterpret_cast<const uint4*>(wt + c1);
                }
                const uint32_t* e0 = reinterpret_cast<const uint32_t*>(&w0);
                const uint32_t* e1 = reinterpret_cast<const uint32_t*>(&w1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[2 * i] *= inv * __uint_as_float(e0[i] << 16);
                    x[2 * i + 1] *= inv * __uint_as_float(e0[i] & 0xFFFF0000u);
                    y[2 * i] *= inv * __uint_as_float(e1[i] << 16);
                    y[2 * i + 1] *= inv * __uint_as_float(e1[i] & 0xFFFF0000u);
                }
            }
            const float2* cs = table + local * half;
            if (which < 2) {
                if (p.interleaved) {
                    if (c0 < p.rot) {
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            const float4 w = *reinterpret_cast<const float4*>(cs + c0 / 2 + i);
                            turn(x[2 * i], x[2 * i + 1], w.x, w.y);
                            turn(x[2 * i + 2], x[2 * i + 3], w.z, w.w);
                        }
                    }
                    if (c1 < p.rot) {
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            const float4 w = *reinterpret_cast<const float4*>(cs + c1 / 2 + i);
                            turn(y[2 * i], y[2 * i + 1], w.x, w.y);
                            turn(y[2 * i + 2], y[2 * i + 3], w.z, w.w);
                        }
                    }
                } else if (li < turned) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float4 w = *reinterpret_cast<const float4*>(cs + li * 8 + i);
                        turn(x[i], y[i], w.x, w.y);
                        turn(x[i + 1], y[i + 1], w.z, w.w);
                    }
                }
            }
            if (h >= heads || (cell < 0 && which)) continue;
            T* dst = which == 0 ? static_cast<T*>(p.q_out) + t * p.qo_stride + (long long)h * HD
                     : which == 1 ? kv.k + cell + (h - p.nq) * kv.head_stride
                                  : kv.v + cell + (h - p.nq - p.nkv) * kv.head_stride;
            uint32_t r[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r[i] = cell < 0 ? 0u : pack2<T>(x[2 * i], x[2 * i + 1]);
                r[i + 4] = cell < 0 ? 0u : pack2<T>(y[2 * i], y[2 * i + 1]);
            }
            *reinterpret_cast<uint4*>(dst + c0) = make_uint4(r[0], r[1], r[2], r[3]);
            *reinterpret_cast<uint4*>(dst + c1) = make_uint4(r[4], r[5], r[6], r[7]);
        }
    }
}

// Any head size, pairs that no 16-byte boundary meets, rows of any alignment: one
// CTA per token, a warp per head, a row in shared memory.
template <typename T>
__global__ void __launch_bounds__(128) rope_kernel(RopeParams p, PagedView<T> kv) {
    __shared__ float2 turn[kMaxPagedHeadDim / 2];
    __shared__ float row[4][kMaxPagedHeadDim];
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_wait();
    int slot = p.slots[t];
    if (slot >= kv.num_pages * kv.page_size) {
        if (threadIdx.x == 0) atomicOr(p.err, kErrBadPage);
        slot = -1;
    }
    const int half = p.rot >> 1;
    for (int i = threadIdx.x; i < half; i += blockDim.x) turn[i] = turn_of(p.positions[t], p.inv_freq[i], p.factor);
    __syncthreads();
    const long long cell = slot < 0 ? 0
                                    : (long long)(slot / kv.page_size) * kv.page_stride +
                                          (long long)(slot % kv.page_size) * kv.pos_stride;
    float* x = row[warp];
    for (int h = warp; h < p.nq + 2 * p.nkv; h += 4) {
        const int which = h < p.nq ? 0 : (h < p.nq + p.nkv ? 1 : 2);
        const int kh = h - p.nq - (which == 2 ? p.nkv : 0);
        if (slot < 0 && which) break;
        const T* src = which == 0 ? static_cast<const T*>(p.q) + t * p.q_stride + (long long)h * p.hd
                                  : (which == 1 ? static_cast<const T*>(p.k) + t * p.k_stride
                                                : static_cast<const T*>(p.v) + t * p.v_stride) +
                                        (long long)kh * p.hd;
        T* dst = which == 0 ? static_cast<T*>(p.q_out) + t * p.qo_stride + (long long)h * p.hd
                            : (which == 1 ? kv.k : kv.v) + cell + kh * kv.head_stride;
        if (slot < 0) {
            for (int e = lane; e < p.hd; e += 32) dst[e] = from_float<T>(0.f);
            continue;
        }
        float sum = 0.f;
        for (int e = lane; e < p.hd; e += 32) {
            x[e] = to_float(src[e]);
            sum = fmaf(x[e], x[e], sum);
        }
        if (p.norm) {
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float inv = rsqrtf(sum / (float)p.hd + p.eps);
            const __nv_bfloat16* w = which == 0 ? p.q_weight : (which == 1 ? p.k_weight : nullptr);
            for (int e = lane; e < p.hd; e += 32) x[e] = w ? x[e] * inv * __bfloat162float(w[e]) : x[e] * inv;
        }
        __syncwarp();
        const int turned = which == 2 ? 0 : half;
        for (int i = lane; i < turned; i += 32) {
            const int a = p.interleaved ? 2 * i : i, b = p.interleaved ? 2 * i + 1 : i + half;
            const float2 cs = turn[i];
            const float x0 = x[a], x1 = x[b];
            dst[a] = from_float<T>(x0 * cs.x - x1 * cs.y);
            dst[b] = from_float<T>(x0 * cs.y + x1 * cs.x);
        }
        for (int e = 2 * turned + lane; e < p.hd; e += 32) dst[e] = from_float<T>(x[e]);
        __syncwarp();
    }
}

template <typename T>
tf_status launch_rope(tf_context* ctx, const RopeParams& p, const tf_paged_kv* kv, cudaStream_t cs, const char* name) {
    const PagedView<T> view = paged_view<T>(kv);
    // whole chunks: a power-of-two head size, halves (or pairs) of 16-byte chunks, aligned rows
    const bool chunks = (p.hd == 64 || p.hd == 128 || p.hd == 256 || p.hd == 512) && p.rot % (p.interleaved ? 8 : 16) == 0;
    const bool aligned = aligned16(p.q_weight) && aligned16(p.k_weight) && aligned16(p.q) && aligned16(p.k) && aligned16(p.v) && aligned16(p.q_out) &&
                         (p.T == 1 || (p.q_stride | p.k_stride | p.v_stride | p.qo_stride) % 8 == 0);
    if (!chunks || !aligned) {
        return cuda_check(ctx, launch_overlapped(rope_kernel<T>, p.T, 128, 0, cs, p, view), name);
    }
    // sixteen items a CTA (two a warp, all loads in flight), but a CTA a token while that
    // does not fill the GPU
    const int H = 512 / p.hd, passes = (p.nq + 2 * p.nkv + H - 1) / H;
    const int fit = std::min(16 / std::min(passes, 16), p.rot ? kRopeTable / std::max(1, p.rot / 2) : 16);
    const int tokens = std::max(1, std::min<int>(fit, (int)(p.T / (4ll * ctx->num_sms))));
    const unsigned ctas = (unsigned)(((long long)p.T + tokens - 1) / tokens);
    auto* kernel = p.hd == 64    ? rope_vec_kernel<T, 64>
                   : p.hd == 128 ? rope_vec_kernel<T, 128>
                   : p.hd == 256 ? rope_vec_kernel<T, 256>
                                 : rope_vec_kernel<T, 512>;
    return cuda_check(ctx, launch_overlapped(kernel, ctas, 256, 0, cs, p, view, tokens), name);
}

}  // namespace

extern "C" {

size_t tf_kv_pages_workspace_bytes(uint32_t num_requests) { return (2 + 4 * (size_t)num_requests) * sizeof(int); }

tf_status tf_kv_pages_resize(tf_context* ctx, const void* seq_lens, const void* targets, uint32_t num_requests,
                             void* page_table, uint32_t max_pages, void* free_ring, uint32_t num_pages,
                             const void* free_state, uint32_t page_size, uint32_t position_base, void* seq_lens_out,
                             void* free_state_out, void* token_starts, void* slots, void* positions, void* requests,
                             uint32_t max_tokens, void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "tf_kv_pages_resize";
    tf_status s = enter(ctx, name);
    if (s) return s;
    if (num_requests == 0 || max_pages == 0 || num_pages == 0 || page_size == 0)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: requests, pages per request, pages and page size above 0", name);
    if ((uint64_t)num_pages * page_size > 0x7FFFFFFFull || (uint64_t)num_requests * max_pages > 0x7FFFFFFFull ||
        (uint64_t)max_pages * page_size + position_base > 0x7FFFFFFFull || max_tokens > 0x7FFFFFFFu ||
        num_requests > 0x7FFFFFFu)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE,
                    "%s: slots, table entries, positions and tokens must be below 2^31", name);
    const void* all[] = {seq_lens, targets, page_table, free_ring, free_state, seq_lens_out, free_state_out,
                         token_starts, workspace};
    for (const void* ptr : all) {
        if (!ptr) return fail(ctx, TF_ERR_INVALID_ARG, "%s: null pointer", name);
        if (!aligned4(ptr)) return fail(ctx, TF_ERR_MISALIGNED, "%s: pointers must be 4-byte aligned", name);
    }
    if (max_tokens && (!slots || !positions || !requests))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: null pointer", name);
    if (!aligned4(slots) || !aligned4(positions) || !aligned4(requests))
        return fail(ctx, TF_ERR_MISALIGNED, "%s: pointers must be 4-byte aligned", name);
    if (workspace_bytes < tf_kv_pages_workspace_bytes(num_requests))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes,
                    tf_kv_pages_workspace_bytes(num_requests));
    ResizeParams p;
    p.seq_lens = static_cast<const int*>(seq_lens);
    p.targets = static_cast<const int*>(targets);
    p.table = static_cast<int*>(page_table);
    p.ring = static_cast<int*>(free_ring);
    p.state = static_cast<const int*>(free_state);
    p.lens_out = static_cast<int*>(seq_lens_out);
    p.state_out = static_cast<int*>(free_state_out);
    p.starts = static_cast<int*>(token_starts);
    p.slots = static_cast<int*>(slots);
    p.positions = static_cast<int*>(positions);
    p.requests = static_cast<int*>(requests);
    p.plan = static_cast<int*>(workspace);
    p.starts_at = p.starts;
    p.err = ctx->d_err;
    p.B = (int)num_requests;
    p.max_pages = (int)max_pages;
    p.N = (int)num_pages;
    p.ps = (int)page_size;
    p.base = (int)position_base;
    p.max_tokens = (int)max_tokens;
    p.most = (int)(max_pages * page_size);
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    if (max_tokens <= kSmallTokens && num_requests <= kSmallRequests) {
        return cuda_check(ctx, launch_overlapped(resize_small_kernel, 1, kSmallRequests, 0, cs, p), name);
    }
    const long long work = std::max<long long>(((long long)max_tokens + 3) / 4, 32ll * num_requests);
    const unsigned ctas = (unsigned)std::min<long long>((work + kFillThreads - 1) / kFillThreads, 8ll * ctx->num_sms);
    cudaError_t e = launch_overlapped(resize_plan_kernel, 1, kResizeThreads, 0, cs, p);
    if (e == cudaSuccess) e = launch_overlapped(resize_fill_kernel, ctas, kFillThreads, 0, cs, p);
    return cuda_check(ctx, e, name);
}

tf_status tf_rope_frequencies(uint32_t rotary_dim, double theta, tf_rope_scaling scaling, double factor,
                              double original_context, double low, double high, double* inv_freq,
                              double* attention_factor) {
    if (!inv_freq || !attention_factor || rotary_dim == 0 || rotary_dim % 2 || !(theta > 0.0)) return TF_ERR_INVALID_ARG;
    const bool scaled = scaling != TF_ROPE_SCALE_NONE;
    if (scaled && !(factor > 0.0)) return TF_ERR_INVALID_ARG;
    const bool by_context = scaling == TF_ROPE_SCALE_RAMP || scaling == TF_ROPE_SCALE_BANDS;
    if (by_context && (!(original_context > 0.0) || !(high > low) || !(low > 0.0))) return TF_ERR_INVALID_ARG;
    if (scaling == TF_ROPE_SCALE_RAMP && theta == 1.0) return TF_ERR_INVALID_ARG;  // every pair turns alike
    if (scaling < TF_ROPE_SCALE_NONE || scaling > TF_ROPE_SCALE_BANDS) return TF_ERR_INVALID_ARG;
    const double rot = rotary_dim, tau = 6.283185307179586476925;
    if (scaling == TF_ROPE_SCALE_BASE) {
        if (rotary_dim <= 2) return TF_ERR_UNSUPPORTED_SHAPE;
        theta *= pow(factor, rot / (rot - 2.0));
    }
    *attention_factor = 1.0;
    double ramp_lo = 0, ramp_hi = 0;
    if (scaling == TF_ROPE_SCALE_RAMP) {
        // the pair that makes `turns` turns over the original context
        auto pair_of = [&](double turns) { return rot * log(original_context / (turns * tau)) / (2.0 * log(theta)); };
        ramp_lo = fmax(floor(pair_of(high)), 0.0);
        ramp_hi = fmin(ceil(pair_of(low)), rot - 1.0);
        *attention_factor = factor > 1.0 ? 0.1 * log(factor) + 1.0 : 1.0;
    }
    for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
        const double f = pow(theta, -2.0 * i / rot);
        double slowed = 0.0;  // share of the frequency that is divided by the factor
        if (scaling == TF_ROPE_SCALE_LINEAR) slowed = 1.0;
        if (scaling == TF_ROPE_SCALE_RAMP) slowed = (i - ramp_lo) / fmax(ramp_hi - ramp_lo, 1e-3);
        if (scaling == TF_ROPE_SCALE_BANDS) slowed = 1.0 - (original_context * f / tau - low) / (high - low);
        slowed = fmin(fmax(slowed, 0.0), 1.0);
        inv_freq[i] = slowed > 0.0 ? f / factor * slowed + f * (1.0 - slowed) : f;
    }
    return TF_OK;
}

tf_status tf_rope_kv_write(tf_context* ctx, const void* q, uint64_t q_stride, const void* k, uint64_t k_stride,
                           const void* v, uint64_t v_stride, void* q_out, uint64_t q_out_stride, const tf_paged_kv* kv,
                           const void* slots, const void* positions, const void* inv_freq, uint32_t rotary_dim,
                           tf_rope_layout layout, float attention_factor, int norm, const void* q_weight,
                           const void* k_weight, float eps, uint32_t T, uint32_t num_q_heads, void* stream) {
    const char* name = "tf_rope_kv_write";
    tf_status s = enter(ctx, name);
    if (s) return s;
    s = check_paged_kv(ctx, kv, name);
    if (s) return s;
    if (rotary_dim % 2 || rotary_dim > kv->head_dim)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: rotary_dim must be even and at most head_dim", name);
    if (layout != TF_ROPE_HALF && layout != TF_ROPE_INTERLEAVED)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: unknown layout", name);
    if (T > 0x7FFFFFFFu || num_q_heads > 0xFFFFu || kv->num_kv_heads > 0xFFFFu)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: too many tokens or heads", name);
    if (norm && !(eps >= 0.f)) return fail(ctx, TF_ERR_INVALID_ARG, "%s: eps must not be negative", name);
    if (T == 0) return TF_OK;
    const uint64_t qw = (uint64_t)num_q_heads * kv->head_dim, kw = (uint64_t)kv->num_kv_heads * kv->head_dim;
    if (!k || !v || !slots || !positions || (rotary_dim && !inv_freq) || (num_q_heads && (!q || !q_out)))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: null pointer", name);
    if (T > 1 && (k_stride < kw || v_stride < kw || q_stride < qw || q_out_stride < qw))
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: token strides below the heads' width", name);
    if (!aligned2(q) || !aligned2(k) || !aligned2(v) || !aligned2(q_out) || !aligned4(slots) || !aligned4(positions) ||
        (reinterpret_cast<uintptr_t>(inv_freq) & 7u) || !aligned2(q_weight) || !aligned2(k_weight))
        return fail(ctx, TF_ERR_MISALIGNED, "%s: a pointer is not aligned to its type", name);
    RopeParams p;
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_out = q_out;
    p.q_stride = (long long)q_stride;
    p.k_stride = (long long)k_stride;
    p.v_stride = (long long)v_stride;
    p.qo_stride = (long long)q_out_stride;
    p.slots = static_cast<const int*>(slots);
    p.positions = static_cast<const int*>(positions);
    p.inv_freq = static_cast<const double*>(inv_freq);
    p.q_weight = static_cast<const __nv_bfloat16*>(q_weight);
    p.k_weight = static_cast<const __nv_bfloat16*>(k_weight);
    p.err = ctx->d_err;
    p.factor = attention_factor;
    p.eps = eps;
    p.T = (int)T;
    p.nq = (int)num_q_heads;
    p.nkv = (int)kv->num_kv_heads;
    p.hd = (int)kv->head_dim;
    p.rot = (int)rotary_dim;
    p.interleaved = layout == TF_ROPE_INTERLEAVED;
    p.norm = norm != 0;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    return kv->dtype == TF_DTYPE_F16 ? launch_rope<__half>(ctx, p, kv, cs, name)
                                     : launch_rope<__nv_bfloat16>(ctx, p, kv, cs, name);
}

}  // extern "C"

// tf_prefix_kernels.cuh -- the kernels of tf_shared_prefix_attention and (kTree) tf_tree_attention
// and their launch: attention of a ragged batch behind a shared prefix, over a paged cache.
//
// For a query row at position p, with the keys split in any way into parts i:
//   m_i = max s, d_i = sum e^(s - m_i), o_i = sum e^(s - m_i) v   over the part's visible keys,
//   M = max m_i, D = sum d_i e^(m_i - M), out = sum o_i e^(m_i - M) / D, lse = M + log D,
// so the shared prefix can be one part and the request's own pages another: the
// prefix is read once for the rows of the whole batch (by the tensor cores, or by
// the streaming warps when there are few rows), own keys once each.
//   attention_parts_kernel   all parts of all rows, one CTA per SM, two kinds of work
//   join_parts_kernel        M, D, out and lse of every row that has more than one part
// Measured with both (16 query / 8 KV heads of 256): 256 requests behind 4096
// shared positions with 1 to 1001 of their own, 1.09 GB: 215 to 221 us by machine,
// 5.0 TB/s; 32 behind 2048 with up to 2048, 286 MB: 70 us; 2 behind 317: 18 us (17
// on the GPU: launch, sums over the batch, one unit, join).
#pragma once
#include <math.h>

#include "tf_prefix_stream.cuh"
#include "tf_prefix_tensor.cuh"

namespace tf {
namespace {

constexpr int kThreads = 256;  // of the parts kernel: 8 warps, 255 registers a thread
constexpr int kJoinRows = 128;  // rows a joining CTA looks at, at most

// One warp, one row, key by key: the definition.  Only for rows whose joined
// result is not finite: an infinity or NaN in a key that the row does not see,
// but a neighbour in its tile does, reaches the tile's product as 0 * inf; here
// such a key is not read.
template <typename T, bool kTree>
__device__ __noinline__ void attend_alone(const AttnParams<T, kTree>& p, int b, const Request& r, int j, int h) {
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
    const int end = kTree ? p.prefix_len + r.len : hi, node0 = p.prefix_len + r.len - r.n;
    // (kTree: positions far ahead leave nothing of the history, and the nodes all the same)
    for (int pos = kTree ? min(lo, hi) : lo; pos < end; ++pos) {
        if (kTree && pos >= hi && !sees_node(p.ancestors + (long long)t * p.words, p.words, pos - node0)) continue;
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

// Nanoseconds of an SM that a unit takes, for dealing the SMs to the two kinds
// of work.  A streamed unit is bound by memory: 16 keys of K and V at an SM's
// share of the bandwidth (6450 / 148 bytes a nanosecond).  A tensor unit is 64
// (head_dim 256) or 128 keys for 128 rows: 600 ns by itself, but beside the
// stream its loads take their turn behind the others': 1700 measured, 2300 for 128 keys of 128.
// Fits, not laws; halved / as they are / doubled (us, cold, with a graph's launch):
//   256: 32 decodes behind 2048, 1-2047 own     111 /  84 /  78     128, 1-200   76 / 68 / 82 (behind 4096)
//        256 behind 4096, 1-1000 own            359 / 244 / 248
//   128: 101 behind 1500, 0-900 own              70 /  57 /  61     128, 1-200   45 / 55 / 70
//        256 behind 4096, 1-1000 own            125 / 127 / 142
//    64: 101 behind 1500, 0-900 own              47 /  41 /  43     128, 1-200   41 / 45 / 53
//        256 behind 4096, 1-1000 own             76 /  78 /  86
__host__ __device__ constexpr float few_unit_ns(int hd) { return 16.f * 4.f * hd / 43.6f; }
__host__ __device__ constexpr float many_unit_ns(int hd) { return hd > 128 ? 1700.f : (hd > 64 ? 2300.f : 900.f); }

// kTree: which segment unit u0 is in, where that begins and what its row tiles have; told by the one
// thread that has it among its requests [b0, b1), whose first unit is `before`.
template <typename T, int HD>
__device__ __forceinline__ void find_tree_segment(const AttnParams<T, true>& p, int u0, int b0, int b1, int before,
                                                  int& seg, int& at, int& units) {
    const TreeSegment prefix = tree_segment<T, HD>(p, -1);
    if (threadIdx.x == 0 && u0 < tree_slots(p, prefix)) {
        seg = -1;
        at = 0;
        units = prefix.units;
    }
    for (int b = b0; b < b1; ++b) {
        const TreeSegment s = tree_segment<T, HD>(p, b);
        const int slots = tree_slots(p, s);
        if (u0 >= before && u0 < before + slots) {
            seg = b;
            at = before;
            units = s.units;
        }
        before += slots;
    }
}

// All parts of all rows, one CTA per SM.  Every CTA sums the units of both kinds
// over the batch and finds its share: the first CTAs take the tensor cores' jobs,
// as many as these need to finish when the others have streamed the rest.
// kTensor false: a batch with nothing for the tensor cores, without their 100 KB of
// code (a small call's time is launch, instruction fetches and dependent loads).
template <typename T, int HD, int NT, bool kTensor, bool kTree>
__global__ void __launch_bounds__(kThreads, 1) attention_parts_kernel(const __grid_constant__ AttnParams<T, kTree> p) {
    using S = StreamShape<HD, NT>;
    extern __shared__ uint8_t raw[];
    __shared__ int red[32], s_seg[S::kWarps], s_at[S::kWarps], s_begin[S::kWarps], s_tile, s_tile_at, s_tile_units;
    __shared__ __align__(8) uint64_t full[S::kBars];
    const uint32_t smem = (smem_u32(raw) + 1023u) & ~1023u;
    griddep_wait();
    griddep_launch_dependents();  // the joining kernel may read what this one may
    const int grid = gridDim.x, cta = blockIdx.x;

    // thread i looks after requests [i*per, (i+1)*per) and a share of the row tiles
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(p.B, (int)threadIdx.x * per), b1 = min(p.B, b0 + per);
    int few_before, many_before = 0, many = 0, i0 = 0, i1 = 0, per_row_tile = 0;
    const int few = stream_units<T, HD, NT>(p, red, b0, b1, few_before);
    if (p.window && cta == 0 && threadIdx.x == 0) *p.prefix_first = prefix_first(p);
    if constexpr (kTensor && kTree) {
        many = all_tree_units<T, HD>(p, red, b0, b1, many_before);
    } else if constexpr (kTensor) {
        const bool own = p.max_query * p.G > p.many_above;  // requests may have own keys here
        if (!own && !p.prefix_few) {
            // the prefix alone: the same for every row tile with a token of the batch
            const int live = (int)(((long long)max(0, min(p.starts[p.B], p.T_tokens)) * p.G + kTcRows - 1) / kTcRows);
            per_row_tile = tensor_units<T, HD>(p, 0) * p.nkv;
            many = live * per_row_tile;
        } else if (own) {
            const int row_tiles = (int)(((long long)p.T_tokens * p.G + kTcRows - 1) / kTcRows);
            const int per_tile = (row_tiles + kThreads - 1) / kThreads;
            i0 = min(row_tiles, (int)threadIdx.x * per_tile);
            i1 = min(row_tiles, i0 + per_tile);
            many = all_tensor_units<T, HD>(p, red, i0, i1, many_before);
        }
    }
    int many_ctas = 0;
    if (many) {
        const float m = many * many_unit_ns(HD);
        float f = few * few_unit_ns(HD);
        // a small share: its warps wait for latencies, not for bandwidth (256 decodes behind 4096 with
        // 1 to 30 own positions, head_dim 64: 45 us, 59 without; other batches the same, also with six)
        if (f * 10.f < m) f *= 3.f;
        many_ctas = few ? max(1, min(grid - 1, (int)(grid * (m / (m + f))))) : grid;
        many_ctas = min(many_ctas, many);
    }
    // no worker without a unit (a part is read back for every worker between a job's
    // first and last), and two at least where there are: a part more costs the joining
    // kernel about what a unit costs here; few workers are spread over the CTAs
    const int few_ctas = grid - many_ctas, workers = min((few + 1) / 2, few_ctas * S::kWarps);
    if (cta < many_ctas) {
        if constexpr (kTensor) {
            __shared__ TensorBarriers bar;
            const int u0 = unit_begin(cta, many, many_ctas), u1 = unit_begin(cta + 1, many, many_ctas);
            if constexpr (kTree) {
                find_tree_segment<T, HD>(p, u0, b0, b1, many_before, s_tile, s_tile_at, s_tile_units);
            } else if (per_row_tile) {
                if (threadIdx.x == 0) {
                    s_tile = u0 / per_row_tile;
                    s_tile_at = u0 / per_row_tile * per_row_tile;
                    s_tile_units = per_row_tile / p.nkv;
                }
            } else {
                int at = many_before;
                for (int i = i0; i < i1; ++i) {
                    const int units = tensor_units<T, HD>(p, i);
                    if (u0 >= at && u0 < at + units * p.nkv) {
                        s_tile = i;
                        s_tile_at = at;
                        s_tile_units = units;
                    }
                    at += units * p.nkv;
                }
            }
            __syncthreads();
            tensor_cta<T, HD>(p, smem, bar, u0, u1, s_tile, s_tile_at, s_tile_units, cta);
        }
        return;
    }
    const int mine = cta - many_ctas;  // this CTA's workers: mine, mine + few_ctas, ...
    if (mine >= workers) return;
    if (threadIdx.x < S::kWarps) s_begin[threadIdx.x] = unit_begin(min(mine + (int)threadIdx.x * few_ctas, workers), few, workers);
    __syncthreads();
    {
        StreamCursor c;
        c.seg = -1;
        stream_segment<T, HD, NT>(p, c);
        const int prefix_units = c.row_tiles * c.tiles * p.nkv;
        if (threadIdx.x < S::kWarps && s_begin[threadIdx.x] < prefix_units) {
            s_seg[threadIdx.x] = -1;
            s_at[threadIdx.x] = 0;
        }
        int at = few_before;
        for (c.seg = b0; c.seg < b1; ++c.seg) {
            stream_segment<T, HD, NT>(p, c);
            const int units = c.row_tiles * c.tiles * p.nkv;
            for (int w = 0; units && w < S::kWarps; ++w) {
                const int u = s_begin[w];
                if (u >= at && u < at + units) {
                    s_seg[w] = c.seg;
                    s_at[w] = at;
                }
            }
            at += units;
        }
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kBars; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5;
    const int worker = mine + warp * few_ctas;
    if (warp >= S::kWarps || worker >= workers) return;
    const int u0 = s_begin[warp], u1 = unit_begin(worker + 1, few, workers);
    StreamCursor cur;
    cur.seg = s_seg[warp];
    stream_segment<T, HD, NT>(p, cur);
    const int in = u0 - s_at[warp];
    cur.tile = in % cur.tiles;
    cur.rt = in / cur.tiles % cur.row_tiles;
    cur.kvh = in / cur.tiles / cur.row_tiles;
    stream_warp<T, HD, NT>(p, smem + warp * S::kTiles * S::kTile, full + warp * S::kTiles, cur, u0, u1, worker);
}

// kTree, requests of more than eight rows among them: everything on the tensor cores, without the
// streaming warps' code and without counting their units.  A few requests of one or two nodes beside
// such trees stream no faster than this (61 requests of 1 to 5 nodes, eight query heads a KV head: 55
// us with those of one node streamed, their warps ending long after the tiles, 39 this way); 200
// requests of which one has more take 225 instead of 156 us (16 / 8 heads of 256).
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) tree_tiles_kernel(const __grid_constant__ AttnParams<T, true> p) {
    extern __shared__ uint8_t raw[];
    __shared__ int red[32], s_seg, s_at, s_units;
    __shared__ TensorBarriers bar;
    griddep_wait();
    griddep_launch_dependents();  // the joining kernel may read what this one may
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min(p.B, (int)threadIdx.x * per), b1 = min(p.B, b0 + per);
    if (p.window) {  // the first prefix position that any row sees
        if (threadIdx.x == 0) shared_prefix_first() = p.prefix_len;
        __syncthreads();
        int first = p.prefix_len;
        for (int b = b0; b < b1; ++b) {
            const Request r = request_of(p, b);
            if (r.used) first = min(first, seen_from(p, r));
        }
        if (first < p.prefix_len) atomicMin(&shared_prefix_first(), first);
        __syncthreads();
        if (blockIdx.x == 0 && threadIdx.x == 0) *p.prefix_first = prefix_first(p);
    }
    int before;
    const int units = all_tree_units<T, HD>(p, red, b0, b1, before), ctas = min((int)gridDim.x, units), cta = blockIdx.x;
    if (cta >= ctas) return;
    const int u0 = unit_begin(cta, units, ctas), u1 = unit_begin(cta + 1, units, ctas);
    find_tree_segment<T, HD>(p, u0, b0, b1, before, s_seg, s_at, s_units);
    __syncthreads();
    tensor_cta<T, HD>(p, (smem_u32(raw) + 1023u) & ~1023u, bar, u0, u1, s_seg, s_at, s_units, cta);
}

// The parts of one row: own keys' first and cont, then (prefix or tensor
// cores') first and cont; cont places are a worker's rows apart.
struct RowParts {
    int n[4], place[4];
    bool own_many;  // kTree: the own keys' parts are the tensor cores'
    int row;
    int b, j;  // request and token in it; b = the batch's size: a row of zeros
};

// The workers of a row's parts are among those that there are places for.  They always are where
// a worker has written them; where none has (a wait gave up), the workspace may hold anything.
__device__ __forceinline__ bool parts_exist(const Parts& p, int first_of, int last_of) {
    const int first = first_of >> p.shift;
    return first >= 0 && last_of >= first && last_of < p.places;
}

// Joins the parts of every row.  A thread finds the parts of a row (rows that
// are finished drop out; the others in any order), a warp adds them up.  Bound by
// latency: two rounds of dependent loads to find a row's parts, then two for each
// row of a warp.  So as many CTAs as fit: 3 an SM with 32 registers of loads in
// flight (58,000 rows of which a third have two parts, with the parts kernel: 205
// us; 218 with 2 an SM and twice the loads; 229 without dropping finished rows
// before the warps take theirs; by itself, cold, 29 us).
template <typename T, int HD, bool kTree>
__global__ void __launch_bounds__(256, 3) join_parts_kernel(const __grid_constant__ AttnParams<T, kTree> p, int rows_per_cta) {
    __shared__ RowParts rows[kJoinRows];
    __shared__ int left;
    const int lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * rows_per_cta, n_rows = min(rows_per_cta, p.T_tokens * p.nq - row0);
    if (threadIdx.x == 0) left = 0;
    __syncthreads();
    const int row = row0 + threadIdx.x;
    const bool mine = threadIdx.x < n_rows;  // (a thread for each: kJoinRows <= threads)
    static_assert(kJoinRows <= 256);
    RowParts x = {};
    Request r = {};
    bool many = false, own = false, seen = false;
    x.b = p.B;
    if (mine) {
        // what the caller wrote is complete: the parts kernel lets this one start after its own wait
        const int t = row / p.nq;
        // most batches have one token a request, and then b = t
        x.b = min(t, p.B - 1);
        if (!(p.starts[x.b] <= t && t < p.starts[x.b + 1])) x.b = request_at(p, t);
        if (x.b < p.B) {
            r = request_of(p, x.b);
            x.j = t - r.start;
            if (x.j < 0) x.b = p.B;  // before the first request: a row of zeros
        }
        if (x.b < p.B) {
            int lo, hi;
            seen_by(p, r, x.j, lo, hi);
            many = is_many(p, r);
            own = (kTree || !many) && r.len > own_lo(p, r);
            seen = hi > lo;
        }
    }
    griddep_wait();
    if (mine) {
        bool done = false;
        x.row = row;
        // (read together, used where it is there)
        const Parts& second = p.prefix_few ? p.few : p.many;  // whose places the second two parts have
        const int own_first = p.few.first_of[row], own_last = p.few.last_of[row];
        const int other_first = p.many.first_of[row], other_last = p.many.last_of[row];
        const float mark = (kTree ? p.few : p.many).first_md[row].x;
        const bool other =
            x.b < p.B && (p.prefix_len > (p.window ? *p.prefix_first : 0) || (!kTree && many && seen));
        const bool lost = (own && !parts_exist(kTree && many ? p.many : p.few, own_first, own_last)) ||
                          (other && !parts_exist(second, other_first, other_last));
        if (x.b < p.B && (x.j >= r.used || lost)) {
            atomicOr(p.err, kErrBadPage);
            x.b = p.B;
        } else if (x.b < p.B) {
            if (own) {
                const int shift = kTree && many ? p.many.shift : p.few.shift, c0 = own_first >> shift;
                x.own_many = kTree && many;
                x.n[0] = 1;
                x.place[0] = row;
                x.n[1] = own_last - c0;
                x.place[1] = own_first + (1 << shift);
                if (kTree && many && !other && own_last == c0) {  // written where it was computed, as below
                    x.n[0] = mark == mark ? 0 : -1;
                    done = mark == mark;
                }
            }
            if (other) {
                const int c0 = other_first >> second.shift;
                x.n[2] = 1;
                x.place[2] = row;
                x.n[3] = other_last - c0;
                x.place[3] = other_first + (1 << second.shift);
                if (!kTree && many && other_last == c0) {  // written where it was computed, unless it was not finite
                    x.n[2] = 0;
                    x.n[0] = mark == mark ? 0 : -1;
                    done = mark == mark;
                }
            }
        }
        if (!done) rows[atomicAdd(&left, 1)] = x;
    }
    __syncthreads();
    for (int i = threadIdx.x >> 5; i < left; i += blockDim.x >> 5) {
        const RowParts& x = rows[i];
        const int row = x.row, t = row / p.nq, h = row - t * p.nq;
        T* out = p.out + t * p.out_stride + (long long)h * p.hd;
        const int n0 = max(0, x.n[0]), n1 = n0 + x.n[1], n2 = n1 + x.n[2], n = n2 + x.n[3];
        float top = -INFINITY, d = 0.f;
        constexpr int E = HD > 128 ? HD / 128 : 1;  // 16-byte pieces of a lane
        float4 o[E];
#pragma unroll
        for (int u = 0; u < E; ++u) o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int base = 0; base < n; base += 32) {
            // lane i has part base + i
            const int part = base + lane;
            const float* src = nullptr;
            float2 md = make_float2(-INFINITY, 0.f);
            if (part < n) {
                const int k = part < n0 ? 0 : (part < n1 ? 1 : (part < n2 ? 2 : 3));
                const int at = part - (k == 0 ? 0 : (k == 1 ? n0 : (k == 2 ? n1 : n2)));
                const bool own_cont = (k == 1 && !(kTree && x.own_many)) || (k == 3 && p.prefix_few);
                const long long place = x.place[k] + (long long)at * (own_cont ? 1 << p.few.shift : kTcRows);
                src = (k == 0 ? p.few.first : (k == 2 ? p.many.first : (own_cont ? p.few.cont : p.many.cont))) + place * p.hd;
                md = (k == 0 ? p.few.first_md : (k == 2 ? p.many.first_md : (own_cont ? p.few.cont_md : p.many.cont_md)))[place];
            }
            float now = md.x;
            for (int s = 16; s; s >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, s));
            now = fmaxf(now, top);
            const float ref = now == -INFINITY ? 0.f : now;
            const float w = exp2_approx(md.x - ref);
            float sum = md.y * w;
            for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
            const float keep = exp2_approx(top - ref);
            d = d * keep + sum;
            top = now;
            if (base) {
#pragma unroll
                for (int u = 0; u < E; ++u) {
                    o[u].x *= keep;
                    o[u].y *= keep;
                    o[u].z *= keep;
                    o[u].w *= keep;
                }
            }
            const int here = min(32, n - base);
            constexpr int kFly = 8 / E;  // parts whose loads are in flight together
            for (int k0 = 0; k0 < here; k0 += kFly) {
                float4 v[kFly][E];
                float wk[kFly];
#pragma unroll
                for (int k = 0; k < kFly; ++k) {
                    const int l = min(k0 + k, 31);
                    wk[k] = __shfl_sync(0xffffffffu, w, l);
                    const float* from = reinterpret_cast<const float*>(
                        __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), l));
#pragma unroll
                    for (int u = 0; u < E; ++u) {
                        const int e = u * 128 + lane * 4;
                        v[k][u] = k0 + k < here && e < p.hd ? *reinterpret_cast<const float4*>(from + e)
                                                            : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    if (k0 + k >= here) wk[k] = 0.f;
                }
#pragma unroll
                for (int k = 0; k < kFly; ++k)
#pragma unroll
                    for (int u = 0; u < E; ++u) {
                        o[u].x = fmaf(v[k][u].x, wk[k], o[u].x);
                        o[u].y = fmaf(v[k][u].y, wk[k], o[u].y);
                        o[u].z = fmaf(v[k][u].z, wk[k], o[u].z);
                        o[u].w = fmaf(v[k][u].w, wk[k], o[u].w);
                    }
            }
        }
        const float inv = d == 0.f ? 0.f : 1.f / d;
        bool fine = isfinite(d) && x.n[0] >= 0;
#pragma unroll
        for (int u = 0; u < E; ++u) {
            o[u].x *= inv;
            o[u].y *= inv;
            o[u].z *= inv;
            o[u].w *= inv;
            fine &= isfinite(o[u].x) && isfinite(o[u].y) && isfinite(o[u].z) && isfinite(o[u].w);
        }
        if (!__all_sync(0xffffffffu, fine)) {
            attend_alone(p, x.b, request_of(p, x.b), x.j, h);
            continue;
        }
#pragma unroll
        for (int u = 0; u < E; ++u) {
            const int e = u * 128 + lane * 4;
            if (e < p.hd)
                *reinterpret_cast<uint2*>(out + e) =
                    make_uint2(Pair<T>::pack(o[u].x, o[u].y), Pair<T>::pack(o[u].z, o[u].w));
        }
        if (lane == 0 && p.lse) p.lse[row] = d == 0.f ? -INFINITY : (top + log2f(d)) * kLn2;
    }
}

// ---- sizes and the workspace ---------------------------------------------------------
// Rows per KV head up to which a request streams its keys (again for every job's
// worth of rows, but then out of L2), and up to which the whole batch does so with
// the prefix.  Beyond, the tensor cores' 128-row tile costs less.
constexpr int kFewRows = 64, kFewPrefixRows = 32;

struct Shape {
    int hd, nt, few_rows;
    bool prefix_few, tensor;  // tensor: there may be work for the tensor cores
    bool tiles;               // trees: everything is
    int many_above;
};

// Column tiles for `rows` query rows of a job: one up to eight rows, beyond
// that as many as a warp's registers hold (512 / head_dim).
Shape shape_of_call(const tf_paged_kv* kv, uint32_t nq, uint32_t T, uint32_t prefix_len, uint32_t max_query, bool tree) {
    const long long G = nq / kv->num_kv_heads, own = std::min<long long>(max_query, T) * G;
    Shape s;
    s.hd = kv->head_dim <= 64 ? 64 : (kv->head_dim <= 128 ? 128 : (kv->head_dim <= 256 ? 256 : 512));
    s.nt = own <= 8 || tree ? 1 : std::min(4, 512 / s.hd);
    s.tiles = tree && s.hd <= 256 && own > 8;
    s.few_rows = s.nt * 8;
    const bool can = s.hd <= 256;
    s.prefix_few = !can || (T * G <= kFewPrefixRows && !s.tiles);
    s.many_above = !can ? 0x7FFFFFFF : (s.tiles ? 0 : (tree ? s.few_rows : kFewRows));
    s.tensor = can && ((prefix_len && !s.prefix_few) || own > s.many_above);
    return s;
}

struct Layout {
    size_t first[2], first_md[2], cont[2], cont_md[2], first_of[2], last_of[2], prefix_first, bytes;
};

Layout layout_of(const tf_context* ctx, const tf_paged_kv* kv, uint32_t nq, uint32_t T, const Shape& s) {
    Layout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) & ~(size_t)255;
        return here;
    };
    const size_t rows = (size_t)T * nq;
    const size_t cont[2] = {(size_t)ctx->num_sms * (kThreads / 32) * s.few_rows, (size_t)ctx->num_sms * kTcRows};  // (Parts::places)
    for (int k = 0; k < 2; ++k) {
        l.first_of[k] = take(rows * sizeof(int));
        l.last_of[k] = take(rows * sizeof(int));
        l.first_md[k] = take(rows * sizeof(float2));
        l.cont_md[k] = take(cont[k] * sizeof(float2));
        l.first[k] = take(rows * kv->head_dim * sizeof(float));
        l.cont[k] = take(cont[k] * kv->head_dim * sizeof(float));
    }
    l.prefix_first = take(sizeof(int));
    l.bytes = at;
    return l;
}

// The pool in boxes of `keys` keys and `blocks` 64-dim blocks; false when it
// cannot be described.  With one block a box, the dims of a head are not split
// (dims beyond head_dim arrive as zeros).
bool pool_map(CUtensorMap* m, const tf_paged_kv* kv, const void* base, uint32_t keys, uint32_t blocks) {
    memset(m, 0, sizeof(*m));
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const bool split = blocks > 0;
    cuuint64_t dims[5] = {split ? 64 : kv->head_dim, kv->page_size, split ? kv->head_dim / 64 : 1, kv->num_kv_heads,
                          kv->num_pages};
    cuuint64_t strides[4] = {kv->position_stride * 2, 128, kv->head_stride * 2, kv->page_stride * 2};
    for (int i = 0; i < 4; ++i) {
        if (dims[i + 1] == 1) strides[i] = 128;  // never used
        if (strides[i] >= (1ull << 40)) return false;
    }
    cuuint32_t box[5] = {64, keys, split ? blocks : 1, 1, 1};
    cuuint32_t es[5] = {1, 1, 1, 1, 1};
    return fn(m, kv->dtype == TF_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
              const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, int NT, bool kTensor, bool kTree>
tf_status launch_parts(tf_context* ctx, const AttnParams<T, kTree>& p, cudaStream_t cs, const char* name) {
    constexpr int kMany = kTensor ? TensorShape<HD>::kSmem : 0, kFew = StreamShape<HD, NT>::kSmem;
    constexpr int kSmem = kMany > kFew ? kMany : kFew;
    static bool configured[64] = {};  // per instantiation, per device
    const int dev = ctx->device & 63;
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(attention_parts_kernel<T, HD, NT, kTensor, kTree>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return cuda_check(ctx, e, name);
        configured[dev] = true;
    }
    return cuda_check(ctx, launch_overlapped(attention_parts_kernel<T, HD, NT, kTensor, kTree>, ctx->num_sms, kThreads, kSmem, cs, p),
                      name);
}

template <typename T, int HD>
tf_status launch_tiles(tf_context* ctx, const AttnParams<T, true>& p, cudaStream_t cs, const char* name) {
    constexpr int kSmem = TensorShape<HD>::kSmem;
    static bool configured[64] = {};  // per instantiation, per device
    const int dev = ctx->device & 63;
    if (!configured[dev]) {
        cudaError_t e =
            cudaFuncSetAttribute(tree_tiles_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return cuda_check(ctx, e, name);
        configured[dev] = true;
    }
    return cuda_check(ctx, launch_overlapped(tree_tiles_kernel<T, HD>, ctx->num_sms, kThreads, kSmem, cs, p), name);
}

template <typename T, bool kTree>
tf_status launch(tf_context* ctx, const AttnParams<T, kTree>& p, const Shape& s, cudaStream_t cs, const char* name) {
    tf_status st = TF_OK;
    auto parts = [&](auto hd, auto nt) {
        constexpr int HD = decltype(hd)::value, NT = kTree ? 1 : decltype(nt)::value;
        if constexpr (HD <= 256 && kTree) {
            if (s.tiles) return launch_tiles<T, HD>(ctx, p, cs, name);
        }
        if constexpr (HD <= 256) {
            if (s.tensor) return launch_parts<T, HD, NT, true>(ctx, p, cs, name);
        }
        return launch_parts<T, HD, NT, false>(ctx, p, cs, name);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    if (s.hd == 64)
        st = s.nt == 1 ? parts(integral_constant<int, 64>(), one) : parts(integral_constant<int, 64>(), four);
    else if (s.hd == 128)
        st = s.nt == 1 ? parts(integral_constant<int, 128>(), one) : parts(integral_constant<int, 128>(), four);
    else if (s.hd == 256)
        st = s.nt == 1 ? parts(integral_constant<int, 256>(), one) : parts(integral_constant<int, 256>(), two);
    else
        st = parts(integral_constant<int, 512>(), one);
    if (st) return st;
    // a warp per row while that fills the GPU; then more rows a CTA, in four rounds of CTAs
    const int rows = p.T_tokens * p.nq;
    // (trees: in one round, since to find a row's request takes a bisection, which the first round does
    // while the parts are still computed: 11520 rows join in 11 us, 16 in four rounds)
    const int per = std::min(kJoinRows, std::max(8, (rows / (ctx->num_sms * (kTree ? 3 : 12)) + 7) / 8 * 8));
    const unsigned ctas = (unsigned)((rows + per - 1) / per);
    cudaError_t e;
    if (s.hd <= 128)
        e = launch_overlapped(join_parts_kernel<T, 128, kTree>, ctas, 256, 0, cs, p, per);
    else if (s.hd == 256)
        e = launch_overlapped(join_parts_kernel<T, 256, kTree>, ctas, 256, 0, cs, p, per);
    else
        e = launch_overlapped(join_parts_kernel<T, 512, kTree>, ctas, 256, 0, cs, p, per);
    return cuda_check(ctx, e, name);
}

// What a call needs beside the cache and the lengths (kTree: the last three).
struct AttentionCall {
    const void* q;
    uint64_t q_stride;
    const void* prefix_pages;
    uint32_t prefix_len;
    const void* page_table;
    uint32_t max_pages;
    const void* seq_lens;
    const void* token_starts;
    uint32_t num_requests, max_query, T, num_q_heads;
    float scale;
    uint32_t window;
    void* out;
    uint64_t out_stride;
    void* lse;
    void* workspace;
    size_t workspace_bytes;
    const void* ancestors;
    uint32_t words;
    const void* positions;
};

template <bool kTree>
tf_status attention_call(tf_context* ctx, const tf_paged_kv* kv, const AttentionCall& c, cudaStream_t cs,
                         const char* name) {
    const uint32_t T = c.T, num_requests = c.num_requests, num_q_heads = c.num_q_heads, prefix_len = c.prefix_len,
                   max_pages = c.max_pages, window = c.window;
    const uint64_t q_stride = c.q_stride, out_stride = c.out_stride;
    const void *q = c.q, *prefix_pages = c.prefix_pages, *page_table = c.page_table, *seq_lens = c.seq_lens,
               *token_starts = c.token_starts;
    void *out = c.out, *lse = c.lse, *workspace = c.workspace;
    const float scale = c.scale;
    const size_t workspace_bytes = c.workspace_bytes;
    uint32_t max_query = c.max_query;
    max_query = std::min(max_query, T);  // no request has more
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
    if constexpr (kTree) {
        if (c.words > 0xFFFFu || c.words * 32 < max_query || max_query > 256)
            return fail(ctx, TF_ERR_INVALID_ARG, "%s: trees of up to 256 nodes, a bit for each in %u words", name, c.words);
        // a node's ancestors are then inside its window
        if (window && (window < max_query || !c.positions))
            return fail(ctx, TF_ERR_INVALID_ARG, "%s: a window takes positions, and is no smaller than a tree", name);
        if (!c.ancestors) return fail(ctx, TF_ERR_INVALID_ARG, "%s: null pointer", name);
        if (!aligned4(c.ancestors) || !aligned4(c.positions))
            return fail(ctx, TF_ERR_MISALIGNED, "%s: pointers must be 4-byte aligned", name);
        if ((uint64_t)T * c.words > 0x7FFFFFFFull)
            return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: words must be below 2^31", name);
    }
    const uint64_t G = num_q_heads / kv->num_kv_heads;
    const Shape shape = shape_of_call(kv, num_q_heads, T, prefix_len, max_query, kTree);
    // an int counts the units: streamed ones, smaller than the tensor cores', or, of tiles alone, theirs (a row
    // tile has two jobs at most, prefix and own keys)
    const uint64_t unit_rows = shape.tiles ? kTcRows : shape.few_rows;
    const uint64_t unit_keys = !shape.tiles ? 16 : (shape.hd > 128 ? TensorShape<256>::kKeys : TensorShape<128>::kKeys);
    const uint64_t row_tiles = T * G / unit_rows + std::min<uint64_t>(T, num_requests);
    const uint64_t tiles = (uint64_t)max_pages * kv->page_size / unit_keys + prefix_len / unit_keys + 2;
    if (row_tiles * (tiles + (kTree ? 2 * kJobUnits : 0)) * kv->num_kv_heads > 0x7FFFFFFFull)
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: too many keys", name);
    const Layout l = layout_of(ctx, kv, num_q_heads, T, shape);
    const size_t need = l.bytes;
    if (workspace_bytes < need)
        return fail(ctx, TF_ERR_INVALID_ARG, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes, need);

    KvMaps maps;
    const uint32_t run = std::min<uint32_t>(kMaxRun, kv->page_size & (0u - kv->page_size));
    const bool wide = run == 8 && kv->head_dim % 64 == 0;
    const uint32_t blocks = wide ? shape.hd / 64 : 0;
    if (!pool_map(&maps.k, kv, kv->k, run, blocks) || !pool_map(&maps.v, kv, kv->v, run, blocks) ||
        !pool_map(&maps.v_row, kv, kv->v, 1, 0))
        return fail(ctx, TF_ERR_UNSUPPORTED_SHAPE, "%s: the pool's sizes and strides cannot be described to TMA", name);

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
        p.ancestors = static_cast<const uint32_t*>(c.ancestors);
        p.positions = static_cast<const int*>(c.positions);
        p.words = (int)c.words;
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
        p.prefix_few = shape.prefix_few;
        p.many_above = shape.many_above;
        uint8_t* w = static_cast<uint8_t*>(workspace);
        Parts* parts[2] = {&p.few, &p.many};
        for (int k = 0; k < 2; ++k) {
            parts[k]->first = reinterpret_cast<float*>(w + l.first[k]);
            parts[k]->first_md = reinterpret_cast<float2*>(w + l.first_md[k]);
            parts[k]->cont = reinterpret_cast<float*>(w + l.cont[k]);
            parts[k]->cont_md = reinterpret_cast<float2*>(w + l.cont_md[k]);
            parts[k]->first_of = reinterpret_cast<int*>(w + l.first_of[k]);
            parts[k]->last_of = reinterpret_cast<int*>(w + l.last_of[k]);
        }
        p.prefix_first = reinterpret_cast<int*>(w + l.prefix_first);
        p.few.places = ctx->num_sms * (kThreads / 32);
        p.many.places = ctx->num_sms;
        p.few.shift = 2 + (shape.nt == 1 ? 1 : (shape.nt == 2 ? 2 : 3));  // log2(8 nt)
        p.many.shift = 7;
        p.run_shift = run == 8 ? 3 : (run == 4 ? 2 : (run == 2 ? 1 : 0));
        p.page_shift = p.g_shift = -1;
        for (int i = 0; i < 31; ++i) {
            if (kv->page_size == (1u << i)) p.page_shift = i;
            if (G == (1u << i)) p.g_shift = i;
        }
        p.wide = wide;
        p.maps = maps;
    };
    if (kv->dtype == TF_DTYPE_F16) {
        AttnParams<__half, kTree> p;
        fill(p);
        return launch(ctx, p, shape, cs, name);
    }
    AttnParams<__nv_bfloat16, kTree> p;
    fill(p);
    return launch(ctx, p, shape, cs, name);
}

}  // namespace
}  // namespace tf

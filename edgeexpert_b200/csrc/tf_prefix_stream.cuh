// tf_prefix_stream.cuh -- the attention of few query rows over many keys: each
// request's own pages (and the shared prefix, when the whole batch has few rows).
//
// HBM-bound: K and V are read once, 4 * head_dim bytes a key, for 4 * head_dim
// * rows operations.  Everything serves the stream of loads:
//   * the units (64 keys of one request, KV head and row tile) are dealt evenly
//     and contiguously, whatever the lengths; a CTA's stream of loads runs on
//     across the requests it covers;
//   * a warp owns 16 of a unit's keys and a ring of its own, filled by cp.async
//     up to S - 1 units ahead, so warps wait for nobody until a job ends; page
//     ids are looked up one unit before their loads are issued;
//   * scores are S^T = K Q^T and outputs O^T = V^T P^T: keys and dims fill the
//     16-row side of mma.sync m16n8k16 and the few query rows its 8 columns, so
//     one to eight rows cost one column tile and the accumulator of 256 dims is
//     64 registers.  P^T comes from S^T by transposing 8x8 tiles in registers.
// The tensor cores run at a few percent here; tcgen05's 64-row tiles would be
// nearly empty.
#pragma once
#include "tf_prefix_attention.cuh"

namespace tf {

template <typename T>
__device__ __forceinline__ void mma_16x8(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16x8<__half>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16x8<__nv_bfloat16>(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t r[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int HD, int NT>
struct StreamShape {
    static constexpr int kWarps = HD > 256 ? 2 : 4;
    static constexpr int kKeys = kWarps * 16;                  // keys of a unit
    static constexpr int kRows = NT * 8;                       // query rows of a job
    static constexpr int kTile = 16 * HD * 2;                  // a warp's K (or V) tile, bytes
    static constexpr int kStages = HD == 64 ? 6 : 3;           // K and V tiles per warp
    static constexpr int kCtas = HD >= 256 ? 1 : 2;            // per SM
    static constexpr int kJoinLd = 66;                         // floats per row while warps are joined
    static constexpr int kRing = kWarps * kStages * 2 * kTile;
    static constexpr int kSmem = kRing + kWarps * kRows * (kJoinLd + 2) * 4 + 1024;
};

// Where a CTA is in its range of units.
struct StreamCursor {
    int seg;             // request, or -1: the prefix
    int kvh, rt, tile;   // KV head, row tile, key tile
    int row_tiles, tiles;
    int lo, hi;          // keys of the segment
};

template <typename T, int HD, int NT>
__device__ __forceinline__ void stream_segment(const AttnParams<T>& p, StreamCursor& c) {
    using S = StreamShape<HD, NT>;
    if (c.seg < 0) {
        const int rows = p.prefix_by_stream ? max(0, min(p.starts[p.B], p.T_tokens)) * p.G : 0;
        c.lo = p.prefix_lo;
        c.hi = p.prefix_len;
        c.row_tiles = (rows + S::kRows - 1) / S::kRows;
    } else {
        const Request r = request_of(p, c.seg);
        c.lo = own_lo(p, r);
        c.hi = r.len;
        c.row_tiles = by_tensor(p, r) ? 0 : (r.used * p.G + S::kRows - 1) / S::kRows;
    }
    c.tiles = c.row_tiles ? (c.hi - c.lo + S::kKeys - 1) / S::kKeys : 0;
}

template <typename T, int HD, int NT>
__device__ __forceinline__ void stream_advance(const AttnParams<T>& p, StreamCursor& c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.rt < c.row_tiles) return;
    c.rt = 0;
    if (++c.kvh < p.nkv) return;
    c.kvh = 0;
    do {
        ++c.seg;
        if (c.seg >= p.B) return;
        stream_segment<T, HD, NT>(p, c);
    } while (c.tiles == 0);
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(StreamShape<HD, NT>::kWarps * 32, StreamShape<HD, NT>::kCtas)
    attention_few_rows_kernel(const __grid_constant__ AttnParams<T> p) {
    using S = StreamShape<HD, NT>;
    constexpr int kWarps = S::kWarps, kRows = S::kRows, kStages = S::kStages, CPR = HD / 8;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    float* join = reinterpret_cast<float*>(smem + S::kRing);         // [warp][row][kJoinLd]
    float* join_md = join + kWarps * kRows * S::kJoinLd;             // [warp][row][2]
    __shared__ int red[32], s_seg, s_at;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;

    // ---- which units are mine -------------------------------------------------
    // thread i sums the units of requests [i*per, (i+1)*per); the one whose sum
    // contains my first unit finds the request
    int U, u0, u1;
    StreamCursor cur;
    {
        StreamCursor c;
        c.seg = -1;
        stream_segment<T, HD, NT>(p, c);
        const int prefix_units = c.row_tiles * c.tiles * p.nkv;
        const int per = (p.B + blockDim.x - 1) / blockDim.x;
        const int b0 = min(p.B, (int)threadIdx.x * per), b1 = min(p.B, b0 + per);
        int sum = 0;
        for (c.seg = b0; c.seg < b1; ++c.seg) {
            stream_segment<T, HD, NT>(p, c);
            sum += c.row_tiles * c.tiles * p.nkv;
        }
        int at = prefix_units + block_scan(sum, red, &U);
        U += prefix_units;
        u0 = unit_begin(blockIdx.x, U, gridDim.x);
        u1 = unit_begin(blockIdx.x + 1, U, gridDim.x);
        if (threadIdx.x == 0 && (u0 < prefix_units || U == 0)) {
            s_seg = -1;
            s_at = 0;
        }
        for (c.seg = b0; c.seg < b1; ++c.seg) {
            stream_segment<T, HD, NT>(p, c);
            const int units = c.row_tiles * c.tiles * p.nkv;
            if (blockIdx.x == 0) p.stream.base[c.seg] = at;
            if (u0 >= at && u0 < at + units) {
                s_seg = c.seg;
                s_at = at;
            }
            at += units;
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) p.stream.base[p.B] = U;
        __syncthreads();
        if (u0 >= u1) return;
        cur.seg = s_seg;
        stream_segment<T, HD, NT>(p, cur);
        const int in = u0 - s_at;
        cur.tile = in % cur.tiles;
        cur.rt = in / cur.tiles % cur.row_tiles;
        cur.kvh = in / cur.tiles / cur.row_tiles;
    }
    StreamCursor ahead = cur;  // the unit whose page ids are looked up next
    int left_ahead = u1 - u0;

    // ---- loads ------------------------------------------------------------------
    const uint32_t ring = smem_u32(smem) + warp * kStages * 2 * S::kTile;
    long long next_off = 0;     // lane < 16: element offset of its key's row
    uint32_t next_mask = 0;     // which of the 16 keys exist
    auto look_up = [&]() {
        next_mask = 0;
        if (left_ahead <= 0) return;
        const int pos = ahead.lo + ahead.tile * S::kKeys + warp * 16 + (lane & 15);
        bool ok = pos < ahead.hi;
        next_off = 0;
        if (ok) {
            const int at = pos / p.kv.page_size;
            const int page = ahead.seg < 0 ? p.prefix_pages[at] : p.table[(long long)ahead.seg * p.max_pages + at];
            ok = page >= 0 && page < p.kv.num_pages;
            if (ok)
                next_off = page * p.kv.page_stride + (pos - at * p.kv.page_size) * p.kv.pos_stride +
                           ahead.kvh * p.kv.head_stride;
            else
                atomicOr(p.err, kErrBadPage);
        }
        next_mask = __ballot_sync(0xffffffffu, ok) & 0xFFFFu;
        --left_ahead;
        stream_advance<T, HD, NT>(p, ahead);
    };
    auto issue = [&](int stage) {  // loads of the keys last looked up
        const uint32_t dst = ring + stage * 2 * S::kTile;
#pragma unroll
        for (int i = 0; i < 16 * CPR / 32; ++i) {
            const int chunk = i * 32 + lane, row = chunk / CPR, c = chunk % CPR;
            const long long off = __shfl_sync(0xffffffffu, next_off, row);
            const int bytes = ((next_mask >> row) & 1) && c * 8 < p.hd ? 16 : 0;
            const long long at = bytes ? off + c * 8 : 0;
            const uint32_t to = dst + row * (HD * 2) + ((c ^ (row & 7)) << 4);
            cp_async16(to, p.kv.k + at, bytes);
            cp_async16(to + S::kTile, p.kv.v + at, bytes);
        }
    };

    look_up();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        issue(i);
        cp_async_commit();
        look_up();
    }

    // ---- the job's rows -----------------------------------------------------------
    uint32_t qf[HD / 16][NT][2];
    int row_lo[NT][2], row_hi[NT][2];
    float m[NT][2], d[NT][2], acc[HD / 16][NT][4];
    const float sc = p.scale * kLog2e;
    int job_rows = 0, first_token = 0;
    auto begin_job = [&]() {
        const bool prefix = cur.seg < 0;
        Request r;
        if (prefix) {
            job_rows = max(0, min(p.starts[p.B], p.T_tokens)) * p.G;
            first_token = 0;
        } else {
            r = request_of(p, cur.seg);
            job_rows = r.used * p.G;
            first_token = r.start;
        }
        const int row0 = cur.rt * kRows;
        job_rows -= row0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int rq = row0 + nt * 8 + g;  // the row whose q this lane holds
            const bool ok = nt * 8 + g < job_rows;
            const T* qr = p.q + (long long)(first_token + rq / p.G) * p.q_stride + (cur.kvh * p.G + rq % p.G) * p.hd;
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int e = ks * 16 + 2 * tq + 8 * i;
                    qf[ks][nt][i] = ok && e < p.hd ? *reinterpret_cast<const uint32_t*>(qr + e) : 0u;
                }
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // rows whose scores it holds
                const int rs = row0 + nt * 8 + 2 * tq + i;
                int lo = 0, hi = 0;
                if (nt * 8 + 2 * tq + i < job_rows) {
                    const int j = rs / p.G;
                    if (prefix) {
                        const int b = request_at(p, j);
                        if (b < p.B) {
                            const Request rb = request_of(p, b);
                            if (j - rb.start < rb.used) seen_by(p, rb, j - rb.start, lo, hi);
                        }
                    } else {
                        seen_by(p, r, j, lo, hi);
                        lo -= p.prefix_len;
                        hi -= p.prefix_len;
                    }
                }
                row_lo[nt][i] = lo;
                row_hi[nt][i] = min(hi, cur.hi);
                m[nt][i] = -INFINITY;
                d[nt][i] = 0.f;
            }
#pragma unroll
            for (int mt = 0; mt < HD / 16; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[mt][nt][i] = 0.f;
        }
    };

    // Joins the warps and writes the job's part.
    bool from_start = cur.tile == 0;
    auto end_job = [&]() {
        const int row0 = cur.rt * kRows;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float s = d[nt][i];
                for (int o = 4; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (g == 0) {
                    float* md = join_md + (warp * kRows + nt * 8 + 2 * tq + i) * 2;
                    md[0] = m[nt][i];
                    md[1] = s;
                }
            }
        __syncthreads();
        float fac[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = -INFINITY;
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, join_md[(w * kRows + nt * 8 + 2 * tq + i) * 2]);
                fac[nt][i] = m[nt][i] == -INFINITY ? 0.f : exp2_approx(m[nt][i] - top);
            }
        auto place = [&](int r) -> long long {  // row of `first` or `cont`
            if (!from_start) return (long long)blockIdx.x * p.stream.rows + r;
            const int row = row0 + r;
            return (long long)(first_token + row / p.G) * p.nq + cur.kvh * p.G + row % p.G;
        };
        // a row's part of the prefix goes where the tensor kernel would have put it
        const Parts& to = cur.seg < 0 ? p.tensor : p.stream;
        float* po = from_start ? to.first : p.stream.cont;
        float2* pm = from_start ? to.first_md : p.stream.cont_md;
        for (int r = threadIdx.x; r < min(kRows, job_rows); r += blockDim.x) {
            float top = -INFINITY, sum = 0.f;
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, join_md[(w * kRows + r) * 2]);
            for (int w = 0; w < kWarps; ++w) {
                const float mw = join_md[(w * kRows + r) * 2];
                if (mw != -INFINITY) sum += join_md[(w * kRows + r) * 2 + 1] * exp2_approx(mw - top);
            }
            pm[place(r)] = make_float2(top, sum);
        }
#pragma unroll
        for (int mt0 = 0; mt0 < HD / 16; mt0 += 4) {  // 64 dims at a time
            if (mt0) __syncthreads();
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        join[(warp * kRows + nt * 8 + 2 * tq + (i & 1)) * S::kJoinLd + u * 16 + g + 8 * (i >> 1)] =
                            acc[mt0 + u][nt][i] * fac[nt][i & 1];
            __syncthreads();
            for (int x = threadIdx.x; x < kRows * 64; x += blockDim.x) {
                const int r = x >> 6, e = x & 63;
                if (r >= job_rows || mt0 * 16 + e >= p.hd) continue;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) v += join[(w * kRows + r) * S::kJoinLd + e];
                po[place(r) * p.hd + mt0 * 16 + e] = v;
            }
        }
        __syncthreads();
    };

    // ---- one unit -------------------------------------------------------------------
    const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_chunk = lane >> 4;      // K: keys x dims
    const int v_row = (lane & 7) + ((lane >> 4) & 1) * 8, v_chunk = (lane >> 3) & 1;  // V: dims x keys
    int stage = 0;
    for (int u = u0; u < u1; ++u) {
        if (u == u0 || cur.tile == 0) begin_job();
        const int fill = stage == 0 ? kStages - 1 : stage - 1;
        issue(fill);
        cp_async_commit();
        look_up();
        cp_async_wait<kStages - 1>();
        __syncwarp();

        const uint32_t kt = ring + stage * 2 * S::kTile, vt = kt + S::kTile;
        float s[NT][4], s2[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][i] = s2[nt][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
            uint32_t a[4];
            ldsm4(a, kt + k_row * (HD * 2) + (((ks * 2 + k_chunk) ^ (k_row & 7)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16x8<T>(ks & 1 ? s2[nt] : s[nt], a, qf[ks][nt][0], qf[ks][nt][1]);
        }
        const int key0 = cur.lo + cur.tile * S::kKeys + warp * 16;
        uint32_t pf[NT][2];
        bool grew = false;
        float keep[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = key0 + g + 8 * (i >> 1);
                const bool ok = key >= row_lo[nt][i & 1] && key < row_hi[nt][i & 1];
                s[nt][i] = ok ? (s[nt][i] + s2[nt][i]) * sc : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float top = fmaxf(s[nt][i], s[nt][i + 2]);
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = fmaxf(top, m[nt][i]);
                keep[nt][i] = m[nt][i] == -INFINITY ? 1.f : exp2_approx(m[nt][i] - top);
                grew |= top > m[nt][i];
                m[nt][i] = top;
                const float ref = top == -INFINITY ? 0.f : top;
                s[nt][i] = exp2_approx(s[nt][i] - ref);
                s[nt][i + 2] = exp2_approx(s[nt][i + 2] - ref);
                d[nt][i] = d[nt][i] * keep[nt][i] + (s[nt][i] + s[nt][i + 2]);
            }
            // weights go to the tensor cores in the cache's type (their sum is of the unrounded ones)
            pf[nt][0] = transpose8x8(Pair<T>::pack(s[nt][0], s[nt][1]));
            pf[nt][1] = transpose8x8(Pair<T>::pack(s[nt][2], s[nt][3]));
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int mt = 0; mt < HD / 16; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[mt][nt][i] *= keep[nt][i & 1];
        }
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            uint32_t a[4];
            ldsm4_t(a, vt + v_row * (HD * 2) + (((mt * 2 + v_chunk) ^ (v_row & 7)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16x8<T>(acc[mt][nt], a, pf[nt][0], pf[nt][1]);
        }
        __syncwarp();  // before this stage is filled again
        stage = stage == kStages - 1 ? 0 : stage + 1;
        if (cur.tile == cur.tiles - 1 || u == u1 - 1) {
            end_job();
            from_start = true;
        }
        stream_advance<T, HD, NT>(p, cur);
    }
    cp_async_wait<0>();
}

}  // namespace tf

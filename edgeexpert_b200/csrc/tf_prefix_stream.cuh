// tf_prefix_stream.cuh -- the attention of few query rows over many keys: each
// request's own pages (and the shared prefix, when the whole batch has few rows).
//
// HBM-bound: K and V are read once, 4 * head_dim bytes a key, for 4 * head_dim
// * rows operations.  Everything serves the stream of loads:
//   * the units (16 keys of one request, KV head and row tile) are dealt evenly
//     and contiguously to the warps, whatever the lengths.  A warp works for
//     itself: its ring of K and V tiles is filled by its own TMA loads, which run
//     on across the jobs it covers, so no warp ever waits for another and one
//     that begins or ends a job leaves the memory to the rest;
//   * page ids are looked up one unit before their loads are issued;
//   * scores are S^T = K Q^T and outputs O^T = V^T P^T: keys and dims fill the
//     16-row side of mma.sync m16n8k16 and the few query rows its 8 columns, so
//     one to eight rows cost one column tile and the accumulator of 256 dims is
//     64 registers.  P^T comes from S^T by transposing 8x8 tiles in registers.
// The tensor cores run at a few percent here; tcgen05's 64-row tiles would be
// nearly empty.
// Measured (16 query / 8 KV heads of 256, fp16): 256 requests of 500 keys on
// average, no prefix, 1.05 GB: 207 us with the join, 5.1 TB/s; the warps end
// between 137 and 208 us, 175 on average (the SMs do not get equal shares of the
// memory).  Shares taken from a counter for the last 40 % instead: 183 us, but 2
// to 11 us more for smaller batches (the counter's reset, restarts of the rings).
// Four warps a CTA on the keys of one job, joined in shared memory: 71 us instead
// of 55 us for 32 requests of 1024 keys (every join stopped all four).
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
    static constexpr int kWarps = HD > 256 ? 4 : 8;  // that stream
    static constexpr int kKeys = 16;                 // keys of a unit
    static constexpr int kRows = NT * 8;             // query rows of a job
    static constexpr int kTile = kKeys * HD * 2;     // bytes of a K (or V) tile
    static constexpr int kTiles = HD >= 256 ? 3 : (HD == 128 ? 6 : 10);  // a warp's ring, K and V tiles in turn
    static constexpr int kSmem = kWarps * kTiles * kTile + 1024;
    static constexpr int kBars = kWarps * kTiles;
};

// Where a warp is in its range of units.
struct StreamCursor {
    int seg;             // request, or -1: the prefix
    int kvh, rt, tile;   // KV head, row tile, key tile
    int row_tiles, tiles;
    int lo, hi;          // keys of the segment; lo is rounded down to a box
    int from;            // the first that any row sees
};

// Rows that have the prefix here.
template <typename T>
__device__ __forceinline__ int stream_prefix_rows(const AttnParams<T>& p) {
    return p.prefix_few ? max(0, min(p.starts[p.B], p.T_tokens)) * p.G : 0;
}

template <typename T, int HD, int NT>
__device__ __forceinline__ void stream_segment(const AttnParams<T>& p, StreamCursor& c) {
    using S = StreamShape<HD, NT>;
    if (c.seg < 0) {
        const int rows = stream_prefix_rows(p);
        c.from = prefix_first(p);
        c.hi = p.prefix_len;
        c.row_tiles = (rows + S::kRows - 1) / S::kRows;
    } else {
        const Request r = request_of(p, c.seg);
        c.from = own_lo(p, r);
        c.hi = r.len;
        c.row_tiles = is_many(p, r) ? 0 : (r.used * p.G + S::kRows - 1) / S::kRows;
    }
    c.lo = c.from & ~(kMaxRun - 1);
    c.tiles = c.row_tiles && c.hi > c.from ? (c.hi - c.lo + S::kKeys - 1) / S::kKeys : 0;
}

// The first unit of the next job.
template <typename T, int HD, int NT>
__device__ __noinline__ StreamCursor stream_next_job(const AttnParams<T>& p, StreamCursor c) {
    c.tile = 0;
    if (++c.rt < c.row_tiles) return c;
    c.rt = 0;
    if (++c.kvh < p.nkv) return c;
    c.kvh = 0;
    do {
        ++c.seg;
        if (c.seg >= p.B) return c;
        stream_segment<T, HD, NT>(p, c);
    } while (c.tiles == 0);
    return c;
}
template <typename T, int HD, int NT>
__device__ __forceinline__ void stream_advance(const AttnParams<T>& p, StreamCursor& c) {
    if (++c.tile >= c.tiles) c = stream_next_job<T, HD, NT>(p, c);
}

// The units of the whole batch; `before` those of the requests before this
// thread's own [b0, b1).  With a window also the first prefix position that any row sees.
template <typename T, int HD, int NT>
__device__ __forceinline__ int stream_units(const AttnParams<T>& p, int* red, int b0, int b1, int& before) {
    using S = StreamShape<HD, NT>;
    if (p.window) {
        if (threadIdx.x == 0) shared_prefix_first() = p.prefix_len;
        __syncthreads();
    }
    const int rows = stream_prefix_rows(p);
    StreamCursor c;
    int sum = 0, total, first = p.prefix_len;
    for (c.seg = b0; c.seg < b1; ++c.seg) {
        stream_segment<T, HD, NT>(p, c);
        sum += c.row_tiles * c.tiles * p.nkv;
        if (p.window) {
            const Request r = request_of(p, c.seg);
            int lo = first, hi;
            if (r.used) seen_by(p, r, 0, lo, hi);
            first = min(first, lo);
        }
    }
    if (p.window && first < p.prefix_len) atomicMin(&shared_prefix_first(), first);
    before = block_scan(sum, red, &total);
    const int prefix_units = (rows + S::kRows - 1) / S::kRows * prefix_tiles(p, S::kKeys) * p.nkv;
    before += prefix_units;
    return prefix_units + total;
}

// One warp: units [u0, u1) beginning at `cur`, as worker `worker`.
template <typename T, int HD, int NT>
__device__ __forceinline__ void stream_warp(const AttnParams<T>& p, uint32_t ring, uint64_t* full, StreamCursor cur,
                                            int u0, int u1, int worker) {
    using S = StreamShape<HD, NT>;
    constexpr int kRows = S::kRows, R = S::kTiles, kGroup8 = HD / 64 * 1024;  // bytes of eight keys
    const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;

    // ---- loads ------------------------------------------------------------------
    StreamCursor ahead = cur;  // the unit whose page ids are looked up next
    int left = u1 - u0;        // units not looked up yet
    TileKeys<16> next, now;  // the unit after the one being loaded, and that one
    int next_head = 0, now_head = 0;
    bool next_own = true, now_own = true;  // own keys that no other row tile reads
    auto look_up = [&]() {
        next_head = ahead.kvh;
        next_own = ahead.seg >= 0 && ahead.row_tiles == 1;
        next = look_up_keys<16>(p, ahead.seg, ahead.lo + ahead.tile * S::kKeys, ahead.from, left > 0 ? ahead.hi : 0);
        if (left-- > 0) stream_advance<T, HD, NT>(p, ahead);
    };
    int fill = 0;  // ring place of the next tile to load
    bool v_next = false;
    auto load_tile = [&]() {
        if (!v_next) {
            now = next;
            now_head = next_head;
            now_own = next_own;
            check_keys(p, now);
        }
        load_tile_keys<HD, 16>(p, v_next, ring + fill * S::kTile, now_head, now, full + fill,
                               now_own);
        if (!v_next) look_up();
        v_next = !v_next;
        fill = fill == R - 1 ? 0 : fill + 1;
    };
    look_up();
    // A tile's loads: bounded like every wait, and given up by the whole warp or by none of it.
    // A warp that gives up issues no more loads and leaves its jobs; the error is reported.
    int slot = 0;
    uint32_t phase = 0;
    auto landed = [&]() { return __all_sync(0xffffffffu, mbar_wait_limited(full + slot, phase, p.err)) != 0; };
    auto taken = [&]() {
        if (++slot == R) {
            slot = 0;
            phase ^= 1;
        }
    };
#pragma unroll 1
    for (int i = 0; i < R - 1; ++i) load_tile();

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
            const int tq0 = token_of(p, rq);
            const T* qr = p.q + (long long)(first_token + tq0) * p.q_stride + (cur.kvh * p.G + rq - tq0 * p.G) * p.hd;
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
                    const int j = token_of(p, rs);
                    if (prefix) {
                        const int b = request_at(p, j);
                        if (b < p.B) {
                            const Request rb = request_of(p, b);
                            if (is_used(rb, j - rb.start)) seen_by(p, rb, j - rb.start, lo, hi);
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

    // The job's part, straight from the registers: eight lanes write the 32
    // bytes of eight dims of a row.
    bool from_start = cur.tile == 0;
    auto end_job = [&]() {
        const bool to_end = cur.tile == cur.tiles - 1;
        // a row's part of the prefix goes where the tensor cores' would be
        const Parts& to = cur.seg < 0 ? p.many : p.few;
        float* po = from_start ? to.first : p.few.cont;
        float2* pm = from_start ? to.first_md : p.few.cont_md;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = nt * 8 + 2 * tq + i, row = cur.rt * kRows + r;
                const int tr = token_of(p, row);
                const long long of = (long long)(first_token + tr) * p.nq + cur.kvh * p.G + row - tr * p.G;
                const long long place = from_start ? of : (long long)worker * kRows + r;
                float sum = d[nt][i];
                for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (r >= job_rows) continue;
                if (g == 0) {
                    pm[place] = make_float2(m[nt][i], sum);
                    if (from_start) to.first_of[of] = worker * kRows + r;
                    if (to_end) to.last_of[of] = worker;
                }
                float* dst = po + place * p.hd + g;
#pragma unroll
                for (int mt = 0; mt < HD / 16; ++mt) {
                    if (mt * 16 < p.hd) dst[mt * 16] = acc[mt][nt][i];
                    if (mt * 16 + 8 < p.hd) dst[mt * 16 + 8] = acc[mt][nt][i + 2];
                }
            }
    };

    // ---- units ------------------------------------------------------------------------
    const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_chunk = lane >> 4;        // K: keys x dims
    const int v_row = (lane & 7) + ((lane >> 4) & 1) * 8, v_chunk = (lane >> 3) & 1;  // V: dims x keys
    bool ok = true;
    for (int u = u0; u < u1; ++u) {
        if (u == u0 || cur.tile == 0) begin_job();
        __syncwarp();  // the tile before this one has been read by every lane
        load_tile();
        ok = landed();
        if (!ok) break;
        const uint32_t kt = ring + slot * S::kTile;
        taken();
        float s[NT][4], s2[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nt][i] = s2[nt][i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
            uint32_t a[4];
            ldsm4(a, kt + (k_row >> 3) * kGroup8 + (ks >> 2) * 1024 + (k_row & 7) * 128 + ((((ks & 3) * 2 + k_chunk) ^ (k_row & 7)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16x8<T>(ks & 1 ? s2[nt] : s[nt], a, qf[ks][nt][0], qf[ks][nt][1]);
        }
        const int key0 = cur.lo + cur.tile * S::kKeys;
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
            // weights go to the tensor cores in the cache's type, which their product with V has to have;
            // each is off by half an ulp of it, their sum is of the unrounded ones
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
        __syncwarp();  // K has been read
        load_tile();
        ok = landed();
        if (!ok) break;
        const uint32_t vt = ring + slot * S::kTile;
        taken();
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            uint32_t a[4];
            ldsm4_t(a, vt + (v_row >> 3) * kGroup8 + (mt >> 2) * 1024 + (v_row & 7) * 128 + ((((mt & 3) * 2 + v_chunk) ^ (v_row & 7)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16x8<T>(acc[mt][nt], a, pf[nt][0], pf[nt][1]);
        }
        if (cur.tile == cur.tiles - 1 || u == u1 - 1) {
            end_job();
            from_start = true;
        }
        stream_advance<T, HD, NT>(p, cur);
    }
    // what was loaded ahead (zeros) lands before the CTA may end; after a wait that gave up, what
    // lands within one more such time
    const long long since = clock64();
    for (int i = 0; i < (ok ? R - 1 : R); ++i) {
        mbar_wait_limited(full + slot, phase, p.err, since);
        taken();
    }
}

}  // namespace tf

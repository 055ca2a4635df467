// tf_prefix_tensor.cuh -- attention of many query rows on the tcgen05 tensor
// cores: the shared prefix for the rows of the whole batch at once, and the own
// keys of requests with many rows (prompts).
//
// A job is 128 query rows of one KV head (row = token * G + head in the group,
// over all tokens of the batch, so a tile may hold several requests); its keys
// are the prefix and then, one after the other, the own keys of those of its
// requests that are this kernel's.  Rows mask what is not theirs.
//
// Tensor memory (512 columns): O (HD), Q (HD/2, 16-bit pairs), two score
// buffers (N each) whose first N/2 columns take the 16-bit weights P once the
// scores are read.  Both products read their A operand from tensor memory, so
// shared memory carries each K and V tile once in and once out:
//   S = Q K^T     A = Q (TMEM), B = K tile [keys][dims], K-major
//   O += P V      A = P (TMEM), B = V tile [keys][dims], MN-major
// Roles: warps 0-3 a row per thread (softmax, Q in, O out), warp 4 issues the
// MMAs, warps 5 and 6 fetch K and V by page into rings of 128-byte-swizzled tiles.
// Scores of tile i+1 are computed while the softmax of tile i runs.
// Bound: MMAs alone take 1030 clocks a unit of 64 keys of 256 (measured, S and O
// interleaved); with all SMs at work a unit takes 1600 inside a job, because K and
// V tiles arrive at 40 bytes a clock and SM, 10.6 TB/s over all SMs, from L2.  24
// prompts of 1 to 300 tokens behind 2050 shared positions (16/8 heads of 256): 217
// us with the join, 595 TFLOP/s; 116 units a CTA from 9 us on, ending at 151 to
// 178 us, 1.33 us a unit with the changes of job (Q in, pipeline drained, O out).
// Pairs of CTAs (cta_group::2) halve the bytes, but the second CTA's weights have
// to be reported to the first every unit: 257 us at best, against 231 then.
// Beside the stream a unit takes about 1.7 us, waiting for loads behind the
// stream's; bringing tiles into L2 ten units ahead made it 1.9.
// O is rescaled only when a row's maximum has grown by more than 2^8 over the
// one its sums refer to: weights stay below 256, sums in fp32, and the quotient
// at the end does not depend on the reference.  P is rounded to the cache's type,
// as the product with V needs it; d sums the unrounded weights.  With that the
// results for prompts of N(0, 1) keys and values are off by 2.9e-4 (fp16, relative
// to the largest) where fp32 weights and a rounded result give 2.1e-4.
#pragma once
#include "tf_prefix_attention.cuh"
#include "tf_umma.cuh"

namespace tf {

template <int HD>
struct TensorShape {
    static constexpr int kKeys = HD > 128 ? 64 : 128;     // keys of a unit
    static constexpr int kSlot = kKeys * HD * 2;          // bytes of a K or V tile
    static constexpr int kSlots = HD > 64 ? 3 : 4;        // of K, and as many of V behind them
    static constexpr int kSmem = 2 * kSlots * kSlot + 1024;
    static constexpr int kColO = 0, kColQ = HD, kColS = HD + HD / 2;
};

// tcgen05 pieces that only this kernel uses
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

#define TF_R32(r) \
    "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),     \
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),   \
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),   \
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        TF_R32(r)
        : "memory");
}
#undef TF_R32

// 32 columns of this warp's lanes, without waiting for them
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld_wait(float (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    // the values may only be used from here on
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}

// Descriptors of a tile [group of 8 keys][64-dim block][8 keys][128 bytes], 16-byte
// chunk c of a row stored at c ^ (row % 8).  K-major (K tile): keys are N, `stride`
// from one group of eight to the next.  MN-major (V tile): keys are K, 64-wide
// blocks of N `leading` bytes apart, groups of eight keys `stride` bytes apart.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t leading, uint32_t stride) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 |
           (uint64_t)1u << 46 | (uint64_t)2u << 61;
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t attention_idesc(int n, bool b_mn_major) {
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kTcRows >> 4) << 24);
}

// The keys of one row tile, segment by segment.
struct TensorCursor {
    int seg, last;   // -1: prefix, else request; the tile's last request
    int tile, tiles; // key tile of the segment
    int lo, hi;      // keys of the segment; lo is rounded down to a box
    int from;        // the first that any row sees
};

// Requests of row tile i: [first, last], first > last when it has no tokens.
template <typename T>
__device__ __forceinline__ void requests_of_tile(const AttnParams<T>& p, int i, int& first, int& last) {
    const long long rows = (long long)p.T_tokens * p.G, row0 = (long long)i * kTcRows;
    first = request_at(p, (int)(row0 / p.G));
    last = min(p.B - 1, request_at(p, (int)((min(rows, row0 + kTcRows) - 1) / p.G)));
}

template <typename T, int HD>
__device__ __forceinline__ void tensor_segment(const AttnParams<T>& p, int i, TensorCursor& c) {
    c.tile = 0;
    if (c.seg < 0) {
        c.from = prefix_first(p);
        c.hi = p.prefix_few ? c.from : p.prefix_len;
    } else {
        const Request r = request_of(p, c.seg);
        c.from = c.hi = 0;
        if (is_many(p, r)) {
            // its tokens in the tile, and what they see of its own keys
            const int j0 = max(0, (int)((long long)i * kTcRows / p.G) - r.start);
            const int j1 = min(r.used, (int)((((long long)i + 1) * kTcRows - 1) / p.G) + 1 - r.start);
            if (j0 < j1) {
                int lo, hi, unused;
                seen_by(p, r, j0, lo, unused);
                seen_by(p, r, j1 - 1, unused, hi);
                c.from = max(0, min(r.len, lo - p.prefix_len));
                c.hi = max(c.from, min(r.len, hi - p.prefix_len));
            }
        }
    }
    c.lo = c.from & ~(kMaxRun - 1);
    c.tiles = c.hi > c.from ? (c.hi - c.lo + TensorShape<HD>::kKeys - 1) / TensorShape<HD>::kKeys : 0;
}

// First segment with keys of row tile i at or behind c.seg; false if none.
template <typename T, int HD>
__device__ __forceinline__ bool tensor_seek(const AttnParams<T>& p, int i, TensorCursor& c) {
    for (;;) {
        if (c.seg > c.last || (c.seg >= 0 && p.max_query * p.G <= p.many_above)) return false;
        tensor_segment<T, HD>(p, i, c);
        if (c.tiles) return true;
        if (c.seg < 0) {
            int first, last;
            requests_of_tile(p, i, first, last);
            c.seg = first;
        } else {
            ++c.seg;
        }
    }
}
// The first unit of the next segment.
template <typename T, int HD>
__device__ __noinline__ TensorCursor tensor_next_segment(const AttnParams<T>& p, int i, TensorCursor c) {
    if (c.seg < 0) {
        int first, last;
        requests_of_tile(p, i, first, last);
        c.seg = first;
    } else {
        ++c.seg;
    }
    tensor_seek<T, HD>(p, i, c);
    return c;
}
template <typename T, int HD>
__device__ __forceinline__ void tensor_advance(const AttnParams<T>& p, int i, TensorCursor& c) {
    if (++c.tile >= c.tiles) c = tensor_next_segment<T, HD>(p, i, c);
}
// The cursor at the `skip`-th unit of row tile i.
template <typename T, int HD>
__device__ __noinline__ TensorCursor tensor_begin(const AttnParams<T>& p, int i, int skip) {
    TensorCursor c;
    int first;
    requests_of_tile(p, i, first, c.last);
    c.seg = -1;
    while (tensor_seek<T, HD>(p, i, c) && skip >= c.tiles) {
        skip -= c.tiles;
        c.seg = c.seg < 0 ? first : c.seg + 1;
    }
    c.tile = skip;
    return c;
}
template <typename T, int HD>
__device__ __noinline__ int tensor_units(const AttnParams<T>& p, int i) {
    if (p.max_query * p.G <= p.many_above) {  // the prefix alone, for any tile with a token of the batch
        return (int)((long long)i * kTcRows / p.G) < p.starts[p.B] ? prefix_tiles(p, TensorShape<HD>::kKeys) : 0;
    }
    TensorCursor c;
    int first, units = 0;
    requests_of_tile(p, i, first, c.last);
    if (first > c.last) return 0;
    c.seg = -1;
    while (tensor_seek<T, HD>(p, i, c)) {
        units += c.tiles;
        c.seg = c.seg < 0 ? first : c.seg + 1;
    }
    return units;
}

// The units of all row tiles; `before` those before this thread's own [i0, i1).
template <typename T, int HD>
__device__ __forceinline__ int all_tensor_units(const AttnParams<T>& p, int* red, int i0, int i1, int& before) {
    int sum = 0, total;
    for (int i = i0; i < i1; ++i) sum += tensor_units<T, HD>(p, i) * p.nkv;
    before = block_scan(sum, red, &total);
    return total;
}

struct TensorBarriers {
    uint64_t full[2][4], empty[2][4], s_full[2],  // [K, V][slot]
        p_full[2], o_done[2], q_full, drained;
    uint32_t tmem;
    volatile int dead;
};

// One CTA: units [u0, u1) of worker `worker`; the first is in row tile `tile`,
// which begins at unit `tile_at` and has `tile_units` units a KV head.
template <typename T, int HD>
__device__ __forceinline__ void tensor_cta(const AttnParams<T>& p, uint32_t ring, TensorBarriers& bar, int u0, int u1,
                                           int tile0, int tile_at, int tile_units, int worker) {
    using S = TensorShape<HD>;
    constexpr int N = S::kKeys;
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kSlots; ++i) {
            for (int kv = 0; kv < 2; ++kv) {
                mbar_init(&bar.full[kv][i], 1);
                mbar_init(&bar.empty[kv][i], 1);
            }
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar.s_full[i], 1);
            mbar_init(&bar.p_full[i], 128);
            mbar_init(&bar.o_done[i], 1);
        }
        mbar_init(&bar.q_full, 128);
        mbar_init(&bar.drained, 1);
        fence_mbar_init();
        bar.dead = 0;
    }
    if (warp == 4) tmem_alloc(&bar.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem;

    // Bounded waits: about two seconds, or until another warp gave up.
    auto wait = [&](uint64_t* b, uint32_t parity) -> bool {
        if (mbar_try_wait(b, parity)) return true;
        const long long since = clock64();
        while (!mbar_try_wait(b, parity)) {
            if (bar.dead) return false;
            if (clock64() - since > 4000000000ll) {
                bar.dead = 1;
                atomicOr(p.err, kErrMbarTimeout);
                return false;
            }
        }
        return true;
    };
    // For warps that stay together: given up by the whole warp or by none of it (votes and tensor
    // memory instructions with lanes missing would wait for them for good).
    auto wait_warp = [&](uint64_t* b, uint32_t parity) { return __all_sync(0xffffffffu, wait(b, parity)) != 0; };
    // Every role walks the CTA's jobs: (row tile, KV head, units [from, to) of `units`).
    struct Job {
        int tile, kvh, units, from, to;
    };
    auto first_job = [&]() {
        Job j;
        const int in = u0 - tile_at;
        j.tile = tile0;
        j.units = tile_units;
        j.kvh = in / j.units;
        j.from = in % j.units;
        j.to = min(j.units, j.from + u1 - u0);
        return j;
    };
    auto next_job = [&](Job& j, int u) {  // u: units done
        j.from = 0;
        if (++j.kvh == p.nkv) {
            j.kvh = 0;
            do {
                j.units = tensor_units<T, HD>(p, ++j.tile);
            } while (j.units == 0);
        }
        j.to = min(j.units, u1 - u);
    };

    if (warp > 6) {
        // no work
    } else if (warp >= 5) {
        // ---- loaders: warp 5 K, warp 6 V, tile after tile -------------------------------
        const int kv = warp - 5;
        int it = 0;
        bool ok = true;
        Job job = first_job();
        for (int u = u0; ok && u < u1;) {
            TensorCursor c = tensor_begin<T, HD>(p, job.tile, job.from);
            TileKeys<N> next = look_up_keys<N>(p, c.seg, c.lo + c.tile * N, c.from, c.hi);
            for (int x = job.from; ok && x < job.to; ++x, ++it) {
                TileKeys<N> now = next;
                check_keys(p, now);
                if (x + 1 < job.to) {
                    tensor_advance<T, HD>(p, job.tile, c);
                    next = look_up_keys<N>(p, c.seg, c.lo + c.tile * N, c.from, c.hi);
                }
                const int slot = it % S::kSlots;
                ok = wait_warp(&bar.empty[kv][slot], ((it / S::kSlots) & 1) ^ 1);
                if (ok)
                    load_tile_keys<HD, N>(p, kv != 0, ring + (kv * S::kSlots + slot) * S::kSlot, job.kvh, now,
                                          &bar.full[kv][slot], false);
            }
            u += job.to - job.from;
            if (u < u1) next_job(job, u);
        }
        // what is in flight lands before the CTA may end: also what nobody waits for any more because
        // another warp gave up
        const long long since = clock64();
        const int issued = ok ? it : it - 1;
        for (int i = max(0, issued - S::kSlots); i < issued; ++i)
            mbar_wait_limited(&bar.full[kv][i % S::kSlots], (i / S::kSlots) & 1, p.err, since);
    } else if (warp == 4) {
        // ---- MMA issue: one elected thread ------------------------------------------
        if (elect_one()) {
            constexpr uint32_t kGroup8 = HD / 64 * 1024;  // bytes of eight keys
            constexpr uint32_t idesc_s = attention_idesc<T>(N, false), idesc_o = attention_idesc<T>(HD, true);
            struct Place {  // in a ring
                int slot = 0;
                uint32_t phase = 0;
                __device__ __forceinline__ void next() {
                    if (++slot == S::kSlots) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            } k, v;
            uint32_t s_buf = 0, p_buf = 0, p_phase = 0, q_phase = 0;  // score buffers of the next S and P
            bool ok = true;
            auto scores = [&]() {  // S = Q K^T of the next K tile
                const uint32_t base = ring + k.slot * S::kSlot, to = tmem + S::kColS + s_buf * N;
#pragma unroll 1  // four at a time: short enough to stay in the scheduler's instruction cache
                for (int b = 0; b < HD / 64; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        umma_f16_ts(to, tmem + S::kColQ + b * 32 + i * 8, tile_desc(base + b * 1024 + i * 32, 16, kGroup8),
                                    idesc_s, b > 0 || i > 0);
                umma_commit(&bar.s_full[s_buf]);
                umma_commit(&bar.empty[0][k.slot]);
                k.next();
                s_buf ^= 1;
            };
            Job job = first_job();
            for (int u = u0; ok && u < u1;) {
                const int n = job.to - job.from;
                ok = wait(&bar.q_full, q_phase) && wait(&bar.full[0][k.slot], k.phase);
                if (!ok) break;
                tc_fence_after();
                scores();
                // The scores of unit x + 1, then O += P V of unit x: the softmax of x + 1 runs beside
                // the second and the scores of x + 2.  About five MMAs can be queued, so behind PV's (128
                // clocks each) there is time for the waits before the next scores, and behind those
                // (32 clocks each) only for one: everything but the weights is waited for up front.
                for (int x = 0; x < n; ++x) {
                    const bool more = x + 1 < n;
                    ok = wait(&bar.full[1][v.slot], v.phase) && (!more || wait(&bar.full[0][k.slot], k.phase));
                    if (!ok) break;
                    tc_fence_after();
                    // S of unit x + 1 lies over P of unit x - 1: its product is over before that is overwritten
                    // (queued MMAs run in order, but only for one accumulator is that promised; 0.5 % slower)
                    if (more && x > 0) ok = wait(&bar.o_done[p_buf ^ 1], p_phase ^ p_buf ^ 1);
                    if (!ok) break;
                    if (more) scores();
                    ok = wait(&bar.p_full[p_buf], p_phase);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t base = ring + (S::kSlots + v.slot) * S::kSlot, p_at = tmem + S::kColS + p_buf * N;
#pragma unroll
                    for (int ks = 0; ks < N / 16; ++ks)
                        umma_f16_ts(tmem + S::kColO, p_at + ks * 8, tile_desc(base + ks * 2 * kGroup8, 1024, kGroup8),
                                    idesc_o, ks > 0 || x > 0);
                    umma_commit(&bar.empty[1][v.slot]);
                    umma_commit(&bar.o_done[p_buf]);
                    v.next();
                    p_phase ^= p_buf;
                    p_buf ^= 1;
                }
                q_phase ^= 1;
                u += n;
                if (u < u1) next_job(job, u);
            }
            // tensor memory is given back only when no MMA uses it, also after a wait that gave up
            umma_commit(&bar.drained);
            mbar_wait_limited(&bar.drained, 0, p.err);
        }
        __syncwarp();
    } else {
        // ---- a row per thread -------------------------------------------------------
        const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);  // this warp's lanes
        const float sc = p.scale * kLog2e;
        int uc = 0;
        bool ok = true;
        // O holds everything up to unit uc - 1.  A barrier for even and one for odd units:
        // a commit covers all earlier MMAs, so the scores of unit uc being there means that
        // the phase before the one waited for here (unit uc - 3) is over.
        auto o_ready = [&]() { return wait_warp(&bar.o_done[(uc - 1) & 1], ((uc - 1) >> 1) & 1); };
        Job job = first_job();
        for (int u = u0; ok && u < u1;) {
            const long long row = (long long)job.tile * kTcRows + threadIdx.x;
            const bool exists = row < (long long)p.T_tokens * p.G;
            const int t = exists ? (int)(row / p.G) : 0, h = job.kvh * p.G + (int)(row % p.G);
            int b = p.B, row_lo = 0, row_hi = 0;
            bool own = false;  // its own keys are this kernel's too
            if (exists) b = request_at(p, t);
            if (b < p.B) {
                const Request r = request_of(p, b);
                if (is_used(r, t - r.start)) {
                    seen_by(p, r, t - r.start, row_lo, row_hi);
                    own = is_many(p, r);
                } else {
                    b = p.B;
                }
            }
            const bool live = b < p.B;
            {  // Q to tensor memory
                const T* q = p.q + t * p.q_stride + (long long)h * p.hd;
#pragma unroll
                for (int c = 0; c < HD / 2; c += 32) {
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint4 x = make_uint4(0u, 0u, 0u, 0u);
                        if (live && c * 2 + i * 8 < p.hd) x = *reinterpret_cast<const uint4*>(q + c * 2 + i * 8);
                        w[4 * i] = x.x;
                        w[4 * i + 1] = x.y;
                        w[4 * i + 2] = x.z;
                        w[4 * i + 3] = x.w;
                    }
                    tmem_st32(mine + S::kColQ + c, w);
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&bar.q_full);
            }
            float m = -INFINITY, d = 0.f;
            TensorCursor c = tensor_begin<T, HD>(p, job.tile, job.from);
            for (int x = job.from; x < job.to; ++x, ++uc) {
                const int buf = uc & 1;
                ok = wait_warp(&bar.s_full[buf], (uc >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t scol = mine + S::kColS + buf * N;
                // the keys of this tile that the row sees: [lo, hi) of 0..N
                const int key0 = c.lo + c.tile * N;
                int lo = row_lo, hi = row_hi;
                if (c.seg >= 0) {
                    lo = b == c.seg ? lo - p.prefix_len : 0;
                    hi = b == c.seg ? hi - p.prefix_len : 0;
                }
                lo = max(0, lo - key0);
                hi = min(min(hi, c.hi) - key0, N);
                float s[N];
                if (__any_sync(0xffffffffu, hi > lo)) {
#pragma unroll
                    for (int i = 0; i < N; i += 32) tmem_ld32_async(scol + i, s + i);
                    tmem_ld_wait(s);
                    if (!__all_sync(0xffffffffu, lo == 0 && hi == N)) {
#pragma unroll
                        for (int i = 0; i < N; ++i) s[i] = i >= lo && i < hi ? s[i] : -INFINITY;
                    }
                    float top4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int i = 4; i < N; ++i) top4[i & 3] = fmaxf(top4[i & 3], s[i]);
                    const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])) * sc;
                    if (__any_sync(0xffffffffu, top > m + 8.f)) {
                        const float now = fmaxf(m, top);
                        const float f = m == -INFINITY ? 1.f : exp2_approx(m - now);
                        d *= f;
                        m = now;
                        if (x > job.from) {
                            ok = o_ready();
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll
                            for (int i = 0; i < HD; i += 32) {
                                float o[32];
                                tmem_ld32_async(mine + S::kColO + i, o);
                                tmem_ld_wait(o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] *= f;
                                tmem_st32(mine + S::kColO + i, reinterpret_cast<uint32_t*>(o));
                            }
                        }
                    }
                    const float ref = m == -INFINITY ? 0.f : m;
                    float d4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < N; i += 64) {
                        uint32_t w[32];
#pragma unroll
                        for (int e = 0; e < 64; e += 2) {
                            const float a = exp2_approx(fmaf(s[i + e], sc, -ref));
                            const float z = exp2_approx(fmaf(s[i + e + 1], sc, -ref));
                            d4[e & 2] += a;
                            d4[(e & 2) + 1] += z;
                            w[e / 2] = Pair<T>::pack(a, z);
                        }
                        tmem_st32(scol + i / 2, w);
                    }
                    d += (d4[0] + d4[1]) + (d4[2] + d4[3]);
                } else {
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) w[i] = 0u;
#pragma unroll
                    for (int i = 0; i < N / 2; i += 32) tmem_st32(scol + i, w);
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&bar.p_full[buf]);
                if (x + 1 < job.to) tensor_advance<T, HD>(p, job.tile, c);
            }
            // ---- the job's part, or the result where nothing else belongs to it ------
            ok = ok && o_ready();
            if (!ok) break;
            tc_fence_after();
            const bool whole = job.from == 0 && job.to == job.units;
            const bool final = whole && own;
            const long long of = (long long)t * p.nq + h;
            const long long at = job.from == 0 ? of : (long long)worker * kTcRows + threadIdx.x;
            float* po = (job.from == 0 ? p.many.first : p.many.cont) + at * p.hd;
            const float inv = d == 0.f ? 0.f : 1.f / d;
            bool fine = isfinite(d);
#pragma unroll
            for (int i = 0; i < HD; i += 32) {
                float o[32];
                tmem_ld32_async(mine + S::kColO + i, o);
                tmem_ld_wait(o);
                if (!live) continue;
                if (final) {
                    T* out = p.out + t * p.out_stride + (long long)h * p.hd;
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float a = o[e + 2 * k] * inv, z = o[e + 2 * k + 1] * inv;
                            fine &= isfinite(a) && isfinite(z);
                            w[k] = Pair<T>::pack(a, z);
                        }
                        if (i + e < p.hd) *reinterpret_cast<uint4*>(out + i + e) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        if (i + e < p.hd)
                            *reinterpret_cast<float4*>(po + i + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            if (live) {
                if (job.from == 0) p.many.first_of[of] = worker * kTcRows + threadIdx.x;
                if (job.to == job.units) p.many.last_of[of] = worker;
                if (final) {
                    if (p.lse) p.lse[at] = d == 0.f ? -INFINITY : (m + log2f(d)) * kLn2;
                    // NaN here asks the joining kernel to compute the row by itself
                    p.many.first_md[at] = make_float2(fine ? 0.f : __int_as_float(0x7fffffff), 0.f);
                } else {
                    (job.from == 0 ? p.many.first_md : p.many.cont_md)[at] = make_float2(m, d);
                }
            }
            tc_fence_before();
            u += job.to - job.from;
            if (u < u1) next_job(job, u);
        }
    }
    __syncthreads();
    if (warp == 4) tmem_dealloc(tmem, 512);
}

}  // namespace tf

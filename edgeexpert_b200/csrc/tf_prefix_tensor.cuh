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
// MMAs, warps 5-6 gather K and V by page into a ring of 128-byte-swizzled tiles.
// Scores of tile i+1 are computed while the softmax of tile i runs.
// O is rescaled only when a row's maximum has grown by more than 2^8 over the
// one its sums refer to: weights stay below 256, sums in fp32, and the quotient
// at the end does not depend on the reference.
#pragma once
#include "tf_prefix_attention.cuh"
#include "tf_umma.cuh"

namespace tf {

template <int HD>
struct TensorShape {
    static constexpr int kKeys = HD > 128 ? 64 : 128;     // keys of a unit
    static constexpr int kSlot = kKeys * HD * 2;          // bytes of a K or V tile
    static constexpr int kSlots = HD > 64 ? 6 : 8;
    static constexpr int kSmem = kSlots * kSlot + 1024;
    static constexpr int kColO = 0, kColQ = HD, kColS = HD + HD / 2;
    static constexpr int kLoaders = 2;                    // warps; with two warps at most on a scheduler,
    static constexpr int kThreads = 160 + 32 * kLoaders;  // a thread may have 255 registers
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

// Descriptors of a tile [HD/64 blocks][keys][128 bytes], 16-byte chunk c of a
// row stored at c ^ (row % 8).  K-major (K tile): rows are N, 8-row groups 1024
// bytes apart.  MN-major (V tile): rows are K, 8-row groups 1024 bytes apart
// (stride offset), 64-wide blocks of N `block` bytes apart (leading offset).
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t leading) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
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
    int lo, hi;      // keys of the segment
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
        c.lo = p.prefix_lo;
        c.hi = p.prefix_by_stream ? p.prefix_lo : p.prefix_len;
    } else {
        const Request r = request_of(p, c.seg);
        c.lo = c.hi = 0;
        if (by_tensor(p, r)) {
            // its tokens in the tile, and what they see of its own keys
            const int j0 = max(0, (int)((long long)i * kTcRows / p.G) - r.start);
            const int j1 = min(r.used, (int)((((long long)i + 1) * kTcRows - 1) / p.G) + 1 - r.start);
            if (j0 < j1) {
                int lo, hi, unused;
                seen_by(p, r, j0, lo, unused);
                seen_by(p, r, j1 - 1, unused, hi);
                c.lo = max(0, min(r.len, lo - p.prefix_len));
                c.hi = max(c.lo, min(r.len, hi - p.prefix_len));
            }
        }
    }
    c.tiles = (c.hi - c.lo + TensorShape<HD>::kKeys - 1) / TensorShape<HD>::kKeys;
}

// First segment with keys of row tile i at or behind c.seg; false if none.
template <typename T, int HD>
__device__ __forceinline__ bool tensor_seek(const AttnParams<T>& p, int i, TensorCursor& c) {
    for (;;) {
        if (c.seg > c.last || (c.seg >= 0 && p.max_query * p.G <= p.tensor_above)) return false;
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
template <typename T, int HD>
__device__ __forceinline__ void tensor_advance(const AttnParams<T>& p, int i, TensorCursor& c) {
    if (++c.tile < c.tiles) return;
    if (c.seg < 0) {
        int first, last;
        requests_of_tile(p, i, first, last);
        c.seg = first;
    } else {
        ++c.seg;
    }
    tensor_seek<T, HD>(p, i, c);
}
// The cursor at the `skip`-th unit of row tile i.
template <typename T, int HD>
__device__ __forceinline__ TensorCursor tensor_begin(const AttnParams<T>& p, int i, int skip) {
    TensorCursor c;
    int first;
    requests_of_tile(p, i, first, c.last);
    c.seg = -1;
    while (tensor_seek<T, HD>(p, i, c) && skip >= c.tiles) {
        skip -= c.tiles;
        c.tile = c.tiles - 1;
        if (c.seg < 0)
            c.seg = first;
        else
            ++c.seg;
    }
    c.tile = skip;
    return c;
}
template <typename T, int HD>
__device__ __forceinline__ int tensor_units(const AttnParams<T>& p, int i) {
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

template <typename T, int HD>
__global__ void __launch_bounds__(TensorShape<HD>::kThreads, 1)
    attention_many_rows_kernel(const __grid_constant__ AttnParams<T> p) {
    using S = TensorShape<HD>;
    constexpr int N = S::kKeys, CPR = HD / 8;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t full[S::kSlots], empty[S::kSlots], s_full[2], p_full[2], o_done[2], q_full,
        drained;
    __shared__ uint32_t s_tmem;
    __shared__ int red[32], s_tile, s_at, s_units;
    __shared__ volatile int s_dead;
    const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row_tiles = (int)(((long long)p.T_tokens * p.G + kTcRows - 1) / kTcRows);

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kSlots; ++i) {
            mbar_init(&full[i], S::kLoaders);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_done[i], 1);
        }
        mbar_init(&q_full, 128);
        mbar_init(&drained, 1);
        fence_mbar_init();
        s_dead = 0;
        s_units = 0;
    }
    // ---- which units are mine: sums over the row tiles, as in the stream kernel ----
    int U, u0, u1;
    {
        const int per = (row_tiles + blockDim.x - 1) / blockDim.x;
        const int i0 = min(row_tiles, (int)threadIdx.x * per), i1 = min(row_tiles, i0 + per);
        int sum = 0;
        for (int i = i0; i < i1; ++i) sum += tensor_units<T, HD>(p, i) * p.nkv;
        int at = block_scan(sum, red, &U);
        u0 = unit_begin(blockIdx.x, U, gridDim.x);
        u1 = unit_begin(blockIdx.x + 1, U, gridDim.x);
        for (int i = i0; i < i1; ++i) {
            const int units = tensor_units<T, HD>(p, i);
            if (blockIdx.x == 0) p.tensor.base[i] = at;
            if (u0 >= at && u0 < at + units * p.nkv) {
                s_tile = i;
                s_at = at;
                s_units = units;
            }
            at += units * p.nkv;
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) p.tensor.base[row_tiles] = U;
    }
    if (u0 >= u1) return;  // the same for the whole CTA
    if (warp == 4) tmem_alloc(&s_tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    // Bounded waits: about a second, or until another warp gave up.
    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        for (uint32_t i = 0; i < kSpinLimit; ++i) {
            if (mbar_try_wait_sleep(bar, parity, 1000u)) return true;
            if (s_dead) return false;
        }
        s_dead = 1;
        atomicOr(p.err, kErrMbarTimeout);
        return false;
    };
    // Every role walks the CTA's jobs: (row tile, KV head, units [from, to) of `units`).
    struct Job {
        int tile, kvh, units, from, to;
    };
    auto first_job = [&]() {
        Job j;
        const int in = u0 - s_at;
        j.tile = s_tile;
        j.units = s_units;
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

    if (warp >= 5) {
        // ---- loaders: tile after tile, K then V ---------------------------------
        const int lw = warp - 5;
        constexpr int kRows = N / S::kLoaders;          // of a tile, per warp
        constexpr int kLag = 2;                         // tiles between a copy's issue and its hand-over
        int it = 0;
        bool ok = true;
        auto hand_over = [&](int tile) {
            fence_proxy_async_smem();  // the copies are read by the tensor cores
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[tile % S::kSlots]);
        };
        Job job = first_job();
        for (int u = u0; ok && u < u1;) {
            TensorCursor c = tensor_begin<T, HD>(p, job.tile, job.from);
            for (int x = job.from; ok && x < job.to; ++x) {
                long long off[kRows / 32];  // element offsets of the keys lane, lane + 32, ...
                uint32_t mask[kRows / 32];  // which of them exist
#pragma unroll
                for (int w = 0; w < kRows / 32; ++w) {
                    const int pos = c.lo + c.tile * N + lw * kRows + w * 32 + lane;
                    bool have = false;
                    off[w] = 0;
                    if (pos < c.hi) {
                        const int at = pos / p.kv.page_size;
                        const int page = c.seg < 0 ? p.prefix_pages[at] : p.table[(long long)c.seg * p.max_pages + at];
                        have = page >= 0 && page < p.kv.num_pages;
                        if (have)
                            off[w] = page * p.kv.page_stride + (pos - at * p.kv.page_size) * p.kv.pos_stride +
                                     job.kvh * p.kv.head_stride;
                        else
                            atomicOr(p.err, kErrBadPage);
                    }
                    mask[w] = __ballot_sync(0xffffffffu, have);
                }
#pragma unroll 1
                for (int kv = 0; kv < 2 && ok; ++kv, ++it) {
                    const int slot = it % S::kSlots;
                    ok = wait(&empty[slot], ((it / S::kSlots) & 1) ^ 1);
                    if (!ok) break;
                    const T* src = kv ? p.kv.v : p.kv.k;
                    const uint32_t dst = ring + slot * S::kSlot;
                    constexpr int kPer = 32 * CPR / 32;  // copies of 32 rows, per lane
#pragma unroll
                    for (int w = 0; w < kRows / 32; ++w)
#pragma unroll 8
                        for (int i = 0; i < kPer; ++i) {
                            const int chunk = i * 32 + lane, rr = chunk / CPR, ch = chunk % CPR;
                            const int row = lw * kRows + w * 32 + rr;
                            const long long o = __shfl_sync(0xffffffffu, off[w], rr);
                            const int bytes = ((mask[w] >> rr) & 1) && ch * 8 < p.hd ? 16 : 0;
                            cp_async16(dst + (ch >> 3) * (N * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4),
                                       src + (bytes ? o + ch * 8 : 0), bytes);
                        }
                    cp_async_commit();
                    if (it >= kLag) {
                        cp_async_wait<kLag>();
                        hand_over(it - kLag);
                    }
                }
                if (x + 1 < job.to) tensor_advance<T, HD>(p, job.tile, c);
            }
            u += job.to - job.from;
            if (u < u1) next_job(job, u);
        }
        cp_async_wait<0>();
        if (ok)
            for (int tile = max(0, it - kLag); tile < it; ++tile) hand_over(tile);
    } else if (warp == 4) {
        // ---- MMA issue: one thread ------------------------------------------------
        if (lane == 0) {
            constexpr uint32_t idesc_s = attention_idesc<T>(N, false), idesc_o = attention_idesc<T>(HD, true);
            int uc = 0, jobs = 0;  // units and jobs so far
            bool ok = true;
            auto scores = [&](int x) {  // S[x % 2] = Q K^T of the CTA's x-th unit
                const int it = 2 * x, slot = it % S::kSlots;
                if (!wait(&full[slot], (it / S::kSlots) & 1)) return false;
                tc_fence_after();
                const uint32_t base = ring + slot * S::kSlot;
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks)
                    umma_f16_ts(tmem + S::kColS + (x & 1) * N, tmem + S::kColQ + ks * 8,
                                tile_desc(base + (ks >> 2) * (N * 128) + (ks & 3) * 32, 16), idesc_s, ks > 0);
                umma_commit(&empty[slot]);
                umma_commit(&s_full[x & 1]);
                return true;
            };
            Job job = first_job();
            for (int u = u0; ok && u < u1;) {
                const int n = job.to - job.from;
                ok = wait(&q_full, jobs & 1);
                tc_fence_after();
                ok = ok && scores(uc);
                for (int x = 0; ok && x < n; ++x) {
                    if (x + 1 < n) ok = scores(uc + x + 1);
                    const int it = 2 * (uc + x) + 1, slot = it % S::kSlots;
                    ok = ok && wait(&p_full[(uc + x) & 1], ((uc + x) >> 1) & 1) &&
                         wait(&full[slot], (it / S::kSlots) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t base = ring + slot * S::kSlot;
#pragma unroll
                    for (int ks = 0; ks < N / 16; ++ks)
                        umma_f16_ts(tmem + S::kColO, tmem + S::kColS + ((uc + x) & 1) * N + ks * 8,
                                    tile_desc(base + ks * 2048, N * 128), idesc_o, x > 0 || ks > 0);
                    umma_commit(&empty[slot]);
                    umma_commit(&o_done[(uc + x) & 1]);
                }
                uc += n;
                ++jobs;
                u += n;
                if (u < u1) next_job(job, u);
            }
            // tensor memory is given back only when no MMA uses it, also after a wait that gave up
            umma_commit(&drained);
            for (uint32_t i = 0; i < kSpinLimit && !mbar_try_wait_sleep(&drained, 0, 1000u); ++i) {
            }
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
        auto o_ready = [&]() { return wait(&o_done[(uc - 1) & 1], ((uc - 1) >> 1) & 1); };
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
                if (t - r.start < r.used) {
                    seen_by(p, r, t - r.start, row_lo, row_hi);
                    own = by_tensor(p, r);
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
                mbar_arrive(&q_full);
            }
            float m = -INFINITY, d = 0.f;
            TensorCursor c = tensor_begin<T, HD>(p, job.tile, job.from);
            for (int x = job.from; x < job.to; ++x, ++uc) {
                const int buf = uc & 1;
                ok = wait(&s_full[buf], (uc >> 1) & 1);
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
                mbar_arrive(&p_full[buf]);
                if (x + 1 < job.to) tensor_advance<T, HD>(p, job.tile, c);
            }
            // ---- the job's part, or the result where nothing else belongs to it ------
            ok = ok && o_ready();
            if (!ok) break;
            tc_fence_after();
            const bool whole = job.from == 0 && job.to == job.units;
            const bool final = whole && own;
            const long long at = job.from == 0 ? (long long)t * p.nq + h
                                               : (long long)blockIdx.x * kTcRows + threadIdx.x;
            float* po = (job.from == 0 ? p.tensor.first : p.tensor.cont) + at * p.hd;
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
                if (final) {
                    if (p.lse) p.lse[at] = d == 0.f ? -INFINITY : (m + log2f(d)) * kLn2;
                    // NaN here asks the joining kernel to compute the row by itself
                    p.tensor.first_md[at] = make_float2(fine ? 0.f : __int_as_float(0x7fffffff), 0.f);
                } else {
                    (job.from == 0 ? p.tensor.first_md : p.tensor.cont_md)[at] = make_float2(m, d);
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

// Attention of n <= 64 new rows (one token, or drafted tokens under a tree mask) to a bfloat16 or INT8 cache that already holds their own
// keys and values:  o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max),  j over the positions before `pos` and those
// of the new rows that row i's mask names.
//
// The G query heads of a key/value head and the n rows are G n query rows that read the same keys: they meet the cache in one pass.  Up to
// 16 of them run here, more on tcgen05 (scmx_cache_attn_tc.cu).  The products are taken transposed, S^T = K Q^T and O^T = V^T P^T (mma.sync m16n8k16, bfloat16, float32 sums): keys
// and values are the 16-row operand, query rows come eight at a time, so one row costs eight and an INT8 code is converted once for
// all rows.  The positions are cut into ranges, one CTA each; in a CTA every warp takes blocks of 16 positions of its own, brought into its own ring
// in shared memory by asynchronous copies, and keeps a running maximum, sum and output in registers.  The maximum is only raised when a
// score exceeds it by 2^8, so that most blocks neither exchange nor rescale anything.  The warps' states are joined in shared memory, the
// ranges' through the cluster's shared memory where the ranges of a key/value head are one cluster (few positions), by a second launch otherwise.
// INT8 codes become operands exactly, keys bfloat16 like the queries, values float16; a position's key scale multiplies its scores, the log2 of its value
// scale is added to them (CA_SHIFT), so that weights are float16.  Over bfloat16 a weight is two operands, what it rounds to and the rest (2^-16 of it):
// the second product costs 1 to 5 %, a single one made the output's error 0.0023 where rounding it costs 0.0016.
// Measured on a B200, one token, 8 key/value heads of 128: 1500 bfloat16 positions 5.4 us, launch latency and one round of loads; 65537 INT8
// positions 28.8 us, 4.8 TB/s, of which 5 us start, drain and join; within the ranges the conversions' integer operations keep the warps as busy as
// the loads.
#include <cooperative_groups.h>
#include "scmx_cache_attn.cuh"

namespace cg = cooperative_groups;

namespace scmx {

// NT: groups of eight query rows.  Warps: what registers and shared memory allow; INT8 needs more of them, its conversions are latency.
template <int D, bool I8, int NT>
struct CaShape {
    static constexpr int ROWS = 8 * NT;
    static constexpr int WARPS = !I8 ? 8 : NT == 1 ? 16 : 12;
    static constexpr int THREADS = 32 * WARPS;
    static constexpr int ROW = I8 ? D : 2 * D;                        // bytes of a vector
    static constexpr int BLOCK = CA_KEYS * ROW;                       // 16 keys or values
    static constexpr int STAGE = 2 * BLOCK + (I8 ? 128 : 0);          // keys, values, their scales
    static constexpr int STAGES = 3;
    static constexpr int RING = STAGE * STAGES;
    static constexpr int PITCH = D + 4;                               // a warp's state when the warps are joined: rows of values, then maxima and sums
    static constexpr int STATE = ROWS * (PITCH + 2) * 4;
    static constexpr int WARP = ((RING > STATE ? RING : STATE) + 127) / 128 * 128;
    static constexpr int TOTAL = WARP * WARPS + ROWS * (D + 2) * 4;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte offset of 16-byte piece c of vector r in a block: pieces are permuted within groups of eight so that the eight vectors of a matrix
// load, and the vectors of one INT8 value load, lie in different banks.
template <int ROW>
__device__ __forceinline__ int ca_at(int r, int c) {
    if constexpr (ROW == 64) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    return r * ROW + ((c ^ (r & 7)) << 4);
}
// An 8 x 8 matrix of 16-bit values, a row to four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
    return d;
}
template <int D, bool I8, int NT>
__global__ void __launch_bounds__(CaShape<D, I8, NT>::THREADS, 1) cache_attn_kernel(const __grid_constant__ CaArgs a) {
    using L = CaShape<D, I8, NT>;
    constexpr int ROW = L::ROW, PIECES = ROW / 16, KSTEPS = D / 16, MT = D / 16, WARPS = L::WARPS;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int kvh = blockIdx.x, split = blockIdx.y, G = a.G, R = G * a.n, row0 = blockIdx.z * L::ROWS;
    const int64_t pos = ca_pos(a.pos_dev, a.pos, a.cap, a.n), T = pos + a.n, chunk = ca_chunk(T, a.nsplit, a.unit);
    const int64_t t0 = split * chunk, t1 = t0 + chunk < T ? t0 + chunk : T;
    if (t0 >= T && !a.cluster) return;
    const unsigned char* kb = static_cast<const unsigned char*>(a.k) + ((int64_t)kvh * a.cap + t0) * ROW;
    const unsigned char* vb = static_cast<const unsigned char*>(a.v) + ((int64_t)kvh * a.cap + t0) * ROW;
    unsigned char* ring = smem_raw + warp * L::WARP;
    const uint32_t ring_s = smem_u32(ring);
    const int nkeys = t1 > t0 ? (int)(t1 - t0) : 0, nblocks = (nkeys + CA_KEYS - 1) / CA_KEYS, ntail = (int)(pos - t0 < nkeys ? pos - t0 : nkeys);      // keys from ntail on are new rows (negative: from before t0)

    // copies of block b: pieces lane, lane + 32, .. of 16 bytes; a warp covers whole vectors with each, whose places repeat after DIST
    constexpr int COPIES = CA_KEYS * PIECES / 32, RSTEP = 32 / PIECES, DIST = RSTEP >= 8 ? 1 : 8 / RSTEP;
    const int lr0 = lane / PIECES;
    int at[DIST];
#pragma unroll
    for (int p = 0; p < DIST; ++p) at[p] = ca_at<ROW>(lr0 + p * RSTEP, lane % PIECES);
    auto load = [&](int b, int stage) {
        if (b < nblocks) {
            const uint32_t dst = ring_s + stage * L::STAGE;
            const int left = nkeys - b * CA_KEYS;
            const unsigned char *ksrc = kb + (int64_t)b * L::BLOCK + lane * 16, *vsrc = vb + (int64_t)b * L::BLOCK + lane * 16;
            if (left >= CA_KEYS) {
#pragma unroll
                for (int p = 0; p < COPIES; ++p) {
                    const uint32_t to = dst + at[p % DIST] + p / DIST * (DIST * RSTEP * ROW);
                    cp_async16(to, ksrc + p * 512, true);
                    cp_async16(to + L::BLOCK, vsrc + p * 512, true);
                }
            } else {
#pragma unroll
                for (int p = 0; p < COPIES; ++p) {
                    const uint32_t to = dst + at[p % DIST] + p / DIST * (DIST * RSTEP * ROW);
                    const bool on = lr0 + p * RSTEP < left;
                    cp_async16(to, on ? ksrc + p * 512 : kb, on);
                    cp_async16(to + L::BLOCK, on ? vsrc + p * 512 : vb, on);
                }
            }
            if constexpr (I8) {
                const bool on = (lane & 15) < left;
                const float* s = (lane < 16 ? a.ks : a.vs) + (int64_t)kvh * a.cap + t0 + (on ? b * CA_KEYS + (lane & 15) : 0);
                cp_async4(dst + 2 * L::BLOCK + 4 * lane, s, on);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int s = 0; s < L::STAGES - 1; ++s) load(warp + s * WARPS, s);

    // query rows, as the B operand: row g of each group of eight (rows past the last are read from row 0 and cleared, so that no load waits for another)
    uint2 qf[NT][KSTEPS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = row0 + 8 * nt + g, rr = r < R ? r : 0, tok = ca_tok(a, rr);
        const uint16_t* qp = a.q + (int64_t)(kvh * G + rr - tok * G) * a.q_hs + (int64_t)tok * a.q_rs;
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
            if constexpr (I8) qf[nt][s] = *reinterpret_cast<const uint2*>(qp + 16 * s + 4 * t4);
            else qf[nt][s] = make_uint2(*reinterpret_cast<const uint32_t*>(qp + 16 * s + 2 * t4), *reinterpret_cast<const uint32_t*>(qp + 16 * s + 8 + 2 * t4));
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
            uint2& w = qf[nt][s];
            if (I8) w = make_uint2(__byte_perm(w.x, w.y, 0x5410), __byte_perm(w.x, w.y, 0x7632));      // values 0 and 2, 1 and 3 of a word of codes
            if (row0 + 8 * nt + g >= R) w = make_uint2(0, 0);
        }

    // rows 2 t4 and 2 t4 + 1 of each group: maximum and sum; output: 16 values of the vectors times eight rows
    float o[MT][NT][4], mx[NT][2], sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            mx[nt][e] = -INFINITY;
            sum[nt][e] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][nt][j] = 0.0f;
    }

    const I8Pairs i8;
    const I8Halves i8h;
    const int lr = lane & 7, lm = lane >> 3;            // row of a matrix load, and which of its four matrices
    int stage = 0;
    float ref = 0.0f;                                   // INT8: log2 of the scale that the warp's values are relative to
    for (int b = warp; b < nblocks; b += WARPS) {
        cp_wait<L::STAGES - 2>();
        __syncwarp();
        load(b + (L::STAGES - 1) * WARPS, stage == 0 ? L::STAGES - 1 : stage - 1);
        const unsigned char* blk = ring + stage * L::STAGE;
        const uint32_t kst = ring_s + stage * L::STAGE, vst = kst + L::BLOCK;
        // scores: keys g and g + 8, rows 2 t4 and 2 t4 + 1
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[nt][j] = 0.0f;
        auto scores = [&](int c, const uint32_t (&w)[4]) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_bf16(s[nt], w, qf[nt][c].x, qf[nt][c].y);
        };
        if constexpr (I8) {
#pragma unroll
            for (int c = 0; c < KSTEPS; c += 2) {
                uint32_t w[4];                          // keys 0-7, keys 8-15 of piece c, the same of piece c + 1
                ldsm4(kst + ca_at<ROW>(lr + 8 * (lm & 1), c + (lm >> 1)), w);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t f[4] = {i8.even(w[2 * e]), i8.even(w[2 * e + 1]), i8.odd(w[2 * e]), i8.odd(w[2 * e + 1])};
                    scores(c + e, f);
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < KSTEPS; ++c) {
                uint32_t w[4];
                ldsm4(kst + ca_at<ROW>(lr + 8 * (lm & 1), 2 * c + (lm >> 1)), w);
                scores(c, w);
            }
        }
        float kf[2] = {a.scale, a.scale}, lg[2] = {0.0f, 0.0f}, inv[2] = {1.0f, 1.0f};
        if constexpr (I8) {
            const float* scales = reinterpret_cast<const float*>(blk + 2 * L::BLOCK);
            if (b == warp) {
                const int key = b * CA_KEYS + (lane & 15);
                const float first[1] = {scales[16 + (lane & 15)]};
                const uint64_t any = (b + 1) * CA_KEYS > ntail ? ca_seen_by_any(a, lane) : 0;
                const bool from[1] = {key < ntail || (key - ntail < a.n && (any >> ((key - ntail) & 63) & 1))};
                ref = ca_reference(first, from);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                kf[h] *= scales[g + 8 * h];
                ca_scale(scales[16 + g + 8 * h], ref, lg[h], inv[h]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[nt][j] = I8 ? fmaf(s[nt][j], kf[j >> 1], lg[j >> 1]) : s[nt][j] * kf[j >> 1];
        const int d0 = b * CA_KEYS - ntail;             // the block's first key, counted from the first new row
        const bool tail = d0 + CA_KEYS > 0;             // some keys are new rows, or past the end
        uint32_t seen = 0xFFFFFFFFu;                    // bit 4 nt + j
        if (tail) {
            seen = 0;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = row0 + 8 * nt + 2 * t4 + e, tok = ca_tok(a, r);
                    if (r < R) {
                        const uint64_t bits = a.mask ? (uint64_t)a.mask[tok] : (2ull << tok) - 1ull;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int d = d0 + g + 8 * h;
                            if (d < 0 || (d < a.n && (bits >> d & 1))) seen |= 1u << (4 * nt + 2 * h + e);
                        }
                    }
                }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!(seen >> (4 * nt + j) & 1)) s[nt][j] = -INFINITY;
        }
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) grow |= fmaxf(s[nt][e], s[nt][2 + e]) > mx[nt][e] + CA_GROWTH;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float m = fmaxf(s[nt][e], s[nt][2 + e]);
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
                    m = fmaxf(m, mx[nt][e]);
                    const float f = mx[nt][e] == -INFINITY ? 0.0f : ca_ex2(mx[nt][e] - m);      // nothing so far: sum and output are zero
                    mx[nt][e] = m;
                    sum[nt][e] *= f;
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        o[i][nt][e] *= f;
                        o[i][nt][2 + e] *= f;
                    }
                }
        }
        uint32_t pb[NT][2], pl[NT][2];                 // weights as an operand; bfloat16: and what its rounding left of them
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float base = mx[nt][e] == -INFINITY ? 0.0f : I8 ? mx[nt][e] - CA_SHIFT : mx[nt][e];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float& x = s[nt][2 * h + e];
                    x = ca_ex2(x - base);
                    if constexpr (I8) {
                        if (!tail || (seen >> (4 * nt + 2 * h + e) & 1)) sum[nt][e] = fmaf(x, inv[h], sum[nt][e]);      // an unseen one's scale may be anything
                    } else {
                        sum[nt][e] += x;
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (I8) {
                    pb[nt][h] = transpose8(pack_f16x2(s[nt][2 * h], s[nt][2 * h + 1]));
                } else {
                    const uint32_t p = pack_bf16x2(s[nt][2 * h], s[nt][2 * h + 1]);
                    pb[nt][h] = transpose8(p);
                    pl[nt][h] = transpose8(pack_bf16x2(s[nt][2 * h] - bf16_lo(p), s[nt][2 * h + 1] - bf16_hi(p)));
                }
            }
        }
        // a value that is not finite must not reach rows that do not see it: such blocks, which only new rows can make, go key by key
        bool odd = false;
        if constexpr (!I8) {
            if (tail) {
#pragma unroll
                for (int i = 0; i < COPIES; ++i) {
                    const uint4 w = *reinterpret_cast<const uint4*>(blk + L::BLOCK + 16 * (32 * i + lane));
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) odd = odd || (u[j] & 0x7F800000u) == 0x7F800000u || (u[j] & 0x7F80u) == 0x7F80u;
                }
                odd = __any_sync(0xffffffffu, odd);
            }
        }
        if (odd) {
#pragma unroll 1
            for (int kk = 0; kk < CA_KEYS; ++kk) {
                const int src = 4 * (kk & 7) + t4;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float lo = __shfl_sync(0xffffffffu, s[nt][e], src), hi = __shfl_sync(0xffffffffu, s[nt][2 + e], src);
                        const uint32_t bits = __shfl_sync(0xffffffffu, seen, src);
                        const float w = kk < 8 ? lo : hi;
                        if (bits >> (4 * nt + (kk < 8 ? 0 : 2) + e) & 1) {
#pragma unroll
                            for (int i = 0; i < MT; ++i)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const float x = bf16_to_f32(*reinterpret_cast<const uint16_t*>(blk + L::BLOCK + ca_at<ROW>(kk, 2 * i + h) + 2 * g));
                                    o[i][nt][2 * h + e] = fmaf(w, x, o[i][nt][2 * h + e]);
                                }
                        }
                    }
            }
        } else if constexpr (I8) {
#pragma unroll
            for (int i = 0; i < MT; i += 2) {           // pairs of values as 16-bit units: keys 0-7, 8-15 of piece i, the same of piece i + 1
                uint32_t w[4];
                ldsm4_t(vst + ca_at<ROW>(lr + 8 * (lm & 1), i + (lm >> 1)), w);
#pragma unroll
                for (int e = 0; e < 2; ++e) {           // operand rows g and g + 8: values 2 g and 2 g + 1 of the piece
                    const uint32_t f[4] = {i8h.even(w[2 * e]), i8h.odd(w[2 * e]), i8h.even(w[2 * e + 1]), i8h.odd(w[2 * e + 1])};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_f16(o[i + e][nt], f, pb[nt][0], pb[nt][1]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint32_t w[4];                          // values 0-7, 8-15 of keys 0-7, the same of keys 8-15
                ldsm4_t(vst + ca_at<ROW>(lr + 8 * (lm >> 1), 2 * i + (lm & 1)), w);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma_bf16(o[i][nt], w, pb[nt][0], pb[nt][1]);
                    mma_bf16(o[i][nt], w, pl[nt][0], pl[nt][1]);
                }
            }
        }
        stage = stage + 1 == L::STAGES ? 0 : stage + 1;
    }
    cp_wait<0>();
    __syncwarp();

    // the warps' states, joined: a warp to a row
    float* st = reinterpret_cast<float*>(ring);
    const float by = I8 ? ca_ex2(ref) : 1.0f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float l = I8 ? sum[nt][e] * CA_DOWN : sum[nt][e];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
            const int r = 8 * nt + 2 * t4 + e;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) st[r * L::PITCH + (I8 ? 16 * i + 2 * g + h : 16 * i + 8 * h + g)] = I8 ? o[i][nt][2 * h + e] * CA_DOWN * by : o[i][nt][2 * h + e];
            if (g == 0) reinterpret_cast<float2*>(st + L::ROWS * L::PITCH)[r] = make_float2(mx[nt][e], l);
        }
    __syncthreads();
    constexpr int E = D / 32;
    const int live = nblocks < WARPS ? nblocks : WARPS, rows = R - row0 < L::ROWS ? R - row0 : L::ROWS;      // warps that had a block; rows of this tile
    const float* states = reinterpret_cast<const float*>(smem_raw);
    float* joined = reinterpret_cast<float*>(smem_raw + WARPS * L::WARP);      // this range's state: values, then maxima and sums
    for (int r = warp; r < rows; r += WARPS) {
        const float2 ml = lane < live ? reinterpret_cast<const float2*>(states + lane * (L::WARP / 4) + L::ROWS * L::PITCH)[r] : make_float2(-INFINITY, 0.0f);
        float m = ml.x, l = ml.y, v[E];
        ca_join<E, 8>(live, m, l, v, [&](int s, float (&z)[E]) { ca_load<E>(states + s * (L::WARP / 4) + r * L::PITCH + lane * E, z); });
        if (a.cluster) {
            ca_store<E>(joined + r * D + lane * E, v);
            if (lane == 0) reinterpret_cast<float2*>(joined + L::ROWS * D)[r] = make_float2(m, l);
        } else if (a.part == nullptr) {
            ca_output<D>(a, kvh, row0 + r, lane, v, l);
        } else {
            const int64_t at = (((int64_t)kvh * gridDim.z + blockIdx.z) * a.nsplit + split) * L::ROWS + r;
            ca_store<E>(a.part + at * D + lane * E, v);
            if (lane == 0) a.part_ml[at] = make_float2(m, l);
        }
    }
    if (a.cluster) {                     // the ranges' states, read where they lie: the rows in turn to the CTAs
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        const int ctas = (int)cl.num_blocks();
        for (int r = (int)cl.block_rank() + ctas * warp; r < rows; r += ctas * WARPS) {
            const float2 ml = lane < ctas ? reinterpret_cast<const float2*>(cl.map_shared_rank(joined, lane) + L::ROWS * D)[r] : make_float2(-INFINITY, 0.0f);
            float m = ml.x, l = ml.y, v[E];
            ca_join<E, 8>(ctas, m, l, v, [&](int s, float (&z)[E]) { ca_load<E>(cl.map_shared_rank(joined, s) + r * D + lane * E, z); });
            ca_output<D>(a, kvh, row0 + r, lane, v, l);
        }
        cl.sync();                       // nobody leaves while its state may still be read
    }
}

// Joins the ranges: a warp to a query row.
template <int D>
__global__ void __launch_bounds__(128) cache_attn_join_kernel(const __grid_constant__ CaArgs a, int tiles, int rows) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, R = a.G * a.n, i = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (i >= a.hk * R) return;
    constexpr int E = D / 32;
    const int kvh = i / R, r = i - kvh * R, tile = r / rows;
    const int64_t T = ca_pos(a.pos_dev, a.pos, a.cap, a.n) + a.n, chunk = ca_chunk(T, a.nsplit, a.unit);
    const int active = ca_ranges(T, chunk);
    const int64_t first = ((int64_t)kvh * tiles + tile) * a.nsplit * rows + (r - tile * rows);
    float m = -INFINITY, l = 0.0f, v[E] = {};
    for (int s0 = 0; s0 < active; s0 += 32) {
        const int count = active - s0 < 32 ? active - s0 : 32;
        const float2 ml = lane < count ? a.part_ml[first + (int64_t)(s0 + lane) * rows] : make_float2(-INFINITY, 0.0f);
        float m2 = ml.x, l2 = ml.y, v2[E];
        ca_join<E, 10>(count, m2, l2, v2, [&](int s, float (&z)[E]) { ca_load<E>(a.part + (first + (int64_t)(s0 + s) * rows) * D + lane * E, z); });
        const float top = fmaxf(m, m2), f1 = m == -INFINITY ? 0.0f : ca_ex2(m - top), f2 = m2 == -INFINITY ? 0.0f : ca_ex2(m2 - top);
        l = l * f1 + l2 * f2;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = (f1 == 0.0f ? 0.0f : v[e] * f1) + (f2 == 0.0f ? 0.0f : v2[e] * f2);
        m = top;
    }
    ca_output<D>(a, kvh, r, lane, v, l);
}

// Whether the ranges of a head are one cluster of at most eight CTAs, which joins them without a second launch (and 6 us sooner on the host), or as many as the device
// has room for.  Device us of a call among others, cluster / two launches, head size 128 (64 alike unless said):
//   All clusters have to run at once: fifteen of eight did (120 CTAs), sixteen waited for one another, 32 of four did.  1000 positions, 2 query rows: 15 key/value heads 5.8 / 7.6, 16 heads
//   9.7 / 7.7, 32 heads 14.5 / 9.0; INT8, 21 rows: 10.1 / 10.0, 18.2 / 10.6, 28.1 / 12.5.  500 positions, 21 rows in clusters of four: 32 heads 10.3 / 11.3.
//   A single range is no cluster: 60 positions 4.5 / 3.4 (one launch), 21 rows 9.2 / 6.7.
//   Few rows, 2 and 16 of them, bfloat16, 1 / 4 / 8 / 15 heads: 8000 positions 8.8 / 17.0, 9.2 / 11.9, 10.0 / 11.8, 13.4 / 15.1 and 12.2 / 19.3, 12.8 / 16.4, 13.8 / 15.3, 16.0 / 17.3;
//   16000 12.9 / 20.2, 13.3 / 14.2, 14.7 / 16.1, 21.9 / 23.6 and 17.5 / 23.8, 18.0 / 18.0, 18.9 / 19.0, 24.8 / 26.4; 24000 and 4 heads 17.8 / 16.7 and 23.7 / 20.4.
//   INT8: 8000 9.3 / 16.9, 10.0 / 11.8, 10.6 / 11.1, 11.6 / 13.4 and 13.3 / 18.9, 13.8 / 15.7, 14.4 / 14.9, 15.1 / 16.7; 12000 and 8 heads 12.9 / 12.8 and 17.3 / 16.2.
//   On tcgen05 tiles that hold copies, 21 and 42 rows, bfloat16: 4000 10.6 / 11.6, 11.5 / 12.6, 12.3 / 13.2, 13.9 / 15.1 and 11.8 / 12.1, 12.5 / 13.6, 13.2 / 13.8, 14.9 / 16.1; 6000 12.7 / 13.6, 13.7 / 13.7,
//   14.6 / 15.7, 16.6 / 17.7 and 14.2 / 14.6, 14.8 / 14.3, 15.6 / 16.2, 17.5 / 19.0; 10000 14.5 / 16.9, 15.0 / 13.2, 16.3 / 16.2 and 15.7 / 17.7, 16.3 / 13.9, 17.3 / 16.7.
//   INT8, 1 / 4 / 8 / 15 heads: 2000 9.4 / 9.8, 9.6 / 9.7, 10.7 / 10.6, 11.5 / 12.2 and 10.9 / 10.6, 11.0 / 10.5, 12.2 / 12.5, 13.1 / 13.8; 4000 11.6 / 11.3, 12.5 / 12.0, 13.3 / 13.6, 14.7 / 15.3 and
//   13.3 / 12.0, 14.2 / 13.1, 14.8 / 14.9, 16.1 / 17.2; 6000 13.9 / 12.7, 15.0 / 14.7, 16.1 / 15.2, 17.6 / 18.9 and 15.8 / 13.7, 16.8 / 16.1, 17.8 / 16.8, 19.4 / 20.6.  Here the device loses up to
//   2 us with few heads, but calls that are not in a graph wait for the host: 42 rows over 6001 positions, 8 heads, 17.0 / 19.5 a call.
//   Full tiles: 84 rows over 4000 positions, 8 heads, 16.3 / 15.0, 256 rows 25.3 / 19.9.
static bool ca_joins_in_cluster(const CaPlan& p, int nsplit, int64_t positions, int hk, bool int8) {
    if (nsplit < 2 || (p.tc && p.copies == 1)) return false;
    if ((int64_t)hk * p.tiles * nsplit > sm_count() * (nsplit == 8 ? 13 : 14) / 16) return false;
    return positions <= (p.tc ? 6144 : int8 ? 8192 : 16384);
}

static CaPlan ca_plan(int64_t positions, int R, int hk, bool int8) {
    CaPlan p;
    p.cluster = 0;
    // Up to 16 query rows two groups of eight read the cache once; more would read it again, and tcgen05's tile has 128 rows.  Device us, mma.sync / tcgen05, head size 128, over 1500, 6000,
    // 20000 and 60000 positions of 8 key/value heads: bfloat16, 16 rows 8.9 / 9.8, 12.2 / 12.2, 21.7 / 21.0, 45.2 / 44.3, 20 rows 12.5 / 10.0, 18.8 / 12.4, 23.0 / 21.1, 48.9 / 44.4; INT8 8.4 / 10.2,
    // 12.6 / 15.8, 18.9 / 25.2, 32.8 / 47.2 and 13.0 / 10.4, 20.6 / 16.0, 23.9 / 25.4, 51.1 / 47.5.  Of 2 heads: bfloat16, 16 rows 7.8 / 8.7, 11.3 / 11.1, 22.3 / 16.2, 27.2 / 23.7, 20 rows 8.0 / 8.8,
    // 11.4 / 11.2, 17.7 / 16.3, 23.9 / 23.7; INT8 8.1 / 9.4, 11.9 / 14.2, 20.1 / 19.5, 23.4 / 30.0 and 8.4 / 9.6, 11.8 / 14.4, 17.2 / 20.3, 24.5 / 30.9.
    p.tc = R > 16;
    if (p.tc) {
        p.nt = R > 128 ? 2 : 1;
        p.copies = R <= 32 ? 4 : R <= 64 ? 2 : 1;
        p.rows = 128 * p.nt / p.copies;
        p.unit = 128;
    } else {
        p.nt = R <= 8 ? 1 : 2;
        p.copies = 1;
        p.rows = 8 * p.nt;
        p.unit = 4 * CA_KEYS;
    }
    p.tiles = (R + p.rows - 1) / p.rows;
    const int64_t most = (positions + p.unit - 1) / p.unit, want = sm_count() / ((int64_t)hk * p.tiles);
    const int64_t s = want < most ? want : most;
    p.nsplit = s < 1 ? 1 : (int)s;
    const int ctas = most >= 8 ? 8 : most >= 3 ? 4 : most == 2 ? 2 : 1;
    if (ca_joins_in_cluster(p, ctas, positions, hk, int8)) {
        p.cluster = 1;
        p.nsplit = ctas;
    }
    if (!p.tc && positions > (int64_t)p.nsplit * p.unit) p.unit = CA_KEYS;      // long enough: ranges end at any block
    return p;
}

template <int D, bool I8, int NT>
static int launch_ca(const CaArgs& a, const CaPlan& p, cudaStream_t st) {
    using L = CaShape<D, I8, NT>;
    static bool configured[64] = {};
    const int dev = current_device();
    SCMX_REQUIRE(dev >= 0, SCMX_ECUDA, "no current CUDA device (ordinal 0..63)");
    if (!configured[dev]) {
        SCMX_CUDA_OK(cudaFuncSetAttribute(cache_attn_kernel<D, I8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL));
        configured[dev] = true;
    }
    SCMX_PDL_OK("cache_attn_kernel", ca_launch(cache_attn_kernel<D, I8, NT>, a.hk, p, L::THREADS, L::TOTAL, st, a));
    return SCMX_OK;
}
template <int D, bool I8>
static int dispatch_ca(const CaArgs& a, const CaPlan& p, cudaStream_t st) { return p.nt == 1 ? launch_ca<D, I8, 1>(a, p, st) : launch_ca<D, I8, 2>(a, p, st); }
static int64_t ca_states(const CaPlan& p, int hk) { return p.nsplit == 1 || p.cluster ? 0 : (int64_t)hk * p.tiles * p.nsplit * p.rows; }      // partial states of query rows

}  // namespace scmx

using namespace scmx;

extern "C" int64_t scmx_cache_attn_scratch(int64_t positions, int n, int hq, int hk, int d) {
    if (positions < 1 || n < 1 || n > CA_MAX_ROWS || hk < 1 || hq < hk || hq % hk || (d != 64 && d != 128)) return 0;
    const int64_t bf16 = ca_states(ca_plan(positions, hq / hk * n, hk, false), hk), int8 = ca_states(ca_plan(positions, hq / hk * n, hk, true), hk);      // either type's
    return (bf16 > int8 ? bf16 : int8) * (d + 2) * 4;
}

extern "C" int scmx_cache_attn(const uint16_t* q, int64_t q_head_stride, int64_t q_row_stride, const void* k, const void* v, const float* k_scales,
                               const float* v_scales, int int8, const int64_t* mask, int n, int64_t pos, const int32_t* pos_dev, int64_t capacity, int hq, int hk,
                               int d, float scale, uint16_t* out, void* scratch, int64_t scratch_bytes, int32_t* status, void* stream) {
    SCMX_REQUIRE(q && k && v && out && status && (!int8 || (k_scales && v_scales)), SCMX_EINVAL, "cache_attn: null buffer");
    SCMX_REQUIRE(n >= 1 && n <= CA_MAX_ROWS, SCMX_ELIMIT, "cache_attn: %d rows (1 .. %d)", n, CA_MAX_ROWS);
    SCMX_REQUIRE(d == 64 || d == 128, SCMX_EINVAL, "cache_attn: head size %d (64 or 128)", d);
    SCMX_REQUIRE(hk > 0 && hq > 0 && hq % hk == 0 && hq / hk <= 4096, SCMX_EINVAL, "cache_attn: hq=%d hk=%d", hq, hk);
    SCMX_REQUIRE(capacity >= n && (pos_dev != nullptr || (pos >= 0 && pos + n <= capacity)), SCMX_EINVAL, "cache_attn: rows %lld .. %lld of a cache of %lld",
                 (long long)pos, (long long)(pos + n), (long long)capacity);
    SCMX_REQUIRE(q_head_stride % 4 == 0 && q_row_stride % 4 == 0 && ((uintptr_t)q & 7) == 0 && ((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0 &&
                     ((uintptr_t)out & 15) == 0, SCMX_EINVAL, "cache_attn: query rows must be 8-byte, caches and the output 16-byte aligned");
    CaArgs a;
    const CaPlan p = ca_plan(pos_dev ? capacity : pos + n, hq / hk * n, hk, int8 != 0);
    a.nsplit = p.nsplit; a.unit = p.unit; a.cluster = p.cluster;
    const int64_t states = ca_states(p, hk), need = states * (d + 2) * 4;
    SCMX_REQUIRE(scratch_bytes >= need && (need == 0 || (scratch && ((uintptr_t)scratch & 15) == 0)), SCMX_EINVAL, "cache_attn: %lld bytes of scratch, %lld needed",
                 (long long)scratch_bytes, (long long)need);
    a.q = q; a.q_hs = q_head_stride; a.q_rs = q_row_stride; a.k = k; a.v = v; a.ks = k_scales; a.vs = v_scales; a.mask = mask; a.pos_dev = pos_dev; a.pos = pos;
    a.part = need ? static_cast<float*>(scratch) : nullptr; a.part_ml = need ? reinterpret_cast<float2*>(a.part + states * d) : nullptr; a.out = out; a.cap = capacity; a.n = n; a.hq = hq; a.hk = hk; a.G = hq / hk; a.inv_g = 1.0f / (float)a.G; a.scale = scale * CA_LOG2E;
    const cudaStream_t st = (cudaStream_t)stream;
    int rc = p.tc ? cache_attn_tc(a, p, d, int8, status, st)
             : d == 128 ? (int8 ? dispatch_ca<128, true>(a, p, st) : dispatch_ca<128, false>(a, p, st))
                        : (int8 ? dispatch_ca<64, true>(a, p, st) : dispatch_ca<64, false>(a, p, st));
    if (rc != SCMX_OK || a.part == nullptr) return rc;
    void (*join)(CaArgs, int, int) = d == 128 ? cache_attn_join_kernel<128> : cache_attn_join_kernel<64>;
    SCMX_PDL_OK("cache_attn_join_kernel", launch_pdl(join, dim3((unsigned)((hq * n + 3) / 4)), dim3(128), 0, st, a, p.tiles, p.rows));
    return SCMX_OK;
}

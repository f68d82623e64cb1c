// Attention of more than 16 query rows (drafted rows times the query heads of a key/value head) to a cache, on tcgen05.  The formula, the cut into
// ranges of positions and the join of the ranges are those of scmx_cache_attn.cu; here a CTA takes 128 or 256 query rows.
//
// Two streams share the tensor core: while it works for one, the other's softmax runs.  With one query tile of 128 rows the streams take the
// key tiles (128 positions) in turn and are joined at the end; with two, each stream has a query tile of its own.  A `unit` is a stream's work
// on one key tile: S = Q K^T (128 x 128, float32 in tensor memory), softmax, O += P V with P (bfloat16; float16 over INT8) read from tensor memory, where
// it overwrites S.
//   warps 0-7     two softmax warpgroups, one per stream, a thread per lane of tensor memory.  The maximum is raised when it has grown by
//                 more than 2^8
//   warps 8-15    (INT8) codes of a tile from memory to operands, exactly, keys to bfloat16 and values to float16; a position's key scale multiplies
//                 its scores, and the log2 of its value scale is added to them (CA_SHIFT).  Vectors are stored with values 1 and 2 of every four exchanged, as the conversion leaves them: queries are
//                 laid out alike, and outputs put back.  Tiles ahead are prefetched into L2
//   last warps    one issues all MMAs (it stays converged, one lane issues), one loads key and value tiles by TMA (bfloat16)
// INT8: registers are shared out by role (setmaxnreg).
// Up to 64 query rows leave lanes idle: a tile then holds two or four copies of them, each copy's threads take a half or a quarter of a tile's
// keys, and their weights for the other keys are zero.  The copies are joined like the streams.  So the softmax of few rows is spread over all
// threads, and the products, which a memory-bound call has time for, stay whole tiles.
// New rows' values that are not finite must not reach rows that do not see them (0 x inf): the threads of a tile that holds new rows clear them
// in shared memory, with the rows behind the last position, and add them at the end to the rows that see them.
// Every mbarrier wait is bounded (status word codes 71..76).
//
// Measured on a B200 (8 key/value heads of 128): 60000 bfloat16 positions 45.2 us with 18 query rows (5.4 TB/s), 51.5 with 128, 68 with 256; INT8 49,
// 63 and 107 us.  bfloat16 up to 128 rows waits for memory.  A pair of units of 256 rows takes 3400 cycles, and its bytes arrive in 2800: a stream's
// scores, softmax (2050 cycles, half of them the exponentials' rate) and product follow on one another, and two streams are what tensor memory
// holds, although half of a stream's columns of scores are free while its softmax runs.  A second softmax thread per row, or a third of the exponentials from a cubic, changed less than 2 %.  INT8 adds
// the scales and the conversions: 6000 cycles for a pair, with 48 % of the issue slots used and loads' latency the most frequent stall; half of its exponents wait in tensor memory (all loaded and scaled twice: 67 us, not 63).  Weights in halves against whole tiles: 256 rows 72 -> 70 us, INT8 65 -> 62 us at
// 128 rows; for bfloat16 at 128 rows, which has its two streams on different tiles, 16.9 -> 17.6 us at 8000 positions, so there they stay whole.
#include <cooperative_groups.h>
#include "mixers/mix_tc.cuh"
#include "scmx_cache_attn.cuh"

namespace cg = cooperative_groups;

namespace scmx {

constexpr int CT_TILE = 128 * 128;        // bytes of a [128 rows x 64 bfloat16] block
constexpr uint32_t IDESC_BF16 = 1u << 7 | 1u << 10;      // types of A and B in an instruction descriptor: bfloat16, 0 for float16
constexpr int CT_SCALES = 8;              // tiles whose scales are held
constexpr int CT_AHEAD = 6;               // tiles that are prefetched into L2

template <int D, bool I8, int MQ>
struct CtSmem {
    static constexpr int KB = D / 64;
    static constexpr int KS = D == 64 ? 4 : I8 || MQ == 2 ? 2 : 3;            // stages of keys
    static constexpr int VS = D == 64 ? 4 : MQ == 2 ? 2 : 3;                  // stages of values
    static constexpr int Q_OFF = 0;
    static constexpr int K_OFF = Q_OFF + MQ * KB * CT_TILE;
    static constexpr int V_OFF = K_OFF + KS * KB * CT_TILE;
    static constexpr int SC_OFF = V_OFF + VS * KB * CT_TILE;                  // [CT_SCALES][keys' scales, values' log2, values' reciprocals][128] float
    static constexpr int BAR_OFF = SC_OFF + (I8 ? CT_SCALES * 1536 : 0);
    // kfull, kempty [KS], vfull, vempty [VS], scales [CT_SCALES], S [2], P [2][halves], O [2], queries
    static constexpr int NBAR = 2 * KS + 2 * VS + (I8 ? CT_SCALES : 0) + 9;
    // threads; INT8: registers of a thread by role, together no more than the block is launched with
    static constexpr int THREADS = I8 ? 640 : 320, LAUNCH_REGS = 96, SOFT_REGS = 136, CONV_REGS = 72, MISC_REGS = 56;
    static_assert(256 * SOFT_REGS + 256 * CONV_REGS + 128 * MISC_REGS <= 640 * LAUNCH_REGS, "registers of a block");
    static constexpr int MISC_OFF = BAR_OFF + 8 * NBAR;
    static constexpr int TOTAL = MISC_OFF + 32 + 1024;
    static constexpr int PITCH = D + 4;                                       // outputs of 256 lanes from Q_OFF on, then maxima and sums, in place of operands
    static constexpr int ML_OFF = Q_OFF + 256 * PITCH * 4;
    static_assert(ML_OFF + 2048 <= SC_OFF, "joined outputs fit the operands' memory");
    static_assert(TOTAL <= 232448, "shared memory of an SM");
};

// 16 registers of a thread -> 16 consecutive 32-bit columns of its lane.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
          "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
// 16 columns of a lane into registers, waited for.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Bits of 32 keys, the first `b` positions after the first new row (negative: before it), that a row with these bits sees.
__device__ __forceinline__ uint32_t ct_seen(uint64_t bits, int b) {
    if (b <= -32) return 0xFFFFFFFFu;
    if (b < 0) return (uint32_t)(bits << -b) | ((1u << -b) - 1u);
    return b < 64 ? (uint32_t)(bits >> b) : 0u;
}

template <bool UP, int N>
__device__ __forceinline__ void set_regs() {
    if (UP) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// MQ: query tiles; COPIES of the rows in a tile (1 with two tiles).
template <int D, bool I8, int MQ, int COPIES>
__global__ void __launch_bounds__(CtSmem<D, I8, MQ>::THREADS, 1)
    cache_attn_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CaArgs a, int32_t* status,
                         uint64_t wait_ns) {
    using L = CtSmem<D, I8, MQ>;
    constexpr int KB = L::KB, KS = L::KS, VS = L::VS;
    constexpr int RP = 128 / COPIES, ROWS = MQ * RP, NCH = 4 / COPIES;      // rows of a tile, of the CTA; 32-key pieces of a thread
    constexpr int HALVES = COPIES == 1 && (I8 || MQ == 2) ? 2 : 1;      // weights handed over in halves: the first's product runs while the second is computed
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sbase = smem_u32(smem), bars = sbase + L::BAR_OFF;
    const uint32_t b_kf = bars, b_ke = b_kf + 8 * KS, b_vf = b_ke + 8 * KS, b_ve = b_vf + 8 * VS, b_sc = b_ve + 8 * VS, b_s = b_sc + (I8 ? 8 * CT_SCALES : 0),
                   b_p = b_s + 16, b_o = b_p + 32, b_q = b_o + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::MISC_OFF + 4);
    uint32_t* bad = reinterpret_cast<uint32_t*>(smem + L::MISC_OFF + 8);      // new rows with values that are not finite
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, tid = threadIdx.x;

    if (tid == 0) {
        if (!I8) {
            prefetch_map(&tmK);
            prefetch_map(&tmV);
        }
        for (int i = 0; i < L::NBAR; ++i) {
            const uint32_t b = bars + 8 * i;
            const bool converted = I8 && ((b >= b_kf && b < b_ke) || (b >= b_vf && b < b_ve) || (b >= b_sc && b < b_s));      // one arrival per converting warp
            mbar_init(b, b == b_q || converted ? 8 : b >= b_p && b < b_o ? 4 : 1);                                          // weights: one per softmax warp
        }
        *abort_flag = 0;
        bad[0] = bad[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        proxy_fence();
    }
    constexpr int MISC = I8 ? 16 : 8;        // first of the last warps: MMAs; the one after it: TMA
    if (warp == MISC) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    pdl_launch_dependents();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    pdl_wait();

    const int kvh = blockIdx.x, split = blockIdx.y, G = a.G, R = G * a.n, row0 = blockIdx.z * ROWS;
    const int64_t pos = ca_pos(a.pos_dev, a.pos, a.cap, a.n), T = pos + a.n, chunk = ca_chunk(T, a.nsplit, a.unit);
    const int64_t t0 = split * chunk, t1 = t0 + chunk < T ? t0 + chunk : T;
    const int nkeys = t1 > t0 ? (int)(t1 - t0) : 0, ntiles = (nkeys + 127) / 128, units = ntiles * MQ;
    const int dnew = (int)(t0 - pos > -(int64_t)nkeys - 64 ? t0 - pos : -(int64_t)nkeys - 64);      // the range's first key, counted from the first new row

    int fail = 0;

    if (warp > MISC) {
        if (I8) set_regs<false, L::MISC_REGS>();
        if (!I8 && warp == MISC + 1 && lane == 0) {
            for (int j = 0; j < ntiles; ++j) {
                const int key = (int)t0 + 128 * j, ks = j % KS, vs = j % VS;
                if (int w = mbar_wait(b_ke + 8 * ks, ((j / KS) & 1) ^ 1, abort_flag, wait_ns)) { fail = w == 1 ? 71 : -1; break; }
                mbar_expect_tx(b_kf + 8 * ks, KB * CT_TILE);
                for (int c = 0; c < KB; ++c) tma_load_3d(sbase + L::K_OFF + (ks * KB + c) * CT_TILE, &tmK, c * 128, key, kvh, b_kf + 8 * ks);
                if (int w = mbar_wait(b_ve + 8 * vs, ((j / VS) & 1) ^ 1, abort_flag, wait_ns)) { fail = w == 1 ? 71 : -1; break; }
                mbar_expect_tx(b_vf + 8 * vs, KB * CT_TILE);
                for (int c = 0; c < KB; ++c) tma_load_3d(sbase + L::V_OFF + (vs * KB + c) * CT_TILE, &tmV, c * 128, key, kvh, b_vf + 8 * vs);
                // the queries first: behind all stages' loads of all multiprocessors they arrive 3 us later
                if (j == 0)
                    if (int w = mbar_wait(b_q, 0, abort_flag, wait_ns)) { fail = w == 1 ? 71 : -1; break; }
            }
        }
    } else if (warp == MISC) {
        if (I8) set_regs<false, L::MISC_REGS>();
        const uint32_t on = elect_lane();
        const uint32_t idesc_s = umma_idesc_bf16(128, 128), idesc_o = (umma_idesc_bf16(128, D) | IDESC_B_MN) & ~(I8 ? IDESC_BF16 : 0u);      // (INT8: float16)
        int kt = -1, vt = -1;            // last tiles that were waited for
        auto wait = [&](uint32_t bar, uint32_t parity, int code) -> bool {
            if (!wait_warp(bar, parity, abort_flag, wait_ns, code, fail)) return false;
            tc_fence_after();
            return true;
        };
        auto scores = [&](int u) -> bool {
            const int m = u & 1, j = MQ == 2 ? u >> 1 : u, ks = j % KS;
            if (j != kt && !wait(b_kf + 8 * ks, (j / KS) & 1, 72)) return false;
            kt = j;
            const uint32_t q = sbase + L::Q_OFF + (MQ == 2 ? m * KB : 0) * CT_TILE;
#pragma unroll
            for (int c = 0; c < KB; ++c) {
                const uint64_t da = umma_desc(q + c * CT_TILE), db = umma_desc(sbase + L::K_OFF + (ks * KB + c) * CT_TILE);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_bf16(on, tmem + 128 * m, da + 2 * k, db + 2 * k, idesc_s, c + k > 0);
            }
            umma_commit(on, b_s + 8 * m);
            if (MQ == 1 || m == 1) umma_commit(on, b_ke + 8 * ks);
            return true;
        };
        bool ok = units == 0 || (wait(b_q, 0, 72) && scores(0));
        if (ok && units > 1) ok = scores(1);
        for (int u = 0; u < units && ok; ++u) {
            const int m = u & 1, j = MQ == 2 ? u >> 1 : u, vs = j % VS;
            const uint64_t dv = umma_desc_mn(sbase + L::V_OFF + vs * KB * CT_TILE, CT_TILE);
#pragma unroll
            for (int h = 0; h < HALVES && ok; ++h) {
                if (!(ok = wait(b_p + 16 * m + 8 * h, (u >> 1) & 1, 73))) break;
                if (h == 0 && j != vt && !(ok = wait(b_vf + 8 * vs, (j / VS) & 1, 72))) break;
                vt = j;
#pragma unroll
                for (int k = 8 / HALVES * h; k < 8 / HALVES * (h + 1); ++k)
                    umma_bf16_ts(on, tmem + 256 + 128 * m, tmem + 128 * m + 8 * k, dv + 128 * k, idesc_o, k > 0 ? 1u : (uint32_t)(u > 1));
            }
            if (!ok) break;
            if (MQ == 1 || m == 1) umma_commit(on, b_ve + 8 * vs);
            if (u + 2 >= units) umma_commit(on, b_o + 8 * m);
            else ok = scores(u + 2);
        }
        if (!on) fail = fail > 0 ? -1 : fail;      // one lane reports
    } else if (warp < 8) {
        if (I8) set_regs<true, L::SOFT_REGS>();
        // queries: K-major tiles with the 128-byte swizzle, four values of a row to a lane; a negative scale is taken by the queries
        if (ntiles) {
            constexpr int LPR = D / 4, RPW = 32 / LPR, PER = ROWS / (8 * RPW);      // lanes of a row, rows of a warp's load, loads of a warp
            const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
            const int ql = lane % LPR;
            constexpr int BATCH = PER < 8 ? PER : 8;       // loads of a warp that are in flight together
#pragma unroll 1
            for (int i0 = 0; i0 < PER; i0 += BATCH) {
                uint2 x[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {          // nothing here waits for a load: rows past the last read row 0
                    const int r = row0 + ((i0 + i) * 8 + warp) * RPW + lane / LPR, rr = r < R ? r : 0, qt = ca_tok(a, rr);
                    x[i] = __ldg(reinterpret_cast<const uint2*>(a.q + (int64_t)(kvh * G + rr - qt * G) * a.q_hs + (int64_t)qt * a.q_rs + 4 * ql));
                }
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int r = ((i0 + i) * 8 + warp) * RPW + lane / LPR;
                    uint2 w = I8 ? make_uint2(__byte_perm(x[i].x, x[i].y, 0x5410), __byte_perm(x[i].x, x[i].y, 0x7632)) : x[i];
                    w.x = row0 + r < R ? w.x ^ flip : 0u;
                    w.y = row0 + r < R ? w.y ^ flip : 0u;
#pragma unroll
                    for (int c = 0; c < COPIES; ++c) {
                        const int to = r + c * RP;
                        *reinterpret_cast<uint2*>(smem + L::Q_OFF + (to / 128 * KB + ql / 16) * CT_TILE + to % 128 * 128 + ((((ql & 15) >> 1) ^ (to & 7)) << 4) + (ql & 1) * 8) = w;
                    }
                }
            }
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(b_q);
        }
        const int m = warp >> 2 & 1, zero = warp >> 3, q = warp & 3, l = 32 * q + lane, copy = l / RP, row = row0 + (MQ == 2 ? 128 * m : 0) + l % RP, tok = ca_tok(a, row);
        const uint32_t lane_base = (uint32_t)(32 * q) << 16, ts = tmem + 128 * m + lane_base, to = tmem + 256 + 128 * m + lane_base;
        // The thread's first key of a tile.  `zero` keeps it from being a constant with one copy, where the compiler then orders the loads of the two
        // streams worse (60000 positions, 256 rows, bfloat16 70.3 us and not 68.2; INT8 125 and not 114 when scores were scaled twice)
        const int c0 = copy * (128 / COPIES) + zero * 64;
        uint64_t bits = 0;
        if (row < R) {
            bits = a.mask ? (uint64_t)a.mask[tok] : (2ull << tok) - 1ull;
            if (a.n < 64) bits &= (1ull << a.n) - 1ull;
        }
        // scores times this are exponents of 2 (INT8: the key scales have it).  Not zero, which would make hidden scores, -inf, NaN
        const float sl = I8 ? 1.0f : fmaxf(fabsf(a.scale), 1.17549435e-38f);
        float mx = -1e30f, sum = 0.0f;
        for (int u = m; u < units; u += 2) {
            const int j = MQ == 2 ? u >> 1 : u, d0 = dnew + 128 * j;
            const bool tail = d0 + 128 > 0;                     // some keys are new rows, or past the end
            const float* scales = reinterpret_cast<const float*>(smem + L::SC_OFF) + (j & (CT_SCALES - 1)) * 384 + c0;
            int w = mbar_wait(b_s + 8 * m, (u >> 1) & 1, abort_flag, wait_ns);
            if (I8 && !w) w = mbar_wait(b_sc + 8 * (j & (CT_SCALES - 1)), (j / CT_SCALES) & 1, abort_flag, wait_ns);
            if (__any_sync(0xffffffffu, w)) { fail = w == 1 ? 74 : -1; break; }
            tc_fence_after();
            // scores of piece c: 32 keys in pairs, as exponents of 2 once multiplied by sl; unseen ones -inf
            auto finish = [&](uint32_t (&v)[32], int c) {
                if constexpr (I8) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(scales + 32 * c + i), g = *reinterpret_cast<const float4*>(scales + 128 + 32 * c + i);
                        const float2 x = unpack2(fma2(pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), pack2(f.x, f.y), pack2(g.x, g.y)));
                        const float2 y = unpack2(fma2(pack2(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), pack2(f.z, f.w), pack2(g.z, g.w)));
                        v[i] = __float_as_uint(x.x);
                        v[i + 1] = __float_as_uint(x.y);
                        v[i + 2] = __float_as_uint(y.x);
                        v[i + 3] = __float_as_uint(y.y);
                    }
                }
                if (tail) {
                    const uint32_t seen = ct_seen(bits, d0 + c0 + 32 * c);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!(seen >> i & 1)) v[i] = 0xFF800000u;
                }
            };
            // the scores stay in registers between the two passes; where those are too few, only the first half does, and the second waits as exponents in its place
            constexpr int HELD = I8 && NCH > 2 ? 2 : NCH;
            uint32_t r[HELD][32];
            float tm = -INFINITY;
#pragma unroll
            for (int half = NCH / HELD - 1; half >= 0; --half) {
#pragma unroll
                for (int e = 0; e < HELD; ++e) tmem_ld32(ts + c0 + 32 * (HELD * half + e), r[e]);
#pragma unroll
                for (int e = 0; e < HELD; ++e) tmem_ld_fence(r[e]);
#pragma unroll
                for (int e = 0; e < HELD; ++e) {
                    uint32_t(&v)[32] = r[e];
                    finish(v, HELD * half + e);
                    float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        m0 = fmaxf(m0, fmaxf(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
                        m1 = fmaxf(m1, fmaxf(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])));
                    }
                    tm = fmaxf(tm, fmaxf(m0, m1));
                    if (half > 0) tmem_st32(ts + c0 + 32 * (HELD * half + e), v);
                }
            }
            const bool first = u == m, grow = first || (tm - mx) * sl > CA_GROWTH;
            if (__any_sync(0xffffffffu, grow)) {
                const float mn = grow ? fmaxf(mx, tm) : mx, f = ex2_approx((mx - mn) * sl);
                mx = mn;
                if (!first) sum *= f;
                if (!first) {      // S complete implies the stream's last product complete: MMAs of one thread finish in order
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {      // few registers: the scores wait in theirs
                        uint32_t v[16];
                        tmem_ld16(to + 16 * c, v);
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                        tmem_st16(to + 16 * c, v);
                    }
                }
            }
            const bool clear = !I8 && tail;                     // values are cleared first
            auto hand_over = [&](int h) {
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b_p + 16 * m + 8 * h);
            };
            const float off = I8 ? CA_SHIFT - mx : -mx * sl;
            const uint64_t sl2 = pack2(sl, sl), off2 = pack2(off, off);
            uint64_t s2[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                uint32_t(&v)[32] = r[c % HELD];
                if (c > 0 && c % HELD == 0) {
#pragma unroll
                    for (int e = 0; e < HELD; ++e) tmem_ld_fence(r[e]);
                }
                const uint32_t seen = tail ? ct_seen(bits, d0 + c0 + 32 * c) : 0xFFFFFFFFu;
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const uint64_t z = pack2(__uint_as_float(v[i + e]), __uint_as_float(v[i + e + 1]));
                        const float2 y = unpack2(I8 ? add2(z, off2) : fma2(z, sl2, off2));
                        x[e] = ex2_approx(y.x);
                        x[e + 1] = ex2_approx(y.y);
                        if (!I8) s2[e / 2] = add2(s2[e / 2], pack2(x[e], x[e + 1]));
                    }
                    if constexpr (I8) {
                        float4 f = *reinterpret_cast<const float4*>(scales + 256 + 32 * c + i);
                        if (tail) {                                           // an unseen position's scale may be anything
                            if (!(seen >> i & 1)) f.x = 0.0f;
                            if (!(seen >> i & 2)) f.y = 0.0f;
                            if (!(seen >> i & 4)) f.z = 0.0f;
                            if (!(seen >> i & 8)) f.w = 0.0f;
                        }
                        s2[0] = fma2(pack2(x[0], x[1]), pack2(f.x, f.y), s2[0]);
                        s2[1] = fma2(pack2(x[2], x[3]), pack2(f.z, f.w), s2[1]);
                    }
                    pk[i / 2] = I8 ? pack_f16x2(x[0], x[1]) : pack_bf16x2(x[0], x[1]);
                    pk[i / 2 + 1] = I8 ? pack_f16x2(x[2], x[3]) : pack_bf16x2(x[2], x[3]);
                }
                if (c + HELD < NCH) {
                    if (c == 0) tmem_st_wait();
                    tmem_ld32(ts + c0 + 32 * (c + HELD), v);
                }
                tmem_st16(ts + c0 / 2 + 16 * c, pk);
                if (HALVES == 2 && c == NCH / 2 - 1 && !clear) hand_over(0);
            }
            const float2 sum0 = unpack2(s2[0]), sum1 = unpack2(s2[1]);
            if (COPIES > 1) {            // weights of the other copies' keys
                uint32_t z[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] = 0;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c / NCH != copy) tmem_st16(ts + 16 * c, z);
            }
            sum += (sum0.x + sum0.y) + (sum1.x + sum1.y);
            if (clear && (MQ == 1 || m == 0)) {      // a thread per position
                w = mbar_wait(b_vf + 8 * (j % VS), (j / VS) & 1, abort_flag, wait_ns);
                if (__any_sync(0xffffffffu, w)) { fail = w == 1 ? 74 : -1; break; }
                const int d = d0 + l;
                if (d >= 0) {
                    bool odd = false;
#pragma unroll
                    for (int c = 0; c < KB; ++c) {
                        uint4* p = reinterpret_cast<uint4*>(smem + L::V_OFF + (j % VS * KB + c) * CT_TILE + l * 128);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint4 x = p[i];
                            uint32_t v[4] = {x.x, x.y, x.z, x.w};
                            bool any = d >= a.n;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const bool lo = (v[e] & 0x7F80u) == 0x7F80u, hi = (v[e] & 0x7F800000u) == 0x7F800000u;
                                if (lo || d >= a.n) v[e] &= 0xFFFF0000u;
                                if (hi || d >= a.n) v[e] &= 0x0000FFFFu;
                                any |= lo || hi;
                            }
                            odd |= any;
                            if (any) p[i] = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                    }
                    if (odd && d < a.n) atomicOr(bad + (d >> 5), 1u << (d & 31));
                }
                proxy_fence();
            }
            if (HALVES == 2 && clear) hand_over(0);
            hand_over(HALVES - 1);
        }
        // both streams' products are complete before the operands' memory is used again
        if (fail == 0) {
            int w = units > 0 ? mbar_wait(b_o, 0, abort_flag, wait_ns) : 0;
            if (!w && units > 1) w = mbar_wait(b_o + 8, 0, abort_flag, wait_ns);
            if (__any_sync(0xffffffffu, w)) fail = w == 1 ? 75 : -1;
            tc_fence_after();
        }
        // every lane's output to shared memory, where the states of a row's copies and streams are joined
        constexpr int STATES = MQ == 2 ? 1 : 2 * COPIES, PIECES = D / 4;
        const bool mine = fail == 0 && units > m;
        float* out = reinterpret_cast<float*>(smem + L::Q_OFF);
        float2* ml = reinterpret_cast<float2*>(smem + L::ML_OFF);
        const int slot = 128 * m + l;
        ml[slot] = mine && sum != 0.0f ? make_float2(mx * sl, I8 ? sum * CA_DOWN : sum) : make_float2(-INFINITY, 0.0f);
        const float by = I8 && mine ? ca_ex2(*reinterpret_cast<const float*>(smem + L::MISC_OFF + 16)) : 1.0f;
        for (int c = 0; c < D / 32 && mine; ++c) {
            uint32_t v[32];
            tmem_ld32(to + 32 * c, v);
            tmem_ld_fence(v);
            float4* p = reinterpret_cast<float4*>(out + slot * L::PITCH + 32 * c);
#pragma unroll
            for (int i = 0; i < 8; ++i)      // INT8: values 1 and 2 of four change places again
                p[i] = I8 ? make_float4(__uint_as_float(v[4 * i]) * CA_DOWN * by, __uint_as_float(v[4 * i + 2]) * CA_DOWN * by, __uint_as_float(v[4 * i + 1]) * CA_DOWN * by, __uint_as_float(v[4 * i + 3]) * CA_DOWN * by)
                          : make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const int rows = units == 0 ? 0 : R - row0 < ROWS ? R - row0 : ROWS;
        const int64_t first = (((int64_t)kvh * gridDim.z + blockIdx.z) * a.nsplit + split) * ROWS;
        auto state = [](int r, int s) { return MQ == 2 ? r : (s & 1) * 128 + (s >> 1) * RP + r; };
        // a thread to a row: what each of its states is multiplied by (in place of its maximum), the row's maximum and sum
        float top = -INFINITY, total = 0.0f;
        if (tid < rows) {
#pragma unroll
            for (int s = 0; s < STATES; ++s) top = fmaxf(top, ml[state(tid, s)].x);
#pragma unroll
            for (int s = 0; s < STATES; ++s) {
                float2& z = ml[state(tid, s)];
                const float f = z.x == -INFINITY ? 0.0f : ex2_approx(z.x - top);
                total += z.y * f;
                z.x = f;
            }
            if (a.part != nullptr) a.part_ml[first + tid] = make_float2(top, total);
            ml[tid].y = total;               // (state 0 is row tid itself)
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const uint64_t odd = (uint64_t)bad[1] << 32 | bad[0];
#pragma unroll 1
        for (int i0 = tid; i0 < rows * PIECES; i0 += 4 * 256) {
            float4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * 256 < rows * PIECES ? i0 + k * 256 : i0, r = i / PIECES, c = i % PIECES;
                v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int s = 0; s < STATES; ++s) {
                    const int at = state(r, s);
                    const float f = ml[at].x;
                    float4 x = *reinterpret_cast<const float4*>(out + at * L::PITCH + 4 * c);
                    if (f == 0.0f) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);      // nothing seen: the output may not have been written
                    v[k].x = fmaf(x.x, f, v[k].x); v[k].y = fmaf(x.y, f, v[k].y); v[k].z = fmaf(x.z, f, v[k].z); v[k].w = fmaf(x.w, f, v[k].w);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * 256, r = i / PIECES, c = i % PIECES;
                if (i >= rows * PIECES) break;
                const int rr = row0 + r, tk = ca_tok(a, rr);
                float4& y = v[k];
                if (odd) {                       // new rows' values that are not finite, to a row that sees them
                    for (uint64_t b = (a.mask ? (uint64_t)a.mask[tk] : (2ull << tk) - 1ull) & odd; b; b &= b - 1) {
                        const uint16_t* p = static_cast<const uint16_t*>(a.v) + ((int64_t)kvh * a.cap + pos + (__ffsll((long long)b) - 1)) * D + 4 * c;
                        if ((p[0] & 0x7F80u) == 0x7F80u) y.x += bf16_to_f32(p[0]);
                        if ((p[1] & 0x7F80u) == 0x7F80u) y.y += bf16_to_f32(p[1]);
                        if ((p[2] & 0x7F80u) == 0x7F80u) y.z += bf16_to_f32(p[2]);
                        if ((p[3] & 0x7F80u) == 0x7F80u) y.w += bf16_to_f32(p[3]);
                    }
                }
                if (a.cluster) {                 // in place of the row's first state, which no other thread reads here
                    *reinterpret_cast<float4*>(out + r * L::PITCH + 4 * c) = y;
                } else if (a.part != nullptr) {
                    *reinterpret_cast<float4*>(a.part + (first + r) * D + 4 * c) = y;
                } else {
                    const float total = ml[r].y, inv = total == 0.0f ? 0.0f : 1.0f / total;
                    *reinterpret_cast<uint2*>(a.out + (int64_t)tk * a.hq * D + (kvh * G + rr - tk * G) * D + 4 * c) =
                        make_uint2(pack_bf16x2(y.x * inv, y.y * inv), pack_bf16x2(y.z * inv, y.w * inv));
                }
            }
        }
        if (a.cluster) {
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (tid < ROWS) ml[tid] = tid < rows ? make_float2(top, total) : make_float2(-INFINITY, 0.0f);
        }
    } else if (I8) {
        set_regs<false, L::CONV_REGS>();
        // codes to operands: 16 codes of a vector to a thread, CPR threads to a vector, PASSES vectors to a thread
        constexpr int CPR = D / 16, PASSES = 128 * CPR / 256;
        const int t = tid - 256, cc = t % CPR, r0 = t / CPR;
        const I8Pairs i8;
        const I8Halves i8h;
        const int8_t *kc = static_cast<const int8_t*>(a.k) + ((int64_t)kvh * a.cap + t0) * D, *vc = static_cast<const int8_t*>(a.v) + ((int64_t)kvh * a.cap + t0) * D;
        auto load = [&](const int8_t* p, int j, uint4 (&x)[PASSES]) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int r = 128 * j + r0 + i * (256 / CPR);
                x[i] = r < nkeys ? __ldg(reinterpret_cast<const uint4*>(p + (int64_t)r * D + 16 * cc)) : make_uint4(0, 0, 0, 0);
            }
        };
        auto ahead = [&](int j) {                 // a tile's keys (thread 0) and values (thread 32) into L2
            const int n = nkeys - 128 * j < 128 ? nkeys - 128 * j : 128;
            if (n > 0 && (t & ~32) == 0) {
                const int8_t* p = (t ? vc : kc) + (int64_t)128 * j * D;
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(n * D) : "memory");
            }
        };
        auto convert = [&](bool halves, uint8_t* dst, const uint4 (&x)[PASSES]) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int r = r0 + i * (256 / CPR);
                const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                uint32_t o[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[2 * e] = halves ? i8h.even(u[e]) : i8.even(u[e]);
                    o[2 * e + 1] = halves ? i8h.odd(u[e]) : i8.odd(u[e]);
                }
                uint8_t* p = dst + cc / 4 * CT_TILE + r * 128;
                const int e = 2 * (cc & 3), swap = cc >> 2;      // the upper half's stores in the other order: all of a vector's fall on different banks
                const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
                *reinterpret_cast<uint4*>(p + (((e + swap) ^ (r & 7)) << 4)) = swap ? hi : lo;
                *reinterpret_cast<uint4*>(p + (((e + 1 - swap) ^ (r & 7)) << 4)) = swap ? lo : hi;
            }
        };
        // a position's scales: keys' by threads 0-127, values' by the others, loaded a tile ahead
        const float* scales = (t < 128 ? a.ks : a.vs) + (int64_t)kvh * a.cap + t0 + (t & 127);
        const float factor = fabsf(a.scale);
        float ref = 0.0f;                         // log2 of the scale that values are relative to
        if (t >= 128) {
            float first[4];
            bool from[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) first[i] = 32 * i + lane < nkeys ? __ldg(a.vs + (int64_t)kvh * a.cap + t0 + 32 * i + lane) : 0.0f;
            const uint64_t any = dnew + 128 > 0 ? ca_seen_by_any(a, lane) : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = dnew + 32 * i + lane;         // counted from the first new row
                from[i] = d < 0 || (d < a.n && (any >> (d & 63) & 1));
            }
            ref = ca_reference(first, from);
            if (t == 128) *reinterpret_cast<float*>(smem + L::MISC_OFF + 16) = ref;
        }
        auto scale = [&](int j) { return 128 * j + (t & 127) < nkeys ? __ldg(scales + 128 * j) : 0.0f; };
        uint4 xk[PASSES], xv[PASSES];
        for (int j = 1; j < CT_AHEAD; ++j) ahead(j);
        load(kc, 0, xk);
        load(vc, 0, xv);
        float sc = scale(0);
        auto ready = [&](uint32_t empty, int j, int stages) -> bool {
            const int w = mbar_wait(empty + 8 * (j % stages), ((j / stages) & 1) ^ 1, abort_flag, wait_ns);
            if (__any_sync(0xffffffffu, w)) { fail = w == 1 ? 76 : -1; return false; }
            return true;
        };
        auto done = [&](uint32_t full) {
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(full);
        };
        for (int j = 0; j < ntiles; ++j) {
            ahead(j + CT_AHEAD);
            if (!ready(b_ke, j, KS)) break;
            convert(false, smem + L::K_OFF + j % KS * KB * CT_TILE, xk);
            float* own = reinterpret_cast<float*>(smem + L::SC_OFF) + (j & (CT_SCALES - 1)) * 384 + t;
            if (t < 128) own[0] = sc * factor;
            else ca_scale(sc, ref, own[0], own[128]);
            if (j + 1 < ntiles) load(kc, j + 1, xk);
            sc = scale(j + 1);
            done(b_kf + 8 * (j % KS));
            if (lane == 0) mbar_arrive(b_sc + 8 * (j & (CT_SCALES - 1)));
            if (!ready(b_ve, j, VS)) break;
            convert(true, smem + L::V_OFF + j % VS * KB * CT_TILE, xv);
            if (j + 1 < ntiles) load(vc, j + 1, xv);
            done(b_vf + 8 * (j % VS));
        }
    }

    if (fail > 0) {
        if (atomicCAS(status, 0, fail) == 0) {
            status[1] = blockIdx.x;
            status[2] = threadIdx.x;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (a.cluster) {                     // the ranges' states, read where they lie: the rows in turn to the CTAs, a warp to a row
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        constexpr int E = D / 32;
        const int ctas = (int)cl.num_blocks(), rows = R - row0 < ROWS ? R - row0 : ROWS;
        float* out = reinterpret_cast<float*>(smem + L::Q_OFF);
        float2* ml = reinterpret_cast<float2*>(smem + L::ML_OFF);
        for (int r = (int)cl.block_rank() + ctas * warp; r < rows; r += ctas * (L::THREADS / 32)) {
            const float2 z = lane < ctas ? cl.map_shared_rank(ml, lane)[r] : make_float2(-INFINITY, 0.0f);
            float m = z.x, l = z.y, v[E];
            ca_join<E, 8>(ctas, m, l, v, [&](int s, float (&z)[E]) { ca_load<E>(cl.map_shared_rank(out, s) + r * L::PITCH + lane * E, z); });
            ca_output<D>(a, kvh, row0 + r, lane, v, l);
        }
        cl.sync();                       // nobody leaves while its state may still be read
    }
    if (*abort_flag) {
        const uint64_t begin = globaltimer_ns();
        while (globaltimer_ns() - begin < 200000ull) __nanosleep(1000);   // 0.2 ms for outstanding TMA writes
        __syncthreads();
    }
    if (warp == MISC) tmem_dealloc(tmem, 512);
}

template <int D, bool I8, int MQ, int COPIES>
static int launch_ct(const CUtensorMap& k, const CUtensorMap& v, const CaArgs& a, const CaPlan& p, int32_t* status, cudaStream_t st) {
    using L = CtSmem<D, I8, MQ>;
    static bool configured[64] = {};
    const int dev = current_device();
    SCMX_REQUIRE(dev >= 0, SCMX_ECUDA, "no current CUDA device (ordinal 0..63)");
    if (!configured[dev]) {
        SCMX_CUDA_OK(cudaFuncSetAttribute(cache_attn_tc_kernel<D, I8, MQ, COPIES>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL));
        configured[dev] = true;
    }
    SCMX_PDL_OK("cache_attn_tc_kernel", ca_launch(cache_attn_tc_kernel<D, I8, MQ, COPIES>, a.hk, p, L::THREADS, L::TOTAL, st, k, v, a, status, (uint64_t)g_wait_limit_ns));
    return SCMX_OK;
}
template <int D, bool I8>
static int dispatch_ct(const CUtensorMap& k, const CUtensorMap& v, const CaArgs& a, const CaPlan& p, int32_t* status, cudaStream_t st) {
    if (p.nt == 2) return launch_ct<D, I8, 2, 1>(k, v, a, p, status, st);
    return p.copies == 4 ? launch_ct<D, I8, 1, 4>(k, v, a, p, status, st) : p.copies == 2 ? launch_ct<D, I8, 1, 2>(k, v, a, p, status, st)
                                                                                         : launch_ct<D, I8, 1, 1>(k, v, a, p, status, st);
}

int cache_attn_tc(const CaArgs& a, const CaPlan& p, int d, int int8, int32_t* status, cudaStream_t st) {
    SCMX_REQUIRE(a.cap < (1ll << 31) - 128, SCMX_ELIMIT, "cache_attn: a cache of %lld positions", (long long)a.cap);
    CUtensorMap k, v;
    if (int8) {
        memset(&k, 0, sizeof(k));            // codes are loaded by threads
        memset(&v, 0, sizeof(v));
    } else {
        int rc = make_map_planes(&k, a.k, a.hk, a.cap, 2 * d, 2 * d, 2ll * d * a.cap, 128);
        if (!rc) rc = make_map_planes(&v, a.v, a.hk, a.cap, 2 * d, 2 * d, 2ll * d * a.cap, 128);
        if (rc) return rc;
    }
    if (d == 128) return int8 ? dispatch_ct<128, true>(k, v, a, p, status, st) : dispatch_ct<128, false>(k, v, a, p, status, st);
    return int8 ? dispatch_ct<64, true>(k, v, a, p, status, st) : dispatch_ct<64, false>(k, v, a, p, status, st);
}

}  // namespace scmx

// Attention of n <= 64 new rows (one token, or drafted tokens under a tree mask) to a bfloat16 or INT8 cache that already holds their own
// keys and values:  o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - max),  j over the positions before `pos` and those
// of the new rows that row i's mask names.
//
// The G query heads of a key/value head and the n rows are G n query rows that read the same keys: tiles of 16 of them meet the cache in
// one pass (mma.sync m16n8k16, bfloat16, float32 sums).  The positions are cut into ranges, one CTA each; in a CTA every warp takes blocks of
// 16 positions of its own, brought into its own ring in shared memory by asynchronous copies, and keeps a running maximum, sum and output
// in registers.  The warps' states are joined in shared memory, the ranges' by a second launch.
// INT8 codes become bfloat16 exactly (8 significant bits); a position's key scale multiplies its scores, its value scale its weights.
#include "scmx_common.cuh"
#include "scmx_ptx.cuh"

namespace scmx {

constexpr int CA_WARPS = 8, CA_THREADS = 32 * CA_WARPS, CA_KEYS = 16, CA_ROWS = 16;
constexpr int CA_MAX_ROWS = 64;
constexpr float CA_LOG2E = 1.4426950408889634f;

struct CaArgs {
    const uint16_t* q;               // bf16, heads q_hs and rows q_rs elements apart
    const void *k, *v;               // [hk, cap, d] bf16 or int8
    const float *ks, *vs;            // [hk, cap] (INT8)
    const int64_t* mask;             // [n] or null: row i sees rows 0 .. i
    const int32_t* pos_dev;
    float* part;                     // [hk, tiles, nsplit, 16, D + 2] or null (nsplit 1)
    uint16_t* out;                   // bf16 [n, hq d]
    int64_t q_hs, q_rs, pos, cap;
    int n, hq, hk, nsplit;
    float scale;                     // times log2(e)
};

// Positions of a call and of one range: ranges are multiples of 128, so a short cache uses the first few only.
__device__ __forceinline__ int64_t ca_pos(const int32_t* pos_dev, int64_t pos, int64_t cap, int n) {
    int64_t p = pos_dev ? (int64_t)pos_dev[0] : pos;
    return p < 0 ? 0 : p > cap - n ? cap - n : p;
}
__device__ __forceinline__ int64_t ca_chunk(int64_t T, int nsplit) {
    const int64_t c = (T + nsplit - 1) / nsplit;
    return (c + CA_KEYS * CA_WARPS - 1) / (CA_KEYS * CA_WARPS) * (CA_KEYS * CA_WARPS);
}

template <int D, bool I8>
struct CaSmem {
    static constexpr int ROW = I8 ? D : 2 * D;                        // bytes of a vector
    static constexpr int BLOCK = CA_KEYS * ROW;                       // 16 keys or values
    static constexpr int STAGE = 2 * BLOCK + (I8 ? 128 : 0);          // keys, values, their scales
    static constexpr int STAGES = 3;
    static constexpr int RING = STAGE * STAGES;
    static constexpr int STATE = CA_ROWS * (D + 2) * 4;               // a warp's state when the warps are joined
    static constexpr int WARP = RING > STATE ? RING : STATE;
    static constexpr int TOTAL = WARP * CA_WARPS;
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
// Byte offset of 16-byte piece c of vector r in a block: pieces are permuted within groups of eight so that the eight vectors of a matrix
// load, and the vectors of one INT8 value load, lie in different banks.
template <int ROW>
__device__ __forceinline__ int ca_at(int r, int c) {
    if constexpr (ROW == 64) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    return r * ROW + ((c ^ (r & 7)) << 4);
}
// Two INT8 codes in the low bytes of the halves of w (the other bytes are ignored) -> two bfloat16, exactly: a code below 128 is the low
// bits of the significand of 128 + code; its sign bit falls on the exponent's low bit, so 128 or 256 is taken off.
__device__ __forceinline__ uint32_t i8x2_bf16(uint32_t w) {
    const uint32_t x = (w & 0x007F007Fu) | 0x43004300u, y = (w & 0x00800080u) | 0x43004300u;
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
    return d;
}

template <int D, bool I8>
__global__ void __launch_bounds__(CA_THREADS) cache_attn_kernel(const CaArgs a) {
    using L = CaSmem<D, I8>;
    constexpr int ROW = L::ROW, PIECES = ROW / 16, KSTEPS = D / 16, NT = D / 8;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int kvh = blockIdx.x, split = blockIdx.y, G = a.hq / a.hk, R = G * a.n;
    const int64_t pos = ca_pos(a.pos_dev, a.pos, a.cap, a.n), T = pos + a.n, chunk = ca_chunk(T, a.nsplit);
    const int64_t t0 = split * chunk, t1 = t0 + chunk < T ? t0 + chunk : T;
    if (t0 >= T) return;
    const unsigned char* kb = static_cast<const unsigned char*>(a.k) + (int64_t)kvh * a.cap * ROW;
    const unsigned char* vb = static_cast<const unsigned char*>(a.v) + (int64_t)kvh * a.cap * ROW;
    unsigned char* ring = smem_raw + warp * L::WARP;
    const uint32_t ring_s = smem_u32(ring);

    // query rows g and g + 8 of this tile, as the A operand
    int row[2], tok[2];
    uint64_t sees[2];
    uint32_t qf[KSTEPS][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        row[h] = blockIdx.z * CA_ROWS + g + 8 * h;
        const bool on = row[h] < R;
        tok[h] = on ? row[h] / G : 0;
        sees[h] = !on ? 0ull : a.mask ? (uint64_t)a.mask[tok[h]] : (2ull << tok[h]) - 1ull;
        const uint16_t* qp = a.q + (int64_t)(kvh * G + (on ? row[h] - tok[h] * G : 0)) * a.q_hs + (int64_t)tok[h] * a.q_rs;
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
            if constexpr (I8) {       // the four values that one word of codes holds
                const uint2 w = *reinterpret_cast<const uint2*>(qp + 16 * s + 4 * t4);
                qf[s][h] = on ? w.x : 0u;
                qf[s][2 + h] = on ? w.y : 0u;
            } else {
                const uint32_t lo = *reinterpret_cast<const uint32_t*>(qp + 16 * s + 2 * t4), hi = *reinterpret_cast<const uint32_t*>(qp + 16 * s + 8 + 2 * t4);
                qf[s][h] = on ? lo : 0u;
                qf[s][2 + h] = on ? hi : 0u;
            }
        }
    }

    const int64_t nblocks = (t1 - t0 + CA_KEYS - 1) / CA_KEYS;
    auto load = [&](int64_t b, int stage) {
        if (b < nblocks) {
            const int64_t key0 = t0 + b * CA_KEYS;
            const uint32_t dst = ring_s + stage * L::STAGE;
#pragma unroll
            for (int p = 0; p < CA_KEYS * PIECES / 32; ++p) {
                const int i = p * 32 + lane, r = i / PIECES, c = i % PIECES;
                const bool on = key0 + r < t1;
                const int64_t off = (on ? key0 + r : t0) * ROW + 16 * c;
                cp_async16(dst + ca_at<ROW>(r, c), kb + off, on);
                cp_async16(dst + L::BLOCK + ca_at<ROW>(r, c), vb + off, on);
            }
            if constexpr (I8) {
                const bool on = key0 + (lane & 15) < t1;
                const float* s = (lane < 16 ? a.ks : a.vs) + (int64_t)kvh * a.cap + (on ? key0 + (lane & 15) : t0);
                cp_async4(dst + 2 * L::BLOCK + 4 * lane, s, on);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int s = 0; s < L::STAGES - 1; ++s) load(warp + s * CA_WARPS, s);

    float o[NT][4], mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;

    int stage = 0;
    for (int64_t b = warp; b < nblocks; b += CA_WARPS) {
        cp_wait<L::STAGES - 2>();
        __syncwarp();
        load(b + (L::STAGES - 1) * CA_WARPS, stage == 0 ? L::STAGES - 1 : stage - 1);
        const unsigned char* blk = ring + stage * L::STAGE;
        const uint32_t kst = ring_s + stage * L::STAGE, vst = kst + L::BLOCK;
        const float* scales = reinterpret_cast<const float*>(blk + 2 * L::BLOCK);
        const int64_t key0 = t0 + b * CA_KEYS;
        // scores of 16 rows and 2 x 8 keys
        float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
        const int lr = lane & 7, lm = lane >> 3;        // row of a matrix load, and which of its four matrices
        if constexpr (I8) {
#pragma unroll
            for (int c = 0; c < KSTEPS; c += 2) {
                uint32_t w[4];                          // keys 0-7 pieces c, c + 1, keys 8-15 pieces c, c + 1
                ldsm4(kst + ca_at<ROW>(lr + 8 * (lm >> 1), c + (lm & 1)), w);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        mma_bf16(s[j], qf[c + e], i8x2_bf16(__byte_perm(w[2 * j + e], 0, 0x4140)), i8x2_bf16(__byte_perm(w[2 * j + e], 0, 0x4342)));
            }
        } else {
#pragma unroll
            for (int c = 0; c < KSTEPS; ++c) {
                uint32_t w[4];
                ldsm4(kst + ca_at<ROW>(lr + 8 * (lm >> 1), 2 * c + (lm & 1)), w);
                mma_bf16(s[0], qf[c], w[0], w[1]);
                mma_bf16(s[1], qf[c], w[2], w[3]);
            }
        }
        // the thread's keys: 2 t4, 2 t4 + 1 of each group of eight
        float vsc[2][2];
        bool vis[2][2][2];                              // row half, key group, key
        const bool tail = key0 + CA_KEYS > pos;         // some keys are new rows, or past the end
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int kk = 8 * j + 2 * t4 + e;
                float f = a.scale;
                if constexpr (I8) {
                    f *= scales[kk];
                    vsc[j][e] = scales[16 + kk];
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    bool v = true;
                    if (tail) {
                        const int64_t d = key0 + kk - pos;
                        v = row[h] < R && (d < 0 || (d < a.n && ((sees[h] >> d) & 1)));
                    }
                    vis[h][j][e] = v;
                    s[j][2 * h + e] = v ? s[j][2 * h + e] * f : -INFINITY;
                }
            }
        uint32_t pa[4];
        float p[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float m = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const float mn = fmaxf(mx[h], m);
            const float base = mn == -INFINITY ? 0.0f : mn;
            if (__any_sync(0xffffffffu, mn > mx[h])) {
                const float f = exp2f(mx[h] - base);
                sum[h] *= f;
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    o[i][2 * h] *= f;
                    o[i][2 * h + 1] *= f;
                }
                mx[h] = mn;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float x = exp2f(s[j][2 * h + e] - base);
                    sum[h] += x;
                    p[j][2 * h + e] = I8 ? (vis[h][j][e] ? x * vsc[j][e] : 0.0f) : x;
                }
            pa[h] = pack_bf16x2(p[0][2 * h], p[0][2 * h + 1]);
            pa[2 + h] = pack_bf16x2(p[1][2 * h], p[1][2 * h + 1]);
        }
        // a value that is not finite must not reach rows that do not see it: such blocks, which only new rows can make, go key by key
        bool odd = false;
        if constexpr (!I8) {
            if (tail) {
#pragma unroll
                for (int i = 0; i < CA_KEYS * PIECES / 32; ++i) {
                    const uint4 w = *reinterpret_cast<const uint4*>(blk + L::BLOCK + 16 * (32 * i + lane));
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) odd = odd || (u[j] & 0x7F800000u) == 0x7F800000u || (u[j] & 0x7F80u) == 0x7F80u;
                }
                odd = __any_sync(0xffffffffu, odd);
            }
        }
        if (odd) {
#pragma unroll
            for (int kk = 0; kk < CA_KEYS; ++kk) {
                const int j = kk >> 3, e = kk & 1, src = (lane & ~3) | ((kk & 7) >> 1);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float w = __shfl_sync(0xffffffffu, p[j][2 * h + e], src);
                    const bool on = __shfl_sync(0xffffffffu, (int)vis[h][j][e], src) != 0;
                    if (on) {
#pragma unroll
                        for (int i = 0; i < NT; ++i) {
                            const uint32_t x = *reinterpret_cast<const uint32_t*>(blk + L::BLOCK + ca_at<ROW>(kk, i) + 4 * t4);
                            o[i][2 * h] = fmaf(w, bf16_lo(x), o[i][2 * h]);
                            o[i][2 * h + 1] = fmaf(w, bf16_hi(x), o[i][2 * h + 1]);
                        }
                    }
                }
            }
        } else if constexpr (I8) {
#pragma unroll
            for (int cg = 0; cg < D / 32; ++cg) {       // 32 values: a thread's word holds values 4 g .. of its four keys
                uint32_t w[4];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    w[r] = *reinterpret_cast<const uint32_t*>(blk + L::BLOCK + ca_at<ROW>(2 * t4 + (r & 1) + 8 * (r >> 1), 2 * cg + (g >> 2)) + 4 * (g & 3));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    mma_bf16(o[4 * cg + j], pa, i8x2_bf16(__byte_perm(w[0], w[1], 0x4400 + j * 0x1111)), i8x2_bf16(__byte_perm(w[2], w[3], 0x4400 + j * 0x1111)));
            }
        } else {
#pragma unroll
            for (int i = 0; i < NT; i += 2) {
                uint32_t w[4];
                ldsm4_t(vst + ca_at<ROW>(lr + 8 * (lm & 1), i + (lm >> 1)), w);
                mma_bf16(o[i], pa, w[0], w[1]);
                mma_bf16(o[i + 1], pa, w[2], w[3]);
            }
        }
        stage = stage + 1 == L::STAGES ? 0 : stage + 1;
    }
    cp_wait<0>();
    __syncwarp();

    // the warps' states, joined: output in the operand's order of values
    float* st = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
        float* r = st + (g + 8 * h) * (D + 2);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = I8 ? 32 * (i >> 2) + 8 * t4 + 4 * e + (i & 3) : 8 * i + 2 * t4 + e;
                r[d] = o[i][2 * h + e];
            }
        if (t4 == 0) {
            r[D] = mx[h];
            r[D + 1] = sum[h];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < CA_ROWS * D; i += CA_THREADS) {
        const int r = i / D, d = i - r * D, rr = blockIdx.z * CA_ROWS + r;
        if (rr >= R) break;
        float m = -INFINITY, l = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < CA_WARPS; ++w) m = fmaxf(m, reinterpret_cast<const float*>(smem_raw + w * L::WARP)[r * (D + 2) + D]);
#pragma unroll
        for (int w = 0; w < CA_WARPS; ++w) {
            const float* x = reinterpret_cast<const float*>(smem_raw + w * L::WARP) + r * (D + 2);
            const float f = x[D] == -INFINITY ? 0.0f : exp2f(x[D] - m);
            l += x[D + 1] * f;
            v += f == 0.0f ? 0.0f : x[d] * f;
        }
        if (a.part != nullptr) {
            float* y = a.part + ((((int64_t)kvh * gridDim.z + blockIdx.z) * a.nsplit + split) * CA_ROWS + r) * (D + 2);
            y[d] = v;
            if (d == 0) {
                y[D] = m;
                y[D + 1] = l;
            }
        } else {
            const int tk = rr / G, hd = kvh * G + rr - tk * G;
            a.out[(int64_t)tk * a.hq * D + hd * D + d] = f32_to_bf16(l == 0.0f ? 0.0f : v / l);
        }
    }
}

// Joins the ranges: one warp per query row.
template <int D>
__global__ void __launch_bounds__(128) cache_attn_join_kernel(const CaArgs a, int tiles) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, G = a.hq / a.hk, R = G * a.n;
    const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (i >= a.hk * R) return;
    const int kvh = i / R, r = i - kvh * R, tile = r / CA_ROWS;
    const int64_t T = ca_pos(a.pos_dev, a.pos, a.cap, a.n) + a.n, chunk = ca_chunk(T, a.nsplit);
    const int active = (int)((T + chunk - 1) / chunk);
    const float* x = a.part + (((int64_t)kvh * tiles + tile) * a.nsplit * CA_ROWS + r % CA_ROWS) * (D + 2);
    constexpr int STRIDE = CA_ROWS * (D + 2), E = D / 32;
    float m = -INFINITY;
    for (int s = 0; s < active; ++s) m = fmaxf(m, x[(int64_t)s * STRIDE + D]);
    float l = 0.0f, v[E] = {};
    for (int s = 0; s < active; ++s) {
        const float* y = x + (int64_t)s * STRIDE;
        const float f = y[D] == -INFINITY ? 0.0f : exp2f(y[D] - m);
        if (f == 0.0f) continue;
        l += y[D + 1] * f;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += y[lane * E + e] * f;
    }
    const int tk = r / G, hd = kvh * G + r - tk * G;
    uint16_t* o = a.out + (int64_t)tk * a.hq * D + hd * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(o + e) = l == 0.0f ? 0u : pack_bf16x2(v[e] / l, v[e + 1] / l);
}

// Ranges of positions: as many CTAs as multiprocessors, none shorter than one block for every warp.
static int ca_splits(int64_t positions, int hk, int tiles) {
    const int64_t most = (positions + CA_KEYS * CA_WARPS - 1) / (CA_KEYS * CA_WARPS), want = sm_count() / ((int64_t)hk * tiles);
    const int64_t s = want < most ? want : most;
    return s < 1 ? 1 : (int)s;
}

template <int D, bool I8>
static int launch_ca(const CaArgs& a, int tiles, cudaStream_t st) {
    using L = CaSmem<D, I8>;
    static bool configured[64] = {};
    const int dev = current_device();
    SCMX_REQUIRE(dev >= 0, SCMX_ECUDA, "no current CUDA device (ordinal 0..63)");
    if (!configured[dev]) {
        SCMX_CUDA_OK(cudaFuncSetAttribute(cache_attn_kernel<D, I8>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL));
        configured[dev] = true;
    }
    SCMX_PDL_OK("cache_attn_kernel", launch_pdl(cache_attn_kernel<D, I8>, dim3((unsigned)a.hk, (unsigned)a.nsplit, (unsigned)tiles), dim3(CA_THREADS),
                                                (size_t)L::TOTAL, st, a));
    if (a.part != nullptr)
        SCMX_PDL_OK("cache_attn_join_kernel", launch_pdl(cache_attn_join_kernel<D>, dim3((unsigned)((a.hq * a.n + 3) / 4)), dim3(128), 0, st, a, tiles));
    return SCMX_OK;
}

}  // namespace scmx

using namespace scmx;

extern "C" int64_t scmx_cache_attn_scratch(int64_t positions, int n, int hq, int hk, int d) {
    if (positions < 1 || n < 1 || n > CA_MAX_ROWS || hk < 1 || hq < hk || hq % hk || (d != 64 && d != 128)) return 0;
    const int tiles = (hq / hk * n + CA_ROWS - 1) / CA_ROWS, ns = ca_splits(positions, hk, tiles);
    return ns == 1 ? 0 : (int64_t)hk * tiles * ns * CA_ROWS * (d + 2) * 4;
}

extern "C" int scmx_cache_attn(const uint16_t* q, int64_t q_head_stride, int64_t q_row_stride, const void* k, const void* v, const float* k_scales,
                               const float* v_scales, int int8, const int64_t* mask, int n, int64_t pos, const int32_t* pos_dev, int64_t capacity, int hq, int hk,
                               int d, float scale, uint16_t* out, void* scratch, int64_t scratch_bytes, void* stream) {
    SCMX_REQUIRE(q && k && v && out && (!int8 || (k_scales && v_scales)), SCMX_EINVAL, "cache_attn: null buffer");
    SCMX_REQUIRE(n >= 1 && n <= CA_MAX_ROWS, SCMX_ELIMIT, "cache_attn: %d rows (1 .. %d)", n, CA_MAX_ROWS);
    SCMX_REQUIRE(d == 64 || d == 128, SCMX_EINVAL, "cache_attn: head size %d (64 or 128)", d);
    SCMX_REQUIRE(hk > 0 && hq > 0 && hq % hk == 0, SCMX_EINVAL, "cache_attn: hq=%d hk=%d", hq, hk);
    SCMX_REQUIRE(capacity >= n && (pos_dev != nullptr || (pos >= 0 && pos + n <= capacity)), SCMX_EINVAL, "cache_attn: rows %lld .. %lld of a cache of %lld",
                 (long long)pos, (long long)(pos + n), (long long)capacity);
    SCMX_REQUIRE(q_head_stride % 4 == 0 && q_row_stride % 4 == 0 && ((uintptr_t)q & 7) == 0 && ((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0 &&
                     ((uintptr_t)out & 3) == 0, SCMX_EINVAL, "cache_attn: query rows must be 8-byte and caches 16-byte aligned");
    CaArgs a;
    const int tiles = (hq / hk * n + CA_ROWS - 1) / CA_ROWS;
    a.nsplit = ca_splits(pos_dev ? capacity : pos + n, hk, tiles);
    const int64_t need = scmx_cache_attn_scratch(pos_dev ? capacity : pos + n, n, hq, hk, d);
    SCMX_REQUIRE(scratch_bytes >= need && (need == 0 || (scratch && ((uintptr_t)scratch & 15) == 0)), SCMX_EINVAL, "cache_attn: %lld bytes of scratch, %lld needed",
                 (long long)scratch_bytes, (long long)need);
    a.q = q; a.q_hs = q_head_stride; a.q_rs = q_row_stride; a.k = k; a.v = v; a.ks = k_scales; a.vs = v_scales; a.mask = mask; a.pos_dev = pos_dev; a.pos = pos;
    a.part = need ? static_cast<float*>(scratch) : nullptr; a.out = out; a.cap = capacity; a.n = n; a.hq = hq; a.hk = hk; a.scale = scale * CA_LOG2E;
    const cudaStream_t st = (cudaStream_t)stream;
    if (d == 128) return int8 ? launch_ca<128, true>(a, tiles, st) : launch_ca<128, false>(a, tiles, st);
    return int8 ? launch_ca<64, true>(a, tiles, st) : launch_ca<64, false>(a, tiles, st);
}

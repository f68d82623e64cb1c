// What the two kernels of attention to a cache share: arguments, the cut into ranges of positions.
#pragma once
#include <string.h>
#include "scmx_common.cuh"
#include "scmx_ptx.cuh"

namespace scmx {

constexpr int CA_KEYS = 16;             // positions of a block
constexpr int CA_MAX_ROWS = 64;
constexpr float CA_LOG2E = 1.4426950408889634f;
constexpr float CA_GROWTH = 8.0f;      // log2 of how far a weight may exceed one before the maximum is raised
// INT8: a weight and its value's scale s are one power of 2, w = 2^(score + log2(s / r) - max), whose maximum the rows keep, r the geometric mean of the scales of the
// first positions; what is summed is w / (s / r), and outputs are multiplied by r at the end.  So w never exceeds 2^8 whatever the scales, and it goes to
// the product as float16 (the codes are exact in it), 2^6 larger: from 2^14 down to 2^-24, 2^-12 of a weight off where bfloat16 is 2^-8.  Sums and outputs leave
// 2^20 smaller, so that large values times r stay finite.
constexpr float CA_SHIFT = 6.0f, CA_LEAST = -90.0f, CA_ZERO = -64.0f, CA_DOWN = 9.5367431640625e-07f;

struct CaArgs {
    const uint16_t* q;               // bf16, heads q_hs and rows q_rs elements apart
    const void *k, *v;               // [hk, cap, d] bf16 or int8
    const float *ks, *vs;            // [hk, cap] (INT8)
    const int64_t* mask;             // [n] or null: row i sees rows 0 .. i
    const int32_t* pos_dev;
    float* part;                     // sums of weighted values [hk, tiles, nsplit, rows of a CTA, D], or null (nsplit 1)
    float2* part_ml;                 // their maxima (exponents of 2) and sums of weights, [hk, tiles, nsplit, rows]
    uint16_t* out;                   // bf16 [n, hq d]
    int64_t q_hs, q_rs, pos, cap;
    int n, hq, hk, G, nsplit, unit, cluster;      // cluster: the ranges' CTAs are one, and join their states themselves
    float scale;                     // times log2(e)
    float inv_g;                     // 1 / G, G = hq / hk
};

// First new row's position, and positions of one range: whole units, so a short cache uses the first few ranges only.
__device__ __forceinline__ int64_t ca_pos(const int32_t* pos_dev, int64_t pos, int64_t cap, int n) {
    int64_t p = pos_dev ? (int64_t)pos_dev[0] : pos;
    return p < 0 ? 0 : p > cap - n ? cap - n : p;
}
__device__ __forceinline__ int64_t ca_chunk(int64_t T, int nsplit, int unit) {
    if (T < (1ll << 31) - 4096) {        // 64-bit divisions are hundreds of cycles before a kernel's first load
        const uint32_t c = ((uint32_t)T + nsplit - 1) / (uint32_t)nsplit;
        return (c + unit - 1) & ~(uint32_t)(unit - 1);      // units are powers of two
    }
    const int64_t c = (T + nsplit - 1) / nsplit;
    return (c + unit - 1) / unit * unit;
}
__device__ __forceinline__ int ca_ranges(int64_t T, int64_t chunk) { return T < (1ll << 31) ? (int)(((uint32_t)T + (uint32_t)chunk - 1) / (uint32_t)chunk) : (int)((T + chunk - 1) / chunk); }
// The new row of a query row: row / G.  Exact: row + 1/2 is at least 1 / (2 G) of its size away from whole multiples of G, rows are below 2^18 (64 rows of 4096 heads).
__device__ __forceinline__ int ca_tok(const CaArgs& a, int row) { return (int)(((float)row + 0.5f) * a.inv_g); }

__device__ __forceinline__ float ca_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// New rows that some query row sees.
__device__ __forceinline__ uint64_t ca_seen_by_any(const CaArgs& a, int lane) {
    uint64_t bits = a.mask == nullptr ? ~0ull : (lane < a.n ? (uint64_t)a.mask[lane] : 0ull) | (lane + 32 < a.n ? (uint64_t)a.mask[lane + 32] : 0ull);
    bits = (uint64_t)__reduce_or_sync(0xffffffffu, (uint32_t)(bits >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)bits);
    return a.n < 64 ? bits & ((1ull << a.n) - 1ull) : bits;
}
// log2 r from PER scales of every lane, those that `from` names: positions before the new rows, which every row sees, and the new rows that some row sees.  What nobody sees may
// hold any scale, and must not set the range that the others have.  The mean of the logarithms: one scale far from all others moves it least (a vector that is not finite, or of
// zeros, does not count).
template <int PER>
__device__ __forceinline__ float ca_reference(const float (&s)[PER], const bool (&from)[PER]) {
    int sum = 0, count = 0;      // of sixteenths: r need not be the mean exactly, and whole numbers are added over a warp in one instruction
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        float lg;
        asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lg) : "f"(s[i]));
        if (from[i] && lg > -INFINITY && lg < INFINITY) {
            sum += __float2int_rn(lg * 16.0f);
            ++count;
        }
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    count = PER == 1 ? __popc(__ballot_sync(0xffffffffu, count)) : __reduce_add_sync(0xffffffffu, count);
    return count ? rintf(__fdividef((float)sum, 16.0f * (float)count)) : 0.0f;
}
// log2(s / r) and r / s of a value's scale, 2^-20 off at most; below 2^-90 r the sums' range ends (above, at 2^106 r), and a weight counts in its row's sum down to 2^-132 of the largest
// weight times the two scales' ratio.  A vector of zeros has scale 0: any other is right for it, and a small one keeps its weight out of the maximum (with r, a score 28 powers of two above
// all others left these so few bits that the output was half wrong), one not too small keeps it in the sum.
__device__ __forceinline__ void ca_scale(float s, float ref, float& lg, float& inv) {
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lg) : "f"(s));
    lg = s == 0.0f ? CA_ZERO : s != s ? s : fmaxf(lg - ref, CA_LEAST);
    inv = ca_ex2(-lg);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
// E = D / 32 consecutive values of a row to a lane.
template <int E> struct CaVec;
template <> struct CaVec<2> { typedef float2 type; };
template <> struct CaVec<4> { typedef float4 type; };
template <int E>
__device__ __forceinline__ void ca_load(const float* p, float (&v)[E]) {
    const typename CaVec<E>::type x = *reinterpret_cast<const typename CaVec<E>::type*>(p);
    memcpy(v, &x, sizeof(x));
}
template <int E>
__device__ __forceinline__ void ca_store(float* p, const float (&v)[E]) {
    typename CaVec<E>::type x;
    memcpy(&x, v, sizeof(x));
    *reinterpret_cast<typename CaVec<E>::type*>(p) = x;
}
// A query row of the output, v / total (zeros where nothing was seen).
template <int D>
__device__ __forceinline__ void ca_output(const CaArgs& a, int kvh, int row, int lane, const float (&v)[D / 32], float total) {
    const int tok = ca_tok(a, row);
    uint32_t* o = reinterpret_cast<uint32_t*>(a.out + (int64_t)tok * a.hq * D + (kvh * a.G + row - tok * a.G) * D) + lane * (D / 64);
#pragma unroll
    for (int e = 0; e < D / 32; e += 2) o[e / 2] = total == 0.0f ? 0u : pack_bf16x2(v[e] / total, v[e + 1] / total);
}
// Joins partial softmax states of one row by a whole warp: state s < count (count <= 32) has its maximum and sum in lane s's (m, l); values(s, v) gives the lane's E
// values of it.  (m, l) become the joined maximum and sum, in every lane.
template <int E, int BATCH, typename Values>
__device__ __forceinline__ void ca_join(int count, float& m, float& l, float (&v)[E], Values values) {
    const float top = warp_max(m), f = m == -INFINITY ? 0.0f : ca_ex2(m - top);
    float total = l * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.0f;
    for (int s = 0; s < count; s += BATCH) {
        float z[BATCH][E];
#pragma unroll
        for (int j = 0; j < BATCH; ++j)
            if (s + j < count) values(s + j, z[j]);
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const float w = __shfl_sync(0xffffffffu, f, (s + j) & 31);
            if (s + j < count && w != 0.0f)
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = fmaf(z[j][e], w, v[e]);
        }
    }
    m = top;
    l = total;
}

// How a call is cut.  tc: by the tcgen05 kernel, `nt` query tiles of 128 in a CTA and `copies` of the rows in a tile; otherwise nt groups of eight query rows.
// `rows` query rows in a CTA, `tiles` of them, `nsplit` ranges of positions that are multiples of `unit`.
struct CaPlan { int tc, nt, copies, rows, tiles, nsplit, unit, cluster; };

// Launches one CTA for every key/value head, range and tile; the ranges of a head as a cluster where they join their states themselves.
template <typename... KArgs, typename... Args>
inline cudaError_t ca_launch(void (*kernel)(KArgs...), int hk, const CaPlan& p, int threads, int smem, cudaStream_t st, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)hk, (unsigned)p.nsplit, (unsigned)p.tiles);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (g_use_pdl) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (p.cluster) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = attr[cfg.numAttrs].val.clusterDim.z = 1;
        attr[cfg.numAttrs++].val.clusterDim.y = p.nsplit;
    }
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

int cache_attn_tc(const CaArgs& a, const CaPlan& p, int d, int int8, int32_t* status, cudaStream_t st);

}  // namespace scmx

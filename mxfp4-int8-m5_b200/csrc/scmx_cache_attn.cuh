// What the two kernels of attention to a cache share: arguments, the cut into ranges of positions.
#pragma once
#include "scmx_common.cuh"
#include "scmx_ptx.cuh"

namespace scmx {

constexpr int CA_KEYS = 16;             // positions of a block
constexpr int CA_MAX_ROWS = 64;
constexpr float CA_LOG2E = 1.4426950408889634f;
constexpr float CA_GROWTH = 8.0f;      // log2 of how far a weight may exceed one before the maximum is raised

struct CaArgs {
    const uint16_t* q;               // bf16, heads q_hs and rows q_rs elements apart
    const void *k, *v;               // [hk, cap, d] bf16 or int8
    const float *ks, *vs;            // [hk, cap] (INT8)
    const int64_t* mask;             // [n] or null: row i sees rows 0 .. i
    const int32_t* pos_dev;
    float* part;                     // [hk, tiles, nsplit, rows of a tile, D + 2] or null (nsplit 1)
    uint16_t* out;                   // bf16 [n, hq d]
    int64_t q_hs, q_rs, pos, cap;
    int n, hq, hk, nsplit, unit;
    float scale;                     // times log2(e)
};

// First new row's position, and positions of one range: whole units, so a short cache uses the first few ranges only.
__device__ __forceinline__ int64_t ca_pos(const int32_t* pos_dev, int64_t pos, int64_t cap, int n) {
    int64_t p = pos_dev ? (int64_t)pos_dev[0] : pos;
    return p < 0 ? 0 : p > cap - n ? cap - n : p;
}
__device__ __forceinline__ int64_t ca_chunk(int64_t T, int nsplit, int unit) {
    const int64_t c = (T + nsplit - 1) / nsplit;
    return (c + unit - 1) / unit * unit;
}

// How a call is cut.  tc: by the tcgen05 kernel, `nt` query tiles of 128 in a CTA and `copies` of the rows in a tile; otherwise nt groups of eight query rows.
// `rows` query rows in a CTA, `tiles` of them, `nsplit` ranges of positions that are multiples of `unit`.
struct CaPlan { int tc, nt, copies, rows, tiles, nsplit, unit; };

int cache_attn_tc(const CaArgs& a, const CaPlan& p, int d, int int8, int32_t* status, cudaStream_t st);

}  // namespace scmx

// Verification of drafted tokens: which rows of a tree of drafts the target accepts, from its logits and given random numbers, and the
// token after them.  Row 0 is the last chosen token, row c continues row parents[c] < c.  At a node with target probabilities p, its children
// are tested in ascending order: child c with token x is accepted if u[c] q(x) < p(x), q the draft's probabilities (1 where there are none);
// a rejected child leaves p <- max(p - q, 0) / Z (or p without x).  Where no child is left, the token is the first whose
// cumulative probability exceeds u[0].  Accepted paths and tokens follow the target's distribution whatever the draft proposed.
// Temperature 0: a child is accepted if it is the largest logit of its parent (the lowest index of equal ones), which is also the token.
//
// The maxima and sums of all rows are a pass over the logits by the whole device (memory-bound); one cluster then walks the tree, which needs one
// logit per drafted row.  Where drafts have probabilities, it reads a node's row again when a rejected child has a sibling to be tested on what
// is left (float32 weights: this mass decides tests whose border a relative error of 1e-6 moves by as much; all such masses ahead, a cluster
// to a node, took 19 us of the whole device where a pass of the walk takes 3).  The last token's weights, sums and cumulative
// probabilities are float64: between 100000 neighbours float32 sums would pick another token once in a hundred draws.
//
// Measured on a B200: greedy, 5 rows of 32000 bfloat16 logits, 4.9 us (two launches); 21 rows of 50304 float32 logits by temperature 11.5 us, of which the two launches and the cluster's start and
// barriers are 8.6 (one row of 8 logits), the last node's pass 1; 64 rows of 151936 with the draft's probabilities 23.8 us from memory, 17.1 from L2, against 9 us for all bytes once: the
// walk is a chain of dependent passes over single rows, 3 us each, 8 us in a row of 151936, and all of the tree's rows are not its path's.  63 children of one node, all rejected: 30 us without
// probabilities, 450 with them at 50304.
#include <cooperative_groups.h>
#include "scmx_common.cuh"

namespace cg = cooperative_groups;

namespace scmx {

constexpr int VF_ROWS = 64, VF_THREADS = 256, VF_VECS = 4;                  // first launch: 256 x 4 vectors of 8 logits per CTA
constexpr int VF_SLICE = VF_THREADS * VF_VECS * 8;
constexpr int VW_CTAS = 16, VW_THREADS = 512, VW_WARPS = VW_THREADS / 32;   // walk: a cluster of 16 CTAs, or 8 where the device has no room for one
constexpr int VW_CACHE = 200 * 1024;                                        // bytes of weights and probabilities that a CTA of it keeps

struct VfPart {          // of a slice of a row: maximum and sum of 2^((x - max) c), or the key of its largest logit
    union { double sum; unsigned long long key; };
    float max, pad;
};

struct VfArgs {
    const void* logits;              // [n, V], rows ld elements apart
    const float* probs;              // [n, V], rows ldp apart, or null
    const int64_t* tokens;
    const int32_t* parents;
    const float* u;
    VfPart* part;                    // [n, slices]
    int32_t *rows, *count;
    int64_t* token;
    int64_t ld, ldp;
    int n, V, slices;
    float c;                         // log2(e) / temperature
    double cd;                       // 1 / temperature
};

__device__ __forceinline__ float vf_get(const uint16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float vf_get(const float* p) { return *p; }

// Eight values from index 8 v of a row of V; those past its end are -inf (`fill`).
__device__ __forceinline__ void vf_load(const uint16_t* row, int v, int V, float fill, float (&x)[8]) {
    const uint16_t* p = row + 8 * (int64_t)v;
    if (8 * v + 8 <= V && ((uintptr_t)p & 15) == 0) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = bf16_lo(u[j]);
            x[2 * j + 1] = bf16_hi(u[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 8 * v + j < V ? vf_get(p + j) : fill;
    }
}
__device__ __forceinline__ void vf_load(const float* row, int v, int V, float fill, float (&x)[8]) {
    const float* p = row + 8 * (int64_t)v;
    if (8 * v + 8 <= V && ((uintptr_t)p & 15) == 0) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 8 * v + j < V ? p[j] : fill;
    }
}

// The weight of a logit against its row's maximum in float32, the same in all launches.
__device__ __forceinline__ float vf_weight(float x, float m, float c) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(__fmul_rn(__fsub_rn(x, m), c)));
    return y;
}

// Keys order like (value, lower index first); NaN counts as the largest.
__device__ __forceinline__ unsigned long long vf_key(float f, uint32_t i) {
    const uint32_t u = __float_as_uint(f == 0.0f ? 0.0f : f);
    const uint32_t r = f != f ? 0xFFFFFFFFu : u & 0x80000000u ? ~u : u | 0x80000000u;
    return (unsigned long long)r << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ unsigned long long vf_warp_max(unsigned long long k) {
    const uint32_t hi = (uint32_t)(k >> 32), m = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t lo = __reduce_max_sync(0xffffffffu, hi == m ? (uint32_t)k : 0u);
    return (unsigned long long)m << 32 | lo;
}

// grid (slices, n)
template <typename T, bool GREEDY>
__global__ void __launch_bounds__(VF_THREADS) verify_rows_kernel(const __grid_constant__ VfArgs a) {
    __shared__ float red[33];
    __shared__ double dred[33];
    __shared__ unsigned long long kred[VF_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const T* row = static_cast<const T*>(a.logits) + (int64_t)blockIdx.y * a.ld;
    const int v0 = blockIdx.x * (VF_SLICE / 8) + threadIdx.x;
    float x[VF_VECS][8];
#pragma unroll
    for (int i = 0; i < VF_VECS; ++i) vf_load(row, v0 + i * VF_THREADS, a.V, -INFINITY, x[i]);
    VfPart* out = a.part + (int64_t)blockIdx.y * a.slices + blockIdx.x;
    if constexpr (GREEDY) {
        unsigned long long k = 0;
#pragma unroll
        for (int i = 0; i < VF_VECS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = 8 * (v0 + i * VF_THREADS) + j;
                if (e < a.V) k = max(k, vf_key(x[i][j], (uint32_t)e));
            }
        k = vf_warp_max(k);
        if ((threadIdx.x & 31) == 0) kred[threadIdx.x >> 5] = k;
        __syncthreads();
        if (threadIdx.x < 32) {
            k = vf_warp_max(threadIdx.x < VF_THREADS / 32 ? kred[threadIdx.x] : 0ull);
            if (threadIdx.x == 0) out->key = k;
        }
    } else {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < VF_VECS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, x[i][j]);
        m = block_max(m, red);
        double s = 0.0;
        if (m != -INFINITY) {
#pragma unroll
            for (int i = 0; i < VF_VECS; ++i) {
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = vf_weight(x[i][j], m, a.c);
                s += (double)(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
            }
        }
        s = block_sum(s, dred);
        if (threadIdx.x == 0) {
            out->sum = s;
            out->max = m;
        }
    }
}

// A warp to a row for the slices' keys, then one thread walks.
__global__ void __launch_bounds__(1024) verify_greedy_kernel(const __grid_constant__ VfArgs a) {
    __shared__ int best[VF_ROWS], parent[VF_ROWS], path[VF_ROWS], length;
    __shared__ int64_t token[VF_ROWS];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid < a.n) {
        parent[tid] = a.parents[tid];
        token[tid] = a.tokens[tid];
        path[tid] = -1;
    }
    for (int r = tid >> 5; r < a.n; r += 32) {
        unsigned long long k = 0;
        for (int s = lane; s < a.slices; s += 32) k = max(k, a.part[(int64_t)r * a.slices + s].key);
        k = vf_warp_max(k);
        if (lane == 0) best[r] = (int)(0xFFFFFFFFu - (uint32_t)k);
    }
    __syncthreads();
    if (tid == 0) {
        int node = 0, count = 1;
        path[0] = 0;
        for (int c = 1; c < a.n; ++c)
            if (parent[c] == node && token[c] == best[node]) path[count++] = node = c;
        length = count;
        *a.token = best[node];
    }
    __syncthreads();
    if (tid < a.n) a.rows[tid] = path[tid];
    if (tid == 0) *a.count = length;
}

// e^x for x <= 0 in float64, relative error below 1e-13: 2^(k / 64) by a table, e^r of the rest, |r| < ln 2 / 128, by its Taylor series.  The library's function is
// correct to the last bit and took half of the walk's time.
__device__ __forceinline__ double vf_exp(double x, const double* table) {
    const double big = 6755399441055744.0;                   // 1.5 2^52: adding it rounds to a whole number, whose low bits are those of the sum
    const double t = fma(x, 92.332482616893656877, big);     // 64 / ln 2
    const int k = __double2loint(t);
    const double r = fma(t - big, -0.010830424696249145, x); // ln 2 / 64
    const double p = fma(r, fma(r, fma(r, fma(r, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0), 1.0) * table[k & 63];
    const double e = __hiloint2double(__double2hiint(p) + ((k >> 6) << 20), __double2loint(p));
    return x >= -700.0 ? e : x != x ? x : 0.0;               // no branch: eight of these run side by side
}

// Maximum and sum of a row from its slices, by a warp.
__device__ __forceinline__ void vf_row_sum(const VfArgs& a, int row, float& m, double& sum) {
    const int lane = threadIdx.x & 31;
    const VfPart* part = a.part + (int64_t)row * a.slices;
    VfPart p;
    p.sum = 0.0;
    p.max = -INFINITY;
    if (lane < a.slices) p = part[lane];
    for (int s = lane + 32; s < a.slices; s += 32) {
        const VfPart z = part[s];
        const float mn = fmaxf(p.max, z.max);
        if (mn != -INFINITY) p.sum = p.sum * (double)vf_weight(p.max, mn, a.c) + z.sum * (double)vf_weight(z.max, mn, a.c);
        p.max = mn;
    }
    m = warp_max(p.max);
    sum = warp_sum(p.max == -INFINITY ? 0.0 : p.sum * (double)vf_weight(p.max, m, a.c));
}
// A thread's share -> the cluster's sum in every thread; warps' and CTAs' shares stay in warp_part and parts[turn].  Shares are pushed to the other CTAs, so
// that after the barrier everything is near.  turn alternates: a share is not overwritten before everybody has passed the next barrier.
template <int WARPS>
__device__ __forceinline__ double vf_reduce(cg::cluster_group& cl, double s, double* warp_part, double (*parts)[VW_CTAS], int& turn) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = (int)cl.num_blocks();
    s = warp_sum(s);
    turn ^= 1;
    __syncthreads();
    if (lane == 0) warp_part[warp] = s;
    __syncthreads();
    if (warp == 0) {
        const double t = warp_sum(lane < WARPS ? warp_part[lane] : 0.0);
        if (lane < ctas) *cl.map_shared_rank(&parts[turn][cl.block_rank()], lane) = t;
    }
    cl.sync();
    double t = 0.0;
    for (int r = 0; r < ctas; ++r) t += parts[turn][r];
    return t;
}

template <typename T, bool PROBS>
__global__ void __launch_bounds__(VW_THREADS) verify_walk_kernel(const __grid_constant__ VfArgs a, int per, int cached) {
    extern __shared__ double cache[];            // weights of the last node [vector of a lane, value, lane], then its probabilities (float)
    __shared__ int parent[VF_ROWS], tok[VF_ROWS], path[VF_ROWS], gone[VF_ROWS];
    __shared__ unsigned long long children[VF_ROWS];
    __shared__ float u[VF_ROWS], top[VF_ROWS], weight[VF_ROWS], prob[VF_ROWS];
    __shared__ double mass[VF_ROWS], left[VF_ROWS + 1], warp_part[VW_WARPS], parts[2][VW_CTAS], table[64];
    pdl_launch_dependents();
    if (threadIdx.x < 64) {
        table[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
        children[threadIdx.x] = 0;
    }
    pdl_wait();
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), ctas = (int)cl.num_blocks(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* logits = static_cast<const T*>(a.logits);
    // every CTA holds what the walk needs: a warp to a row
    if (tid < a.n) {
        u[tid] = a.u[tid];
        const int up = a.parents[tid];
        parent[tid] = tid > 0 && up >= 0 && up < tid ? up : -1;
        const int64_t x = a.tokens[tid];
        tok[tid] = x >= 0 && x < a.V ? (int)x : -1;
    }
#pragma unroll
    for (int i = 0; i < VF_ROWS / VW_WARPS; ++i) {      // side by side: a row's sum is a chain of exchanges
        const int r = warp + i * VW_WARPS;
        float m;
        double s;
        vf_row_sum(a, r < a.n ? r : 0, m, s);
        if (lane == 0) {
            top[r] = m;
            mass[r] = s;
        }
    }
    __syncthreads();
    if (tid < a.n) {
        float w = 0.0f, q = 1.0f;
        const int up = parent[tid], x = tok[tid];
        if (up >= 0) atomicOr(&children[up], 1ull << tid);
        if (up >= 0 && x >= 0) {
            w = top[up] == -INFINITY ? 0.0f : vf_weight(vf_get(logits + (int64_t)up * a.ld + x), top[up], a.c);
            if (PROBS) q = a.probs[(int64_t)up * a.ldp + x];
        }
        weight[tid] = w;
        prob[tid] = q;
    }
    __syncthreads();

    cl.sync();                       // shares are pushed to CTAs that run

    const int nvec = (a.V + 7) / 8, w0 = (rank * VW_WARPS + warp) * per, w1 = min(w0 + per, nvec), steps = (per + 31) / 32;      // a warp's vectors of a row
    int node = 0, count = 1, nrej = 0, turn = 0;
    // the mass that rejections with probabilities leave of the node; left[r]: the mass before rejection r
    auto rough = [&]() {
        const T* row = logits + (int64_t)node * a.ld;
        const float *probs = a.probs + (int64_t)node * a.ldp, m = top[node];
        double s = 0.0;
        constexpr int BATCH = 3;         // loads in flight together
        for (int v = w0 + lane; v < w1; v += 32 * BATCH) {
            float x[BATCH][8], q[BATCH][8];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                vf_load(row, v + 32 * i < w1 ? v + 32 * i : nvec, a.V, -INFINITY, x[i]);      // (nvec: past the end, all -inf)
                vf_load(probs, v + 32 * i < w1 ? v + 32 * i : nvec, a.V, 0.0f, q[i]);
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[i][j] = m == -INFINITY ? 0.0f : vf_weight(x[i][j], m, a.c);
            for (int r = 0; r < nrej; ++r) {
                const float l = (float)left[r];
#pragma unroll
                for (int i = 0; i < BATCH; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[i][j] = fmaxf(fmaf(-q[i][j], l, x[i][j]), 0.0f);
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) s += (double)(((x[i][0] + x[i][1]) + (x[i][2] + x[i][3])) + ((x[i][4] + x[i][5]) + (x[i][6] + x[i][7])));
        }
        return vf_reduce<VW_WARPS>(cl, s, warp_part, parts, turn);
    };

    // the walk: every thread takes the same steps
    double now = mass[0];            // mass of the node's residual weights
    if (tid == 0) path[0] = 0;
    for (unsigned long long todo = children[0]; todo;) {
        const int c = __ffsll((long long)todo) - 1;
        todo &= todo - 1;
        double w = (double)weight[c];
        if (PROBS) {
            for (int r = 0; r < nrej; ++r) w = fmax(w - (double)prob[c] * left[r], 0.0);
        } else {
            for (int r = 0; r < nrej; ++r)
                if (gone[r] == tok[c]) w = 0.0;
        }
        if ((double)u[c] * (double)prob[c] * now < w) {
            if (tid == 0) path[count] = c;
            node = c;
            ++count;
            nrej = 0;
            now = mass[c];
            todo = children[c];
        } else if (PROBS) {
            __syncthreads();
            if (tid == 0) left[nrej] = now;
            __syncthreads();
            ++nrej;
            if (todo) {              // otherwise nothing is tested on what is left
                const double rest = rough();
                if (rest > 0.0) now = rest;
                else --nrej;
            }
        } else if (w > 0.0 && now - w > 0.0) {
            __syncthreads();
            if (tid == 0) gone[nrej] = tok[c];
            __syncthreads();
            ++nrej;
            now -= w;
        }
    }

    // the last node's weights in float64; a CTA keeps its share of them, and of the probabilities, in shared memory
    const int tests = nrej;
    double *mine = cache + (size_t)warp * steps * 256 + lane, *mine_q = mine + (size_t)VW_WARPS * steps * 256;
    const float* probs = PROBS ? a.probs + (int64_t)node * a.ldp : nullptr;
    const double m0 = (double)top[node];
    auto first = [&](int v, double (&w)[8]) {        // before any rejection with probabilities
        float x[8];
        vf_load(logits + (int64_t)node * a.ld, v, a.V, -INFINITY, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = x[j] == -INFINITY ? 0.0 : vf_exp(((double)x[j] - m0) * a.cd, table);
        if (!PROBS)
            for (int r = 0; r < tests; ++r)
                if (gone[r] >> 3 == v)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if ((gone[r] & 7) == j) w[j] = 0.0;
    };
    auto reject = [&](double (&w)[8], const double (&q)[8], double mass_before) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double t = fma(-q[j], mass_before, w[j]);
            w[j] = t > 0.0 ? t : 0.0;
        }
    };
    // the weights after `kept` rejections (masses before them in left[]), of which the last may still be missing in the cache (done < kept), and one more
    auto residual = [&](int v, int done, int kept, bool more, double (&w)[8]) {
        const int at = (v - w0) / 32 * 256;
        double q[8];
        if (cached) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = mine[at + j * 32];
            if (PROBS && (done < kept || more))
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = mine_q[at + j * 32];
        } else {
            first(v, w);
            done = 0;
            if (PROBS && (kept || more)) {
                float y[8];
                vf_load(probs, v, a.V, 0.0f, y);
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = (double)y[j];
            }
        }
        if (PROBS && done < kept) {
            for (int r = done; r < kept; ++r) reject(w, q, left[r]);
            if (cached)
#pragma unroll
                for (int j = 0; j < 8; ++j) mine[at + j * 32] = w[j];
        }
        if (PROBS && more) reject(w, q, left[kept]);
    };
    auto sum8 = [](const double (&w)[8]) { return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])); };
    double s = 0.0;
#pragma unroll 2
    for (int v = w0 + lane; v < w1; v += 32) {
        double w[8];
        float y[8];
        if (PROBS && cached && tests) vf_load(probs, v, a.V, 0.0f, y);
        first(v, w);
        if (cached) {
            const int at = (v - w0) / 32 * 256;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                mine[at + j * 32] = w[j];
                if (PROBS && tests) mine_q[at + j * 32] = (double)y[j];
            }
        }
        s += sum8(w);
    }
    now = vf_reduce<VW_WARPS>(cl, s, warp_part, parts, turn);
    int kept = 0, done = 0;          // rejections in left[], and in the cached weights
    bool last = false;               // whether the shares are those after left[kept]
    if (PROBS) {
        for (int r = 0; r < tests; ++r) {
            if (tid == 0) left[kept] = now;
            __syncthreads();
            s = 0.0;
            for (int v = w0 + lane; v < w1; v += 32) {
                double w[8];
                residual(v, done, kept, true, w);
                s += sum8(w);
            }
            done = kept;
            const double rest = vf_reduce<VW_WARPS>(cl, s, warp_part, parts, turn);
            last = rest > 0.0;
            if (!last) {             // a rejection that leaves nothing is none, and so are the later ones: the shares are made again without it
                s = 0.0;
                for (int v = w0 + lane; v < w1; v += 32) {
                    double w[8];
                    residual(v, done, kept, false, w);
                    s += sum8(w);
                }
                now = vf_reduce<VW_WARPS>(cl, s, warp_part, parts, turn);
                break;
            }
            now = rest;
            if (r + 1 < tests) ++kept;
        }
    }
    // the owner of the target: the first CTA, warp and element whose cumulative weight exceeds it (the last with any where roundings leave none)
    const double target = (double)u[0] * now;
    double before = 0.0, own_before = 0.0;
    int owner = -1;
    bool found = false;
    for (int r = 0; r < ctas; ++r) {
        const double t = parts[turn][r];
        if (t > 0.0 && !found) {
            owner = r;
            own_before = before;
            found = before + t > target;
        }
        before += t;
    }
    if (!(now > 0.0 && now < INFINITY)) owner = -1;      // a NaN or +inf among the logits: every share may be a number but the one that has it
    if (rank == 0 && warp == 1) {
        for (int i = lane; i < a.n; i += 32) a.rows[i] = i < count ? path[i] : -1;
        if (lane == 0) {
            *a.count = count;
            if (owner < 0) *a.token = 0;       // no probabilities
        }
    }
    if (rank == owner) {
        double b = own_before, start = own_before;
        int ow = -1;
        found = false;
        for (int w = 0; w < VW_WARPS; ++w) {
            const double t = warp_part[w];
            if (t > 0.0 && !found) {
                ow = w;
                start = b;
                found = b + t > target;
            }
            b += t;
        }
        if (warp == ow) {
            int best = 0;
            bool hit_found = false;
            for (int v0 = w0; v0 < w1 && !hit_found; v0 += 32) {
                double w[8];
                const int v = v0 + lane;
                if (v < w1) residual(v, done, kept, last, w);
                else
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = 0.0;
                const double t = sum8(w);
                double inc = t;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double z = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += z;
                }
                double run = start + inc - t;
                int hit = -1, last = -1;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    run += w[j];
                    if (w[j] > 0.0) {
                        last = 8 * v + j;
                        if (hit < 0 && run > target) hit = 8 * v + j;
                    }
                }
                const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
                if (hits) {
                    best = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
                    hit_found = true;
                } else if (any) {
                    best = __shfl_sync(0xffffffffu, last, 31 - __clz(any));
                }
                start += __shfl_sync(0xffffffffu, inc, 31);
            }
            if (lane == 0) *a.token = best;
        }
    }
    cl.sync();              // nobody leaves while a share may still be pushed to it
}

template <typename T, bool PROBS>
static int launch_walk(const VfArgs& a, cudaStream_t st) {
    static int clusters[64] = {};        // CTAs of the walking cluster, by device
    const int dev = current_device();
    SCMX_REQUIRE(dev >= 0, SCMX_ECUDA, "no current CUDA device (ordinal 0..63)");
    void (*kern)(VfArgs, int, int) = verify_walk_kernel<T, PROBS>;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = VW_CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(VW_CTAS);
    cfg.blockDim = dim3(VW_THREADS);
    cfg.dynamicSmemBytes = VW_CACHE;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!clusters[dev]) {
        SCMX_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, VW_CACHE));
        int room = 0;
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&room, kern, &cfg) != cudaSuccess) {
            room = 0;
            (void)cudaGetLastError();
        }
        clusters[dev] = room > 0 ? VW_CTAS : VW_CTAS / 2;
    }
    const int ctas = clusters[dev];
    attr[0].val.clusterDim.x = ctas;
    cfg.gridDim = dim3(ctas);
    // vectors of a warp, and what a CTA keeps of its share; a larger vocabulary computes it again for every pass
    const int nvec = (a.V + 7) / 8, per = (nvec + ctas * VW_WARPS - 1) / (ctas * VW_WARPS);
    const int64_t bytes = (int64_t)VW_WARPS * ((per + 31) / 32) * 256 * (PROBS ? 16 : 8);
    const int cached = bytes <= VW_CACHE;
    cfg.dynamicSmemBytes = cached ? bytes : 0;
    cfg.numAttrs = g_use_pdl ? 2 : 1;
    SCMX_PDL_OK("verify_walk_kernel", cudaLaunchKernelEx(&cfg, kern, a, per, cached));
    return SCMX_OK;
}

template <typename T>
static int launch_verify(const VfArgs& a, bool greedy, cudaStream_t st) {
    const dim3 grid((unsigned)a.slices, (unsigned)a.n);
    if (greedy) {
        SCMX_PDL_OK("verify_rows_kernel", launch_pdl(verify_rows_kernel<T, true>, grid, dim3(VF_THREADS), 0, st, a));
        SCMX_PDL_OK("verify_greedy_kernel", launch_pdl(verify_greedy_kernel, dim3(1), dim3(1024), 0, st, a));
        return SCMX_OK;
    }
    SCMX_PDL_OK("verify_rows_kernel", launch_pdl(verify_rows_kernel<T, false>, grid, dim3(VF_THREADS), 0, st, a));
    return a.probs ? launch_walk<T, true>(a, st) : launch_walk<T, false>(a, st);
}

}  // namespace scmx

using namespace scmx;

extern "C" int64_t scmx_verify_scratch(int n, int64_t V) {
    if (n < 1 || n > VF_ROWS || V < 1 || V >= (1ll << 30)) return 0;
    return (int64_t)n * ((V + VF_SLICE - 1) / VF_SLICE) * (int64_t)sizeof(VfPart);
}

extern "C" int scmx_verify(const void* logits, int is_f32, int64_t ld, const int64_t* tokens, const int32_t* parents, const float* u, double temperature,
                           const float* probs, int64_t ldp, int n, int64_t V, int32_t* rows, int32_t* count, int64_t* token, void* scratch, int64_t scratch_bytes,
                           void* stream) {
    SCMX_REQUIRE(n >= 1 && n <= VF_ROWS, SCMX_ELIMIT, "verify: %d rows (1 .. %d)", n, VF_ROWS);
    SCMX_REQUIRE(V >= 1 && V < (1ll << 30) && ld >= V && (probs == nullptr || ldp >= V), SCMX_EINVAL, "verify: %lld logits, rows %lld and %lld apart", (long long)V,
                 (long long)ld, (long long)ldp);
    SCMX_REQUIRE(logits && tokens && parents && rows && count && token, SCMX_EINVAL, "verify: null buffer");
    const bool greedy = temperature == 0.0;
    SCMX_REQUIRE(greedy || (temperature > 0.0 && temperature <= 3.0e38 && 1.45 / temperature <= 3.0e38), SCMX_EINVAL, "verify: temperature %g", temperature);
    SCMX_REQUIRE(greedy || u != nullptr, SCMX_EINVAL, "verify: sampling needs random numbers");
    SCMX_REQUIRE(((uintptr_t)logits & (is_f32 ? 3 : 1)) == 0 && ((uintptr_t)probs & 3) == 0, SCMX_EINVAL, "verify: unaligned buffer");
    const int64_t need = scmx_verify_scratch(n, V);
    SCMX_REQUIRE(scratch && ((uintptr_t)scratch & 15) == 0 && scratch_bytes >= need, SCMX_EINVAL, "verify: %lld bytes of scratch, %lld needed", (long long)scratch_bytes,
                 (long long)need);
    VfArgs a;
    a.logits = logits; a.probs = greedy ? nullptr : probs; a.tokens = tokens; a.parents = parents; a.u = u; a.part = static_cast<VfPart*>(scratch);
    a.rows = rows; a.count = count; a.token = token; a.ld = ld; a.ldp = ldp; a.n = n; a.V = (int)V; a.slices = (int)((V + VF_SLICE - 1) / VF_SLICE);
    a.c = greedy ? 1.0f : (float)(1.4426950408889634 / temperature);
    a.cd = greedy ? 1.0 : 1.0 / temperature;      // (a float32 temperature is 2^-25 off: one of 300 draws from 150000 logits would be another token)
    return is_f32 ? launch_verify<float>(a, greedy, (cudaStream_t)stream) : launch_verify<uint16_t>(a, greedy, (cudaStream_t)stream);
}

// Verification of drafted tokens: which rows of a tree of drafts the target accepts, from its logits and given random numbers, and the
// token after them.  Row 0 is the last chosen token, row c continues row parents[c] < c.  At a node with target probabilities p, its children
// are tested in ascending order: child c with token x is accepted if u[c] q(x) < p(x), q the draft's probabilities (1 where there are none);
// a rejected child leaves p <- max(p - q, 0) / Z (or p without x).  Where no child is left, the token is the first whose
// cumulative probability exceeds u[0].  Accepted paths and tokens follow the target's distribution whatever the draft proposed.
// Temperature 0: a child is accepted if it is the largest logit of its parent (the lowest index of equal ones), which is also the token.
//
// The maxima and sums of all rows are a pass over the logits by the whole device (memory-bound); one cluster then walks the tree, which needs one
// logit per drafted row.  Where drafts have probabilities, a launch between the two finds what rejections leave of every node with more
// than one child, a cluster to a node (float32 weights: this mass decides tests whose border a relative error of 1e-6 moves by as much).
// The last token's weights, sums and cumulative probabilities are float64, made by the walking cluster for its node alone: between 100000
// neighbours float32 sums would pick another token once in a hundred draws.
#include <cooperative_groups.h>
#include "scmx_common.cuh"

namespace cg = cooperative_groups;

namespace scmx {

constexpr int VF_ROWS = 64, VF_THREADS = 256, VF_VECS = 4;                  // first launch: 256 x 4 vectors of 8 logits per CTA
constexpr int VF_SLICE = VF_THREADS * VF_VECS * 8;
constexpr int VM_CTAS = 8, VM_THREADS = 512;                                // masses after rejections: a cluster to a node
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
    double* masses;                  // [n, 64]: what the first, second, .. rejection leaves of a node
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

// The weight of a logit against its row's maximum in float32, the same in both launches.
__device__ __forceinline__ float vf_weight(float x, float m, float c) { return exp2f(__fmul_rn(__fsub_rn(x, m), c)); }

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
    if (!(x >= -700.0)) return x != x ? x : 0.0;
    const double big = 6755399441055744.0;                   // 1.5 2^52: adding it rounds to a whole number, whose low bits are those of the sum
    const double t = fma(x, 92.332482616893656877, big);     // 64 / ln 2
    const int k = __double2loint(t);
    const double r = fma(t - big, -0.010830424696249145, x); // ln 2 / 64
    const double p = fma(r, fma(r, fma(r, fma(r, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0), 1.0) * table[k & 63];
    return __hiloint2double(__double2hiint(p) + ((k >> 6) << 20), __double2loint(p));
}

// Maximum and sum of a row from its slices, by a warp.
__device__ __forceinline__ void vf_row_sum(const VfArgs& a, int row, float& m, double& sum) {
    const int lane = threadIdx.x & 31;
    m = -INFINITY;
    sum = 0.0;
    for (int s0 = 0; s0 < a.slices; s0 += 32) {
        VfPart p;
        p.sum = 0.0;
        p.max = -INFINITY;
        if (s0 + lane < a.slices) p = a.part[(int64_t)row * a.slices + s0 + lane];
        const float mn = fmaxf(m, warp_max(p.max));
        const double w = p.max == -INFINITY ? 0.0 : p.sum * (double)vf_weight(p.max, mn, a.c);
        sum = sum * (m == -INFINITY ? 0.0 : (double)vf_weight(m, mn, a.c)) + warp_sum(w);
        m = mn;
    }
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

// grid (VM_CTAS, n)
template <typename T>
__global__ void __cluster_dims__(VM_CTAS, 1, 1) __launch_bounds__(VM_THREADS) verify_masses_kernel(const __grid_constant__ VfArgs a) {
    __shared__ double warp_part[VM_THREADS / 32], parts[2][VW_CTAS], sum;
    __shared__ float max;
    __shared__ int children;
    pdl_launch_dependents();
    pdl_wait();
    cg::cluster_group cl = cg::this_cluster();
    const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    if (tid < 32) {
        int n = 0;
        for (int c0 = 0; c0 < a.n; c0 += 32) {
            const int c = c0 + lane;
            n += __popc(__ballot_sync(0xffffffffu, c > row && c < a.n && a.parents[c] == row));
        }
        float m;
        double s;
        vf_row_sum(a, row, m, s);
        if (lane == 0) {
            children = n;
            max = m;
            sum = s;
        }
    }
    __syncthreads();
    if (children < 2) return;            // the whole cluster: after an only child's rejection nothing is tested
    cl.sync();                           // shares are pushed to CTAs that run
    const int nvec = (a.V + 7) / 8, per = (nvec + VM_CTAS - 1) / VM_CTAS, v0 = (int)cl.block_rank() * per, v1 = min(v0 + per, nvec);
    const T* logits = static_cast<const T*>(a.logits) + (int64_t)row * a.ld;
    const float* probs = a.probs + (int64_t)row * a.ldp;
    const float m = max;
    double left[2] = {sum, 0.0};         // masses before the first and the second rejection; further ones are read back
    int turn = 0;
    for (int k = 1; k < children; ++k) {
        double s = 0.0;
#pragma unroll 2
        for (int v = v0 + tid; v < v1; v += VM_THREADS) {
            float x[8], q[8];
            vf_load(logits, v, a.V, -INFINITY, x);
            vf_load(probs, v, a.V, 0.0f, q);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = m == -INFINITY ? 0.0f : fmaxf(fmaf(-q[j], (float)left[0], vf_weight(x[j], m, a.c)), 0.0f);
            for (int r = 1; r < k; ++r) {
                const float w = (float)(r == 1 ? left[1] : a.masses[row * VF_ROWS + r - 1]);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = fmaxf(fmaf(-q[j], w, x[j]), 0.0f);
            }
            s += (double)(((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])));
        }
        const double rest = vf_reduce<VM_THREADS / 32>(cl, s, warp_part, parts, turn);
        if (k == 1) left[1] = rest;
        if (tid == 0) a.masses[row * VF_ROWS + k - 1] = rest;      // every CTA stores what it will read
        __syncthreads();
        if (!(rest > 0.0)) break;        // a rejection that leaves nothing is none, and so are the later ones
    }
    cl.sync();                           // nobody leaves while shares may still be pushed to it
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
    for (int r = warp; r < a.n; r += VW_WARPS) {
        float m;
        double s;
        vf_row_sum(a, r, m, s);
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

    // the walk: every thread takes the same steps
    int node = 0, count = 1, nrej = 0, turn = 0;
    double now = mass[0];            // mass of the node's residual weights
    if (tid == 0) path[0] = 0;
    for (unsigned long long todo = children[0]; todo;) {
        const int c = __ffsll((long long)todo) - 1;
        todo &= todo - 1;
        double w = (double)weight[c];
        if (PROBS) {
            for (int r = 0; r < nrej; ++r) w = fmax(w - (double)prob[c] * (r ? a.masses[node * VF_ROWS + r - 1] : mass[node]), 0.0);
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
            const double rest = todo ? a.masses[node * VF_ROWS + nrej] : 1.0;      // the last child's is not tested on
            if (rest > 0.0) {
                ++nrej;
                now = rest;
            }
        } else if (w > 0.0 && now - w > 0.0) {
            __syncthreads();
            if (tid == 0) gone[nrej] = tok[c];
            __syncthreads();
            ++nrej;
            now -= w;
        }
    }

    // the last node's weights in float64, its share of a CTA kept in shared memory
    const int nvec = (a.V + 7) / 8, w0 = (rank * VW_WARPS + warp) * per, w1 = min(w0 + per, nvec), steps = (per + 31) / 32;
    double* mine = cache + (size_t)warp * steps * 256 + lane;
    float* mine_q = reinterpret_cast<float*>(cache + (size_t)VW_WARPS * steps * 256) + (size_t)warp * steps * 256 + lane;
    const float* probs = PROBS ? a.probs + (int64_t)node * a.ldp : nullptr;
    const int tests = nrej;
    auto first = [&](int v, double (&w)[8]) {        // before any rejection with probabilities
        float x[8], q[8];
        vf_load(logits + (int64_t)node * a.ld, v, a.V, -INFINITY, x);
        if (PROBS && cached && tests) vf_load(probs, v, a.V, 0.0f, q);
        const double m = (double)top[node];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = x[j] == -INFINITY ? 0.0 : vf_exp(((double)x[j] - m) * a.cd, table);
        if (!PROBS)
            for (int r = 0; r < tests; ++r)
                if (gone[r] >> 3 == v)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if ((gone[r] & 7) == j) w[j] = 0.0;
        if (cached) {
            const int at = (v - w0) / 32 * 256;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                mine[at + j * 32] = w[j];
                if (PROBS && tests) mine_q[at + j * 32] = q[j];
            }
        }
    };
    auto residual = [&](int v, double (&w)[8]) {     // after nrej of them, once `first` has been through
        if (!cached) {
            first(v, w);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = mine[(v - w0) / 32 * 256 + j * 32];
        }
        if (PROBS && nrej) {
            float q[8];
            if (!cached) vf_load(probs, v, a.V, 0.0f, q);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = mine_q[(v - w0) / 32 * 256 + j * 32];
            for (int r = 0; r < nrej; ++r) {
                const double m = left[r];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const double t = fma(-(double)q[j], m, w[j]);
                    w[j] = t > 0.0 ? t : 0.0;
                }
            }
        }
    };
    auto sum8 = [](const double (&w)[8]) { return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])); };
    double s = 0.0;
#pragma unroll 2
    for (int v = w0 + lane; v < w1; v += 32) {
        double w[8];
        first(v, w);
        s += sum8(w);
    }
    now = vf_reduce<VW_WARPS>(cl, s, warp_part, parts, turn);
    if (PROBS) {
        nrej = 0;
        for (int r = 0; r < tests; ++r) {
            if (tid == 0) left[nrej] = now;
            __syncthreads();
            ++nrej;
            for (;;) {
                s = 0.0;
                for (int v = w0 + lane; v < w1; v += 32) {
                    double w[8];
                    residual(v, w);
                    s += sum8(w);
                }
                const double rest = vf_reduce<VW_WARPS>(cl, s, warp_part, parts, turn);
                if (rest > 0.0) {
                    now = rest;
                    break;
                }
                if (nrej == 0) break;
                --nrej;                  // a rejection that leaves nothing is none: the shares are made again without it
            }
            if (!(now > 0.0)) break;
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
    if (rank == 0 && warp == 1) {
        for (int i = lane; i < a.n; i += 32) a.rows[i] = i < count ? path[i] : -1;
        if (lane == 0) {
            *a.count = count;
            if (owner < 0) *a.token = 0;       // no probabilities: all logits -inf, or not numbers
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
            bool done = false;
            for (int v0 = w0; v0 < w1 && !done; v0 += 32) {
                double w[8];
                const int v = v0 + lane;
                if (v < w1) residual(v, w);
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
                    done = true;
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
    const int64_t bytes = (int64_t)VW_WARPS * ((per + 31) / 32) * 256 * (PROBS ? 12 : 8);
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
    if (a.probs == nullptr) return launch_walk<T, false>(a, st);
    if (a.n > 2) SCMX_PDL_OK("verify_masses_kernel", launch_pdl(verify_masses_kernel<T>, dim3(VM_CTAS, (unsigned)a.n), dim3(VM_THREADS), 0, st, a));
    return launch_walk<T, true>(a, st);
}

}  // namespace scmx

using namespace scmx;

extern "C" int64_t scmx_verify_scratch(int n, int64_t V) {
    if (n < 1 || n > VF_ROWS || V < 1 || V >= (1ll << 30)) return 0;
    return (int64_t)n * (((V + VF_SLICE - 1) / VF_SLICE) * (int64_t)sizeof(VfPart) + VF_ROWS * 8);
}

extern "C" int scmx_verify(const void* logits, int is_f32, int64_t ld, const int64_t* tokens, const int32_t* parents, const float* u, float temperature,
                           const float* probs, int64_t ldp, int n, int64_t V, int32_t* rows, int32_t* count, int64_t* token, void* scratch, int64_t scratch_bytes,
                           void* stream) {
    SCMX_REQUIRE(n >= 1 && n <= VF_ROWS, SCMX_ELIMIT, "verify: %d rows (1 .. %d)", n, VF_ROWS);
    SCMX_REQUIRE(V >= 1 && V < (1ll << 30) && ld >= V && (probs == nullptr || ldp >= V), SCMX_EINVAL, "verify: %lld logits, rows %lld and %lld apart", (long long)V,
                 (long long)ld, (long long)ldp);
    SCMX_REQUIRE(logits && tokens && parents && rows && count && token, SCMX_EINVAL, "verify: null buffer");
    const bool greedy = temperature == 0.0f;
    SCMX_REQUIRE(greedy || (temperature > 0.0f && temperature <= 3.0e38f && 1.0f / temperature <= 3.0e38f), SCMX_EINVAL, "verify: temperature %g", (double)temperature);
    SCMX_REQUIRE(greedy || u != nullptr, SCMX_EINVAL, "verify: sampling needs random numbers");
    SCMX_REQUIRE(((uintptr_t)logits & (is_f32 ? 3 : 1)) == 0 && ((uintptr_t)probs & 3) == 0, SCMX_EINVAL, "verify: unaligned buffer");
    const int64_t need = scmx_verify_scratch(n, V);
    SCMX_REQUIRE(scratch && ((uintptr_t)scratch & 15) == 0 && scratch_bytes >= need, SCMX_EINVAL, "verify: %lld bytes of scratch, %lld needed", (long long)scratch_bytes,
                 (long long)need);
    VfArgs a;
    a.logits = logits; a.probs = greedy ? nullptr : probs; a.tokens = tokens; a.parents = parents; a.u = u; a.part = static_cast<VfPart*>(scratch); a.masses = reinterpret_cast<double*>(a.part + n * ((V + VF_SLICE - 1) / VF_SLICE));
    a.rows = rows; a.count = count; a.token = token; a.ld = ld; a.ldp = ldp; a.n = n; a.V = (int)V; a.slices = (int)((V + VF_SLICE - 1) / VF_SLICE);
    a.c = greedy ? 1.0f : (float)(1.4426950408889634 / (double)temperature);
    a.cd = greedy ? 1.0 : 1.0 / (double)temperature;
    return is_f32 ? launch_verify<float>(a, greedy, (cudaStream_t)stream) : launch_verify<uint16_t>(a, greedy, (cudaStream_t)stream);
}

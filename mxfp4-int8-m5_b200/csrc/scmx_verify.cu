// Verification of drafted tokens: which rows of a tree of drafts the target accepts, from its logits and given random numbers, and the
// token after them.  Row 0 is the last chosen token, row c continues row parents[c] < c.  At a node with target probabilities p, its children
// are tested in ascending order: child c with token x is accepted if u[c] q(x) < p(x), q the draft's probabilities (1 where there are none);
// a rejected child leaves p <- max(p - q, 0) / Z (or p without x).  Where no child is left, the token is the first whose
// cumulative probability exceeds u[0].  Accepted paths and tokens follow the target's distribution whatever the draft proposed.
// Temperature 0: a child is accepted if it is the largest logit of its parent (the lowest index of equal ones), which is also the token.
//
// Two launches: the maxima and sums of all rows, a pass over the logits by the whole device (memory-bound), and one cluster that walks the
// tree.  The walk needs one logit per drafted row; whole rows are read again only where a draft with probabilities is rejected and for the
// last token.  Those sums and the cumulative probabilities are float64, so that a token is decided by the numbers and not by roundings.
#include <cooperative_groups.h>
#include "scmx_common.cuh"

namespace cg = cooperative_groups;

namespace scmx {

constexpr int VF_ROWS = 64, VF_THREADS = 256, VF_VECS = 4;                  // first launch: 256 x 4 vectors of 8 logits per CTA
constexpr int VF_SLICE = VF_THREADS * VF_VECS * 8;
constexpr int VW_CTAS = 8, VW_THREADS = 512, VW_WARPS = VW_THREADS / 32;     // second launch

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
__global__ void __launch_bounds__(VF_THREADS) verify_rows_kernel(const VfArgs a) {
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

// Rows and count of the accepted path, by one thread.
__device__ __forceinline__ void vf_write_path(const VfArgs& a, const int* path, int count) {
    for (int i = 0; i < a.n; ++i) a.rows[i] = i < count ? path[i] : -1;
    *a.count = count;
}

__global__ void __launch_bounds__(VF_ROWS) verify_greedy_kernel(const VfArgs a) {
    __shared__ int best[VF_ROWS], parent[VF_ROWS], path[VF_ROWS];
    __shared__ int64_t token[VF_ROWS];
    pdl_launch_dependents();
    pdl_wait();
    const int i = threadIdx.x;
    if (i < a.n) {
        unsigned long long k = 0;
        for (int s = 0; s < a.slices; ++s) k = max(k, a.part[(int64_t)i * a.slices + s].key);
        best[i] = (int)(0xFFFFFFFFu - (uint32_t)k);
        parent[i] = a.parents[i];
        token[i] = a.tokens[i];
    }
    __syncthreads();
    if (i != 0) return;
    int node = 0, count = 1;
    path[0] = 0;
    for (int c = 1; c < a.n; ++c)
        if (parent[c] == node && token[c] == best[node]) path[count++] = node = c;
    vf_write_path(a, path, count);
    *a.token = best[node];
}

template <typename T, bool PROBS>
__global__ void __cluster_dims__(VW_CTAS, 1, 1) __launch_bounds__(VW_THREADS) verify_walk_kernel(const VfArgs a) {
    __shared__ int parent[VF_ROWS], tok[VF_ROWS], path[VF_ROWS], gone[VF_ROWS];
    __shared__ float u[VF_ROWS], top[VF_ROWS], weight[VF_ROWS], prob[VF_ROWS];
    __shared__ double mass[VF_ROWS], left[VF_ROWS + 1], warp_part[VW_WARPS], cta_part[2];
    pdl_launch_dependents();
    pdl_wait();
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T* logits = static_cast<const T*>(a.logits);
    // every CTA holds what the walk needs
    if (tid < a.n) {
        float m = -INFINITY;
        for (int s = 0; s < a.slices; ++s) m = fmaxf(m, a.part[(int64_t)tid * a.slices + s].max);
        double sum = 0.0;
        if (m != -INFINITY)
            for (int s = 0; s < a.slices; ++s) {
                const VfPart p = a.part[(int64_t)tid * a.slices + s];
                if (p.max != -INFINITY) sum += p.sum * (double)vf_weight(p.max, m, a.c);
            }
        top[tid] = m;
        mass[tid] = sum;
        u[tid] = a.u[tid];
        const int up = a.parents[tid];
        parent[tid] = tid > 0 && up >= 0 && up < tid ? up : -1;
        const int64_t x = a.tokens[tid];
        tok[tid] = x >= 0 && x < a.V ? (int)x : -1;
    }
    __syncthreads();
    if (tid < a.n) {
        float w = 0.0f, q = 1.0f;
        const int up = parent[tid], x = tok[tid];
        if (up >= 0 && x >= 0) {
            w = top[up] == -INFINITY ? 0.0f : vf_weight(vf_get(logits + (int64_t)up * a.ld + x), top[up], a.c);
            if (PROBS) q = a.probs[(int64_t)up * a.ldp + x];
        }
        weight[tid] = w;
        prob[tid] = q;
    }
    __syncthreads();

    const int nvec = (a.V + 7) / 8, per = ((nvec + VW_CTAS * VW_WARPS - 1) / (VW_CTAS * VW_WARPS) + 31) / 32 * 32;      // vectors of a warp
    const int w0 = (rank * VW_WARPS + warp) * per, w1 = min(w0 + per, nvec);
    int node = 0, count = 1, nrej = 0, turn = 0;
    // eight residual weights of the node in float64: left[r] is the mass before rejection r
    auto residual = [&](int v, double (&w)[8]) {
        float x[8], q[8];
        vf_load(logits + (int64_t)node * a.ld, v, a.V, -INFINITY, x);
        if (PROBS && nrej) vf_load(a.probs + (int64_t)node * a.ldp, v, a.V, 0.0f, q);
        const double m = (double)top[node];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = x[j] == -INFINITY ? 0.0 : exp(((double)x[j] - m) * a.cd);
            if (PROBS) {
                for (int r = 0; r < nrej; ++r) w[j] = fmax(w[j] - (double)q[j] * left[r], 0.0);
            } else {
                for (int r = 0; r < nrej; ++r)
                    if (gone[r] == 8 * v + j) w[j] = 0.0;
            }
        }
    };
    // its sum over the vocabulary; every thread gets it, and the warps' and CTAs' shares stay
    auto total = [&]() {
        double s = 0.0;
        for (int v = w0 + lane; v < w1; v += 32) {
            double w[8];
            residual(v, w);
            s += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        }
        s = warp_sum(s);
        turn ^= 1;
        __syncthreads();
        if (lane == 0) warp_part[warp] = s;
        __syncthreads();
        if (tid == 0) {
            double t = 0.0;
            for (int w = 0; w < VW_WARPS; ++w) t += warp_part[w];
            cta_part[turn] = t;
        }
        cl.sync();
        double t = 0.0;
        for (int r = 0; r < VW_CTAS; ++r) t += *cl.map_shared_rank(&cta_part[turn], r);
        return t;
    };

    // the walk: every thread takes the same steps
    double now = mass[0];            // mass of the node's residual weights
    bool fresh = false;              // whether `now` and the shares are those of `total`
    if (tid == 0) path[0] = 0;
    for (int c = 1; c < a.n; ++c) {
        if (parent[c] != node) continue;
        double w = (double)weight[c];
        if (PROBS) {
            if (!fresh && nrej) now = total(), fresh = true;
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
            fresh = false;
        } else if (PROBS) {
            if (!fresh) now = total(), fresh = true;         // the exact mass, of which the draft's share is taken
            __syncthreads();
            if (tid == 0) left[nrej] = now;
            __syncthreads();
            ++nrej;
            const double rest = total();
            if (rest > 0.0) now = rest;
            else --nrej, fresh = false;
        } else if (w > 0.0 && now - w > 0.0) {
            __syncthreads();
            if (tid == 0) gone[nrej] = tok[c];
            __syncthreads();
            ++nrej;
            now -= w;
        }
    }
    if (!fresh) now = total();
    // the owner of the target: the first CTA, warp and element whose cumulative weight exceeds it (the last with any where roundings leave none)
    const double target = (double)u[0] * now;
    double before = 0.0, own_before = 0.0;
    int owner = -1;
    bool found = false;
    for (int r = 0; r < VW_CTAS && !found; ++r) {
        const double s = *cl.map_shared_rank(&cta_part[turn], r);
        if (s > 0.0) {
            owner = r;
            own_before = before;
            found = before + s > target;
        }
        before += s;
    }
    if (rank == 0 && tid == 0) {
        vf_write_path(a, path, count);
        if (owner < 0) *a.token = 0;       // no probabilities: all logits -inf, or not numbers
    }
    if (rank == owner) {
        double b = own_before, mine = own_before;
        int ow = -1;
        found = false;
        for (int w = 0; w < VW_WARPS && !found; ++w) {
            const double s = warp_part[w];
            if (s > 0.0) {
                ow = w;
                mine = b;
                found = b + s > target;
            }
            b += s;
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
                double s = 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) s += w[j];
                double inc = s;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double t = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += t;
                }
                double run = mine + inc - s;
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
                mine += __shfl_sync(0xffffffffu, inc, 31);
            }
            if (lane == 0) *a.token = best;
        }
    }
    cl.sync();              // nobody leaves while its share may still be read
}

template <typename T>
static int launch_verify(const VfArgs& a, bool greedy, cudaStream_t st) {
    const dim3 grid((unsigned)a.slices, (unsigned)a.n);
    if (greedy) {
        SCMX_PDL_OK("verify_rows_kernel", launch_pdl(verify_rows_kernel<T, true>, grid, dim3(VF_THREADS), 0, st, a));
        SCMX_PDL_OK("verify_greedy_kernel", launch_pdl(verify_greedy_kernel, dim3(1), dim3(VF_ROWS), 0, st, a));
        return SCMX_OK;
    }
    SCMX_PDL_OK("verify_rows_kernel", launch_pdl(verify_rows_kernel<T, false>, grid, dim3(VF_THREADS), 0, st, a));
    SCMX_PDL_OK("verify_walk_kernel", launch_pdl(a.probs ? verify_walk_kernel<T, true> : verify_walk_kernel<T, false>, dim3(VW_CTAS), dim3(VW_THREADS), 0, st, a));
    return SCMX_OK;
}

}  // namespace scmx

using namespace scmx;

extern "C" int64_t scmx_verify_scratch(int n, int64_t V) {
    if (n < 1 || n > VF_ROWS || V < 1 || V >= (1ll << 30)) return 0;
    return (int64_t)n * ((V + VF_SLICE - 1) / VF_SLICE) * (int64_t)sizeof(VfPart);
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
    a.logits = logits; a.probs = greedy ? nullptr : probs; a.tokens = tokens; a.parents = parents; a.u = u; a.part = static_cast<VfPart*>(scratch);
    a.rows = rows; a.count = count; a.token = token; a.ld = ld; a.ldp = ldp; a.n = n; a.V = (int)V; a.slices = (int)((V + VF_SLICE - 1) / VF_SLICE);
    a.c = greedy ? 1.0f : (float)(1.4426950408889634 / (double)temperature);
    a.cd = greedy ? 1.0 : 1.0 / (double)temperature;
    return is_f32 ? launch_verify<float>(a, greedy, (cudaStream_t)stream) : launch_verify<uint16_t>(a, greedy, (cudaStream_t)stream);
}

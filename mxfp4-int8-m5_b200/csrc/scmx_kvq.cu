// INT8 key/value cache: vectors of new tokens are quantized as they are written, cached rows are read back as bfloat16, and the rows of
// accepted drafts are moved together.  A head's vector at one position has one float32 scale: s = amax / 127, code = rint(x (1 / s)),
// the recipe of the activations' INT8.  Bound by memory: every value is loaded and stored once.  Measured on a B200: 2048 tokens of 8 heads
// of 128 written and read back in 7.2 us (two launches and 21 MB that stay in L2); 333 tokens written behind 29667 and all 30000 of 16
// heads read back in 60.1 us, 375 MB at 6.2 TB/s.  With 1, 2 and 4 vectors of a thread in flight the two take 7.8, 7.2, 7.5 us and 61.1, 60.1,
// 61.1 us.  A call for one token is its launch, 1.5 us.
#include "scmx_common.cuh"

namespace scmx {

constexpr int KV_THREADS = 256, KV_TURNS = 2;      // vectors of a thread whose loads are in flight together

struct KvWriteArgs {
    const uint16_t *k, *v;           // bf16 [hk, L, d]
    int64_t k_hs, k_rs, v_hs, v_rs;  // head and row strides in elements
    int8_t *kc, *vc;                 // [hk, cap, d]
    float *ks, *vs;                  // [hk, cap]
    const int32_t* pos_dev;
    int64_t pos, cap;
    int L, hk, d;
};

// A vector belongs to G lanes of 8 values each (G the power of two from d / 8 on).  blockIdx: rows, heads, keys or values.
template <int G>
__global__ void __launch_bounds__(KV_THREADS) kv_append_kernel(const __grid_constant__ KvWriteArgs a) {
    constexpr int ROWS = KV_THREADS / G;
    pdl_launch_dependents();
    pdl_wait();
    const bool val = blockIdx.z != 0;
    const int l = threadIdx.x % G, first = blockIdx.x * (ROWS * KV_TURNS) + threadIdx.x / G;
    const int64_t pos = a.pos_dev ? (int64_t)a.pos_dev[0] : a.pos, rs = val ? a.v_rs : a.k_rs;
    for (int head = blockIdx.y; head < a.hk; head += gridDim.y) {
        const uint16_t* src = (val ? a.v + head * a.v_hs : a.k + head * a.k_hs) + 8 * l;
        uint4 w[KV_TURNS];
#pragma unroll
        for (int i = 0; i < KV_TURNS; ++i) {
            const int row = first + i * ROWS;
            w[i] = make_uint4(0, 0, 0, 0);
            if (row < a.L && 8 * l < a.d) w[i] = *reinterpret_cast<const uint4*>(src + row * rs);
        }
        int8_t* codes = (val ? a.vc : a.kc) + head * a.cap * a.d + 8 * l;
        float* scales = (val ? a.vs : a.ks) + head * a.cap;
#pragma unroll
        for (int i = 0; i < KV_TURNS; ++i) {
            if (blockIdx.x * (ROWS * KV_TURNS) + i * ROWS >= a.L) break;
            const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            uint32_t top = 0;                // magnitudes of bfloat16 order like their bits, infinities and NaN last
#pragma unroll
            for (int j = 0; j < 4; ++j) top = max(top, max(u[j] & 0x7FFFu, (u[j] >> 16) & 0x7FFFu));
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            float s, qi;
            kv_scale(top, s, qi);
            const int row = first + i * ROWS;
            const int64_t at = pos + row;
            if (row >= a.L || 8 * l >= a.d || at < 0 || at >= a.cap) continue;      // a device-side position beyond the cache: the row is dropped
            uint32_t q[2] = {0, 0};
            if (qi > 0.0f) {
                q[0] = quant4(bf16_lo(u[0]), bf16_hi(u[0]), bf16_lo(u[1]), bf16_hi(u[1]), qi);
                q[1] = quant4(bf16_lo(u[2]), bf16_hi(u[2]), bf16_lo(u[3]), bf16_hi(u[3]), qi);
            }
            *reinterpret_cast<uint2*>(codes + at * a.d) = make_uint2(q[0], q[1]);
            if (l == 0) scales[at] = s;
        }
    }
}

struct KvReadArgs {
    const int8_t *kc, *vc;
    const float *ks, *vs;
    uint16_t *k, *v;                 // bf16 [hk, n, d]
    int64_t start, cap, n;
    int hk, d, pieces, rows;         // pieces of 16 values of a vector; vectors that a CTA takes in a turn
};

// A lane takes 16 codes; codes become bfloat16 exactly, and their product with the scale is rounded once.  Its 32 bytes leave in one store: two
// stores of 16 each fill half a sector, and reading 30000 positions takes 77 us instead of 60.
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const __grid_constant__ KvReadArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const I8Pairs i8;
    const bool val = blockIdx.z != 0;
    const int r = threadIdx.x / a.pieces, l = threadIdx.x - r * a.pieces;
    if (r >= a.rows) return;
    for (int head = blockIdx.y; head < a.hk; head += gridDim.y) {
        const int8_t* codes = (val ? a.vc : a.kc) + (head * a.cap + a.start) * a.d + 16 * l;
        const float* scales = (val ? a.vs : a.ks) + head * a.cap + a.start;
        uint16_t* out = (val ? a.v : a.k) + head * a.n * a.d + 16 * l;
        const int64_t first = (int64_t)blockIdx.x * a.rows * KV_TURNS + r;
        uint4 c[KV_TURNS];
        float s[KV_TURNS];
#pragma unroll
        for (int i = 0; i < KV_TURNS; ++i) {
            const int64_t row = first + i * a.rows;
            if (row < a.n) {
                c[i] = *reinterpret_cast<const uint4*>(codes + row * a.d);
                s[i] = scales[row];
            }
        }
#pragma unroll
        for (int i = 0; i < KV_TURNS; ++i) {
            const int64_t row = first + i * a.rows;
            if (row >= a.n) continue;
            const uint32_t u[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t even = i8.even(u[j]), odd = i8.odd(u[j]);
                o[2 * j] = pack_bf16x2(__fmul_rn(bf16_lo(even), s[i]), __fmul_rn(bf16_lo(odd), s[i]));
                o[2 * j + 1] = pack_bf16x2(__fmul_rn(bf16_hi(even), s[i]), __fmul_rn(bf16_hi(odd), s[i]));
            }
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + row * a.d), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]), "r"(o[4]),
                         "r"(o[5]), "r"(o[6]), "r"(o[7])
                         : "memory");
        }
    }
}

constexpr int KEEP_LAYERS = 64, KEEP_ROWS = 64, KEEP_THREADS = 128;

struct KvKeepArgs {
    scmx_kv_layer layer[KEEP_LAYERS];
    const int32_t* rows;             // [n]
    const int32_t* pos_dev;
    int64_t pos, cap;
    int n, row_bytes;
};

// One CTA per (head, layer, keys or values): every kept row is loaded before the first one is stored, so rows may change places.  Bound by its
// launch and two dependent loads: 3 rows in 16 layers 2.8 us, 9 rows in 28 layers 4.2 us.
__global__ void __launch_bounds__(KEEP_THREADS) kv_keep_kernel(const __grid_constant__ KvKeepArgs a) {
    constexpr int PER = KEEP_ROWS * 32 / KEEP_THREADS;      // 16-byte pieces of a thread: rows of 512 bytes at most
    pdl_launch_dependents();
    pdl_wait();
    const scmx_kv_layer ly = a.layer[blockIdx.y];
    const int64_t pos = a.pos_dev ? (int64_t)a.pos_dev[0] : a.pos;
    if (pos < 0 || pos + a.n > a.cap) return;
    const int tid = threadIdx.x, pieces = a.row_bytes / 16;
    char* base = static_cast<char*>(blockIdx.z ? ly.v : ly.k) + ((int64_t)blockIdx.x * a.cap + pos) * a.row_bytes;
    float* scales = blockIdx.z ? ly.vs : ly.ks;
    auto source = [&](int j) { const int r = __ldg(a.rows + j); return r >= 0 && r < a.n ? r : j; };
    uint4 w[PER];
    float s = 0.0f;
    int from = tid;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const int i = p * KEEP_THREADS + tid, j = i / pieces;
        const int r = j < a.n ? source(j) : j;
        if (r != j) w[p] = *reinterpret_cast<const uint4*>(base + (int64_t)r * a.row_bytes + 16 * (i - j * pieces));
    }
    if (scales != nullptr) {
        scales += (int64_t)blockIdx.x * a.cap + pos;
        if (tid < a.n) {
            from = source(tid);
            s = scales[from];
        }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const int i = p * KEEP_THREADS + tid, j = i / pieces;
        if (j < a.n && source(j) != j) *reinterpret_cast<uint4*>(base + (int64_t)j * a.row_bytes + 16 * (i - j * pieces)) = w[p];
    }
    if (scales != nullptr && tid < a.n && from != tid) scales[tid] = s;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace scmx

using namespace scmx;

extern "C" int scmx_kv_append(const uint16_t* k, int64_t k_head_stride, int64_t k_row_stride, const uint16_t* v, int64_t v_head_stride,
                              int64_t v_row_stride, int64_t L, int hk, int d, int64_t pos, const int32_t* pos_dev, int64_t capacity, int8_t* k_codes,
                              float* k_scales, int8_t* v_codes, float* v_scales, void* stream) {
    SCMX_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, SCMX_EINVAL, "kv_append: head size %d (a multiple of 16 up to 256)", d);
    SCMX_REQUIRE(hk > 0 && L >= 0 && L < (1ll << 31) && capacity >= 1, SCMX_EINVAL, "kv_append: L=%lld hk=%d capacity=%lld", (long long)L, hk, (long long)capacity);
    SCMX_REQUIRE(pos_dev != nullptr || (pos >= 0 && pos + L <= capacity), SCMX_EINVAL, "kv_append: rows %lld .. %lld of a cache of %lld", (long long)pos,
                 (long long)(pos + L), (long long)capacity);
    if (L == 0) return SCMX_OK;      // (tensors of no elements have no address)
    SCMX_REQUIRE(k && v && k_codes && k_scales && v_codes && v_scales, SCMX_EINVAL, "kv_append: null buffer");
    SCMX_REQUIRE(k_head_stride % 8 == 0 && k_row_stride % 8 == 0 && v_head_stride % 8 == 0 && v_row_stride % 8 == 0 && aligned16(k) && aligned16(v) &&
                     aligned16(k_codes) && aligned16(v_codes), SCMX_EINVAL, "kv_append: vectors must start on 16-byte boundaries");
    KvWriteArgs a;
    a.k = k; a.v = v; a.k_hs = k_head_stride; a.v_hs = v_head_stride; a.k_rs = k_row_stride; a.v_rs = v_row_stride;
    a.kc = k_codes; a.vc = v_codes; a.ks = k_scales; a.vs = v_scales;
    a.pos_dev = pos_dev; a.pos = pos; a.cap = capacity; a.L = (int)L; a.hk = hk; a.d = d;
    const int G = d <= 16 ? 2 : d <= 32 ? 4 : d <= 64 ? 8 : d <= 128 ? 16 : 32;
    void (*kern)(KvWriteArgs) = G == 2 ? kv_append_kernel<2> : G == 4 ? kv_append_kernel<4> : G == 8 ? kv_append_kernel<8> : G == 16 ? kv_append_kernel<16>
                                                                                                                               : kv_append_kernel<32>;
    const int per = KV_THREADS / G * KV_TURNS;
    SCMX_PDL_OK("kv_append_kernel", launch_pdl(kern, dim3((unsigned)((L + per - 1) / per), (unsigned)(hk < 65535 ? hk : 65535), 2), dim3(KV_THREADS), 0,
                                               (cudaStream_t)stream, a));
    return SCMX_OK;
}

extern "C" int scmx_kv_read(const int8_t* k_codes, const float* k_scales, const int8_t* v_codes, const float* v_scales, int64_t start, int64_t n, int hk, int d,
                            int64_t capacity, uint16_t* k, uint16_t* v, void* stream) {
    SCMX_REQUIRE(hk > 0 && n >= 0 && start >= 0 && start + n <= capacity, SCMX_EINVAL, "kv_read: rows %lld .. %lld of a cache of %lld", (long long)start,
                 (long long)(start + n), (long long)capacity);
    SCMX_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, SCMX_EINVAL, "kv_read: head size %d (a multiple of 16 up to 256)", d);
    if (n == 0) return SCMX_OK;
    SCMX_REQUIRE(k && v && k_codes && k_scales && v_codes && v_scales, SCMX_EINVAL, "kv_read: null buffer");
    SCMX_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 32 == 0 && aligned16(k_codes) && aligned16(v_codes), SCMX_EINVAL,
                 "kv_read: codes must be 16-byte aligned, outputs 32-byte");
    KvReadArgs a;
    a.kc = k_codes; a.vc = v_codes; a.ks = k_scales; a.vs = v_scales; a.k = k; a.v = v;
    a.start = start; a.cap = capacity; a.n = n; a.hk = hk; a.d = d; a.pieces = d / 16; a.rows = KV_THREADS / a.pieces;
    const int64_t blocks = (n + a.rows * KV_TURNS - 1) / (a.rows * KV_TURNS);
    SCMX_REQUIRE(blocks < (1ll << 31), SCMX_ELIMIT, "kv_read: %lld rows", (long long)n);
    SCMX_PDL_OK("kv_read_kernel", launch_pdl(kv_read_kernel, dim3((unsigned)blocks, (unsigned)(hk < 65535 ? hk : 65535), 2), dim3(KV_THREADS), 0,
                                             (cudaStream_t)stream, a));
    return SCMX_OK;
}

extern "C" int scmx_kv_keep(const scmx_kv_layer* layers, int n_layers, const int32_t* rows, int n, int64_t pos, const int32_t* pos_dev, int hk, int d,
                            int64_t capacity, int int8, void* stream) {
    SCMX_REQUIRE(n_layers >= 0 && (n_layers == 0 || layers != nullptr) && rows, SCMX_EINVAL, "kv_keep: %d layers", n_layers);
    SCMX_REQUIRE(n >= 1 && n <= KEEP_ROWS, SCMX_ELIMIT, "kv_keep: %d rows (1 .. %d)", n, KEEP_ROWS);
    SCMX_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, SCMX_EINVAL, "kv_keep: head size %d (a multiple of 16 up to 256)", d);
    SCMX_REQUIRE(hk > 0 && capacity >= n && (pos_dev != nullptr || (pos >= 0 && pos + n <= capacity)), SCMX_EINVAL, "kv_keep: rows %lld .. %lld of a cache of %lld",
                 (long long)pos, (long long)(pos + n), (long long)capacity);
    for (int i = 0; i < n_layers; ++i)
        SCMX_REQUIRE(layers[i].k && layers[i].v && aligned16(layers[i].k) && aligned16(layers[i].v) && (!int8 || (layers[i].ks && layers[i].vs)), SCMX_EINVAL,
                     "kv_keep: layer %d: null or unaligned buffer", i);
    KvKeepArgs a;
    a.rows = rows; a.pos_dev = pos_dev; a.pos = pos; a.cap = capacity; a.n = n; a.row_bytes = int8 ? d : 2 * d;
    for (int i0 = 0; i0 < n_layers; i0 += KEEP_LAYERS) {
        const int m = n_layers - i0 < KEEP_LAYERS ? n_layers - i0 : KEEP_LAYERS;
        for (int i = 0; i < m; ++i) {
            a.layer[i] = layers[i0 + i];
            if (!int8) a.layer[i].ks = a.layer[i].vs = nullptr;
        }
        SCMX_PDL_OK("kv_keep_kernel", launch_pdl(kv_keep_kernel, dim3((unsigned)hk, (unsigned)m, 2), dim3(KEEP_THREADS), 0, (cudaStream_t)stream, a));
    }
    return SCMX_OK;
}

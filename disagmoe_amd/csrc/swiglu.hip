// The gradient of the gated activation h = g s p, s = 1 / (1 + exp(-g)) (g: gate, p: up), on the fp32 sums [g | p] that
// the product has kept:
//
//   dp = dh g s,   dg = dh p s (1 + g (1 - s))
//
// Bound by memory: 10 bytes read and 4 written per element of h.  The sums are kept in 32 bits because their rounding to
// bf16 would reach both gradients that are taken of du (relative error of dx and dW 3.1e-3 instead of 2.3e-3, of which
// 1.7e-3 is their own rounding).  du is rounded once, to feed the matrix cores.  The rows behind the last expert's belong
// to nobody: the gradient of the block's input is zero there, du is left as it is.  A lane takes 8 columns, so that every
// access is whole 16-byte vectors (5 loads in flight, 2 stores).  Measured: 8192 rows of 14336: 288 us = 5.7 TB/s of the
// 1.64 GB; 49152 of 1408: 169 us, 5.7 TB/s.  zero_behind_kernel with nothing behind: 2 - 5 us, a launch.
#include "common.h"

namespace dmoe {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kSwThreads = 256;

// Rows that belong to an expert: the sum of the sizes, at most `rows` (the same value in every lane of a wavefront).
__device__ __forceinline__ int64_t rows_in_use(const int64_t *batch_sizes, int E, int64_t rows) {
    int64_t n = 0;
    for (int e = lane_id(); e < E; e += kWave) {
        const int64_t v = batch_sizes[e];
        n += v < 0 ? 0 : (v > rows ? rows : v);
    }
#pragma unroll
    for (int s = kWave / 2; s > 0; s >>= 1) n += __shfl_xor(n, s, kWave);
    return n < rows ? n : rows;
}

// Zeros in the rows [used, rows) of c.
__device__ __forceinline__ void zero_rows(u32x4 *__restrict__ c, int64_t used, int64_t rows, int64_t vecs) {
    for (int64_t i = used * vecs + (int64_t)blockIdx.x * kSwThreads + threadIdx.x; i < rows * vecs; i += (int64_t)gridDim.x * kSwThreads)
        c[i] = u32x4{0, 0, 0, 0};
}

__global__ __launch_bounds__(kSwThreads) void swiglu_backward_kernel(const u32x4 *__restrict__ dh, const f32x4 *__restrict__ u,
                                                                    u32x4 *__restrict__ du, const int64_t *__restrict__ batch_sizes,
                                                                    int E, int64_t rows, int vecs, u32x4 *__restrict__ da, int64_t da_vecs) {
    const int64_t used = rows_in_use(batch_sizes, E, rows), items = used * vecs;
    if (da != nullptr) zero_rows(da, used, rows, da_vecs);
    for (int64_t i = (int64_t)blockIdx.x * kSwThreads + threadIdx.x; i < items; i += (int64_t)gridDim.x * kSwThreads) {
        const int64_t r = i / vecs;
        const int64_t at = r * 2 * vecs + (i - r * vecs);
        const u32x4 d = __builtin_nontemporal_load(dh + i);
        f32x4 g[2], p[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            g[y] = __builtin_nontemporal_load(u + 2 * at + y);
            p[y] = __builtin_nontemporal_load(u + 2 * (at + vecs) + y);
        }
        u32x4 dg, dp;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float og[2], op[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const float dv = y ? __uint_as_float(d[x] & 0xffff0000u) : __uint_as_float(d[x] << 16);
                const float gv = g[x / 2][2 * (x & 1) + y], pv = p[x / 2][2 * (x & 1) + y];
                const float s = __builtin_amdgcn_rcpf(1.f + __expf(-gv));
                const float ds = dv * s;
                op[y] = ds * gv;
                og[y] = ds * pv * (1.f + gv * (1.f - s));
            }
            dg[x] = pack_bf16x2(og[0], og[1]);
            dp[x] = pack_bf16x2(op[0], op[1]);
        }
        du[at] = dg;
        du[at + vecs] = dp;
    }
}

__global__ __launch_bounds__(kSwThreads) void zero_behind_kernel(u32x4 *__restrict__ c, const int64_t *__restrict__ batch_sizes,
                                                                int E, int64_t rows, int64_t vecs) {
    zero_rows(c, rows_in_use(batch_sizes, E, rows), rows, vecs);
}

static int check_rows_of(const char *who, const int64_t *batch_sizes, int64_t rows, int E, int64_t I) {
    DMOE_REQUIRE(rows >= 0 && rows < (1ll << 31), DMOE_ERR_SHAPE, "%s: rows=%lld outside [0, 2^31)", who, (long long)rows);
    DMOE_REQUIRE(E > 0 && E <= 1024, DMOE_ERR_SHAPE, "%s: E=%d outside [1, 1024]", who, E);
    DMOE_REQUIRE(I > 0 && I < (1ll << 23) && I % 8 == 0, DMOE_ERR_SHAPE, "%s: rows of %lld elements must be a positive multiple of 8",
                 who, (long long)I);
    DMOE_REQUIRE(batch_sizes != nullptr, DMOE_ERR_ARG, "%s: null pointer", who);
    return DMOE_OK;
}

static unsigned blocks_of(int64_t vectors) {
    const int64_t want = (vectors + kSwThreads - 1) / kSwThreads, most = (int64_t)device_cus() * 16;
    return (unsigned)(want < most ? want : most);
}

int launch_swiglu_backward(const void *dh, const float *u, void *du, const int64_t *batch_sizes, int64_t rows, int E, int64_t I,
                           void *da, int64_t K, hipStream_t stream) {
    hipLaunchKernelGGL(swiglu_backward_kernel, dim3(blocks_of(rows * (I / 8))), dim3(kSwThreads), 0, stream, (const u32x4 *)dh,
                       (const f32x4 *)u, (u32x4 *)du, batch_sizes, E, rows, (int)(I / 8), (u32x4 *)da, K / 8);
    DMOE_LAUNCH_CHECK("swiglu_backward_kernel");
    return DMOE_OK;
}

}  // namespace dmoe

using namespace dmoe;

extern "C" int dmoe_zero_rows_behind(void *c, const int64_t *batch_sizes, int64_t rows, int E, int64_t d, int dtype, void *stream) {
    DMOE_REQUIRE(dtype == DMOE_BF16 || dtype == DMOE_FP16, DMOE_ERR_DTYPE, "dmoe_zero_rows_behind: dtype %d", dtype);
    const int rc = check_rows_of("dmoe_zero_rows_behind", batch_sizes, rows, E, d);
    if (rc != DMOE_OK) return rc;
    if (rows == 0) return DMOE_OK;
    DMOE_REQUIRE(c != nullptr && ((uintptr_t)c & 15) == 0, DMOE_ERR_ARG, "dmoe_zero_rows_behind: null or unaligned pointer");
    // (most often there is nothing to do: one workgroup per compute unit finds out soonest)
    const unsigned blocks = blocks_of(rows * (d / 8)), cus = (unsigned)device_cus();
    hipLaunchKernelGGL(zero_behind_kernel, dim3(blocks < cus ? blocks : cus), dim3(kSwThreads), 0, (hipStream_t)stream,
                       (u32x4 *)c, batch_sizes, E, rows, d / 8);
    DMOE_LAUNCH_CHECK("zero_behind_kernel");
    return DMOE_OK;
}

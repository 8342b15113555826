// 4-bit weights: quantisation, the way back to bf16, and which form of the product a launch takes (w4.h).
#include "w4.h"

namespace dmoe {

// One wavefront packs one tile: lane 16 g + r holds the 32 weights of column r at k = 32 j + 8 g + i, which a group's
// lanes (4 per column) share the extremes of.  Without zero points s = max |w| / 7 and q = round(w / s) + 8; with them
// s = (max(w, 0) - min(w, 0)) / 15 and z = round(-min(w, 0) / s), so that a weight of zero stays one.  s is rounded to
// bf16 first and the codes follow the rounded one.  Bound by its scattered 2-byte reads; weights are packed once.
__global__ __launch_bounds__(kWave) void w4_quant_kernel(const uint16_t *__restrict__ w, char *__restrict__ codes, uint16_t *__restrict__ scales,
                                                        uint8_t *__restrict__ zeros, int K, int N, int nt, int kt, int group) {
    const int lane = lane_id(), r = lane & 15, g16 = lane >> 4;
    const int64_t tile = blockIdx.x;
    const int c = (int)(tile % kt);
    const int64_t et = tile / kt;
    const int n = (int)(et % nt) * kW4Cols + r;
    const uint16_t *we = w + (et / nt) * K * N;
    float v[4][8], lo[4], hi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        lo[j] = hi[j] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = c * kW4Chunk + j * 32 + g16 * 8 + i;
            v[j][i] = n < N && k < K ? bf16_to_f32(we[(int64_t)k * N + n]) : 0.f;
            lo[j] = fminf(lo[j], v[j][i]);
            hi[j] = fmaxf(hi[j], v[j][i]);
        }
#pragma unroll
        for (int s = 16; s < kWave; s <<= 1) {                 // the 4 lanes of a column
            lo[j] = fminf(lo[j], __shfl_xor(lo[j], s, kWave));
            hi[j] = fmaxf(hi[j], __shfl_xor(hi[j], s, kWave));
        }
    }
    const int steps = group / 32;                              // k-steps that share a scale
    if (steps > 1) {
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
            if (s >= steps) continue;
            float l2[4], h2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { l2[j] = fminf(lo[j], lo[j ^ s]); h2[j] = fmaxf(hi[j], hi[j ^ s]); }
#pragma unroll
            for (int j = 0; j < 4; ++j) { lo[j] = l2[j]; hi[j] = h2[j]; }
        }
    }
    uint32_t words[4];
    const int ng = kW4Chunk / group;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float s = zeros != nullptr ? (hi[j] - lo[j]) / 15.f : fmaxf(hi[j], -lo[j]) / 7.f;
        const uint16_t bits = f32_to_bf16(s);
        s = bf16_to_f32(bits);
        const float inv = s > 0.f ? 1.f / s : 0.f;
        const float z = zeros != nullptr ? fminf(15.f, rintf(-lo[j] * inv)) : 8.f;
        words[j] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = fminf(15.f, fmaxf(0.f, rintf(v[j][i] * inv) + z));
            words[j] |= (uint32_t)q << (4 * ((i >> 1) + 4 * (i & 1)));
        }
        if (j % steps == 0 && g16 == 0) {
            const int64_t at = tile * (kW4Cols * ng) + (r >> 2) * (ng * 4) + (j / steps) * 4 + (r & 3);
            const bool there = n < N && c * kW4Chunk + j * 32 < K;
            scales[at] = there ? bits : 0;
            if (zeros != nullptr) zeros[at] = there ? (uint8_t)z : 0;
        }
    }
    // columns and k past the end have code 0 and scale 0
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n >= N || c * kW4Chunk + j * 32 + g16 * 8 >= K) words[j] = 0;
    *(u32x4 *)(codes + tile * kW4TileBytes + lane * 16) = u32x4{words[0], words[1], words[2], words[3]};
}

// out [E, N, K] = (q - z) s, rounded once to bf16; a wavefront takes tiles of one run of columns.  Only the experts that
// have rows, if batch_sizes is given.
__global__ __launch_bounds__(256) void w4_dequant_kernel(const char *__restrict__ codes, const char *__restrict__ scales, const char *__restrict__ zeros,
                                                        uint16_t *__restrict__ out, const int64_t *__restrict__ batch_sizes, int K, int N,
                                                        int nt, int kt, int group) {
    const int lane = lane_id(), r = lane & 15, g16 = lane >> 4;
    const int e = blockIdx.z;
    if (batch_sizes != nullptr && batch_sizes[e] <= 0) return;
    const int c = blockIdx.x * 4 + threadIdx.x / kWave, t = blockIdx.y;
    const int n = t * kW4Cols + r;
    if (c >= kt || n >= N) return;
    const int64_t tile = ((int64_t)e * nt + t) * kt + c;
    const u32x4 q = *(const u32x4 *)(codes + tile * kW4TileBytes + lane * 16);
    const int ng = kW4Chunk / group;
    uint16_t *row = out + ((int64_t)e * N + n) * K;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int k = c * kW4Chunk + j * 32 + g16 * 8;
        if (k >= K) continue;
        const int64_t at = tile * (kW4Cols * ng) + (r >> 2) * (ng * 4) + (j * 32 / group) * 4 + (r & 3);
        const float s = bf16_to_f32(((const uint16_t *)scales)[at]);
        const float z = zeros != nullptr ? (float)((const uint8_t *)zeros)[at] : 8.f;
        u32x4 v;
#pragma unroll
        for (int p = 0; p < 4; ++p)
            v[p] = pack_bf16x2(((float)((q[j] >> (4 * p)) & 15u) - z) * s, ((float)((q[j] >> (4 * p + 16)) & 15u) - z) * s);
        *(u32x4 *)(row + k) = v;
    }
}

static int check_w4(const char *who, int E, int64_t K, int64_t N, int group) {
    DMOE_REQUIRE(E > 0 && E <= kMaxGroups, DMOE_ERR_SHAPE, "%s: E=%d outside [1, %d]", who, E, kMaxGroups);
    DMOE_REQUIRE(K > 0 && K < (1ll << 22) && K % 8 == 0, DMOE_ERR_SHAPE, "%s: K=%lld must be a positive multiple of 8", who, (long long)K);
    DMOE_REQUIRE(N > 0 && N < (1ll << 20) && N % 8 == 0, DMOE_ERR_SHAPE, "%s: N=%lld must be a positive multiple of 8 below 2^20", who, (long long)N);
    DMOE_REQUIRE(group == 32 || group == 64 || group == 128, DMOE_ERR_ARG, "%s: groups of %d (32, 64 or 128)", who, group);
    return DMOE_OK;
}

static bool aligned(const void *p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

static int tiles_of(int64_t n, int tile) { return (int)((n + tile - 1) / tile); }

struct W4Form {
    bool wide;        // through bf16 weights and the bf16 product
    int tile_rows;
    int m_tiles;
};
// Rows per expert decide.  The direct form reads the codes once for every row tile of an expert; past kWideRows rows the
// bf16 product on weights that are written out first is the faster one.
constexpr int kWideRows = 192;
static W4Form choose_w4(int64_t rows, int E, const int64_t *host_sizes) {
    long long busy = E < rows ? E : rows;
    if (host_sizes != nullptr) {
        busy = 0;
        for (int e = 0; e < E; ++e) busy += host_sizes[e] > 0;
    }
    if (busy < 1) busy = 1;
    const long long avg = (rows + busy - 1) / busy;
    W4Form f;
    f.wide = avg > kWideRows;
    f.tile_rows = avg <= 16 ? 16 : (avg <= 32 ? 32 : 64);
    // row tiles: those of the sizes, or at most one short one for every expert with rows
    long long m = rows / f.tile_rows + (E < rows ? E : rows);
    if (host_sizes != nullptr) {
        long long left = rows;
        m = 0;
        for (int e = 0; e < E; ++e) {
            long long n = host_sizes[e] < 0 ? 0 : host_sizes[e];
            if (n > left) n = left;
            left -= n;
            m += (n + f.tile_rows - 1) / f.tile_rows;
        }
    }
    f.m_tiles = (int)(m > 0 ? m : 1);
    return f;
}

static int gmm_w4(const char *who, const void *a, const void *codes, const void *scales, const void *zeros, int group, void *c,
                  const int64_t *batch_sizes, int64_t rows, int E, int64_t K, int64_t n_out, bool swiglu, void *wide, size_t wide_bytes,
                  void *state, void *workspace, size_t workspace_bytes, const int64_t *host_batch_sizes, void *stream) {
    const int64_t N = swiglu ? 2 * n_out : n_out;
    DMOE_REQUIRE(n_out % 8 == 0, DMOE_ERR_SHAPE, "%s: %lld columns must be a multiple of 8", who, (long long)n_out);
    int rc = check_w4(who, E, K, N, group);
    if (rc != DMOE_OK) return rc;
    DMOE_REQUIRE(rows >= 0 && rows < (1ll << 31), DMOE_ERR_SHAPE, "%s: rows=%lld outside [0, 2^31)", who, (long long)rows);
    DMOE_REQUIRE(batch_sizes != nullptr && codes != nullptr && scales != nullptr, DMOE_ERR_ARG, "%s: null pointer", who);
    DMOE_REQUIRE(rows == 0 || (a != nullptr && c != nullptr), DMOE_ERR_ARG, "%s: null pointer", who);
    DMOE_REQUIRE(aligned(a, 16) && aligned(codes, 16) && aligned(scales, 16) && aligned(zeros, 16) && aligned(c, 16) && aligned(wide, 16),
                 DMOE_ERR_ARG, "%s: a pointer is not 16-byte aligned", who);
    if (rows == 0) return DMOE_OK;
    const W4Form f = choose_w4(rows, E, host_batch_sizes);
    if (f.wide && wide != nullptr && wide_bytes >= (size_t)E * N * K * 2) {
        rc = dmoe_w4_dequant(codes, scales, zeros, group, wide, batch_sizes, E, K, N, stream);
        if (rc != DMOE_OK) return rc;
        return swiglu ? dmoe_gmm_swiglu(a, wide, c, batch_sizes, rows, E, K, n_out, 1, DMOE_BF16, state, workspace, workspace_bytes, host_batch_sizes, stream)
                      : dmoe_gmm(a, wide, c, batch_sizes, rows, E, K, N, 1, DMOE_BF16, state, workspace, workspace_bytes, host_batch_sizes, stream);
    }
    W4Args args{(const char *)a, (const char *)codes, (const char *)scales, (const char *)zeros, (char *)c, batch_sizes, rows, E, (int)K, (int)N,
                (int)n_out, tiles_of(N, kW4Cols), tiles_of(K, kW4Chunk), f.m_tiles};
    if (f.tile_rows == 16) return launch_w4_16(args, group, swiglu, (hipStream_t)stream);
    if (f.tile_rows == 32) return launch_w4_32(args, group, swiglu, (hipStream_t)stream);
    return launch_w4_64(args, group, swiglu, (hipStream_t)stream);
}

}  // namespace dmoe

using namespace dmoe;

extern "C" int dmoe_w4_bytes(int E, int64_t K, int64_t N, int group, size_t *code_bytes, size_t *scale_bytes, size_t *zero_bytes) {
    const int rc = check_w4("dmoe_w4_bytes", E, K, N, group);
    if (rc != DMOE_OK) return rc;
    DMOE_REQUIRE(code_bytes && scale_bytes && zero_bytes, DMOE_ERR_ARG, "dmoe_w4_bytes: null output");
    const size_t tiles = (size_t)E * tiles_of(N, kW4Cols) * tiles_of(K, kW4Chunk);
    *code_bytes = tiles * kW4TileBytes;
    *zero_bytes = tiles * kW4Cols * (kW4Chunk / group);
    *scale_bytes = *zero_bytes * 2;
    return DMOE_OK;
}

extern "C" int dmoe_w4_quant(const void *w, int E, int64_t K, int64_t N, int group, void *codes, void *scales, void *zeros, void *stream) {
    const int rc = check_w4("dmoe_w4_quant", E, K, N, group);
    if (rc != DMOE_OK) return rc;
    DMOE_REQUIRE(w && codes && scales, DMOE_ERR_ARG, "dmoe_w4_quant: null pointer");
    DMOE_REQUIRE(aligned(codes, 16) && aligned(scales, 16), DMOE_ERR_ARG, "dmoe_w4_quant: a pointer is not 16-byte aligned");
    const int nt = tiles_of(N, kW4Cols), kt = tiles_of(K, kW4Chunk);
    const long long tiles = (long long)E * nt * kt;
    DMOE_REQUIRE(tiles < (1ll << 31), DMOE_ERR_SHAPE, "dmoe_w4_quant: %lld tiles", tiles);
    hipLaunchKernelGGL(w4_quant_kernel, dim3((unsigned)tiles), dim3(kWave), 0, (hipStream_t)stream, (const uint16_t *)w, (char *)codes,
                       (uint16_t *)scales, (uint8_t *)zeros, (int)K, (int)N, nt, kt, group);
    DMOE_LAUNCH_CHECK("w4_quant_kernel");
    return DMOE_OK;
}

extern "C" int dmoe_w4_dequant(const void *codes, const void *scales, const void *zeros, int group, void *out, const int64_t *batch_sizes,
                               int E, int64_t K, int64_t N, void *stream) {
    const int rc = check_w4("dmoe_w4_dequant", E, K, N, group);
    if (rc != DMOE_OK) return rc;
    DMOE_REQUIRE(codes && scales && out, DMOE_ERR_ARG, "dmoe_w4_dequant: null pointer");
    DMOE_REQUIRE(aligned(codes, 16) && aligned(scales, 16) && aligned(out, 16), DMOE_ERR_ARG, "dmoe_w4_dequant: a pointer is not 16-byte aligned");
    const int nt = tiles_of(N, kW4Cols), kt = tiles_of(K, kW4Chunk);
    DMOE_REQUIRE(nt < 65536, DMOE_ERR_SHAPE, "dmoe_w4_dequant: N=%lld", (long long)N);
    hipLaunchKernelGGL(w4_dequant_kernel, dim3((kt + 3) / 4, nt, E), dim3(256), 0, (hipStream_t)stream, (const char *)codes, (const char *)scales,
                       (const char *)zeros, (uint16_t *)out, batch_sizes, (int)K, (int)N, nt, kt, group);
    DMOE_LAUNCH_CHECK("w4_dequant_kernel");
    return DMOE_OK;
}

extern "C" int dmoe_gmm_w4_wide_bytes(int64_t rows, int E, int64_t K, int64_t N, const int64_t *host_batch_sizes, size_t *bytes) {
    const int rc = check_w4("dmoe_gmm_w4_wide_bytes", E, K, N, 128);
    if (rc != DMOE_OK) return rc;
    DMOE_REQUIRE(bytes != nullptr && rows >= 0 && rows < (1ll << 31), DMOE_ERR_ARG, "dmoe_gmm_w4_wide_bytes: bad rows or null output");
    *bytes = choose_w4(rows, E, host_batch_sizes).wide ? (size_t)E * N * K * 2 : 0;
    return DMOE_OK;
}

extern "C" int dmoe_gmm_w4(const void *a, const void *codes, const void *scales, const void *zeros, int group, void *c,
                           const int64_t *batch_sizes, int64_t rows, int E, int64_t K, int64_t N, void *wide, size_t wide_bytes,
                           void *state, void *workspace, size_t workspace_bytes, const int64_t *host_batch_sizes, void *stream) {
    return gmm_w4("dmoe_gmm_w4", a, codes, scales, zeros, group, c, batch_sizes, rows, E, K, N, false, wide, wide_bytes, state, workspace,
                  workspace_bytes, host_batch_sizes, stream);
}

extern "C" int dmoe_gmm_w4_swiglu(const void *a, const void *codes, const void *scales, const void *zeros, int group, void *h,
                                  const int64_t *batch_sizes, int64_t rows, int E, int64_t K, int64_t I, void *wide, size_t wide_bytes,
                                  void *state, void *workspace, size_t workspace_bytes, const int64_t *host_batch_sizes, void *stream) {
    return gmm_w4("dmoe_gmm_w4_swiglu", a, codes, scales, zeros, group, h, batch_sizes, rows, E, K, I, true, wide, wide_bytes, state, workspace,
                  workspace_bytes, host_batch_sizes, stream);
}

// Grouped products on 4-bit weights with a scale (and a zero point) for every group of 32, 64 or 128 k of a column.
//
//   c[r, n] = sum_k x[r, k] w[n, k],   w[n, k] = (q[n, k] - z[n, k / G]) s[n, k / G]
//
// Decode-sized batches are bound by the weights' bytes, N K / 2 + N K / G (2 or 3) per expert that has rows, so what
// matters is that they stream and that a byte costs few instructions:
//
//   * the codes lie in tiles of 16 columns x 128 k, 1 KiB that a wavefront loads with one 16-byte instruction; lane
//     16 g + r gets column r, its word j the 8 codes of k = 32 j + 8 g ..: an operand of v_mfma_f32_16x16x32_bf16;
//   * a code becomes a bf16 without a conversion: bf16 16.0 has its units at bit 3, so nibble << 3 | 0x4180 is 16 + q
//     exactly, two codes for one shift and one and-or.  The sum over a group then needs 16 + z times the group's sum of
//     x taken off, which one more matrix instruction per k-step gives (weights of 1) to every lane that needs it:
//         c += s (sum (16 + q) x - (16 + z) sum x)
//     once for a group and four results a lane.  The weights are never rounded; the price is a sum whose terms are up to
//     31 instead of 15 times |x|, some two bits of the 24 that fp32 holds;
//   * the wavefronts of a workgroup split k (chunk c goes to wavefront c mod WK, so that they read a contiguous stretch
//     together) and meet in LDS, where the sums are added in the order of the wavefronts: many bytes in flight on a
//     matrix of few columns, no atomics, the same bits every time.
#pragma once
#include "gmm_common.h"

namespace dmoe {

constexpr int kW4Chunk = 128;                 // k of a tile
constexpr int kW4Cols = 16;                   // columns of a tile
constexpr int kW4TileBytes = 1024;

struct W4Args {
    const char *x;
    const char *codes;                        // [E, nt, kt, 1024]
    const char *scales;                       // bf16 [E, nt, kt, 4, 128 / G, 4]
    const char *zeros;                        // uint8, laid out as the scales, or nullptr (8 everywhere)
    char *c;
    const int64_t *batch_sizes;
    int64_t rows;
    int E;
    int K;
    int N;                                    // columns of an expert's weights (2 I for the gated form)
    int n_out;                                // columns of c
    int nt, kt;                               // tiles of an expert along its columns and along k
    int m_tiles;                              // row tiles of the grid
};

__device__ __forceinline__ uint32_t w4_pair(uint32_t word, int p) {   // 16 + q of nibbles p and p + 4 as two bf16
    const uint32_t v = p == 0 ? word << 3 : word >> (4 * p - 3);
    return (v & 0x00780078u) | 0x41804180u;
}

// Row tile number `m` of all experts' row tiles of BM rows: its expert, first row and rows, and how many row tiles there are
// (without one of that number the other results are left as they are).
template <int BM>
__device__ __forceinline__ int w4_locate(const W4Args &p, int m, int &expert, int &row0, int &rows) {
    const int lane = lane_id();
    long long row_carry = 0;
    int tile_carry = 0;
    for (int e0 = 0; e0 < p.E; e0 += kWave) {
        const int e = e0 + lane;
        long long n = e < p.E ? (long long)p.batch_sizes[e] : 0;
        n = n < 0 ? 0 : (n > p.rows ? p.rows : n);
        long long incl = n;
#pragma unroll
        for (int s = 1; s < kWave; s <<= 1) {
            const long long up = __shfl_up(incl, s, kWave);
            if (lane >= s) incl += up;
        }
        long long start = row_carry + incl - n, end = row_carry + incl;
        start = start > p.rows ? p.rows : start;
        end = end > p.rows ? p.rows : end;
        const int mt = (int)((end - start + BM - 1) / BM);
        int tincl = mt;
#pragma unroll
        for (int s = 1; s < kWave; s <<= 1) {
            const int up = __shfl_up(tincl, s, kWave);
            if (lane >= s) tincl += up;
        }
        const unsigned long long behind = __ballot(tile_carry + tincl > m);
        if (behind != 0 && tile_carry <= m) {
            const int at = __ffsll((unsigned long long)behind) - 1;
            const int in = m - (tile_carry + __shfl(tincl - mt, at, kWave));
            expert = __builtin_amdgcn_readfirstlane(e0 + at);
            row0 = __builtin_amdgcn_readfirstlane((int)__shfl(start, at, kWave) + in * BM);
            const int left = __builtin_amdgcn_readfirstlane((int)__shfl(end, at, kWave)) - row0;
            rows = left < BM ? left : BM;
        }
        row_carry += __shfl(incl, kWave - 1, kWave);
        tile_carry += __shfl(tincl, kWave - 1, kWave);
    }
    return __builtin_amdgcn_readfirstlane(tile_carry);
}

// FM row fragments of 16, FG column fragments of 16 per wavefront (SWIGLU: of the result, with as many of the gate and of
// the up columns; SHIFT: the up columns begin in the middle of a tile, one more), WN wavefronts along the columns, WK
// along k.
template <int FM, int FG, int WN, int WK, int G, bool ZERO, bool SWIGLU, bool SHIFT>
__global__ __launch_bounds__(WN *WK *kWave) void gmm_w4_kernel(const W4Args p) {
    constexpr int BM = 16 * FM;
    constexpr int NF = SWIGLU ? 2 * FG + (SHIFT ? 1 : 0) : FG;
    constexpr int NG = kW4Chunk / G;          // groups of a chunk
    constexpr int SG = G / 32;                // k-steps of a group
    constexpr int BN = 16 * FG * WN;          // columns of the result per workgroup
    constexpr int kPart = NF * BM * 16;       // floats that a wavefront brings to the meeting
    static_assert(!SHIFT || SWIGLU, "only the gated form has two runs of columns");
    extern __shared__ __attribute__((aligned(16))) float red[];

    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wn = wave % WN, wk = wave / WN;
    const int l16 = lane & 15, g16 = lane >> 4;

    // workgroup -> (column tile, row tile): the row tiles of a column tile one after the other on one XCD, whose L2 then
    // holds the column tile's codes
    const int id = blockIdx.x;
    const int oct = id / (kXcds * p.m_tiles), in = id - oct * (kXcds * p.m_tiles);
    const int ntile = oct * kXcds + in % kXcds;
    const int n0 = ntile * BN;
    if (n0 >= p.n_out) return;
    // (one round, unless the grid was laid out for sizes that say less than batch_sizes do)
    for (int m_tile = in / kXcds, total = m_tile + 1; m_tile < total; m_tile += p.m_tiles) {
    int e = 0, row0 = 0, rows = 0;
    total = w4_locate<BM>(p, m_tile, e, row0, rows);
    if (m_tile >= total) break;

    // ---- where this wavefront's fragments lie ----
    const int c0 = n0 + wn * (16 * FG);                       // its first column of the result
    constexpr int kScaleTile = kW4Cols * NG;                  // scales of a tile
    const char *code_at[NF], *scale_at[NF], *zero_at[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
        int t = SWIGLU && f >= FG ? (p.n_out + c0) / 16 + (f - FG) : c0 / 16 + f;
        t = t < p.nt ? t : p.nt - 1;                          // past the end: read, never stored
        const size_t tile = ((size_t)e * p.nt + t) * p.kt;
        code_at[f] = p.codes + tile * kW4TileBytes;
        scale_at[f] = p.scales + tile * (kScaleTile * 2);
        zero_at[f] = ZERO ? p.zeros + tile * kScaleTile : nullptr;
    }
    const char *x_at[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int m = i * 16 + l16;
        x_at[i] = p.x + ((size_t)(row0 + (m < rows ? m : rows - 1)) * p.K + g16 * 8) * 2;   // past the end: the last row
    }

    struct Chunk {
        u32x4 q[NF];
        uint32_t s[NF][NG * 2];
        uint32_t z[ZERO ? NF : 1][NG];
        bf16x8 x[FM][4];
    };
    const int whole = p.K / kW4Chunk;                         // chunks that lie inside K
    auto load = [&](Chunk &b, int c) {
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            b.q[f] = *(const u32x4 *)(code_at[f] + (uint32_t)c * kW4TileBytes + lane * 16);
            __builtin_memcpy(b.s[f], scale_at[f] + (uint32_t)c * (kScaleTile * 2) + g16 * (NG * 8), NG * 8);
            if constexpr (ZERO) __builtin_memcpy(b.z[f], zero_at[f] + (uint32_t)c * kScaleTile + g16 * (NG * 4), NG * 4);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u32x4 v = {0, 0, 0, 0};
                if (c < whole || c * kW4Chunk + j * 32 + g16 * 8 < p.K) v = *(const u32x4 *)(x_at[i] + (uint32_t)c * (kW4Chunk * 2) + j * 64);
                __builtin_memcpy(&b.x[i][j], &v, 16);
            }
    };

    f32x4 acc[NF][FM];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[f][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u32x4 one_bits = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    bf16x8 ones;
    __builtin_memcpy(&ones, &one_bits, 16);

    auto compute = [&](const Chunk &b) {
        float xs[FM][NG];                                     // the groups' sums of x in this lane's row
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = g * SG; j < (g + 1) * SG; ++j) t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, b.x[i][j], t, 0, 0, 0);
                xs[i][g] = ZERO ? t[0] : t[0] * 24.f;         // (no zero points: 16 + 8)
            }
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                f32x4 t[FM];
#pragma unroll
                for (int j = g * SG; j < (g + 1) * SG; ++j) {
                    u32x4 w;
#pragma unroll
                    for (int q = 0; q < 4; ++q) w[q] = w4_pair(b.q[f][j], q);
                    bf16x8 wf;
                    __builtin_memcpy(&wf, &w, 16);
#pragma unroll
                    for (int i = 0; i < FM; ++i)
                        t[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, b.x[i][j], j == g * SG ? f32x4{0.f, 0.f, 0.f, 0.f} : t[i], 0, 0, 0);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t pair = b.s[f][g * 2 + x / 2];
                    const float s = __uint_as_float(x & 1 ? pair & 0xffff0000u : pair << 16);
                    const float off = ZERO ? 16.f + (float)((b.z[ZERO ? f : 0][g] >> (8 * x)) & 0xffu) : 0.f;
#pragma unroll
                    for (int i = 0; i < FM; ++i)
                        acc[f][i][x] = fmaf(s, ZERO ? fmaf(-off, xs[i][g], t[i][x]) : t[i][x] - xs[i][g], acc[f][i][x]);
                }
            }
    };

    // one chunk ahead: the next one's loads are on their way while this one is worked on
    Chunk even, odd;
    int c = wk;
    if (c < p.kt) load(even, c);
    for (; c < p.kt; c += 2 * WK) {
        if (c + WK < p.kt) load(odd, c + WK);
        compute(even);
        if (c + 2 * WK < p.kt) load(even, c + 2 * WK);
        if (c + WK < p.kt) compute(odd);
    }

    // ---- the wavefronts that split k meet: red[wk][wn][fragment][row][16 columns] ----
    float *mine = red + (wk * WN + wn) * kPart;
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int i = 0; i < FM; ++i) *(f32x4 *)(mine + (f * BM + i * 16 + l16) * 16 + g16 * 4) = acc[f][i];
    __syncthreads();
    constexpr int kQuads = BN / 4;
    for (int i = threadIdx.x; i < BM * kQuads; i += WN * WK * kWave) {
        const int m = i / kQuads, col = (i - m * kQuads) * 4;
        if (m >= rows || n0 + col >= p.n_out) continue;       // n_out % 8 == 0: 4 columns at once
        const int w = col / (16 * FG), cw = col - w * (16 * FG);
        auto sum = [&](int f, int at) {
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < WK; ++k) v += *(const f32x4 *)(red + (k * WN + w) * kPart + (f * BM + m) * 16 + at);
            return v;
        };
        f32x4 v = sum(cw / 16, cw % 16);
        if constexpr (SWIGLU) {
            const int uc = cw + (SHIFT ? 8 : 0);
            const f32x4 u = sum(FG + uc / 16, uc % 16);
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = silu_mul(v[x], u[x]);
        }
        uint2 pk;
        pk.x = pack_bf16x2(v[0], v[1]);
        pk.y = pack_bf16x2(v[2], v[3]);
        *(uint2 *)((uint16_t *)p.c + (size_t)(row0 + m) * p.n_out + n0 + col) = pk;
    }
    __syncthreads();                                          // read: the next round may bring its sums
    }
}

template <int FM, int FG, int WN, int WK, int G, bool ZERO, bool SWIGLU, bool SHIFT>
static int launch_w4_one(const W4Args &args, hipStream_t stream) {
    constexpr int NF = SWIGLU ? 2 * FG + (SHIFT ? 1 : 0) : FG;
    constexpr int lds = WN * WK * NF * 16 * FM * 16 * (int)sizeof(float);
    static_assert(lds <= 160 * 1024, "LDS of a compute unit");
    auto kern = gmm_w4_kernel<FM, FG, WN, WK, G, ZERO, SWIGLU, SHIFT>;
    static unsigned long long configured = 0;   // devices on which the kernel's LDS size has been raised
    if (lds > 64 * 1024) DMOE_HIP(raise_dynamic_lds((const void *)kern, lds, &configured));
    const int n_tiles = (args.n_out + 16 * FG * WN - 1) / (16 * FG * WN);
    const long long grid = (long long)((n_tiles + kXcds - 1) / kXcds) * kXcds * args.m_tiles;
    DMOE_REQUIRE(grid < (1ll << 31), DMOE_ERR_SHAPE, "gmm_w4: %lld workgroups", grid);
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(WN * WK * kWave), lds, stream, args);
    DMOE_LAUNCH_CHECK("gmm_w4_kernel");
    return DMOE_OK;
}

template <int FM, int FG, int WN, int WK, int G, bool ZERO>
static int launch_w4_form(const W4Args &args, bool swiglu, hipStream_t stream) {
    if (!swiglu) return launch_w4_one<FM, 2 * FG, WN, WK, G, ZERO, false, false>(args, stream);
    if (args.n_out % 16 == 0) return launch_w4_one<FM, FG, WN, WK, G, ZERO, true, false>(args, stream);
    return launch_w4_one<FM, FG, WN, WK, G, ZERO, true, true>(args, stream);
}

template <int FM, int FG, int WN, int WK>
static int launch_w4_rows(const W4Args &args, int group, bool swiglu, hipStream_t stream) {
    const bool zero = args.zeros != nullptr;
    if (group == 32) return zero ? launch_w4_form<FM, FG, WN, WK, 32, true>(args, swiglu, stream) : launch_w4_form<FM, FG, WN, WK, 32, false>(args, swiglu, stream);
    if (group == 64) return zero ? launch_w4_form<FM, FG, WN, WK, 64, true>(args, swiglu, stream) : launch_w4_form<FM, FG, WN, WK, 64, false>(args, swiglu, stream);
    return zero ? launch_w4_form<FM, FG, WN, WK, 128, true>(args, swiglu, stream) : launch_w4_form<FM, FG, WN, WK, 128, false>(args, swiglu, stream);
}

int launch_w4_16(const W4Args &args, int group, bool swiglu, hipStream_t stream);
int launch_w4_32(const W4Args &args, int group, bool swiglu, hipStream_t stream);
int launch_w4_64(const W4Args &args, int group, bool swiglu, hipStream_t stream);

}  // namespace dmoe

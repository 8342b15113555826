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
//     exactly, two codes for one shift and one and-or.  What that is too much, 16 + z times the group's sum of x, comes
//     from one more matrix instruction per k-step, on weights of -24 (z = 8) or -16: its result is what the sums over the
//     group begin with, so without zero points a group costs one fused multiply-add per result and lane:
//         c += s (sum (16 + q) x - 24 sum x)     or     c += s (sum (16 + q) x - 16 sum x - z sum x)
//     The weights are never rounded; the price is a sum whose terms are up to 31 instead of 15 times |x|, some two bits
//     of the 24 that fp32 holds;
//   * the wavefronts of a workgroup split k (chunk c goes to wavefront c mod WK, so that they read a contiguous stretch
//     together) and meet in LDS, where the sums are added in the order of the wavefronts: many bytes in flight on a
//     matrix of few columns, no atomics, the same bits every time.
//
// Measured (gate-up, 8 experts of 4096 x 28672, unless another is named): one token, 2 experts, groups of 128: 24 us, 5.1 TB/s
// of codes and scales; 16 tokens on the down projection (14336 x 4096), zero points: 43.5 us, 5.7 TB/s (vector units busy
// 65 %); 64 experts of 3 rows, 2048 x 2816, groups of 32, zero points: 56 us, 3.7 TB/s (vector units 77 %: the unpacking is the
// bound); 512 rows on skewed experts, groups of 64: 245 us, 491 TFLOP/s (matrix units 31 %, vector units 47 %: a wavefront's
// two kinds of instruction overlap only in part); 1024 rows an expert, groups of 128: 785 - 815 TFLOP/s.
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
    const int64_t *first;                     // the experts before *first are left out (nullptr: none)
};

// 16 + q of nibbles p and p + 4 as two bf16.  The mask sits in a scalar and the 16s in a vector register: an instruction
// with two literals does not exist, and with them the compiler takes two (`mask`, `bias`: w4_constants).
__device__ __forceinline__ uint32_t w4_pair(uint32_t word, int p, uint32_t mask, uint32_t bias) {
    const uint32_t v = p == 0 ? word << 3 : word >> (4 * p - 3);
    return (v & mask) | bias;
}
struct W4Constants {
    uint32_t mask, bias;
};
__device__ __forceinline__ W4Constants w4_constants() {
    W4Constants k;
    asm("s_mov_b32 %0, 0x00780078" : "=s"(k.mask));
    asm("v_mov_b32 %0, 0x41804180" : "=v"(k.bias));
    return k;
}

// Row tile number `m` of all experts' row tiles of BM rows (of the experts that are not left out): its expert, first row and
// rows, and how many row tiles there are (without one of that number the other results are left as they are).
template <int BM>
__device__ __forceinline__ int w4_locate(const W4Args &p, int m, int &expert, int &row0, int &rows) {
    const int lane = lane_id();
    long long row_carry = 0;
    int tile_carry = 0;
    const int first = p.first != nullptr ? (int)*p.first : 0;
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
        const int mt = e < first ? 0 : (int)((end - start + BM - 1) / BM);
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
            expert = e0 + at;
            row0 = (int)__shfl(start, at, kWave) + in * BM;
            const int left = (int)__shfl(end, at, kWave) - row0;
            rows = left < BM ? left : BM;
        }
        row_carry += __shfl(incl, kWave - 1, kWave);
        tile_carry += __shfl(tincl, kWave - 1, kWave);
    }
    return __builtin_amdgcn_readfirstlane(tile_carry);
}

// What a wavefront holds of one chunk of 128 k: the codes, scales and zero points of its NF fragments of 16 columns.
template <int NF, int NG, bool ZERO>
struct W4Weights {
    u32x4 q[NF];
    uint32_t s[NF][NG * 2];
    uint32_t z[ZERO ? NF : 1][NG];
};
// Where they lie (wave-uniform), and how they are loaded.
template <int NF, int NG, bool ZERO>
struct W4Source {
    const char *code_at[NF], *scale_at[NF], *zero_at[NF];
    static constexpr int kScaleTile = kW4Cols * NG;           // scales of a tile
    __device__ __forceinline__ void aim(const W4Args &p, int f, int e, int t) {
        t = t < p.nt ? t : p.nt - 1;                          // past the end: read, never stored
        const size_t tile = ((size_t)e * p.nt + t) * p.kt;
        code_at[f] = p.codes + tile * kW4TileBytes;
        scale_at[f] = p.scales + tile * (kScaleTile * 2);
        zero_at[f] = ZERO ? p.zeros + tile * kScaleTile : nullptr;
    }
    __device__ __forceinline__ void load_codes(W4Weights<NF, NG, ZERO> &b, int f, int c, int lane) const {
        b.q[f] = *(const u32x4 *)(code_at[f] + ((uint32_t)c * kW4TileBytes + lane * 16));
    }
    __device__ __forceinline__ void load_scales(W4Weights<NF, NG, ZERO> &b, int f, int c, int lane) const {
        __builtin_memcpy(b.s[f], scale_at[f] + ((uint32_t)c * (kScaleTile * 2) + (lane >> 4) * (NG * 8)), NG * 8);
        if constexpr (ZERO) __builtin_memcpy(b.z[f], zero_at[f] + ((uint32_t)c * kScaleTile + (lane >> 4) * (NG * 4)), NG * 4);
    }
    __device__ __forceinline__ void load(W4Weights<NF, NG, ZERO> &b, int c, int lane) const {
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            load_codes(b, f, c, lane);
            load_scales(b, f, c, lane);
        }
    }
};

// acc[f][i] += the products of a chunk's weights with the row fragments x(i, j) of its k-steps j
template <int FM, int NF, int NG, bool ZERO, typename X>
__device__ __forceinline__ void w4_chunk(f32x4 (&acc)[NF][FM], const W4Weights<NF, NG, ZERO> &b, const W4Constants &k, X &&x_of) {
    constexpr int SG = 4 / NG;                                // k-steps of a group
    const uint32_t less = ZERO ? 0xc180c180u : 0xc1c0c1c0u;   // -16 or -24 as two bf16
    const u32x4 less4 = {less, less, less, less};
    bf16x8 lf;
    __builtin_memcpy(&lf, &less4, 16);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        bf16x8 x[FM][SG];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < SG; ++j) x[i][j] = x_of(i, g * SG + j);
        f32x4 base[FM];                                       // -24 (-16) times the group's sum of x in this lane's row
#pragma unroll
        for (int i = 0; i < FM; ++i) base[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = g * SG; j < (g + 1) * SG; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i) base[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lf, x[i][j - g * SG], base[i], 0, 0, 0);
        float less_x[FM];                                     // (ZERO) minus that sum
#pragma unroll
        for (int i = 0; i < FM; ++i) less_x[i] = ZERO ? base[i][0] * 0.0625f : 0.f;
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            f32x4 t[FM];
#pragma unroll
            for (int j = g * SG; j < (g + 1) * SG; ++j) {
                u32x4 w;
#pragma unroll
                for (int q = 0; q < 4; ++q) w[q] = w4_pair(b.q[f][j], q, k.mask, k.bias);
                bf16x8 wf;
                __builtin_memcpy(&wf, &w, 16);
#pragma unroll
                for (int i = 0; i < FM; ++i) t[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, x[i][j - g * SG], j == g * SG ? base[i] : t[i], 0, 0, 0);
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const uint32_t pair = b.s[f][g * 2 + v / 2];
                const float s = __uint_as_float(v & 1 ? pair & 0xffff0000u : pair << 16);
                const float z = ZERO ? (float)((b.z[ZERO ? f : 0][g] >> (8 * v)) & 0xffu) : 0.f;
#pragma unroll
                for (int i = 0; i < FM; ++i) acc[f][i][v] = fmaf(s, ZERO ? fmaf(z, less_x[i], t[i][v]) : t[i][v], acc[f][i][v]);
            }
            __builtin_amdgcn_sched_barrier(0);                // one fragment's sums in registers at a time
        }
    }
}

// The same for tiles of 64 rows of which the first FM * 16 are there, as one pipeline: a matrix instruction occupies its unit
// for 16 cycles and a vector instruction its own for 4, so behind each of the former stand the vector instructions that
// prepare and finish its neighbours: a quarter of the next operand's unpacking, a share of the fold of the fragment before.  A fragment's codes and scales of chunk
// `c_next` are loaded over those of this chunk once they have been used.
template <int FM, int NF, int NG, bool ZERO, typename X>
__device__ __forceinline__ void w4_chunk_64(f32x4 (&acc)[NF][4], W4Weights<NF, NG, ZERO> &b, const W4Source<NF, NG, ZERO> &src, int c_next,
                                            int lane, const W4Constants &k, X &&x_of) {
    constexpr int SG = 4 / NG;                                // k-steps of a group
    constexpr int XB = NG == 1 || ZERO ? 1 : 2;               // groups of x held; the zero points' registers leave room for one
    const uint32_t less = ZERO ? 0xc180c180u : 0xc1c0c1c0u;   // -16 or -24 as two bf16
    const u32x4 less4 = {less, less, less, less};
    bf16x8 lf;
    __builtin_memcpy(&lf, &less4, 16);
    bf16x8 x[XB][SG][FM];
    auto read_x = [&](int g) {
#pragma unroll
        for (int j = 0; j < SG; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i) x[g % XB][j][i] = x_of(i, g * SG + j);
    };
#pragma unroll
    for (int g = 0; g < XB; ++g) read_x(g);
    u32x4 w;
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = w4_pair(b.q[0][0], q, k.mask, k.bias);
    f32x4 t[2][FM], base[FM];
    float less_x[2][FM];                                      // (ZERO) minus the group's sum of x; the group before is still read
    // element v of row fragment i of the sums of (group, fragment) number n
    auto fold = [&](int n, int i, int v) {
        const int g = n / NF, f = n % NF;
        const uint32_t pair = b.s[f][g * 2 + v / 2];
        const float s = __uint_as_float(v & 1 ? pair & 0xffff0000u : pair << 16);
        const float z = ZERO ? (float)((b.z[ZERO ? f : 0][g] >> (8 * v)) & 0xffu) : 0.f;
        acc[f][i][v] = fmaf(s, ZERO ? fmaf(z, less_x[g & 1][i], t[n & 1][i][v]) : t[n & 1][i][v], acc[f][i][v]);
    };
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int j = 0; j < SG; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i)                      // -24 (-16) times the group's sum of x in this lane's row
                base[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lf, x[g % XB][j][i], j == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : base[i], 0, 0, 0);
        if constexpr (ZERO) {
#pragma unroll
            for (int i = 0; i < FM; ++i) less_x[g & 1][i] = base[i][0] * 0.0625f;
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const int n = g * NF + f;
#pragma unroll
            for (int j = 0; j < SG; ++j) {
                // the operand behind this one
                const int fn = j + 1 < SG ? f : (f + 1 < NF ? f + 1 : 0), jn = j + 1 < SG ? g * SG + j + 1 : (f + 1 < NF ? g * SG : (g + 1) * SG);
                const bool more = jn < 4;
                bf16x8 wf;
                __builtin_memcpy(&wf, &w, 16);
                u32x4 wn = w;
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    t[n & 1][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, x[g % XB][j][i], j == 0 ? base[i] : t[n & 1][i], 0, 0, 0);
                    if (more) {
#pragma unroll
                        for (int q = 4 * i / FM; q < 4 * (i + 1) / FM; ++q) wn[q] = w4_pair(b.q[fn][jn], q, k.mask, k.bias);
                    }
                    if (n > 0) {
                        constexpr int kShare = 4 / SG;        // of the 4 FM elements, over SG FM instructions
#pragma unroll
                        for (int u = 0; u < kShare; ++u) {
                            const int at = (j * FM + i) * kShare + u;
                            fold(n - 1, at % FM, at / FM);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                w = wn;
            }
            if (g == NG - 1) {
                src.load_codes(b, f, c_next, lane);
                if (f > 0) src.load_scales(b, f - 1, c_next, lane);
            }
        }
        if (g + XB < NG) read_x(g + XB);
    }
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int i = 0; i < FM; ++i) fold(NG * NF - 1, i, v);
    src.load_scales(b, NF - 1, c_next, lane);
}

// The wavefronts that split k meet: red[wk][wn][fragment][row][16 columns].  Sums in the order of the wavefronts, the
// gated form's activation, one rounding, out by quads of columns.
template <int FM, int FG, int WN, int WK, bool SWIGLU, bool SHIFT, int NF>
__device__ __forceinline__ void w4_finish(const W4Args &p, float *red, const f32x4 (&acc)[NF][FM], int wk, int wn, int row0, int rows, int n0) {
    constexpr int BM = 16 * FM, BN = 16 * FG * WN, kPart = NF * BM * 16;
    const int lane = lane_id(), l16 = lane & 15, g16 = lane >> 4;
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
    __syncthreads();                                          // read: the LDS may be written again
}

// Wavefronts to a SIMD: as many as the registers of the form allow without (many) spills.
constexpr int w4_waves(int FM, int NF) {
    return FM == 1 ? 4 : (FM == 2 && NF <= 4 ? 3 : 2);
}

// FM row fragments of 16, FG column fragments of 16 per wavefront (SWIGLU: of the result, with as many of the gate and of
// the up columns; SHIFT: the up columns begin in the middle of a tile, one more), WN wavefronts along the columns, WK
// along k.  Up to 32 rows (FM 1, 2): the rows come straight from the caches into registers and four (three)
// wavefronts to a SIMD keep loads in flight.  64 rows (FM 4): the sums leave room for two, so weights and rows are fetched a
// round ahead, and all wavefronts bring the WK chunks of a round into LDS, once for the WN wavefronts that read each.
template <int FM, int FG, int WN, int WK, int G, bool ZERO, bool SWIGLU, bool SHIFT>
__global__ __launch_bounds__(WN *WK *kWave) __attribute__((amdgpu_waves_per_eu(w4_waves(FM, SWIGLU ? 2 * FG + (SHIFT ? 1 : 0) : FG))))
void gmm_w4_kernel(const W4Args p) {
    constexpr int BM = 16 * FM;
    constexpr int NF = SWIGLU ? 2 * FG + (SHIFT ? 1 : 0) : FG;
    constexpr int NG = kW4Chunk / G;          // groups of a chunk
    constexpr int BN = 16 * FG * WN;          // columns of the result per workgroup
    constexpr bool kShare = FM > 2;
    static_assert(!SHIFT || SWIGLU, "only the gated form has two runs of columns");
    extern __shared__ __attribute__((aligned(16))) char smem[];

    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wn = wave % WN, wk = wave / WN;
    const int l16 = lane & 15, g16 = lane >> 4;
    const W4Constants consts = w4_constants();

    // workgroup -> (column tile, row tile): the row tiles of a column tile one after the other on one XCD, whose L2 then
    // holds the column tile's codes
    const int id = blockIdx.x;
    const int oct = id / (kXcds * p.m_tiles), in = id - oct * (kXcds * p.m_tiles);
    const int n0 = (oct * kXcds + in % kXcds) * BN;
    if (n0 >= p.n_out) return;
    // (one round, unless the grid was laid out for sizes that say less than batch_sizes do)
    for (int m_tile = in / kXcds, total = m_tile + 1; m_tile < total; m_tile += p.m_tiles) {
        int e = 0, row0 = 0, rows = 0;
        total = w4_locate<BM>(p, m_tile, e, row0, rows);
        if (m_tile >= total) break;
        // (the same in every lane, which the compiler does not see through the search)
        e = __builtin_amdgcn_readfirstlane(e); row0 = __builtin_amdgcn_readfirstlane(row0); rows = __builtin_amdgcn_readfirstlane(rows);
        const int c0 = n0 + wn * (16 * FG);                   // this wavefront's first column of the result
        W4Source<NF, NG, ZERO> src;
#pragma unroll
        for (int f = 0; f < NF; ++f) src.aim(p, f, e, SWIGLU && f >= FG ? (p.n_out + c0) / 16 + (f - FG) : c0 / 16 + f);
        f32x4 acc[NF][FM];
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int i = 0; i < FM; ++i) acc[f][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int whole = p.K / kW4Chunk;                     // chunks that lie inside K

        if constexpr (!kShare) {
            const char *x_at[FM];
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const int m = i * 16 + l16;
                x_at[i] = p.x + ((size_t)(row0 + (m < rows ? m : rows - 1)) * p.K + g16 * 8) * 2;   // past the end: the last row
            }
#pragma unroll 1
            for (int c = wk; c < p.kt; c += WK) {
                W4Weights<NF, NG, ZERO> b;
                src.load(b, c, lane);
                bf16x8 x[FM][4];
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        u32x4 v = {0, 0, 0, 0};
                        if (c < whole || c * kW4Chunk + j * 32 + g16 * 8 < p.K) v = *(const u32x4 *)(x_at[i] + ((uint32_t)c * (kW4Chunk * 2) + j * 64));
                        __builtin_memcpy(&x[i][j], &v, 16);
                    }
                __builtin_amdgcn_sched_barrier(0);            // every load of the chunk is on its way
                w4_chunk<FM>(acc, b, consts, [&](int i, int j) { return x[i][j]; });
            }
        } else {
            // A round brings WK chunks of BM rows x 256 bytes, kept in LDS with the 16-byte piece q of row r at q ^ (r & 15):
            // the 16 rows of an operand read, 256 bytes apart, then lie in different banks.
            constexpr int kRound = WK * BM * 256;
            constexpr int kPieces = kRound / 16 / (WN * WK * kWave);   // of a thread
            static_assert(kPieces * 16 * WN * WK * kWave == kRound, "whole pieces");
            constexpr int kPass = WN * WK * kWave / 16;       // rows that the threads bring at a time, 16 threads each
            static_assert(BM % kPass == 0, "a piece's row is the same in every chunk of the round");
            const int r16 = threadIdx.x / 16, q16 = threadIdx.x % 16;
            const char *x_tile = p.x + (size_t)row0 * p.K * 2;
            uint32_t x_off[BM / kPass];                       // of this thread's rows in the tile; past the end: the last row
#pragma unroll
            for (int u = 0; u < BM / kPass; ++u) {
                const int m = r16 + u * kPass;
                x_off[u] = (uint32_t)(m < rows ? m : rows - 1) * (uint32_t)p.K * 2 + q16 * 16;
            }
            u32x4 px[kPieces];
            auto load_x = [&](int c) {
#pragma unroll
                for (int u = 0; u < kPieces; ++u) {
                    const int ch = c + u / (BM / kPass);
                    px[u] = u32x4{0, 0, 0, 0};
                    if (ch * kW4Chunk + q16 * 8 < p.K) px[u] = *(const u32x4 *)(x_tile + (x_off[u % (BM / kPass)] + (uint32_t)ch * (kW4Chunk * 2)));
                }
            };
            char *const x_to = smem + r16 * 256 + ((q16 ^ (r16 & 15)) << 4);   // rows kPass apart share the place in a row
            auto store_x = [&](int buf) {
#pragma unroll
                for (int u = 0; u < kPieces; ++u) *(u32x4 *)(x_to + buf * kRound + u * (kPass * 256)) = px[u];
            };
            auto rounds = [&](auto fm_tag) {                  // with the row fragments that hold a row
                constexpr int kFrags = decltype(fm_tag)::value;
                W4Weights<NF, NG, ZERO> b;
                load_x(0);
                src.load(b, wk < p.kt ? wk : p.kt - 1, lane);
                store_x(0);
                __syncthreads();
                int buf = 0;
                for (int c = 0; c < p.kt; c += WK, buf ^= 1) {   // the same rounds for every wavefront: they share the barriers
                    const bool more = c + WK < p.kt;
                    if (more) load_x(c + WK);
                    __builtin_amdgcn_sched_barrier(0);
                    if (c + wk < p.kt) {
                        const char *round = smem + buf * kRound + (wk * BM + l16) * 256;
                        const int c_next = c + WK + wk < p.kt ? c + WK + wk : p.kt - 1;   // (behind the last one: loaded, not used)
                        w4_chunk_64<kFrags>(acc, b, src, c_next, lane, consts, [&](int i, int j) {
                            const u32x4 v = *(const u32x4 *)(round + i * (16 * 256) + (((j * 4 + g16) ^ l16) << 4));
                            bf16x8 x;
                            __builtin_memcpy(&x, &v, 16);
                            return x;
                        });
                    }
                    if (more) store_x(buf ^ 1);
                    __syncthreads();
                }
            };
            if (rows > 48) rounds(std::integral_constant<int, 4>{});
            else if (rows > 32) rounds(std::integral_constant<int, 3>{});
            else if (rows > 16) rounds(std::integral_constant<int, 2>{});
            else rounds(std::integral_constant<int, 1>{});
        }
        w4_finish<FM, FG, WN, WK, SWIGLU, SHIFT, NF>(p, (float *)smem, acc, wk, wn, row0, rows, n0);
    }
}

template <int FM, int FG, int WN, int WK, int G, bool ZERO, bool SWIGLU, bool SHIFT>
static int launch_w4_one(const W4Args &args, hipStream_t stream) {
    constexpr int NF = SWIGLU ? 2 * FG + (SHIFT ? 1 : 0) : FG;
    constexpr int meet = WN * WK * NF * 16 * FM * 16 * (int)sizeof(float), rows = FM > 2 ? 2 * WK * 16 * FM * 256 : 0;
    constexpr int lds = meet > rows ? meet : rows;
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
    // Up columns that begin in the middle of a tile cost one fragment more, which is half a wavefront's work again where it
    // holds one column fragment and a quarter where it holds two; two where they leave the registers for as many wavefronts.
    // Measured, one fragment / two, in us: 8 experts of 4096 x 28688, groups of 128: 3 rows 130 / 103, 32 rows 259 / 166; with
    // zero points and groups of 32 (three wavefronts to a SIMD instead of four), 64 experts of 2048 x 2832, 3 rows: 71 / 75;
    // 64 rows (spills), groups of 128: 118 / 151.
    constexpr bool kNarrow = FM == 4 || (FM == 1 && (G == 32 || (G == 64 && ZERO)));
    return launch_w4_one<FM, (kNarrow && FG > 1 ? FG / 2 : FG), WN, WK, G, ZERO, true, true>(args, stream);
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

// 4-bit weights: quantisation, the way back to bf16, and which form of the product a launch takes (w4.h).
#include "w4.h"

namespace dmoe {

// One wavefront packs one tile: lane 16 g + r holds the 32 weights of column r at k = 32 j + 8 g + i, which a group's
// lanes (4 per column) share the extremes of.  Without zero points s = max |w| / 7 and q = round(w / s) + 8; with them
// s = (max(w, 0) - min(w, 0)) / 15 and z = round(-min(w, 0) / s), so that a weight of zero stays one.  s is rounded to
// bf16 first and the codes follow the rounded one; one below the normal numbers is 0.  A group with a weight that is not finite
// has NaN for its scale: codes have no place for such a weight.  Bound by its scattered 2-byte reads
// (8 x 4096 x 28672: 1.1 ms, 2.2 TB/s); weights are packed once.
__global__ __launch_bounds__(kWave) void w4_quant_kernel(const uint16_t *__restrict__ w, char *__restrict__ codes, uint16_t *__restrict__ scales,
                                                        uint8_t *__restrict__ zeros, int K, int N, int nt, int kt, int group) {
    const int lane = lane_id(), r = lane & 15, g16 = lane >> 4;
    const int64_t tile = blockIdx.x;
    const int c = (int)(tile % kt);
    const int64_t et = tile / kt;
    const int n = (int)(et % nt) * kW4Cols + r;
    const uint16_t *we = w + (et / nt) * K * N;
    float v[4][8], lo[4], hi[4];
    int odd[4];                                                // a weight of these is not finite
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        lo[j] = hi[j] = 0.f;
        odd[j] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int k = c * kW4Chunk + j * 32 + g16 * 8 + i;
            v[j][i] = n < N && k < K ? bf16_to_f32(we[(int64_t)k * N + n]) : 0.f;
            lo[j] = fminf(lo[j], v[j][i]);
            hi[j] = fmaxf(hi[j], v[j][i]);
            odd[j] |= !isfinite(v[j][i]);
        }
#pragma unroll
        for (int s = 16; s < kWave; s <<= 1) {                 // the 4 lanes of a column
            lo[j] = fminf(lo[j], __shfl_xor(lo[j], s, kWave));
            hi[j] = fmaxf(hi[j], __shfl_xor(hi[j], s, kWave));
            odd[j] |= __shfl_xor(odd[j], s, kWave);
        }
    }
    const int steps = group / 32;                              // k-steps that share a scale
    if (steps > 1) {
#pragma unroll
        for (int s = 1; s < 4; s <<= 1) {
            if (s >= steps) continue;
            float l2[4], h2[4];
            int o2[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { l2[j] = fminf(lo[j], lo[j ^ s]); h2[j] = fmaxf(hi[j], hi[j ^ s]); o2[j] = odd[j] | odd[j ^ s]; }
#pragma unroll
            for (int j = 0; j < 4; ++j) { lo[j] = l2[j]; hi[j] = h2[j]; odd[j] = o2[j]; }
        }
    }
    uint32_t words[4];
    const int ng = kW4Chunk / group;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        // (a range past fp32 is divided before it is taken)
        const float range = hi[j] - lo[j];
        float s = zeros != nullptr ? (isfinite(range) ? range / 15.f : hi[j] / 15.f - lo[j] / 15.f) : fmaxf(hi[j], -lo[j]) / 7.f;
        if (s < 0x1p-126f) s = 0.f;                            // (its inverse would not be finite)
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
            scales[at] = there ? (odd[j] ? 0x7fc0 : bits) : 0;
            if (zeros != nullptr) zeros[at] = there ? (uint8_t)z : 0;
        }
    }
    // columns and k past the end have code 0 and scale 0
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n >= N || c * kW4Chunk + j * 32 + g16 * 8 >= K) words[j] = 0;
    *(u32x4 *)(codes + tile * kW4TileBytes + lane * 16) = u32x4{words[0], words[1], words[2], words[3]};
}

// The weights of a tile, 16 columns x 128 k, as 16-bit values: a wavefront unpacks them in their lanes' order, passes them
// through 4 KiB of LDS of its own and writes whole lines of [E, N, K], 4 columns of 256 bytes an instruction.  Only the
// experts that have rows, if batch_sizes is given.  Bound by the 2 bytes written per weight: 8 x 4096 x 28672 in 437 us, 5.4
// TB/s of codes and results.
//   HALF false: out = bf16((q - z) s), rounded once.
//   HALF true:  out = fp16((q - z) s / f), col_scale[e, n] = f, the power of two below the column's largest scale: the values
//               are rounded to 11 bits where the 8 of bf16 would show in the product (relative error of the gated form
//               2.5e-3 instead of 1.7e-3, the rounding of its results alone), and f keeps them in fp16's range.
// Rows of `out` are Kp >= K long; what lies behind K is some finite value (it meets zeros there, see w4_half_rows_kernel).
// With slot_sizes, gridDim.y is the number of experts that `out` has room for: its part s takes expert number s of those that have
// rows, and slot_sizes[s] that expert's rows (0 without one), so that a product on the parts finds its rows where they are;
// slot_sizes[gridDim.y] is the first expert that got no part.
template <bool HALF>
__global__ __launch_bounds__(256) void w4_widen_kernel(const char *__restrict__ codes, const uint16_t *__restrict__ scales, const uint8_t *__restrict__ zeros,
                                                      uint16_t *__restrict__ out, float *__restrict__ col_scale, const int64_t *__restrict__ batch_sizes,
                                                      int K, int Kp, int N, int nt, int kt, int group, int E, int64_t *__restrict__ slot_sizes) {
    __shared__ __attribute__((aligned(16))) char stage[4][4096];
    __shared__ uint16_t largest[kW4Cols][16];
    const int lane = lane_id(), r = lane & 15, g16 = lane >> 4, wave = threadIdx.x / kWave;
    const int slot = blockIdx.y, t = blockIdx.x;
    int e = slot;
    if (slot_sizes != nullptr) {
        e = -1;
        int before = 0;
        for (int e0 = 0; e0 < E && e < 0; e0 += kWave) {
            const bool busy = e0 + lane < E && batch_sizes[e0 + lane] > 0;
            const unsigned long long all = __ballot(busy);
            const unsigned long long at = __ballot(busy && before + __popcll(all & ((1ull << lane) - 1)) == slot);
            if (at != 0) e = e0 + __ffsll(at) - 1;
            before += __popcll(all);
        }
        if (t == 0 && threadIdx.x == 0) {
            slot_sizes[slot] = e < 0 ? 0 : batch_sizes[e];
            if (slot + 1 == (int)gridDim.y) slot_sizes[slot + 1] = e < 0 ? E : e + 1;
        }
        if (e < 0) return;
    } else if (batch_sizes != nullptr && batch_sizes[e] <= 0) {
        return;
    }
    const int ng = kW4Chunk / group;
    const int64_t first = ((int64_t)e * nt + t) * kt;          // tile (t, 0) of the expert
    float inv = 1.f;
    if constexpr (HALF) {
        // the column's largest scale, as bf16 bits (scales are not negative): 16 threads a column
        const int col = threadIdx.x / 16;
        uint32_t most = 0;
        for (int i = threadIdx.x % 16; i < kt * ng; i += 16) {
            const uint32_t s = scales[(first + i / ng) * (kW4Cols * ng) + (col >> 2) * (ng * 4) + (i % ng) * 4 + (col & 3)] & 0x7fffu;
            most = s > most ? s : most;
        }
        largest[col][threadIdx.x % 16] = (uint16_t)most;
        __syncthreads();
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = largest[r][i] > top ? largest[r][i] : top;
        int exponent = (int)(top >> 7);
        // (scales below the normal numbers: 2^-126; all zero: 1; infinite: whatever, it stays so)
        exponent = top == 0 ? 127 : (exponent < 1 ? 1 : (exponent > 253 ? 253 : exponent));
        inv = __uint_as_float((uint32_t)(254 - exponent) << 23);
        if (wave == 0 && g16 == 0 && t * kW4Cols + r < N) col_scale[(int64_t)slot * N + t * kW4Cols + r] = __uint_as_float((uint32_t)exponent << 23);
    }
    char *mine = stage[wave];
    for (int c = wave; c < kt; c += 4) {
        const int64_t tile = first + c;
        const u32x4 q = *(const u32x4 *)(codes + tile * kW4TileBytes + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t at = tile * (kW4Cols * ng) + (r >> 2) * (ng * 4) + (j * 32 / group) * 4 + (r & 3);
            const float s = bf16_to_f32(scales[at]) * inv;
            const float z = zeros != nullptr ? (float)zeros[at] : 8.f;
            u32x4 v;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float lo = ((float)((q[j] >> (4 * p)) & 15u) - z) * s, hi = ((float)((q[j] >> (4 * p + 16)) & 15u) - z) * s;
                if constexpr (HALF) {
                    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
                    v[p] = __builtin_bit_cast(uint32_t, (f16x2{(_Float16)lo, (_Float16)hi}));
                } else {
                    v[p] = pack_bf16x2(lo, hi);
                }
            }
            *(u32x4 *)(mine + r * 256 + (((j * 4 + g16) ^ r) << 4)) = v;       // piece p of row r at p ^ r: no bank twice
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = i * 4 + g16, n = t * kW4Cols + row, k = c * kW4Chunk + r * 8;
            const u32x4 v = *(const u32x4 *)(mine + row * 256 + ((r ^ row) << 4));
            if (n < N && k < Kp) __builtin_nontemporal_store(v, (u32x4 *)(out + ((int64_t)slot * N + n) * Kp + k));
        }
    }
}

// out = fp16(x / f), row_scale[r] = f, the power of two below the row's largest magnitude: exact but for values 2^14 times
// smaller than that, which lose what lies below 2^-24 of it.  Rows of `out` are out_vecs >= vecs long, zeros behind the
// values.  One workgroup per row; 8192 rows of 4096 in 24 us, 5.5 TB/s.
__global__ __launch_bounds__(256) void w4_half_rows_kernel(const u32x4 *__restrict__ x, u32x4 *__restrict__ out, float *__restrict__ row_scale, int vecs,
                                                          int out_vecs) {
    __shared__ uint32_t part[4];
    const int64_t row = blockIdx.x;
    uint32_t most = 0;
    for (int i = threadIdx.x; i < vecs; i += 256) {
        const u32x4 v = x[row * vecs + i];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const uint32_t lo = v[p] & 0x7fffu, hi = (v[p] >> 16) & 0x7fffu;
            most = lo > most ? lo : most;
            most = hi > most ? hi : most;
        }
    }
#pragma unroll
    for (int s = kWave / 2; s > 0; s >>= 1) {
        const uint32_t o = __shfl_xor(most, s, kWave);
        most = o > most ? o : most;
    }
    if (lane_id() == 0) part[threadIdx.x / kWave] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) most = part[i] > most ? part[i] : most;
    int exponent = (int)(most >> 7);
    // (values below the normal numbers: 2^-126; a row of zeros: 1; not finite: it stays so)
    exponent = most == 0 ? 127 : (exponent < 1 ? 1 : (exponent > 253 ? 253 : exponent));
    const float inv = __uint_as_float((uint32_t)(254 - exponent) << 23);
    if (threadIdx.x == 0) row_scale[row] = __uint_as_float((uint32_t)exponent << 23);
    for (int i = threadIdx.x; i < out_vecs; i += 256) {
        u32x4 v = {0, 0, 0, 0};
        if (i < vecs) v = x[row * vecs + i];
        u32x4 o;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            o[p] = __builtin_bit_cast(uint32_t, (f16x2{(_Float16)(__uint_as_float(v[p] << 16) * inv), (_Float16)(__uint_as_float(v[p] & 0xffff0000u) * inv)}));
        }
        out[row * out_vecs + i] = o;
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

static size_t up256(size_t n) { return (n + 255) / 256 * 256; }
// Where the form for many rows keeps what it writes: fp16 weights and rows, and their scales.
struct WideLayout {
    size_t weights, col_scales, rows, row_scales, bytes;
    size_t slot_sizes;                                        // behind the others, where not every expert has room
};
static int64_t wide_k(int64_t K) { return (K + 31) / 32 * 32; }   // whole stages of the 256-row tile
static WideLayout wide_layout(int64_t rows, int E, int64_t K_given, int64_t N) {
    const int64_t K = wide_k(K_given);
    WideLayout w;
    w.weights = 0;
    w.col_scales = up256((size_t)E * N * K * 2);
    w.rows = w.col_scales + up256((size_t)E * N * 4);
    w.row_scales = w.rows + up256((size_t)rows * K * 2);
    w.bytes = w.slot_sizes = w.row_scales + up256((size_t)rows * 4);
    return w;
}
static size_t wide_part_bytes(int64_t rows, int experts, int64_t K, int64_t N) {
    return wide_layout(rows, experts, K, N).bytes + up256(((size_t)experts + 1) * sizeof(int64_t));
}
// Experts that `bytes` have room for: E of them, or some (the experts that have rows take the room in turn).
static int wide_experts(int64_t rows, int E, int64_t K, int64_t N, size_t bytes) {
    if (bytes >= wide_layout(rows, E, K, N).bytes) return E;
    int least = 0, most = E;                                  // room for `least`, none for `most`
    while (most - least > 1) {
        const int mid = (least + most) / 2;
        if (bytes >= wide_part_bytes(rows, mid, K, N)) least = mid; else most = mid;
    }
    return least;
}

struct W4Form {
    bool wide;        // through fp16 weights
    int tile_rows;
};
// Rows per expert decide.  The one kernel unpacks the codes again for every 64 rows and folds every group; from some number of
// rows on the product on weights that are written out first is the faster one, the sooner the shorter the groups.  Measured,
// us of the one kernel / through 16-bit weights: K 4096, N 28672, 8 experts, groups of 128: 256 rows 596 / 1203, 512 1144 / 1244,
// 1024 2280 / 1973; groups of 32: 256 rows 774 / 1219, 512 1524 / 1262; K 2048, N 2816, 64 experts, groups of 128: 256 rows
// 381 / 548, 512 748 / 602; groups of 32: 256 rows 480 / 553, 512 951 / 611.  These are many columns, of all experts together.
// Where there are few, the written-out form pays for launches that do not fill the chip and the rule is wrong: plain product, K 4096,
// groups of 128, 1024 / 4096 rows an expert: 1 expert, N 256 33 / 130 and 70 / 138, N 2816 44 / 136 and 158 / 119; 8 experts, N 256
// 130 / 154 and 611 / 243, N 1024 159 / 152 and 620 / 369; K 14336, 1 expert, N 256 95 / 228 and 191 / 280.  (A caller who has such
// a matrix gives no room: 0 wide_bytes.)  And it is one decision for the launch: the experts of a skewed batch share it.
static long long wide_rows(int group) { return group == 128 ? 512 : (group == 64 ? 448 : 384); }
// Row tiles of the one kernel for the experts that have rows but the first `left_out` of them: those of the sizes, or at most one
// short one for every expert with rows.
static int row_tiles_w4(int64_t rows, int E, int tile_rows, int left_out, const int64_t *host_sizes) {
    long long m = rows / tile_rows + (E < rows ? E : rows);
    if (host_sizes != nullptr) {
        long long left = rows;
        m = 0;
        for (int e = 0; e < E; ++e) {
            long long n = host_sizes[e] < 0 ? 0 : host_sizes[e];
            if (n > 0 && left_out-- > 0) { left -= n < left ? n : left; continue; }
            if (n > left) n = left;
            left -= n;
            m += (n + tile_rows - 1) / tile_rows;
        }
    }
    return (int)(m > 0 ? m : 1);
}
static W4Form choose_w4(int64_t rows, int E, int64_t K, int64_t N, int group, const int64_t *host_sizes) {
    long long busy = E < rows ? E : rows;
    if (host_sizes != nullptr) {
        busy = 0;
        for (int e = 0; e < E; ++e) busy += host_sizes[e] > 0;
    }
    if (busy < 1) busy = 1;
    const long long avg = (rows + busy - 1) / busy;
    W4Form f;
    f.wide = avg > wide_rows(group) && wide_k(K) * N * 2 < (1ll << 32);   // (what the 256-row tile takes)
    f.tile_rows = avg <= 16 ? 16 : (avg <= 32 ? 32 : 64);
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
    const W4Form f = choose_w4(rows, E, K, N, group, host_batch_sizes);
    const int nt = tiles_of(N, kW4Cols), kt = tiles_of(K, kW4Chunk);
    const int64_t *left = nullptr;                            // the first expert that had no room
    const int experts = f.wide && wide != nullptr ? wide_experts(rows, E, K, N, wide_bytes) : 0;   // that `wide` has room for
    if (experts > 0) {
        const WideLayout at = wide_layout(rows, experts, K, N);
        char *w = (char *)wide;
        int64_t *slot_sizes = experts < E ? (int64_t *)(w + at.slot_sizes) : nullptr;
        const int64_t Kp = wide_k(K);
        hipLaunchKernelGGL(w4_widen_kernel<true>, dim3(nt, experts), dim3(256), 0, (hipStream_t)stream, (const char *)codes, (const uint16_t *)scales,
                           (const uint8_t *)zeros, (uint16_t *)(w + at.weights), (float *)(w + at.col_scales), batch_sizes, (int)K, (int)Kp, (int)N, nt, kt,
                           group, E, slot_sizes);
        DMOE_LAUNCH_CHECK("w4_widen_kernel");
        hipLaunchKernelGGL(w4_half_rows_kernel, dim3((unsigned)rows), dim3(256), 0, (hipStream_t)stream, (const u32x4 *)a, (u32x4 *)(w + at.rows),
                           (float *)(w + at.row_scales), (int)(K / 8), (int)(Kp / 8));
        DMOE_LAUNCH_CHECK("w4_half_rows_kernel");
        // the sizes of the experts that have room, on the host too
        int64_t host_slots[kMaxGroups];
        if (host_batch_sizes != nullptr && slot_sizes != nullptr) {
            int s = 0;
            for (int e = 0; e < E && s < experts; ++e)
                if (host_batch_sizes[e] > 0) host_slots[s++] = host_batch_sizes[e];
            while (s < experts) host_slots[s++] = 0;
        }
        const HostSizes known(host_batch_sizes != nullptr && slot_sizes != nullptr ? host_slots : host_batch_sizes);
        GmmArgs args{w + at.rows, w + at.weights, (char *)c, slot_sizes != nullptr ? slot_sizes : batch_sizes, (const float *)(w + at.row_scales),
                     (const float *)(w + at.col_scales), rows, experts, (int)Kp, (int)N, (int)n_out};
        rc = bind_state(args, state, workspace, workspace_bytes, (hipStream_t)stream);
        const WorkspaceTurn turn(args);
        if (rc == DMOE_OK) rc = launch_tile256_half(args, swiglu, (hipStream_t)stream);
        if (rc != DMOE_OK || experts >= (E < rows ? E : rows)) return rc;
        left = slot_sizes + experts;
        // (where the host's sizes have nobody left, the launch finds out by itself in a few microseconds)
    }
    W4Args args{(const char *)a, (const char *)codes, (const char *)scales, (const char *)zeros, (char *)c, batch_sizes, rows, E, (int)K, (int)N,
                (int)n_out, nt, kt, row_tiles_w4(rows, E, f.tile_rows, experts, host_batch_sizes), left};
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
    hipLaunchKernelGGL(w4_widen_kernel<false>, dim3(nt, E), dim3(256), 0, (hipStream_t)stream, (const char *)codes, (const uint16_t *)scales,
                       (const uint8_t *)zeros, (uint16_t *)out, (float *)nullptr, batch_sizes, (int)K, (int)K, (int)N, nt, kt, group, E, (int64_t *)nullptr);
    DMOE_LAUNCH_CHECK("w4_widen_kernel");
    return DMOE_OK;
}

extern "C" int dmoe_gmm_w4_wide_bytes(int64_t rows, int E, int64_t K, int64_t N, int group, const int64_t *host_batch_sizes, size_t *bytes) {
    const int rc = check_w4("dmoe_gmm_w4_wide_bytes", E, K, N, group);
    if (rc != DMOE_OK) return rc;
    DMOE_REQUIRE(bytes != nullptr && rows >= 0 && rows < (1ll << 31), DMOE_ERR_ARG, "dmoe_gmm_w4_wide_bytes: bad rows or null output");
    *bytes = choose_w4(rows, E, K, N, group, host_batch_sizes).wide ? wide_layout(rows, E, K, N).bytes : 0;
    return DMOE_OK;
}

extern "C" int dmoe_gmm_w4_wide_bytes_of(int64_t rows, int experts, int64_t K, int64_t N, size_t *bytes) {
    const int rc = check_w4("dmoe_gmm_w4_wide_bytes_of", experts, K, N, 128);
    if (rc != DMOE_OK) return rc;
    DMOE_REQUIRE(bytes != nullptr && rows >= 0 && rows < (1ll << 31), DMOE_ERR_ARG, "dmoe_gmm_w4_wide_bytes_of: bad rows or null output");
    *bytes = wide_part_bytes(rows, experts, K, N);
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

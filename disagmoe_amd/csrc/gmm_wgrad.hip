// Weight gradient of a grouped product: db[e] = a[rows of e]^T @ dc[rows of e], bf16 in and out, fp32 sums.
//
// Bound by the matrix cores (2 rows K N flop) where experts have many rows, by the E K N results that are written where
// they have few.  A work item is a 256 x 256 tile of one expert's result; its contraction runs over the expert's rows, so
// both operands arrive with the contraction as their slow dimension.  Their images in LDS are therefore the same: [32 rows]
// [256 columns], 512 bytes a row, copied there directly (32 KiB a stage, 4 stages, issued 3 stages ahead) and read with
// ds_read_b64_tr_b16, which transposes 4 rows x 16 columns inside 16 lanes, so that two reads are a 32-deep operand of
// v_mfma_f32_16x16x32_bf16.  The order of phases is that of gmm_tile256_kernel: the two wavefronts of a SIMD alternate
// between a stage's operand reads and copies and its 32 MFMAs, handed over by workgroup barriers.
//
// An expert's last stage may reach past its rows.  What lies there belongs to the next expert, or to nobody: the copies
// are aimed at the last row instead (so nothing outside the operands is read), and the lanes that copied write zeros over
// them once they have landed, in both operands, because a zero in one does not silence an infinity in the other.
//
// Measured: 8 experts of 1024 rows, 4096 x 28672: 1796 us, 1071 TFLOP/s (matrix units busy 56 % of the cycles at 1.90 GHz;
// torch's dense product of 8192 cubed runs at 1253 on this card); 64 experts of 768 rows, 2048 x 2816: 584 - 622 us, 910 - 970
// TFLOP/s (24 stages a tile); 8 experts of 128 rows, 1024 x 5632: 32 us for 92 MB of results, 2.9 TB/s.
#include "gmm_direct.h"

namespace dmoe {

// Tile number idx of an expert's result.  Bands of 4 k-tiles, their n-tiles one after the other, a band's k-tiles innermost:
// what shares an operand slice runs side by side on one XCD.
__device__ __forceinline__ void wgrad_tile(int idx, int kt_n, int nt_n, int &k0, int &n0) {
    constexpr int kBand = 4;
    const int band = idx / (kBand * nt_n);
    const int width = kt_n - band * kBand < kBand ? kt_n - band * kBand : kBand;
    const int in = idx - band * kBand * nt_n;
    n0 = (in / width) * 256;
    k0 = (band * kBand + in % width) * 256;
}

__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2)))
void gmm_wgrad_kernel(const GmmArgs p) {
    constexpr int BT = 256, NW = 8, WN = 4;
    constexpr int TM = 128, TN = 64;
    constexpr int FM = TM / 16, FN = TN / 16;            // 8 x 4 accumulators of 16 x 16
    constexpr int CP = 2;                                // copies of 1 KiB per operand, wavefront and stage
    constexpr int kLoads = 2 * CP;
    constexpr int kBlock = NW * 1024;
    constexpr int kImage = BT * kDK * 2;                 // 16 KiB per operand and stage
    constexpr int kStage = 2 * kImage;
    constexpr int kStages = 4;
    extern __shared__ __attribute__((aligned(1024))) char smem[];   // (operand addresses are taken apart by bits below)
    __shared__ int s_tile_start[kMaxGroups + 1];
    __shared__ int s_row_start[kMaxGroups + 1];
    __shared__ long long s_item;

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int E = p.E;

    build_work_list<BT>(p, s_tile_start, s_row_start);
    __syncthreads();

    const int kt_n = (p.K + BT - 1) / BT, nt_n = (p.N + BT - 1) / BT;
    const long long per_expert = (long long)kt_n * nt_n;
    const long long tiles = per_expert * E;
    const int G = gridDim.x;
    const int split = p.split;                             // pieces of every tile's contraction (wgrad_split)
    const long long total = tiles * split;
    const uint32_t pitch_a = (uint32_t)p.K * 2, pitch_d = (uint32_t)p.N * 2;
    const uint32_t smem_addr = lds_addr(smem);
    const int streams = (G % kXcds == 0) ? kXcds : 1;

    auto kn_swizzle = [](int k) { return ((k & 3) << 2) ^ (((k >> 3) & 1) << 1); };
    const int kn_r = 2 * wave + (lane >> 5);               // row of the stage this lane copies; copy i adds 16
    const int kn_chunk = (lane & 31) ^ kn_swizzle(kn_r);   // which 16 bytes of it

    // operand reads: the 16 lanes of a group address 4 rows x 16 columns (see gmm_tile256.h)
    const int l16 = lane & 15, g16 = lane >> 4;
    auto read_off = [&](int slot0) {
        const int col = slot0 + 4 * (l16 & 3);
        const int r = g16 * 8 + (l16 >> 2);
        return r * 512 + (((col >> 3) ^ kn_swizzle(r)) * 16) + (col & 7) * 2;
    };
    // the next fragment is 16 columns, 2 chunks, further on: bits 5 .. 7 of the address, which the swizzle flips and nothing
    // else touches, so fragment i is read at the first one's address ^ 32 i
    const uint32_t fa_0 = smem_addr + read_off(wm * TM), fb_0 = smem_addr + kImage + read_off(wn * TN);

    // ---- state of the item whose copies are being issued ----
    int e = 0, k0 = 0, n0 = 0, rows_e = 0, S = 0, pre = 0;   // (rows_e and S: of its piece)
    int part = -1, split_tile = 0;
    uint64_t a_base = 0, d_base = 0;
    uint32_t a_col = 0, d_col = 0;                         // byte offset of this lane's 16 bytes in a row
    auto open_item = [&](long long q) {
        long long L = item_order(q, G, total);
        if (split > 1) {                                   // the same piece of all tiles side by side
            part = __builtin_amdgcn_readfirstlane((int)(L / tiles));
            L -= part * tiles;
            split_tile = __builtin_amdgcn_readfirstlane((int)L);
        }
        e = __builtin_amdgcn_readfirstlane((int)(L / per_expert));
        const int idx = __builtin_amdgcn_readfirstlane((int)(L - e * per_expert));
        wgrad_tile(idx, kt_n, nt_n, k0, n0);
        int row0 = __builtin_amdgcn_readfirstlane(s_row_start[e]);
        rows_e = __builtin_amdgcn_readfirstlane(s_row_start[e + 1]) - row0;
        S = (rows_e + kDK - 1) / kDK;
        if (split > 1) {                                   // stages [S part / split, S (part + 1) / split) of the tile
            const int lo = (int)((long long)S * part / split), hi = (int)((long long)S * (part + 1) / split);
            row0 += lo * kDK;
            rows_e = (hi < S ? hi * kDK : rows_e) - lo * kDK;
            S = hi - lo;
            if (S == 0) rows_e = 0;
        }
        pre = S < kStages ? S : kStages;
        a_base = to_scalar((uint64_t)(uintptr_t)p.a + (uint64_t)row0 * pitch_a);
        d_base = to_scalar((uint64_t)(uintptr_t)p.b + (uint64_t)row0 * pitch_d);
        const int ca = k0 + kn_chunk * 8, cd = n0 + kn_chunk * 8;
        a_col = (uint32_t)(ca < p.K ? ca : 0) * 2;         // columns past the end read the first one (never stored)
        d_col = (uint32_t)(cd < p.N ? cd : 0) * 2;
    };
    auto issue_copies = [&](int s) {
        const uint32_t lds = smem_addr + (s % kStages) * kStage + wave * 1024;
        const uint64_t ab = to_scalar(a_base + (uint64_t)s * kDK * pitch_a), db = to_scalar(d_base + (uint64_t)s * kDK * pitch_d);
        const int last = rows_e - 1 - s * kDK;             // rows behind it are aimed at it
        static_for<0, CP>([&](auto c_tag) {
            constexpr int c = decltype(c_tag)::value;
            const int r = kn_r + 16 * c;
            const uint32_t rr = (uint32_t)(r < last ? r : last);
            copy_g2lds_16<c * kBlock>(rr * pitch_a + a_col, ab, lds);
            copy_g2lds_16<kImage + c * kBlock>(rr * pitch_d + d_col, db, lds);
        });
    };
    // until at most n stages' copies of this wavefront are outstanding, and kStores stores issued between them
    auto wait_ahead = [&](int n, auto stores_tag) {
        constexpr int st = decltype(stores_tag)::value;
        if (n >= 3) DMOE_WAIT_VMCNT(3 * kLoads + st);
        else if (n == 2) DMOE_WAIT_VMCNT(2 * kLoads + st);
        else if (n == 1) DMOE_WAIT_VMCNT(kLoads + st);
        else DMOE_WAIT_VMCNT(st);
    };
    constexpr std::integral_constant<int, 0> no_stores{};
    constexpr std::integral_constant<int, 16> the_stores{};
    // An item's first three stages are copied before the epilogue of the item before it, the fourth behind it, where the LDS
    // that the epilogue passes its rows through is free again: with contractions of some 30 stages the way there and back
    // would otherwise be a tenth of a tile.  The 16 stores of that epilogue lie between them in the order in which a
    // wavefront's accesses complete, and the waits for stages 1 and 2 need not be waits for the stores too (`behind`: the
    // epilogue wrote a whole tile, so it was 16 of them).
    bool behind = false;
    auto issue_early = [&]() {
        for (int s = 0; s < (pre < 3 ? pre : 3); ++s) issue_copies(s);
    };
    auto issue_late = [&]() {
        if (pre > 3) issue_copies(3);
    };

    unsigned int draw = 0;
    const bool drawer = tid == 0;
    if (drawer) draw = sched_draw(p.sched, streams);
    long long q = blockIdx.x;
    if (q < total) {
        open_item(q);
        issue_early();
        issue_late();
    }

    while (q < total) {
        const int cur_e = e, cur_k0 = k0, cur_n0 = n0, cur_S = S, cur_rows = rows_e, cur_part = part, cur_split_tile = split_tile;
        f32x4 acc[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

        // zeros over the rows of stage s behind the expert's last (this lane's own copies, which have landed)
        auto clear_behind = [&](int s) {
            const int valid = cur_rows - s * kDK;
            __builtin_amdgcn_sched_barrier(0);             // behind the wait
            char *mine = smem + (s % kStages) * kStage + wave * 1024 + lane * 16;
#pragma unroll
            for (int c = 0; c < CP; ++c) {
                if (kn_r + 16 * c < valid) continue;
                *(u32x4 *)(mine + c * kBlock) = u32x4{0, 0, 0, 0};
                *(u32x4 *)(mine + kImage + c * kBlock) = u32x4{0, 0, 0, 0};
            }
        };
        const bool ragged = (cur_rows & (kDK - 1)) != 0;
        bf16x8 fa[FM], fb[FN];
        auto read_operand = [&](bf16x8 &f, uint32_t src) {
            typedef s16x4 __attribute__((address_space(3))) *lds_ptr;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)src);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)(src + 4 * 512));
            const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            __builtin_memcpy(&f, &v, 16);
        };
        // `ahead`: stages behind s + 1 whose copies may still be in flight when s + 1 has to be there
        auto stage = [&](int s, auto refill_tag, int ahead, bool next) {
            constexpr bool kRefill = decltype(refill_tag)::value;
            auto landed = [&]() {
                const bool early = behind && s < 2;        // stage s + 1 was copied before the last epilogue
                if constexpr (kRefill) {
                    if (early) DMOE_WAIT_VMCNT((kStages - 2) * kLoads + 16);
                    else DMOE_WAIT_VMCNT((kStages - 2) * kLoads);
                } else {
                    if (early) wait_ahead(ahead, the_stores);
                    else wait_ahead(ahead, no_stores);
                    if (ragged && s + 1 == cur_S - 1) clear_behind(s + 1);
                }
            };
            const uint32_t slot = (uint32_t)(s % kStages) * kStage;
#pragma unroll
            for (int i = 0; i < FM; ++i) read_operand(fa[i], (fa_0 + slot) ^ (i * 32));
#pragma unroll
            for (int j = 0; j < FN; ++j) read_operand(fb[j], (fb_0 + slot) ^ (j * 32));
            if constexpr (kRefill) issue_copies(s + kStages - 1);
            if (next && wm == 1) landed();
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            static_for<0, FM>([&](auto i_tag) {
                constexpr int i = decltype(i_tag)::value;
#pragma unroll
                for (int jj = 0; jj < FN; ++jj) {
                    const int j = (i & 1) ? FN - 1 - jj : jj;
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
                }
            });
            __builtin_amdgcn_s_setprio(0);
            if (next && wm == 0) landed();
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
        };
        if (cur_S > 0) {
            if (behind) wait_ahead(pre - 1, the_stores);
            else wait_ahead(pre - 1, no_stores);
            if (ragged && cur_S == 1) clear_behind(0);
            __syncthreads();
            if (wm == 1) __syncthreads();                  // the half that runs a phase behind
            auto ahead_of = [&](int s) {                   // stages behind s + 1 that may be in flight when s + 1 has to be there
                const int left = cur_S - 1 - s;
                return left - 1 < kStages - 2 ? left - 1 : kStages - 2;
            };
            stage(0, std::false_type{}, ahead_of(0), cur_S > 1);
            int s = 1;
            for (; s + kStages - 1 < cur_S; ++s) stage(s, std::true_type{}, 0, true);
            for (; s < cur_S; ++s) stage(s, std::false_type{}, ahead_of(s), s + 1 < cur_S);
            if (wm == 0) __syncthreads();
        }
        // ---- the next item and its first copies ----
        if (drawer) s_item = sched_item(draw, streams);
        __syncthreads();                                   // also: the last stage has been read by everyone
        q = (long long)to_scalar((uint64_t)s_item);
        if (q < total) {
            if (drawer) draw = sched_draw(p.sched, streams);
            open_item(q);
            issue_early();
        }

        // ---- epilogue: lane l holds, of fragment (i, j), row i * 16 + l % 16 (of K) and the 4 columns j * 16 + (l / 16) * 4 ..;
        // 32 rows at a time through 4 KiB of LDS that belong to the wavefront, out by whole 128-byte lines ----
        behind = false;
        if (cur_part >= 0) {
            // a piece: its fp32 sums as they lie in the registers, for wgrad_join_kernel
            f32x4 *sums = (f32x4 *)p.partials + (((size_t)cur_part * tiles + cur_split_tile) * NW + wave) * (FM * FN * kWave) + lane;
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) sums[(i * FN + j) * kWave] = acc[i][j];
        } else {
        char *stg = smem + 3 * kStage + wave * 4096;
        // (the rows' addresses as a scalar that moves and one offset per lane: 16 addresses a lane would not stay in registers)
        const bool whole = cur_k0 + BT <= p.K && cur_n0 + BT <= p.N;
        const int out_col = cur_n0 + wn * TN + (lane % 8) * 8;
        const uint32_t out_off = (uint32_t)(lane / 8) * pitch_d + (uint32_t)out_col * 2;
        uint64_t out_row = to_scalar((uint64_t)(uintptr_t)p.c + ((uint64_t)cur_e * p.K + cur_k0 + wm * TM) * pitch_d);
        int rows_left = p.K - cur_k0 - wm * TM;            // of the result, from the one out_row is at
#pragma unroll
        for (int i2 = 0; i2 < FM / 2; ++i2) {
#pragma unroll
            for (int ii = 0; ii < 2; ++ii) {
                const int i = i2 * 2 + ii, row = ii * 16 + l16;
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    uint2 pk;
                    pk.x = pack_bf16x2(acc[i][j][0], acc[i][j][1]);
                    pk.y = pack_bf16x2(acc[i][j][2], acc[i][j][3]);
                    const int cb = j * 32 + g16 * 8;
                    *(uint2 *)(stg + row * 128 + (((cb >> 4) ^ ((row >> 1) & 7)) << 4) + (cb & 8)) = pk;
                }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int row = t * 8 + lane / 8, c = lane % 8;
                const u32x4 val = *(const u32x4 *)(stg + row * 128 + ((c ^ ((row >> 1) & 7)) << 4));
                if (whole || (lane / 8 < rows_left && out_col < p.N)) *(u32x4 *)((char *)out_row + out_off) = val;
                out_row += 8ull * pitch_d;
                rows_left -= 8;
            }
        }

        behind = whole;
        }
        __syncthreads();                                   // the staged rows have been read back by everyone
        if (q < total) issue_late();
    }
    sched_finish(p.sched, drawer, draw, streams, total);
}

// Adds up the pieces of every tile in their order and rounds once: a wavefront per 16 x 64 of the result.
__global__ __launch_bounds__(256) void wgrad_join_kernel(const GmmArgs p, int kt_n, int nt_n) {
    constexpr int NW = 8, FM = 8, FN = 4;
    const long long tiles = (long long)p.E * kt_n * nt_n;
    const long long id = (long long)blockIdx.x * 4 + threadIdx.x / kWave;
    const int lane = threadIdx.x & (kWave - 1), l16 = lane & 15, g16 = lane >> 4;
    const int i = (int)(id % FM), wave = (int)(id / FM % NW);
    const long long tile = id / (FM * NW);
    if (tile >= tiles) return;
    f32x4 acc[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const f32x4 *sums = (const f32x4 *)p.partials + ((size_t)tile * NW + wave) * (FM * FN * kWave) + i * FN * kWave + lane;
    const size_t piece = (size_t)tiles * NW * FM * FN * kWave;
#pragma unroll 4
    for (int k = 0; k < p.split; ++k)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[j] += sums[k * piece + j * kWave];
    // (the tile order of gmm_wgrad_kernel)
    const int e = (int)(tile / ((long long)kt_n * nt_n));
    const int idx = (int)(tile - (long long)e * kt_n * nt_n);
    int k0, n0;
    wgrad_tile(idx, kt_n, nt_n, k0, n0);
    const int row = k0 + (wave / 4) * 128 + i * 16 + l16;
    if (row >= p.K) return;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int col = n0 + (wave % 4) * 64 + j * 16 + g16 * 4;
        if (col >= p.N) continue;                          // N % 8 == 0: 4 columns at once
        uint2 pk;
        pk.x = pack_bf16x2(acc[j][0], acc[j][1]);
        pk.y = pack_bf16x2(acc[j][2], acc[j][3]);
        *(uint2 *)((uint16_t *)p.c + ((size_t)e * p.K + row) * p.N + col) = pk;
    }
}

// A launch whose tiles fill half of the compute units at most cuts their contractions into pieces that fill them, of 8 stages
// (256 rows) or more for an expert of average size, as the workspace has room for.  Joining them is a second, short launch:
// with the pieces counted in and added up by whichever comes last, one compute unit read all pieces of a tile past the caches
// and that took longer than the whole contraction (2 experts of 4096 rows, 512 x 1024: 89 us, 47 us uncut).
static int wgrad_split(const GmmArgs &args, long long tiles, long long cus) {
    if (args.arrive == nullptr || tiles * 2 > cus) return 1;
    const long long room = args.partial_bytes / (256 * 256 * (long long)sizeof(float)), stages = args.rows / ((long long)args.E * kDK);
    long long most = cus / tiles;
    most = most < stages / 8 ? most : stages / 8;
    most = most < room / tiles ? most : room / tiles;
    return most < 2 ? 1 : (int)most;
}

int launch_wgrad(const GmmArgs &given, hipStream_t stream) {
    constexpr int lds = 4 * 2 * 256 * kDK * 2;
    static unsigned long long configured = 0;   // devices on which the kernel's LDS size has been raised
    DMOE_HIP(raise_dynamic_lds((const void *)gmm_wgrad_kernel, lds, &configured));
    GmmArgs args = given;
    const int kt_n = (args.K + 255) / 256, nt_n = (args.N + 255) / 256;
    const long long tiles = (long long)args.E * kt_n * nt_n, cus = device_cus();
    args.split = wgrad_split(args, tiles, cus);
    const long long items = tiles * args.split;
    const long long grid = ((items < cus ? items : cus) + kXcds - 1) / kXcds * kXcds;
    hipLaunchKernelGGL(gmm_wgrad_kernel, dim3((unsigned)grid), dim3(512), lds, stream, args);
    DMOE_LAUNCH_CHECK("gmm_wgrad_kernel");
    if (args.split > 1) {
        hipLaunchKernelGGL(wgrad_join_kernel, dim3((unsigned)(tiles * 16)), dim3(256), 0, stream, args, kt_n, nt_n);
        DMOE_LAUNCH_CHECK("wgrad_join_kernel");
    }
    return DMOE_OK;
}

}  // namespace dmoe

// Global norm of many gradients and their scaling to a largest norm.
//
//   norm = sqrt(sum over all tensors and elements of g^2),  coef = min(1, max_norm / (norm + 1e-6)),  g <- g * coef
//
// Bound by memory: the norm reads every gradient once, the scaling reads and writes it once (and does neither where the
// norm is below the limit).  The list of tensors travels in the launch's arguments (kPerLaunch of them at a time), so
// nothing has to be uploaded, kept alive or looked up by address and a recorded launch holds its own list.  The tensors'
// memory, in whole 16-byte vectors one tensor behind the other, is dealt out to the workgroups in equal stretches; a
// tensor's first and last vector may be partly its own and are then taken element by element.  The scaling walks each
// stretch backwards: what the norm read last is what the last-level cache still has.  Squares are added in 64 bits: they
// are exact there, so neither large nor tiny gradients leave the range, and every workgroup leaves its sum at a place of
// its own that the reader adds up in a fixed order: the same gradients give the same bits.
//
// Measured: 2.82 GB of bf16 in two tensors: norm 468 us (6.0 TB/s), with scaling 1.61 ms (8.5 GB; a copy of 4 GB moves
// 4.9 TB/s); 236 MB of fp32: 37 us warm; 300 mixed tensors of 1 to 200001 elements: 2 x (8.5 + 2.7) us, two tables of 160
// (the host's part, some 80 us of Python, is what a caller waits for there).
#include <algorithm>
#include <exception>
#include <utility>
#include <vector>

#include "common.h"

namespace dmoe {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kGradThreads = 256;
constexpr int kGradSlots = 1024;                 // workgroups of a launch at most = partial sums
constexpr int kLeastVecs = 1024;                 // 16-byte vectors of a workgroup's stretch at least
constexpr int kUnroll = 4;                       // vectors of a thread in flight
constexpr int kPerLaunch = 160;                  // tensors in one launch's arguments (below 4 KiB)
static_assert(kGradSlots * sizeof(double) == DMOE_GRAD_WORKSPACE_BYTES, "workspace as dmoe.h states it");

struct GradTable {
    char *data[kPerLaunch];
    int64_t bytes[kPerLaunch];                   // of a tensor; its type (DMOE_BF16, DMOE_FP16, DMOE_FP32) in the top byte
    int64_t vec_start[kPerLaunch + 1];           // vectors before the tensor
    int n;
};
static_assert(sizeof(GradTable) <= 3900, "launch arguments");
constexpr int64_t kBytesMask = (1ll << 56) - 1;

template <int kType> struct Elem;
template <> struct Elem<DMOE_FP32> {
    static constexpr int kBytes = 4;
    static __device__ __forceinline__ float load(const char *p) { return *(const float *)p; }
    static __device__ __forceinline__ void store(char *p, float v) { *(float *)p = v; }
};
template <> struct Elem<DMOE_BF16> {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ float load(const char *p) { return bf16_to_f32(*(const uint16_t *)p); }
    static __device__ __forceinline__ void store(char *p, float v) { *(uint16_t *)p = f32_to_bf16(v); }
};
template <> struct Elem<DMOE_FP16> {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ float load(const char *p) { return (float)*(const _Float16 *)p; }
    static __device__ __forceinline__ void store(char *p, float v) { *(_Float16 *)p = (_Float16)v; }
};

template <int kType>
__device__ __forceinline__ void unpack(const u32x4 &v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kType == DMOE_FP32) f[i] = __uint_as_float(v[i]);
        else if constexpr (kType == DMOE_BF16) {
            f[2 * i] = __uint_as_float(v[i] << 16);
            f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        } else {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const uint32_t w = v[i];
            f16x2 h;
            __builtin_memcpy(&h, &w, 4);
            f[2 * i] = (float)h[0];
            f[2 * i + 1] = (float)h[1];
        }
    }
}
template <int kType>
__device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kType == DMOE_FP32) v[i] = __float_as_uint(f[i]);
        else if constexpr (kType == DMOE_BF16) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
        else {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const f16x2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]};   // each rounded to nearest even
            uint32_t w;
            __builtin_memcpy(&w, &h, 4);
            v[i] = w;
        }
    }
    return v;
}

// The vectors [v0, v0 + count) of tensor memory [data, data + bytes), vector 0 holding its first byte: whole ones to
// `vec(addresses, whether whole)`, the elements of one that lies partly outside to `one(address)`.  kBackwards: from the
// last to the first.
template <int kType, bool kBackwards, typename Vec, typename One>
__device__ __forceinline__ void for_vectors(char *data, int64_t bytes, int64_t v0, int64_t count, Vec &&vec, One &&one) {
    constexpr int kBytes = Elem<kType>::kBytes;
    constexpr int kStep = kGradThreads * kUnroll;
    char *const base = (char *)((uintptr_t)data & ~(uintptr_t)15) + v0 * 16;
    char *const end = data + bytes;
    for (int64_t i0 = 0; i0 < count; i0 += kStep) {
        char *at[kUnroll];
        bool whole[kUnroll], there[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int64_t k = i0 + u * kGradThreads + threadIdx.x, i = kBackwards ? count - 1 - k : k;
            there[u] = k < count;
            at[u] = base + i * 16;
            whole[u] = there[u] && at[u] >= data && at[u] + 16 <= end;
        }
        vec(at, whole);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            if (whole[u] || !there[u]) continue;
            for (char *p = at[u] < data ? data : at[u]; p < at[u] + 16 && p < end; p += kBytes) one(p);
        }
    }
}

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[kGradThreads / kWave];
#pragma unroll
    for (int s = kWave / 2; s > 0; s >>= 1) v += __shfl_xor(v, s, kWave);
    __syncthreads();                              // an earlier use of `part` has been read
    if (lane_id() == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kGradThreads / kWave; ++i) v += part[i];
    return v;
}

// f(type, data, bytes, first vector, vectors) for the tensors' parts in this workgroup's stretch
template <bool kBackwards, typename F>
__device__ __forceinline__ void for_parts(const GradTable &t, F &&f) {
    const int64_t total = t.vec_start[t.n], share = total / gridDim.x, rest = total % gridDim.x;
    const int64_t b = blockIdx.x, lo = b * share + (b < rest ? b : rest), hi = lo + share + (b < rest ? 1 : 0);
    if (lo >= hi) return;
    const int64_t look = kBackwards ? hi - 1 : lo;
    int at = 0, above = t.n;                      // the last tensor whose first vector is not behind `look`
    while (above - at > 1) {
        const int mid = (at + above) >> 1;
        if (t.vec_start[mid] <= look) at = mid; else above = mid;
    }
    for (; kBackwards ? at >= 0 && t.vec_start[at + 1] > lo : at < t.n && t.vec_start[at] < hi; at += kBackwards ? -1 : 1) {
        const int64_t first = t.vec_start[at], last = t.vec_start[at + 1];
        const int64_t v0 = (lo > first ? lo : first), v1 = (hi < last ? hi : last);
        f((int)(t.bytes[at] >> 56), t.data[at], t.bytes[at] & kBytesMask, v0 - first, v1 - v0);
    }
}

template <int kType>
__device__ __forceinline__ double part_squares(char *data, int64_t bytes, int64_t v0, int64_t count) {
    double sum[kUnroll] = {};
    auto add = [](double &s, float v) { s = fma((double)v, (double)v, s); };
    for_vectors<kType, false>(data, bytes, v0, count,
        [&](char *(&at)[kUnroll], const bool (&whole)[kUnroll]) {
            u32x4 v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                v[u] = u32x4{0, 0, 0, 0};
                if (whole[u]) v[u] = *(const u32x4 *)at[u];
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                float f[8];
                unpack<kType>(v[u], f);
#pragma unroll
                for (int i = 0; i < 16 / Elem<kType>::kBytes; ++i) add(sum[u], f[i]);
            }
        },
        [&](const char *p) { add(sum[0], Elem<kType>::load(p)); });
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// slots[b] (+)= the squares of workgroup b's stretch
__global__ __launch_bounds__(kGradThreads) void grad_squares_kernel(const GradTable t, double *slots, int first) {
    double sum = 0;
    for_parts<false>(t, [&](int type, char *data, int64_t bytes, int64_t v0, int64_t count) {
        if (type == DMOE_FP32) sum += part_squares<DMOE_FP32>(data, bytes, v0, count);
        else if (type == DMOE_BF16) sum += part_squares<DMOE_BF16>(data, bytes, v0, count);
        else sum += part_squares<DMOE_FP16>(data, bytes, v0, count);
    });
    sum = block_sum(sum);
    if (threadIdx.x == 0) slots[blockIdx.x] = first ? sum : slots[blockIdx.x] + sum;
}

__device__ __forceinline__ double norm_of(const double *slots, int n) {
    double v = 0;
    for (int i = threadIdx.x; i < n; i += kGradThreads) v += slots[i];
    return sqrt(block_sum(v));
}

__global__ __launch_bounds__(kGradThreads) void grad_norm_kernel(const double *slots, int n, float *norm) {
    const double v = norm_of(slots, n);
    if (threadIdx.x == 0) *norm = (float)v;
}

template <int kType>
__device__ __forceinline__ void scale_part(char *data, int64_t bytes, int64_t v0, int64_t count, float coef) {
    for_vectors<kType, true>(data, bytes, v0, count,
        [&](char *(&at)[kUnroll], const bool (&whole)[kUnroll]) {
            u32x4 v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (whole[u]) v[u] = *(const u32x4 *)at[u];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (!whole[u]) continue;
                float f[8];
                unpack<kType>(v[u], f);
#pragma unroll
                for (int i = 0; i < 16 / Elem<kType>::kBytes; ++i) f[i] *= coef;
                *(u32x4 *)at[u] = pack<kType>(f);
            }
        },
        [&](char *p) { Elem<kType>::store(p, Elem<kType>::load(p) * coef); });
}

// Every workgroup adds up the partial sums by itself (8 KiB at most, from its XCD's L2) instead of waiting for a launch
// of its own that would; workgroup 0 of the first launch also writes the norm.
__global__ __launch_bounds__(kGradThreads) void grad_scale_kernel(const GradTable t, const double *slots, int n,
                                                                 double max_norm, float *norm) {
    const double total = norm_of(slots, n);
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    const double ratio = max_norm / (total + 1e-6);
    if (ratio >= 1.0) return;                     // (not so where the ratio is NaN: the gradients become NaN then)
    const float coef = (float)ratio;
    for_parts<true>(t, [&](int type, char *data, int64_t bytes, int64_t v0, int64_t count) {
        if (type == DMOE_FP32) scale_part<DMOE_FP32>(data, bytes, v0, count, coef);
        else if (type == DMOE_BF16) scale_part<DMOE_BF16>(data, bytes, v0, count, coef);
        else scale_part<DMOE_FP16>(data, bytes, v0, count, coef);
    });
}

static int check_grads(const char *who, const dmoe_grad *grads, int64_t n, const void *norm, const void *workspace,
                       size_t workspace_bytes) {
    DMOE_REQUIRE(n >= 0, DMOE_ERR_ARG, "%s: %lld tensors", who, (long long)n);
    DMOE_REQUIRE(norm != nullptr && (n == 0 || grads != nullptr), DMOE_ERR_ARG, "%s: null pointer", who);
    DMOE_REQUIRE(workspace != nullptr && workspace_bytes >= DMOE_GRAD_WORKSPACE_BYTES, DMOE_ERR_WORKSPACE,
                 "%s: the workspace needs %d bytes, got %zu", who, DMOE_GRAD_WORKSPACE_BYTES, workspace ? workspace_bytes : 0);
    DMOE_REQUIRE(((uintptr_t)workspace & 7) == 0, DMOE_ERR_WORKSPACE, "%s: the workspace must be 8-byte aligned", who);
    for (int64_t i = 0; i < n; ++i) {
        const dmoe_grad &g = grads[i];
        DMOE_REQUIRE(g.dtype == DMOE_BF16 || g.dtype == DMOE_FP16 || g.dtype == DMOE_FP32, DMOE_ERR_DTYPE,
                     "%s: tensor %lld has dtype %d (bf16, fp16 or fp32)", who, (long long)i, g.dtype);
        DMOE_REQUIRE(g.numel >= 0 && g.numel < (1ll << 42), DMOE_ERR_SHAPE, "%s: tensor %lld has %lld elements", who, (long long)i,
                     (long long)g.numel);
        DMOE_REQUIRE(g.numel == 0 || g.data != nullptr, DMOE_ERR_ARG, "%s: tensor %lld is a null pointer", who, (long long)i);
        DMOE_REQUIRE((uintptr_t)g.data % (g.dtype == DMOE_FP32 ? 4 : 2) == 0, DMOE_ERR_ARG, "%s: tensor %lld is not aligned to its elements",
                     who, (long long)i);
    }
    return DMOE_OK;
}

static int64_t bytes_of(const dmoe_grad &g) { return g.numel * (g.dtype == DMOE_FP32 ? 4 : 2); }

// Tables of up to kPerLaunch tensors, the empty ones left out; at least one table.
static std::vector<GradTable> tables_of(const dmoe_grad *grads, int64_t n, int *blocks) {
    std::vector<GradTable> out;
    GradTable t{};
    int64_t vecs = 0, most = 1;
    auto flush = [&]() {
        t.vec_start[t.n] = vecs;
        if (vecs > most) most = vecs;
        out.push_back(t);
        t.n = 0;
        vecs = 0;
    };
    for (int64_t i = 0; i < n; ++i) {
        if (grads[i].numel == 0) continue;
        if (t.n == kPerLaunch) flush();
        const int64_t bytes = bytes_of(grads[i]);
        t.data[t.n] = (char *)grads[i].data;
        t.bytes[t.n] = bytes | (int64_t)grads[i].dtype << 56;
        t.vec_start[t.n] = vecs;
        ++t.n;
        vecs += ((int64_t)((uintptr_t)grads[i].data & 15) + bytes + 15) / 16;
    }
    if (t.n > 0 || out.empty()) flush();
    most = (most + kLeastVecs - 1) / kLeastVecs;
    *blocks = (int)(most < kGradSlots ? most : kGradSlots);
    return out;
}

static int launch_squares(const std::vector<GradTable> &tables, int blocks, double *slots, hipStream_t stream) {
    for (size_t i = 0; i < tables.size(); ++i) {
        hipLaunchKernelGGL(grad_squares_kernel, dim3(blocks), dim3(kGradThreads), 0, stream, tables[i], slots, i == 0 ? 1 : 0);
        DMOE_LAUNCH_CHECK("grad_squares_kernel");
    }
    return DMOE_OK;
}

}  // namespace dmoe

using namespace dmoe;

extern "C" int dmoe_grad_norm(const dmoe_grad *grads, int64_t n, float *norm, void *workspace, size_t workspace_bytes,
                              void *stream) try {
    int rc = check_grads("dmoe_grad_norm", grads, n, norm, workspace, workspace_bytes);
    if (rc != DMOE_OK) return rc;
    int blocks = 0;
    const std::vector<GradTable> tables = tables_of(grads, n, &blocks);
    rc = launch_squares(tables, blocks, (double *)workspace, (hipStream_t)stream);
    if (rc != DMOE_OK) return rc;
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kGradThreads), 0, (hipStream_t)stream, (const double *)workspace, blocks, norm);
    DMOE_LAUNCH_CHECK("grad_norm_kernel");
    return DMOE_OK;
} catch (const std::exception &e) {
    return fail(DMOE_ERR_ARG, "dmoe_grad_norm: %s", e.what());
}

extern "C" int dmoe_clip_grads(const dmoe_grad *grads, int64_t n, double max_norm, float *norm, void *workspace,
                               size_t workspace_bytes, void *stream) try {
    int rc = check_grads("dmoe_clip_grads", grads, n, norm, workspace, workspace_bytes);
    if (rc != DMOE_OK) return rc;
    DMOE_REQUIRE(max_norm >= 0, DMOE_ERR_ARG, "dmoe_clip_grads: max_norm %g", max_norm);
    // memory that two tensors share would be scaled twice, by workgroups that do not wait for each other
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    spans.reserve((size_t)n);
    for (int64_t i = 0; i < n; ++i)
        if (grads[i].numel > 0) spans.emplace_back((uintptr_t)grads[i].data, (uintptr_t)grads[i].data + (uintptr_t)bytes_of(grads[i]));
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        DMOE_REQUIRE(spans[i].first >= spans[i - 1].second, DMOE_ERR_ARG, "dmoe_clip_grads: two of the tensors share memory");
    int blocks = 0;
    const std::vector<GradTable> tables = tables_of(grads, n, &blocks);
    rc = launch_squares(tables, blocks, (double *)workspace, (hipStream_t)stream);
    if (rc != DMOE_OK) return rc;
    for (size_t i = 0; i < tables.size(); ++i) {
        hipLaunchKernelGGL(grad_scale_kernel, dim3(blocks), dim3(kGradThreads), 0, (hipStream_t)stream, tables[i],
                           (const double *)workspace, blocks, max_norm, i == 0 ? norm : (float *)nullptr);
        DMOE_LAUNCH_CHECK("grad_scale_kernel");
    }
    return DMOE_OK;
} catch (const std::exception &e) {
    return fail(DMOE_ERR_ARG, "dmoe_clip_grads: %s", e.what());
}

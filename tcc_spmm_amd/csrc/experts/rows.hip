// Rows to the experts' order and back, and the gradients (include/experts.h). All of it moves rows: what bounds it is HBM,
// each row read and written once.
//
// A token is held by `lanes` threads of a workgroup, a power of two of them, 8 consecutive elements each; a workgroup takes as
// many tokens as fit. Both ways go token by token: a token's row is read once for all its choices, or its choices' rows
// are added in registers and written once. Rows of the output are stored past the caches, whole lines at a time.
// Measured, 8192 tokens to 8 experts each, 2048 bf16: gather 58 us, 5.2 TB/s of reads and writes; combine 55, 5.5; its
// gradients 111, 5.1. 24 tokens to 4: 3.5 us, a launch's length.
#include "experts.h"
#include "hip_support.h"
#include "blocks/device_blocks.h"

namespace {

using namespace blocks;

constexpr unsigned kThreads = 256;

struct Rows {
    const void *x, *dy;
    void *out, *dweights;
    std::uint64_t xStride, dyStride, outStride;
    const void* weights;
    const std::int32_t *offsets, *places;
    DenseType weightType;
    unsigned tokens, choices, each, experts, width, lanes;
};

__device__ __forceinline__ float weightOf(const Rows& a, unsigned c) {
    if (!a.weights) return 1.0f;
    switch (a.weightType) {
    case DenseType::f32: return static_cast<const float*>(a.weights)[c];
    case DenseType::bf16: return float(static_cast<const __bf16*>(a.weights)[c]);
    default: return float(static_cast<const _Float16*>(a.weights)[c]);
    }
}

// The row of choice c, and whether it has an expert here.
__device__ __forceinline__ unsigned rowOfChoice(const Rows& a, unsigned c, unsigned here, bool& used) {
    const unsigned row = min(unsigned(a.places[c]), a.choices - 1);
    used = row < here;
    return row;
}

// Eight elements as they are.
template <typename T> __device__ __forceinline__ typename Group<T>::Vec raw8(const typename T::Raw* row, unsigned at, unsigned n) {
    typename Group<T>::Vec v = {};
    if (at + 8 <= n) return *reinterpret_cast<const typename Group<T>::Loose*>(row + at);
#pragma unroll
    for (unsigned i = 0; i < 8; ++i)
        if (at + i < n) v[i] = row[at + i];
    return v;
}
template <typename T>
__device__ __forceinline__ void putRaw8(typename T::Raw* row, unsigned at, unsigned n, typename Group<T>::Vec v) {
    if (at + 8 <= n) {
        __builtin_nontemporal_store(v, reinterpret_cast<typename Group<T>::Loose*>(row + at));
    } else {
#pragma unroll
        for (unsigned i = 0; i < 8; ++i)
            if (at + i < n) row[at + i] = v[i];
    }
}

template <typename T> __global__ __launch_bounds__(kThreads) void gatherRows(Rows a) {
    const unsigned token = blockIdx.x * (kThreads / a.lanes) + threadIdx.x / a.lanes;
    const unsigned at = (blockIdx.y * a.lanes + threadIdx.x % a.lanes) * 8;
    if (token >= a.tokens || at >= a.width) return;
    const unsigned here = unsigned(a.offsets[a.experts]);
    const typename Group<T>::Vec v = raw8<T>(static_cast<const typename T::Raw*>(a.x) + token * a.xStride, at, a.width);
    const typename Group<T>::Vec zero = {};
    for (unsigned j = 0; j < a.each; ++j) {
        bool used;
        const unsigned row = rowOfChoice(a, token * a.each + j, here, used);
        putRaw8<T>(static_cast<typename T::Raw*>(a.out) + row * a.outStride, at, a.width, used ? v : zero);
    }
}

template <typename T> __global__ __launch_bounds__(kThreads) void combineRows(Rows a) {
    constexpr unsigned Ahead = 4; // choices whose rows are on their way at a time
    const unsigned token = blockIdx.x * (kThreads / a.lanes) + threadIdx.x / a.lanes;
    const unsigned at = (blockIdx.y * a.lanes + threadIdx.x % a.lanes) * 8;
    if (token >= a.tokens || at >= a.width) return;
    const unsigned here = unsigned(a.offsets[a.experts]);
    float sum[8] = {};
    for (unsigned j = 0; j < a.each; j += Ahead) {
        typename Group<T>::Vec v[Ahead] = {};
        float w[Ahead];
        bool used[Ahead];
#pragma unroll
        for (unsigned u = 0; u < Ahead; ++u) {
            const unsigned c = token * a.each + min(j + u, a.each - 1);
            const unsigned row = rowOfChoice(a, c, here, used[u]);
            w[u] = weightOf(a, c);
            used[u] = used[u] && j + u < a.each;
            if (used[u]) v[u] = raw8<T>(static_cast<const typename T::Raw*>(a.x) + row * a.xStride, at, a.width);
        }
#pragma unroll
        for (unsigned u = 0; u < Ahead; ++u)
            if (used[u])
#pragma unroll
                for (unsigned i = 0; i < 8; ++i) sum[i] = fmaf(w[u], T::get(v[u][i]), sum[i]);
    }
    store8<T>(static_cast<typename T::Raw*>(a.out) + token * a.outStride, at, a.width, sum);
}

// A token's dot products need its whole row: its threads go along it, a batch of choices at a time, and add up.
template <typename T> __global__ __launch_bounds__(kThreads) void combineRowsBackward(Rows a) {
    constexpr unsigned Batch = 8;
    __shared__ float sums[kThreads / kWave][Batch];
    const unsigned t = threadIdx.x, lane = t % a.lanes, token = blockIdx.x * (kThreads / a.lanes) + t / a.lanes;
    const bool in = token < a.tokens;
    const unsigned here = unsigned(a.offsets[a.experts]);
    const typename T::Raw* dy = static_cast<const typename T::Raw*>(a.dy) + std::uint64_t(in ? token : 0) * a.dyStride;
    for (unsigned j0 = 0; j0 < a.each; j0 += Batch) {
        float dots[Batch] = {}, w[Batch];
        unsigned row[Batch];
        bool used[Batch];
#pragma unroll
        for (unsigned u = 0; u < Batch; ++u) {
            const unsigned c = (in ? token : 0) * a.each + min(j0 + u, a.each - 1);
            row[u] = rowOfChoice(a, c, here, used[u]);
            w[u] = weightOf(a, c);
        }
        for (unsigned at = lane * 8; in && at < a.width; at += a.lanes * 8) {
            float g[8];
            const typename Group<T>::Vec d = raw8<T>(dy, at, a.width);
#pragma unroll
            for (unsigned i = 0; i < 8; ++i) g[i] = T::get(d[i]);
            typename Group<T>::Vec v[Batch] = {};
            if (a.dweights)
#pragma unroll
                for (unsigned u = 0; u < Batch; ++u)
                    if (used[u] && j0 + u < a.each)
                        v[u] = raw8<T>(static_cast<const typename T::Raw*>(a.x) + row[u] * a.xStride, at, a.width);
            if (a.out)
#pragma unroll
                for (unsigned u = 0; u < Batch; ++u) {
                    if (j0 + u >= a.each) break;
                    float r[8];
#pragma unroll
                    for (unsigned i = 0; i < 8; ++i) r[i] = used[u] ? w[u] * g[i] : 0.0f;
                    store8<T>(static_cast<typename T::Raw*>(a.out) + row[u] * a.outStride, at, a.width, r);
                }
#pragma unroll
            for (unsigned u = 0; u < Batch; ++u)
                if (used[u] && j0 + u < a.each)
#pragma unroll
                    for (unsigned i = 0; i < 8; ++i) dots[u] = fmaf(g[i], T::get(v[u][i]), dots[u]);
        }
        if (!a.dweights) continue;
        for (unsigned by = min(a.lanes, kWave) / 2; by; by /= 2)
#pragma unroll
            for (unsigned u = 0; u < Batch; ++u) dots[u] += __shfl_xor(dots[u], by);
        if (a.lanes > kWave) {
            __syncthreads();
            if (t % kWave == 0)
#pragma unroll
                for (unsigned u = 0; u < Batch; ++u) sums[t / kWave][u] = dots[u];
            __syncthreads();
            const unsigned first = t / a.lanes * (a.lanes / kWave);
#pragma unroll
            for (unsigned u = 0; u < Batch; ++u) {
                dots[u] = 0.0f;
                for (unsigned k = 0; k < a.lanes / kWave; ++k) dots[u] += sums[first + k][u];
            }
        }
        if (lane || !in) continue;
#pragma unroll
        for (unsigned u = 0; u < Batch; ++u) {
            if (j0 + u >= a.each) break;
            const unsigned c = token * a.each + j0 + u;
            const float d = used[u] ? dots[u] : 0.0f;
            switch (a.weightType) {
            case DenseType::f32: static_cast<float*>(a.dweights)[c] = d; break;
            case DenseType::bf16: static_cast<__bf16*>(a.dweights)[c] = __bf16(d); break;
            default: static_cast<_Float16*>(a.dweights)[c] = _Float16(d); break;
            }
        }
    }
}

// Threads of a row: a power of two, up to a workgroup.
unsigned lanesOf(std::uint32_t width) {
    unsigned lanes = 1;
    while (lanes < kThreads && lanes * 8 < width) lanes *= 2;
    return lanes;
}

Rows rowsOf(const char* where, const ExpertPlan& plan, std::uint32_t width) {
    checkColumns(where, width);
    if (!plan.experts || plan.experts > kMaxExperts) reject(where, "experts must be 1 to 1024");
    if (!plan.each || plan.each > kMaxEach) reject(where, "choices of a token must be 1 to 1024");
    if (plan.choices >> 31) reject(where, "2^31 choices or more");
    if (plan.choices % plan.each) reject(where, "choices are not whole tokens'");
    if (plan.choices) {
        if (!plan.offsets || !plan.places) reject(where, "null plan");
        if ((reinterpret_cast<std::uintptr_t>(plan.offsets) | reinterpret_cast<std::uintptr_t>(plan.places)) % 4)
            reject(where, "plan not aligned to its elements");
    }
    Rows a = {};
    a.offsets = plan.offsets, a.places = plan.places, a.choices = plan.choices, a.each = plan.each, a.experts = plan.experts;
    a.tokens = plan.choices / plan.each, a.width = width, a.lanes = lanesOf(width);
    return a;
}

void checkWeights(const char* where, Rows& a, const void* weights, DenseType type) {
    checkType(where, type);
    if (reinterpret_cast<std::uintptr_t>(weights) % elementBytes(type)) reject(where, "weights not aligned to their type");
    a.weights = weights, a.weightType = type;
}

// Workgroups of all tokens, by runs of a row.
dim3 gridOf(const char* where, const Rows& a, bool whole) {
    const unsigned each = kThreads / a.lanes, groups = (a.tokens + each - 1) / each;
    checkGrid(where, groups, kThreads);
    return dim3(groups, whole ? 1 : (a.width + a.lanes * 8 - 1) / (a.lanes * 8));
}

} // namespace

void gatherExperts(DenseMatrix x, ExpertPlan plan, void* rows, std::uint64_t stride, std::uint32_t width,
                   hipStream_t stream) {
    const char* where = "gather experts";
    Rows a = rowsOf(where, plan, width);
    checkType(where, x.type);
    if (!plan.choices) return;
    checkDense(where, x.data, x.stride, x.type, width);
    checkDense(where, rows, stride, x.type, width);
    a.x = x.data, a.xStride = x.stride, a.out = rows, a.outStride = stride;
    const dim3 grid = gridOf(where, a, false);
    withType(x.type, [&](auto tag) {
        hipLaunchKernelGGL((gatherRows<decltype(tag)>), grid, dim3(kThreads), 0, stream, a);
    });
    checkHip(hipGetLastError());
}

void combineExperts(DenseMatrix rows, ExpertPlan plan, const void* weights, DenseType weightType, void* y,
                    std::uint64_t stride, std::uint32_t width, hipStream_t stream) {
    const char* where = "combine experts";
    Rows a = rowsOf(where, plan, width);
    checkType(where, rows.type);
    checkWeights(where, a, weights, weightType);
    if (!plan.choices) return;
    checkDense(where, rows.data, rows.stride, rows.type, width);
    checkDense(where, y, stride, rows.type, width);
    a.x = rows.data, a.xStride = rows.stride, a.out = y, a.outStride = stride;
    const dim3 grid = gridOf(where, a, false);
    withType(rows.type, [&](auto tag) {
        hipLaunchKernelGGL((combineRows<decltype(tag)>), grid, dim3(kThreads), 0, stream, a);
    });
    checkHip(hipGetLastError());
}

void combineExpertsBackward(DenseMatrix dy, DenseMatrix rows, ExpertPlan plan, const void* weights, DenseType weightType,
                            void* drows, std::uint64_t stride, void* dweights, std::uint32_t width, hipStream_t stream) {
    const char* where = "combine experts backward";
    Rows a = rowsOf(where, plan, width);
    checkType(where, dy.type);
    checkWeights(where, a, weights, weightType);
    if (reinterpret_cast<std::uintptr_t>(dweights) % elementBytes(weightType)) reject(where, "weights not aligned to their type");
    if (!plan.choices) return;
    if (!drows && !dweights) reject(where, "neither the rows' nor the weights' gradient is asked for");
    checkDense(where, dy.data, dy.stride, dy.type, width);
    if (drows) checkDense(where, drows, stride, dy.type, width);
    if (dweights) {
        checkDense(where, rows.data, rows.stride, rows.type, width);
        if (rows.type != dy.type) reject(where, "rows and their sums' gradient must have one type");
    }
    a.dy = dy.data, a.dyStride = dy.stride, a.x = rows.data, a.xStride = rows.stride;
    a.out = drows, a.outStride = stride, a.dweights = dweights;
    const dim3 grid = gridOf(where, a, true);
    withType(dy.type, [&](auto tag) {
        hipLaunchKernelGGL((combineRowsBackward<decltype(tag)>), grid, dim3(kThreads), 0, stream, a);
    });
    checkHip(hipGetLastError());
}

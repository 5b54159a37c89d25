// Activations whose input is kept in 8-bit blocks for the backward pass (include/blocks.h).
//
// One pass each way, bound by HBM: 16 lanes take a block of 128 elements (gated: the gate's block and the
// factor's), 8 a lane. Forward computes y from x itself and the kept blocks from the same registers;
// backward makes x's values from the codes and needs nothing else of the forward pass. Measured: 2,449,029 x 128
// FP32 silu 500 us and back 457, 5.6 and 6.2 TB/s; 16384 x 4096 bf16, gated, 87 and 86 us, 6.2 TB/s; 16384 x 8192
// bf16 silu 133 us, gelu 148 (erf's arithmetic shows), gelu_tanh 135. 333 x 1001: 4.6 us, a launch and its latency.
//
// __expf is off by about its argument times 2^-24 of its value. Where the argument is large, the exponential is
// negligible beside 1 or the result is a small fraction of x; there alone it is off by more than its last bits.
#include "device_blocks.h"
#include "hip_support.h"

namespace {

using namespace blocks;

constexpr unsigned kThreads = 256, kGroups = kThreads / kBlockLanes;

// f(x), and f'(x) where Slope.
template <BlockActivation F, bool Slope> __device__ __forceinline__ void activate(float x, float& f, float& d) {
    if constexpr (F == BlockActivation::silu) {
        const float s = 1.0f / (1.0f + __expf(-x));
        f = x * s;
        if constexpr (Slope) d = s * (1.0f + x * (1.0f - s));
    } else if constexpr (F == BlockActivation::gelu) {
        const float p = 0.5f + 0.5f * erff(x * 0.70710678118654752f);
        f = x * p;
        if constexpr (Slope) d = p + x * 0.39894228040143268f * __expf(-0.5f * x * x);
    } else {
        // tanh(a) = 2 s - 1 with s = 1 / (1 + exp(-2 a)): f = x s
        constexpr float a = 1.5957691216057308f, b = 0.044715f; // 2 sqrt(2 / pi)
        const float q = fminf(x * x, 400.0f); // past |x| = 20 s is 0 or 1, and x^2 may overflow
        const float s = 1.0f / (1.0f + __expf(-a * x * (1.0f + b * q)));
        f = x * s;
        if constexpr (Slope) d = s + x * s * (1.0f - s) * (a + 3.0f * a * b * q);
    }
}

struct Call {
    const void* in; // x, or dy
    std::uint64_t inStride;
    void* out; // y, or dx
    std::uint64_t outStride;
    std::uint8_t *codes, *exponents;
    unsigned items, width, count, magic, expPitch;
};

template <typename T, BlockCodes C>
__device__ __forceinline__ void keepBlock(const Call& a, std::uint64_t row, unsigned block, unsigned lane,
                                          const float (&v)[8]) {
    const unsigned e = exponentOf<C>(rowMax(peakBits(v)));
    storeCodes<T>(a.codes + row * a.count * kBlock + block * kBlock, lane, encode8<C>(v, e));
    if (block + lane < (block + 1 == a.count ? a.expPitch : block + 1))
        a.exponents[row * a.expPitch + block + lane] = std::uint8_t(lane ? 127u : e);
}

template <typename T, BlockCodes C, BlockActivation F, bool Gated>
__global__ __launch_bounds__(kThreads) void activateBlocks(Call a) {
    const unsigned lane = threadIdx.x % kBlockLanes;
    const unsigned item = flatGroup() * kGroups + threadIdx.x / kBlockLanes;
    if (item >= a.items) return;
    const unsigned row = rowOf(item, a.count, a.magic), block = item - row * a.count;
    const unsigned at = block * kBlock;
    const auto* x = static_cast<const typename T::Raw*>(a.in) + row * a.inStride;
    float g[8], u[8], y[8];
    loadBlock<T>(x, at, lane, a.width, g);
    if constexpr (Gated) loadBlock<T>(x + a.width, at, lane, a.width, u);
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
        float d;
        activate<F, false>(g[i], y[i], d);
        if constexpr (Gated) y[i] *= u[i];
    }
    storeBlock<T>(static_cast<typename T::Raw*>(a.out) + row * a.outStride, at, lane, a.width, y);
    if (!a.codes) return;
    if constexpr (Gated) {
        keepBlock<T, C>(a, 2 * std::uint64_t(row), block, lane, g);
        keepBlock<T, C>(a, 2 * std::uint64_t(row) + 1, block, lane, u);
    } else {
        keepBlock<T, C>(a, row, block, lane, g);
    }
}

template <typename T, BlockCodes C>
__device__ __forceinline__ void keptBlock(const Call& a, std::uint64_t row, unsigned block, unsigned lane, float (&v)[8]) {
    const u32x2 q = loadCodes<T>(a.codes + row * a.count * kBlock + block * kBlock, lane);
    decode8<C>(q, scaleOf(a.exponents[row * a.expPitch + block]), v);
}

template <typename T, BlockCodes C, BlockActivation F, bool Gated>
__global__ __launch_bounds__(kThreads) void activateBlocksBackward(Call a) {
    const unsigned lane = threadIdx.x % kBlockLanes;
    const unsigned item = flatGroup() * kGroups + threadIdx.x / kBlockLanes;
    if (item >= a.items) return;
    const unsigned row = rowOf(item, a.count, a.magic), block = item - row * a.count;
    const unsigned at = block * kBlock;
    float dy[8], g[8], u[8];
    loadBlock<T>(static_cast<const typename T::Raw*>(a.in) + row * a.inStride, at, lane, a.width, dy);
    keptBlock<T, C>(a, Gated ? 2 * std::uint64_t(row) : row, block, lane, g);
    if constexpr (Gated) keptBlock<T, C>(a, 2 * std::uint64_t(row) + 1, block, lane, u);
    float dg[8], du[8];
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
        float f, d;
        activate<F, true>(g[i], f, d);
        if constexpr (Gated) {
            dg[i] = dy[i] * u[i] * d;
            du[i] = dy[i] * f;
        } else {
            dg[i] = dy[i] * d;
        }
    }
    auto* dx = static_cast<typename T::Raw*>(a.out) + row * a.outStride;
    storeBlock<T>(dx, at, lane, a.width, dg);
    if constexpr (Gated) storeBlock<T>(dx + a.width, at, lane, a.width, du);
}

template <typename F> void withActivation(BlockActivation k, F f) {
    switch (k) {
    case BlockActivation::silu: f(std::integral_constant<BlockActivation, BlockActivation::silu>{}); break;
    case BlockActivation::gelu: f(std::integral_constant<BlockActivation, BlockActivation::gelu>{}); break;
    case BlockActivation::geluTanh: f(std::integral_constant<BlockActivation, BlockActivation::geluTanh>{}); break;
    }
}

// What both directions check and set up; false if there is nothing to do. `wide` is x or dx.
bool setUp(const char* where, Call& a, const void* narrow, std::uint64_t narrowStride, const void* wide,
           std::uint64_t wideStride, DenseType type, BlockRows kept, bool needKept, BlockActivation f, bool gated,
           std::uint32_t rows, std::uint32_t width) {
    checkColumns(where, width);
    checkRows(where, rows);
    checkType(where, type);
    if (unsigned(f) > 2) reject(where, "unknown activation");
    if (!kept.codes != !kept.exponents) reject(where, "kept codes and exponents come together");
    if (unsigned(kept.type) > 1) reject(where, "unknown code type");
    if (!rows) return false;
    checkDense(where, narrow, narrowStride, type, width);
    checkDense(where, wide, wideStride, type, gated ? 2 * std::uint64_t(width) : width);
    if (needKept || kept.codes) checkCodes(where, kept.codes, kept.exponents);
    a.codes = kept.codes, a.exponents = kept.exponents, a.width = width;
    a.count = (width + kBlock - 1) / kBlock, a.magic = rowMagic(a.count);
    a.expPitch = unsigned(blockExponentPitch(width));
    const std::uint64_t items = std::uint64_t(rows) * a.count;
    if (items >= (std::uint64_t(1) << 32) - kGroups) reject(where, "more than 2^32 blocks");
    a.items = unsigned(items);
    return true;
}

} // namespace

void activationBlocks(DenseMatrix x, BlockActivation f, bool gated, void* y, std::uint64_t yStride, BlockRows keep,
                      std::uint32_t rows, std::uint32_t width, hipStream_t stream) {
    Call a = {};
    if (!setUp("activation blocks", a, y, yStride, x.data, x.stride, x.type, keep, false, f, gated, rows, width)) return;
    a.in = x.data, a.inStride = x.stride, a.out = y, a.outStride = yStride;
    const dim3 grid = flatGrid((a.items + kGroups - 1) / kGroups), threads(kThreads);
    withType(x.type, [&](auto tag) {
        withCodes(keep.type, [&](auto codes) {
            withActivation(f, [&](auto kind) {
                typedef decltype(tag) T;
                if (gated)
                    hipLaunchKernelGGL((activateBlocks<T, decltype(codes)::value, decltype(kind)::value, true>), grid,
                                       threads, 0, stream, a);
                else
                    hipLaunchKernelGGL((activateBlocks<T, decltype(codes)::value, decltype(kind)::value, false>), grid,
                                       threads, 0, stream, a);
            });
        });
    });
    checkHip(hipGetLastError());
}

void activationBlocksBackward(DenseMatrix dy, BlockRows kept, BlockActivation f, bool gated, void* dx,
                              std::uint64_t dxStride, std::uint32_t rows, std::uint32_t width, hipStream_t stream) {
    Call a = {};
    if (!setUp("activation blocks backward", a, dy.data, dy.stride, dx, dxStride, dy.type, kept, true, f, gated, rows,
               width))
        return;
    a.in = dy.data, a.inStride = dy.stride, a.out = dx, a.outStride = dxStride;
    const dim3 grid = flatGrid((a.items + kGroups - 1) / kGroups), threads(kThreads);
    withType(dy.type, [&](auto tag) {
        withCodes(kept.type, [&](auto codes) {
            withActivation(f, [&](auto kind) {
                typedef decltype(tag) T;
                if (gated)
                    hipLaunchKernelGGL((activateBlocksBackward<T, decltype(codes)::value, decltype(kind)::value, true>),
                                       grid, threads, 0, stream, a);
                else
                    hipLaunchKernelGGL((activateBlocksBackward<T, decltype(codes)::value, decltype(kind)::value, false>),
                                       grid, threads, 0, stream, a);
            });
        });
    });
    checkHip(hipGetLastError());
}

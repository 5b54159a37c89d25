// The weight gradient dw = dy^T x from dense dy and the 8-bit blocks of x that the forward pass kept, and
// the bias gradient (include/blocks.h).
//
// Both operands run along the rows, the axis of the sum, so an MFMA operand is a column of each: tiles of
// 64 rows lie in LDS as they do in memory and are read with the transposing LDS load. x is converted to
// bf16 on its way into LDS, exactly, its scales multiplied in. dy goes in as bf16 parts: itself, or for f16 two and
// for f32 three parts of 8 bits each, every part the rest's nearest bf16; their products with x add
// in the same FP32 accumulator, so an f32 gradient keeps its precision at three times the MFMA work.
// The rows are split over workgroups, since a weight has few tiles; each writes its FP32 sums and a second
// kernel adds the splits in order.
#include "device_blocks.h"
#include "hip_support.h"

#include <algorithm>

namespace {

using namespace blocks;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* LdsColumn;

constexpr unsigned kTile = 128, kSteps = 64; // columns of dy and of x; rows of a step
constexpr unsigned kRowBytes = kTile * 2, kPartBytes = kSteps * kRowBytes;

template <typename T> struct Parts { static constexpr unsigned count = 1; };
template <> struct Parts<F16> { static constexpr unsigned count = 2; };
template <> struct Parts<F32> { static constexpr unsigned count = 3; };

// Byte of column c (a multiple of 4) of row r: 32-byte slots of a row are stored in an order that depends
// on the row, so that the 16 rows that a wave's transposing load takes lie in different banks.
__device__ __forceinline__ unsigned slotOf(unsigned r, unsigned c) {
    return r * kRowBytes + ((c / 16) ^ ((r & 3) | ((r >> 1) & 4))) * 32 + c % 16 * 2;
}

// Eight consecutive rows of one column for each lane: rows r0 + 8 * (lane / 16) .., column c0 + lane % 16.
__device__ __forceinline__ bf16x8 columnOf(const std::uint8_t* tile, unsigned r0, unsigned c0, unsigned lane) {
    const unsigned r = r0 + lane / 16 * 8 + lane % 16 / 4, c = c0 + lane % 4 * 4;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsColumn)(tile + slotOf(r, c)));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsColumn)(tile + slotOf(r + 4, c)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(bf16x8, s16x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w});
}

struct Gradient {
    const void* dy;
    std::uint64_t dyStride;
    const std::uint8_t *x, *xe;
    float *dw, *db; // the splits' sums, or the results where there is one split
    unsigned rows, outer, inner, codePitch, expPitch, tilesN, tilesK, rowsPerSplit;
};

template <typename T>
__global__ __launch_bounds__(256) void sumRows(Gradient a) {
    constexpr unsigned P = Parts<T>::count;
    extern __shared__ __align__(1024) std::uint8_t lds[]; // dy's parts, then x
    const unsigned t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    const unsigned tile = blockIdx.x % (a.tilesN * a.tilesK), split = blockIdx.x / (a.tilesN * a.tilesK);
    const unsigned n0 = tile % a.tilesN * kTile, k0 = tile / a.tilesN * kTile;
    const unsigned first = split * a.rowsPerSplit, last = min(first + a.rowsPerSplit, a.rows);
    const auto* dy = static_cast<const typename T::Raw*>(a.dy);
    // A thread takes columns 8 * (t % 16) .. of rows t / 16 + 16 i of dy, and 16 codes of rows t / 8 + 32 i of x.
    const unsigned dyColumn = t % 16 * 8, dyRow = t / 16, xColumn = t % 8 * 16, xRow = t / 8;
    float v[4][8], sums[8] = {};
    u32x4 q[2];
    unsigned e[2];
    auto fetch = [&](unsigned row) {
#pragma unroll
        for (unsigned i = 0; i < 4; ++i) {
            const unsigned r = row + dyRow + 16 * i;
            if (r < last) {
                load8<T>(dy + r * a.dyStride, n0 + dyColumn, a.outer, v[i]);
            } else {
#pragma unroll
                for (unsigned j = 0; j < 8; ++j) v[i][j] = 0.0f;
            }
        }
#pragma unroll
        for (unsigned i = 0; i < 2; ++i) {
            const std::uint64_t r = row + xRow + 32 * i;
            q[i] = u32x4{0, 0, 0, 0};
            e[i] = 127;
            if (r < last) {
                q[i] = *reinterpret_cast<const u32x4*>(a.x + r * a.codePitch + k0 + xColumn);
                e[i] = a.xe[r * a.expPitch + k0 / kBlock];
            }
        }
    };
    auto stash = [&] {
#pragma unroll
        for (unsigned i = 0; i < 4; ++i) {
            float rest[8];
#pragma unroll
            for (unsigned j = 0; j < 8; ++j) rest[j] = v[i][j], sums[j] += v[i][j];
#pragma unroll
            for (unsigned p = 0; p < P; ++p) {
                bf16x8 part;
#pragma unroll
                for (unsigned j = 0; j < 8; ++j) {
                    part[j] = __bf16(rest[j]);
                    if (p + 1 < P) rest[j] -= float(part[j]);
                }
                *reinterpret_cast<bf16x8*>(lds + p * kPartBytes + slotOf(dyRow + 16 * i, dyColumn)) = part;
            }
        }
#pragma unroll
        for (unsigned i = 0; i < 2; ++i) {
            const float s = scaleOf(e[i]);
            std::uint8_t* to = lds + P * kPartBytes;
#pragma unroll
            for (unsigned h = 0; h < 2; ++h) {
                bf16x8 w;
#pragma unroll
                for (unsigned j = 0; j < 2; ++j) {
                    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i][2 * h + j], s, false);
                    const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i][2 * h + j], s, true);
                    w[4 * j] = lo.x, w[4 * j + 1] = lo.y, w[4 * j + 2] = hi.x, w[4 * j + 3] = hi.y;
                }
                *reinterpret_cast<bf16x8*>(to + slotOf(xRow + 32 * i, xColumn + 8 * h)) = w;
            }
        }
    };
    const unsigned wn = wave % 2 * 64, wk = wave / 2 * 64;
    f32x4 acc[4][4] = {}; // dy's columns by x's
    if (first < last) fetch(first);
    for (unsigned row = first; row < last; row += kSteps) {
        stash();
        __syncthreads();
        if (row + kSteps < last) fetch(row + kSteps);
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
            bf16x8 xf[4];
#pragma unroll
            for (unsigned k = 0; k < 4; ++k) xf[k] = columnOf(lds + P * kPartBytes, 32 * h, wk + 16 * k, lane);
#pragma unroll
            for (unsigned n = 0; n < 4; ++n)
#pragma unroll
                for (unsigned p = 0; p < P; ++p) {
                    const bf16x8 df = columnOf(lds + p * kPartBytes, 32 * h, wn + 16 * n, lane);
#pragma unroll
                    for (unsigned k = 0; k < 4; ++k)
                        acc[n][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[k], df, acc[n][k], 0, 0, 0);
                }
        }
        __syncthreads();
    }
    // x was the first operand: a lane has 4 consecutive columns of x for one of dy's.
    float* dw = a.dw + std::uint64_t(split) * a.outer * a.inner;
#pragma unroll
    for (unsigned n = 0; n < 4; ++n) {
        const unsigned row = n0 + wn + 16 * n + lane % 16;
        if (row >= a.outer) continue;
#pragma unroll
        for (unsigned k = 0; k < 4; ++k) {
            const unsigned column = k0 + wk + 16 * k + lane / 16 * 4;
            float* to = dw + std::uint64_t(row) * a.inner + column;
#pragma unroll
            for (unsigned i = 0; i < 4; ++i)
                if (column + i < a.inner) to[i] = acc[n][k][i];
        }
    }
    if (a.db && k0 == 0) {
        // Column sums: the 16 threads with the same columns add theirs through LDS.
        float* part = reinterpret_cast<float*>(lds);
#pragma unroll
        for (unsigned j = 0; j < 8; ++j) part[dyRow * kTile + dyColumn + j] = sums[j];
        __syncthreads();
        if (t < kTile && n0 + t < a.outer) {
            float s = 0.0f;
            for (unsigned r = 0; r < 16; ++r) s += part[r * kTile + t];
            a.db[std::uint64_t(split) * a.outer + n0 + t] = s;
        }
    }
}

// out = the sum of `splits` arrays of n floats, in order.
__global__ __launch_bounds__(256) void addSplits(const float* __restrict__ parts, float* __restrict__ out,
                                                  std::uint64_t n, unsigned splits) {
    const std::uint64_t i = std::uint64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= n) return;
    float s = 0.0f;
    for (unsigned k = 0; k < splits; ++k) s += parts[k * n + i];
    out[i] = s;
}

unsigned splitsOf(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer) {
    const std::uint64_t tiles = std::uint64_t((inner + kTile - 1) / kTile) * ((outer + kTile - 1) / kTile);
    const std::uint64_t steps = (std::uint64_t(rows) + kSteps - 1) / kSteps;
    const std::uint64_t want = (1024 + tiles - 1) / tiles, most = std::max<std::uint64_t>(1, steps / 4);
    return unsigned(std::max<std::uint64_t>(1, std::min(want, most)));
}

} // namespace

std::size_t weightGradBlocksWorkspace(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType) {
    const unsigned splits = splitsOf(rows, inner, outer);
    return splits == 1 ? 0 : std::size_t(splits) * (std::size_t(outer) * inner + outer) * sizeof(float);
}

void weightGradBlocks(DenseMatrix dy, BlockRows x, float* dw, float* db, std::uint32_t rows, std::uint32_t inner,
                      std::uint32_t outer, void* workspace, std::size_t workspaceBytes, hipStream_t stream) {
    const char* where = "weight gradient";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkRows(where, rows);
    checkType(where, dy.type);
    if (x.type != BlockCodes::e4m3) reject(where, "x must have E4M3 codes");
    if (!dw) reject(where, "null weight gradient");
    if (reinterpret_cast<std::uintptr_t>(dw) % 4 || reinterpret_cast<std::uintptr_t>(db) % 4)
        reject(where, "gradients must be float-aligned");
    if (rows) {
        checkDense(where, dy.data, dy.stride, dy.type, outer);
        checkCodes(where, x.codes, x.exponents);
    }
    const unsigned splits = splitsOf(rows, inner, outer);
    const std::size_t need = weightGradBlocksWorkspace(rows, inner, outer, dy.type);
    if (need > workspaceBytes || (need && !workspace)) reject(where, "workspace too small");
    if (reinterpret_cast<std::uintptr_t>(workspace) % 16) reject(where, "workspace must be 16-byte aligned");
    Gradient a = {};
    a.dy = dy.data, a.dyStride = dy.stride, a.x = x.codes, a.xe = x.exponents;
    a.rows = rows, a.outer = outer, a.inner = inner;
    a.codePitch = unsigned(blockCodePitch(inner)), a.expPitch = unsigned(blockExponentPitch(inner));
    a.tilesN = (outer + kTile - 1) / kTile, a.tilesK = (inner + kTile - 1) / kTile;
    const unsigned steps = (rows + kSteps - 1) / kSteps;
    a.rowsPerSplit = std::max(1u, (steps + splits - 1) / splits) * kSteps;
    const std::uint64_t size = std::uint64_t(outer) * inner;
    auto* parts = static_cast<float*>(workspace);
    a.dw = splits == 1 ? dw : parts;
    a.db = !db ? nullptr : splits == 1 ? db : parts + splits * size;
    const std::uint64_t blocks = std::uint64_t(a.tilesN) * a.tilesK * splits;
    if (blocks >> 31) reject(where, "more than 2^31 tiles");
    withType(dy.type, [&](auto tag) {
        typedef decltype(tag) T;
        hipLaunchKernelGGL((sumRows<T>), dim3(unsigned(blocks)), dim3(256), (Parts<T>::count + 1) * kPartBytes, stream,
                           a);
    });
    checkHip(hipGetLastError());
    if (splits > 1) {
        hipLaunchKernelGGL(addSplits, dim3(unsigned((size + 255) / 256)), dim3(256), 0, stream, parts, dw, size, splits);
        if (db)
            hipLaunchKernelGGL(addSplits, dim3((outer + 255) / 256), dim3(256), 0, stream, parts + splits * size, db,
                               std::uint64_t(outer), splits);
        checkHip(hipGetLastError());
    }
}

// Quantization into microscaled 4-bit blocks (include/micro.h), for rows and for weights in tiles, and back.
//
// Rows: 16 lanes take 128 elements, 8 a lane, as in the 8-bit quantizer; a block's peak is two or three DPP steps. Bound by
// HBM: 8192 x 8192 bf16 33 us, 5.1 TB/s of reads and writes, and back 24 us, 7.0 TB/s, part of it from the last cache; 333 x 1001
// 3 us, a launch's length.
//
// Weights in tiles: a workgroup takes 128 x 128 elements, 16 tiles, in registers, finds their peaks through LDS and writes the
// codes and the transposed copy, whose half bytes are turned in LDS. 4097 x 1024 FP32 10.2 us with both, one round of loads,
// peaks and stores that follow each other.
#include "hip_support.h"
#include "micro/device_micro.h"

namespace {

using namespace micro;

constexpr unsigned kThreads = 256;
constexpr unsigned kGroups = kThreads / kBlockLanes;

// A lane's elements, as loadBlock gives them: 8 in a row, all of block lane / 4, or, of FP32, four of each half, of
// blocks lane / 8 and 2 + lane / 8.
template <typename T> constexpr bool kHalves = std::is_same<T, F32>::value;

template <typename T>
__global__ __launch_bounds__(kThreads) void quantizeMicroRows(const typename T::Raw* __restrict__ x, std::uint64_t stride,
                                                               MicroRows out, std::uint64_t expRow, std::uint64_t expNext,
                                                               unsigned items, unsigned columns, unsigned count,
                                                               unsigned magic) {
    const unsigned lane = threadIdx.x % kBlockLanes;
    const unsigned item = flatGroup() * kGroups + threadIdx.x / kBlockLanes;
    if (item >= items) return;
    const unsigned row = rowOf(item, count, magic), step = item - row * count;
    float v[8];
    loadBlock<T>(x + row * stride, step * kStep, lane, columns, v);
    std::uint8_t* codes = out.codes + (std::uint64_t(row) * count + step) * (kStep / 2);
    unsigned e, block;
    if constexpr (kHalves<T>) {
        unsigned lo = 0, hi = 0;
#pragma unroll
        for (unsigned i = 0; i < 4; ++i) {
            lo = max(lo, __float_as_uint(v[i]) & 0x7FFFFFFFu);
            hi = max(hi, __float_as_uint(v[4 + i]) & 0x7FFFFFFFu);
        }
        const unsigned e0 = microExponent(max8(lo)), e1 = microExponent(max8(hi));
        *reinterpret_cast<std::uint16_t*>(codes + lane * 2) = std::uint16_t(microEncode<4>(v, e0));
        *reinterpret_cast<std::uint16_t*>(codes + kStep / 4 + lane * 2) = std::uint16_t(microEncode<4>(v + 4, e1));
        const bool upper = lane / 4 % 2;
        e = upper ? e1 : e0, block = lane / 8 + 2 * upper;
    } else {
        e = microExponent(max4(peakBits(v))), block = lane / 4;
        *reinterpret_cast<unsigned*>(codes + lane * 4) = microEncode<8>(v, e);
    }
    // Four lanes have each block's exponent: one writes it, the others, at the row's last step, fill the dword.
    const unsigned j = lane % 4;
    if (j == 0 || (step + 1 == count && step % 4 + j < 4))
        out.exponents[row * expRow + step / 4 * expNext + exponentAt(step % 4, block) + j] = std::uint8_t(j ? 127u : e);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dequantizeMicroRows(const std::uint8_t* __restrict__ codes,
                                                                 const std::uint8_t* __restrict__ exponents,
                                                                 typename T::Raw* __restrict__ out, std::uint64_t stride,
                                                                 unsigned items, unsigned columns, unsigned count,
                                                                 unsigned magic) {
    const unsigned lane = threadIdx.x % kBlockLanes;
    const unsigned item = flatGroup() * kGroups + threadIdx.x / kBlockLanes;
    if (item >= items) return;
    const unsigned row = rowOf(item, count, magic), step = item - row * count;
    const std::uint8_t* from = codes + (std::uint64_t(row) * count + step) * (kStep / 2);
    const std::uint8_t* exps = exponents + std::uint64_t(row) * ((count + 3) / 4 * 16);
    float v[8];
    if constexpr (kHalves<T>) {
        const float s0 = scaleOf(exps[exponentAt(step, lane / 8)]), s1 = scaleOf(exps[exponentAt(step, 2 + lane / 8)]);
        microDecode4(*reinterpret_cast<const std::uint16_t*>(from + lane * 2), s0, v);
        microDecode4(*reinterpret_cast<const std::uint16_t*>(from + kStep / 4 + lane * 2), s1, v + 4);
    } else {
        const float s = scaleOf(exps[exponentAt(step, lane / 4)]);
        const unsigned q = *reinterpret_cast<const unsigned*>(from + lane * 4);
        microDecode4(q, s, v);
        microDecode4(q >> 16, s, v + 4);
    }
    storeBlock<T>(out + row * stride, step * kStep, lane, columns, v);
}

// Thread t holds eight groups of 8 elements: rows
// i * 16 + t / 16, columns 8 * (t % 16). LDS keeps a byte a code for the transposed copy.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantizeMicroTiles(const typename T::Raw* __restrict__ w, std::uint64_t stride,
                                                                MicroRows out, MicroRows outT, unsigned outer,
                                                                unsigned inner) {
    constexpr unsigned kRowBytes = kStep + 4;
    __shared__ unsigned peaks[kThreads / kWave][4][4]; // of a wave's rows: [wave][row of tiles][column of tiles]
    __shared__ unsigned scales[4][4]; // exponents of the tiles
    __shared__ __align__(16) std::uint8_t turned[kStep * kRowBytes];
    const unsigned t = threadIdx.x, lane = t % kBlockLanes, group = t / kBlockLanes;
    const unsigned across = (inner + kStep - 1) / kStep, up = (outer + kStep - 1) / kStep;
    const unsigned tileX = blockIdx.x % across, tileY = blockIdx.x / across;
    const std::uint64_t first = std::uint64_t(blockIdx.y) * outer, firstT = std::uint64_t(blockIdx.y) * inner;
    float v[8][8];
    unsigned peak[4] = {};
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
        const unsigned row = tileY * kStep + i * 16 + group;
        if (row < outer) {
            load8<T>(w + (first + row) * stride, tileX * kStep + lane * 8, inner, v[i]);
        } else {
#pragma unroll
            for (unsigned j = 0; j < 8; ++j) v[i][j] = 0.0f;
        }
        peak[i / 2] = max(peak[i / 2], peakBits(v[i]));
    }
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
        peak[i] = max4(peak[i]);
        peak[i] = max(peak[i], unsigned(__shfl_xor(int(peak[i]), 16)));
        peak[i] = max(peak[i], unsigned(__shfl_xor(int(peak[i]), 32)));
        if (t % kWave < kBlockLanes && lane % 4 == 0) peaks[t / kWave][i][lane / 4] = peak[i];
    }
    __syncthreads();
    unsigned e[4];
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
        unsigned m = 0;
#pragma unroll
        for (unsigned wave = 0; wave < kThreads / kWave; ++wave) m = max(m, peaks[wave][i][lane / 4]);
        e[i] = microExponent(m);
    }
    const std::uint64_t pitch = across * std::uint64_t(kStep / 2), pitchT = up * std::uint64_t(kStep / 2);
    const unsigned expPitch = (across + 3) / 4 * 16, expPitchT = (up + 3) / 4 * 16;
    const unsigned j = lane % 4;
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
        const unsigned in = i * 16 + group, row = tileY * kStep + in;
        const unsigned q = microEncode<8>(v[i], e[i / 2]);
        if (row < outer) {
            *reinterpret_cast<unsigned*>(out.codes + (first + row) * pitch + tileX * (kStep / 2) + lane * 4) = q;
            if (j == 0 || (tileX + 1 == across && tileX % 4 + j < 4))
                out.exponents[(first + row) * expPitch + exponentAt(tileX, lane / 4) + j] =
                    std::uint8_t(j ? 127u : e[i / 2]);
        }
        if (!outT.codes) continue;
        // A byte a code, four to a dword.
        unsigned bytes[2];
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
            const unsigned c = q >> 16 * h & 0xFFFFu, d = (c | c << 8) & 0x00FF00FFu;
            bytes[h] = (d | d << 4) & 0x0F0F0F0Fu;
        }
        *reinterpret_cast<unsigned*>(turned + in * kRowBytes + lane * 8) = bytes[0];
        *reinterpret_cast<unsigned*>(turned + in * kRowBytes + lane * 8 + 4) = bytes[1];
    }
    if (!outT.codes) return;
    if (t / kBlockLanes == 0 && j == 0)
#pragma unroll
        for (unsigned i = 0; i < 4; ++i) scales[i][lane / 4] = e[i];
    __syncthreads();
    // Two threads a transposed row, 64 codes each.
    const unsigned column = t / 2, half = t % 2, to = tileX * kStep + column;
    if (to >= inner) return;
    u32x4 q[2];
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
        unsigned word = 0;
#pragma unroll
        for (unsigned k = 0; k < 8; ++k)
            word |= unsigned(turned[(half * 64 + i * 8 + k) * kRowBytes + column]) << 4 * k;
        q[i / 4][i % 4] = word;
    }
    std::uint8_t* row = outT.codes + (firstT + to) * pitchT + tileY * (kStep / 2) + half * 32;
    *reinterpret_cast<u32x4*>(row) = q[0];
    *reinterpret_cast<u32x4*>(row + 16) = q[1];
    std::uint8_t* exps = outT.exponents + (firstT + to) * expPitchT;
    const unsigned end = tileY + 1 == up ? 4 : tileY % 4 + 1;
#pragma unroll
    for (unsigned b = 0; b < 2; ++b) {
        const unsigned block = half * 2 + b;
        for (unsigned k = tileY % 4; k < end; ++k)
            exps[tileY / 4 * 16 + block * 4 + k] =
                std::uint8_t(k == tileY % 4 ? scales[block][column / 32] : 127u);
    }
}

unsigned itemsOf(const char* where, std::uint32_t rows, unsigned count) {
    const std::uint64_t items = std::uint64_t(rows) * count;
    if (items >= (std::uint64_t(1) << 32) - kGroups) reject(where, "more than 2^32 runs of 128 elements");
    return unsigned(items);
}

} // namespace

void quantizeMicro(DenseMatrix x, MicroRows out, std::uint32_t rows, std::uint32_t columns, hipStream_t stream) {
    quantizeMicroRowsTo(x, out, false, rows, columns, stream);
}

void quantizeMicroRowsTo(DenseMatrix x, MicroRows out, bool packed, std::uint32_t rows, std::uint32_t columns,
                         hipStream_t stream) {
    const char* where = "quantize micro";
    checkColumns(where, columns);
    checkRows(where, rows);
    if (!rows) return;
    checkDense(where, x.data, x.stride, x.type, columns);
    checkMicro(where, out);
    const unsigned count = (columns + kStep - 1) / kStep, items = itemsOf(where, rows, count);
    const dim3 grid = flatGrid((items + kGroups - 1) / kGroups);
    withType(x.type, [&](auto tag) {
        typedef decltype(tag) T;
        hipLaunchKernelGGL((quantizeMicroRows<T>), grid, dim3(kThreads), 0, stream,
                           static_cast<const typename T::Raw*>(x.data), x.stride, out,
                           packed ? 16 : microExponentPitch(columns), packed ? std::uint64_t(rows) * 16 : 16, items, columns,
                           count, rowMagic(count));
    });
    checkHip(hipGetLastError());
}

void dequantizeMicro(MicroRows x, void* out, DenseType type, std::uint64_t stride, std::uint32_t rows,
                     std::uint32_t columns, hipStream_t stream) {
    const char* where = "dequantize micro";
    checkColumns(where, columns);
    checkRows(where, rows);
    if (!rows) return;
    checkDense(where, out, stride, type, columns);
    checkMicro(where, x);
    const unsigned count = (columns + kStep - 1) / kStep, items = itemsOf(where, rows, count);
    const dim3 grid = flatGrid((items + kGroups - 1) / kGroups);
    withType(type, [&](auto tag) {
        typedef decltype(tag) T;
        hipLaunchKernelGGL((dequantizeMicroRows<T>), grid, dim3(kThreads), 0, stream, x.codes, x.exponents,
                           static_cast<typename T::Raw*>(out), stride, items, columns, count, rowMagic(count));
    });
    checkHip(hipGetLastError());
}

void quantizeWeightMicro(DenseMatrix w, MicroRows out, MicroRows outT, std::uint32_t experts, std::uint32_t outer,
                         std::uint32_t inner, hipStream_t stream) {
    const char* where = "quantize micro weight";
    checkColumns(where, inner);
    checkColumns(where, outer);
    if (!experts || experts > 65535) reject(where, "stacks are of 1 to 65,535 weights");
    checkDense(where, w.data, w.stride, w.type, inner);
    checkMicro(where, out);
    if (!outT.codes != !outT.exponents) reject(where, "transposed codes and exponents come together");
    if (outT.codes) checkMicro(where, outT);
    const std::uint64_t tiles = std::uint64_t((inner + kStep - 1) / kStep) * ((outer + kStep - 1) / kStep);
    checkGrid(where, tiles, kThreads);
    withType(w.type, [&](auto tag) {
        typedef decltype(tag) T;
        hipLaunchKernelGGL((quantizeMicroTiles<T>), dim3(unsigned(tiles), experts), dim3(kThreads), 0, stream,
                           static_cast<const typename T::Raw*>(w.data), w.stride, out, outT, outer, inner);
    });
    checkHip(hipGetLastError());
}

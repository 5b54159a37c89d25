// Quantization into 8-bit blocks (include/blocks.h), for rows and for weights, and back.
//
// Rows: 16 lanes take one block of 128 elements, 8 a lane: one load (two at FP32), the peak by four DPP
// steps inside the lanes' DPP row, one 8-byte store of codes. Bound by HBM: 1,000,000 x 256 bf16 137 us and
// FP32 218, 5.6 and 5.9 TB/s; 8192 x 2048 bf16 11.7 us (four blocks a thread, loaded together, 12.8). Below about
// 1000 x 1024 it is the launch and one load after the other, 3 us. Back: 1,000,000 x 256 FP32 193 us, 6.7 TB/s.
//
// Weights: a workgroup takes one tile of 128 x 128, 64 elements a thread in registers, finds the tile's
// peak through LDS and writes the codes and, for the input gradient, the transposed codes, whose
// bytes are turned in LDS. 8192 x 8192 FP32 72 us with both copies, 5.6 TB/s; 4096 x 1024, one tile a unit, 8.2 us:
// loads, peak and stores follow each other there with nothing to hide them.
#include "device_blocks.h"
#include "hip_support.h"

namespace {

using namespace blocks;

constexpr unsigned kThreads = 256;
constexpr unsigned kGroups = kThreads / kBlockLanes;

template <typename T, BlockCodes C>
__global__ __launch_bounds__(kThreads) void quantizeRowBlocks(const typename T::Raw* __restrict__ x,
                                                               std::uint64_t stride,
                                                               std::uint8_t* __restrict__ codes,
                                                               std::uint8_t* __restrict__ exponents,
                                                               unsigned items, unsigned columns,
                                                               unsigned count, unsigned magic) {
    const unsigned lane = threadIdx.x % kBlockLanes;
    const unsigned item = flatGroup() * kGroups + threadIdx.x / kBlockLanes;
    if (item >= items) return;
    const unsigned codePitch = count * kBlock, exponentPitch = (count + 3) / 4 * 4;
    const unsigned row = rowOf(item, count, magic), block = item - row * count;
    float v[8];
    loadBlock<T>(x + row * stride, block * kBlock, lane, columns, v);
    const unsigned e = exponentOf<C>(rowMax(peakBits(v)));
    storeCodes<T>(codes + std::uint64_t(row) * codePitch + block * kBlock, lane, encode8<C>(v, e));
    // The row's last block fills the exponents up to a multiple of four with it.
    const unsigned end = block + 1 == count ? exponentPitch : block + 1;
    if (block + lane < end)
        exponents[std::uint64_t(row) * exponentPitch + block + lane] = std::uint8_t(lane ? 127u : e);
}

template <typename T, BlockCodes C>
__global__ __launch_bounds__(kThreads) void dequantizeRowBlocks(const std::uint8_t* __restrict__ codes,
                                                                 const std::uint8_t* __restrict__ exponents,
                                                                 typename T::Raw* __restrict__ out,
                                                                 std::uint64_t stride, unsigned items,
                                                                 unsigned columns, unsigned count,
                                                                 unsigned magic) {
    const unsigned lane = threadIdx.x % kBlockLanes;
    const unsigned item = flatGroup() * kGroups + threadIdx.x / kBlockLanes;
    if (item >= items) return;
    const unsigned row = rowOf(item, count, magic), block = item - row * count;
    const std::uint8_t* from = codes + std::uint64_t(row) * count * kBlock + block * kBlock;
    const float scale = scaleOf(exponents[std::uint64_t(row) * ((count + 3) / 4 * 4) + block]);
    float v[8];
    decode8<C>(loadCodes<T>(from, lane), scale, v);
    storeBlock<T>(out + row * stride, block * kBlock, lane, columns, v);
}

// Thread t takes row t / 2's half t % 2 of the tile in eight groups of 8 elements, in the order that
// lets the 16 threads of 8 rows write whole 16-byte chunks. LDS keeps the codes for the transposed copy
// with rows 4 bytes longer than a tile, so that a column's bytes lie in different banks.
template <typename T>
__global__ __launch_bounds__(kThreads) void quantizeWeightTiles(const typename T::Raw* __restrict__ w,
                                                                 std::uint64_t stride, BlockWeightView out,
                                                                 unsigned outer, unsigned inner) {
    constexpr unsigned kRowBytes = kBlock + 4;
    __shared__ unsigned peaks[kThreads / kWave];
    __shared__ __align__(16) std::uint8_t turned[kBlock * kRowBytes];
    const unsigned t = threadIdx.x, lane = t % kBlockLanes, group = t / kBlockLanes;
    const unsigned across = (inner + kBlock - 1) / kBlock, up = (outer + kBlock - 1) / kBlock;
    const unsigned tileX = blockIdx.x % across, tileY = blockIdx.x / across;
    float v[8][8];
    unsigned peak = 0;
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
        const unsigned row = tileY * kBlock + i * 16 + group;
        if (row < outer) {
            load8<T>(w + row * stride, tileX * kBlock + lane * 8, inner, v[i]);
        } else {
#pragma unroll
            for (unsigned j = 0; j < 8; ++j) v[i][j] = 0.0f;
        }
        peak = max(peak, peakBits(v[i]));
    }
    peak = rowMax(peak);
    peak = max(peak, unsigned(__shfl_xor(int(peak), 16)));
    peak = max(peak, unsigned(__shfl_xor(int(peak), 32)));
    if (t % kWave == 0) peaks[t / kWave] = peak;
    __syncthreads();
    peak = max(max(peaks[0], peaks[1]), max(peaks[2], peaks[3]));
    const unsigned e = exponentOf<BlockCodes::e4m3>(peak);
    const std::uint64_t pitch = across * std::uint64_t(kBlock);
    const unsigned expPitch = (across + 3) / 4 * 4, expPitchT = (up + 3) / 4 * 4;
    if (t < 4) {
        if (tileX + t < (tileX + 1 == across ? expPitch : tileX + 1))
            out.exponents[std::uint64_t(tileY) * expPitch + tileX + t] = std::uint8_t(t ? 127u : e);
        if (out.codesT && tileY + t < (tileY + 1 == up ? expPitchT : tileY + 1))
            out.exponentsT[std::uint64_t(tileX) * expPitchT + tileY + t] = std::uint8_t(t ? 127u : e);
    }
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) {
        const unsigned in = i * 16 + group, row = tileY * kBlock + in;
        const u32x2 q = encode8<BlockCodes::e4m3>(v[i], e);
        if (row < outer) *reinterpret_cast<u32x2*>(out.codes + row * pitch + tileX * kBlock + lane * 8) = q;
        if (out.codesT) {
            *reinterpret_cast<unsigned*>(turned + in * kRowBytes + lane * 8) = q.x;
            *reinterpret_cast<unsigned*>(turned + in * kRowBytes + lane * 8 + 4) = q.y;
        }
    }
    if (!out.codesT) return;
    __syncthreads();
    // A thread turns 16 rows of 4 columns, dwords of 4 rows at a time: a transposed row is 8 threads.
    const std::uint64_t pitchT = up * std::uint64_t(kBlock);
    const unsigned column = t / 8 * 4, from = t % 8 * 16;
    u32x4 q[4];
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
        unsigned r[4];
#pragma unroll
        for (unsigned i = 0; i < 4; ++i)
            r[i] = *reinterpret_cast<const unsigned*>(turned + (from + 4 * j + i) * kRowBytes + column);
        const unsigned ab0 = __builtin_amdgcn_perm(r[1], r[0], 0x05010400), ab2 = __builtin_amdgcn_perm(r[1], r[0], 0x07030602);
        const unsigned cd0 = __builtin_amdgcn_perm(r[3], r[2], 0x05010400), cd2 = __builtin_amdgcn_perm(r[3], r[2], 0x07030602);
        q[0][j] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100);
        q[1][j] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302);
        q[2][j] = __builtin_amdgcn_perm(cd2, ab2, 0x05040100);
        q[3][j] = __builtin_amdgcn_perm(cd2, ab2, 0x07060302);
    }
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
        const unsigned to = tileX * kBlock + column + i;
        if (to < inner) *reinterpret_cast<u32x4*>(out.codesT + to * pitchT + tileY * kBlock + from) = q[i];
    }
}

unsigned itemsOf(const char* where, std::uint32_t rows, unsigned count) {
    const std::uint64_t items = std::uint64_t(rows) * count;
    if (items >= (std::uint64_t(1) << 32) - kGroups) reject(where, "more than 2^32 blocks");
    return unsigned(items);
}

} // namespace

void quantizeBlocks(DenseMatrix x, BlockRows out, std::uint32_t rows, std::uint32_t columns, hipStream_t stream) {
    checkColumns("quantize blocks", columns);
    checkRows("quantize blocks", rows);
    if (unsigned(out.type) > 1) reject("quantize blocks", "unknown code type");
    if (!rows) return;
    checkDense("quantize blocks", x.data, x.stride, x.type, columns);
    checkCodes("quantize blocks", out.codes, out.exponents);
    const unsigned count = (columns + kBlock - 1) / kBlock, items = itemsOf("quantize blocks", rows, count);
    const dim3 grid = flatGrid((items + kGroups - 1) / kGroups);
    withType(x.type, [&](auto tag) {
        withCodes(out.type, [&](auto kind) {
            typedef decltype(tag) T;
            hipLaunchKernelGGL((quantizeRowBlocks<T, decltype(kind)::value>), grid, dim3(kThreads), 0, stream,
                               static_cast<const typename T::Raw*>(x.data), x.stride, out.codes, out.exponents, items,
                               columns, count, rowMagic(count));
        });
    });
    checkHip(hipGetLastError());
}

void dequantizeBlocks(BlockRows x, void* out, DenseType type, std::uint64_t stride, std::uint32_t rows,
                      std::uint32_t columns, hipStream_t stream) {
    checkColumns("dequantize blocks", columns);
    checkRows("dequantize blocks", rows);
    if (unsigned(x.type) > 1) reject("dequantize blocks", "unknown code type");
    if (!rows) return;
    checkDense("dequantize blocks", out, stride, type, columns);
    checkCodes("dequantize blocks", x.codes, x.exponents);
    const unsigned count = (columns + kBlock - 1) / kBlock, items = itemsOf("dequantize blocks", rows, count);
    const dim3 grid = flatGrid((items + kGroups - 1) / kGroups);
    withType(type, [&](auto tag) {
        typedef decltype(tag) T;
        auto* data = static_cast<typename T::Raw*>(out);
        if (x.type == BlockCodes::e4m3)
            hipLaunchKernelGGL((dequantizeRowBlocks<T, BlockCodes::e4m3>), grid, dim3(kThreads), 0, stream,
                               x.codes, x.exponents, data, stride, items, columns, count, rowMagic(count));
        else
            hipLaunchKernelGGL((dequantizeRowBlocks<T, BlockCodes::int8>), grid, dim3(kThreads), 0, stream,
                               x.codes, x.exponents, data, stride, items, columns, count, rowMagic(count));
    });
    checkHip(hipGetLastError());
}

void quantizeWeightBlocks(DenseMatrix w, BlockWeightView out, std::uint32_t outer, std::uint32_t inner,
                          hipStream_t stream) {
    const char* where = "quantize weight";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkDense(where, w.data, w.stride, w.type, inner);
    checkCodes(where, out.codes, out.exponents);
    if (!out.codesT != !out.exponentsT) reject(where, "transposed codes and exponents come together");
    if (out.codesT) checkCodes(where, out.codesT, out.exponentsT);
    const std::uint64_t tiles = std::uint64_t((inner + kBlock - 1) / kBlock) * ((outer + kBlock - 1) / kBlock);
    checkGrid(where, tiles, kThreads);
    withType(w.type, [&](auto tag) {
        typedef decltype(tag) T;
        hipLaunchKernelGGL((quantizeWeightTiles<T>), dim3(unsigned(tiles)), dim3(kThreads), 0, stream,
                           static_cast<const typename T::Raw*>(w.data), w.stride, out, outer, inner);
    });
    checkHip(hipGetLastError());
}

// The weight gradient dw = dy^T x from dense dy and the 8-bit blocks of x that the forward pass kept, and
// the bias gradient (include/blocks.h).
//
// Both operands run along the rows, the axis of the sum, so an MFMA operand is a column of each: 64 rows
// of a tile lie in LDS as they do in memory and are read with the transposing LDS load. x is converted to
// bf16 on its way into LDS, its scales multiplied in, exactly for exponents of 3 to 246 (below, bf16's last
// place is 2^-133; above, values end at 2^128). dy goes in as bf16 parts: itself, or for f16 two
// and for f32 three parts of 8 bits each, every part the rest's nearest bf16; their products with x add
// in the same FP32 accumulator, so an f32 gradient keeps its precision at three times the MFMA work.
// The bias gradient is the product of dy with a column of ones, an operand that needs no memory.
// The rows are split over workgroups where a weight has few tiles; each writes its FP32 sums and a second
// kernel adds the splits in order, so repeated calls give the same bits.
#include "device_blocks.h"
#include "hip_support.h"

#include <algorithm>
#include <type_traits>

namespace {

using namespace blocks;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4* LdsColumn;

constexpr unsigned kStep = 64; // rows of a step

template <typename T> struct Parts { static constexpr unsigned count = 1; };
template <> struct Parts<F16> { static constexpr unsigned count = 2; };
template <> struct Parts<F32> { static constexpr unsigned count = 3; };

// A tile of kStep rows of Columns bf16 values in LDS. The 32-byte slots of a row (16 values) are stored in
// an order that depends on the row, its key: a wave's transposing load takes one slot of rows r0 + 8 i + j
// (i, j < 4), which 64 banks of 4 bytes serve in two turns if they spread over all of them.
// (Pairs: for operands of 32 columns half a wave takes two slots of four rows at a time.)
template <unsigned Columns, bool Pairs = false> struct Tile {
    static constexpr unsigned rowBytes = Columns * 2, bytes = kStep * rowBytes;
    static __device__ __forceinline__ unsigned key(unsigned r) {
        if constexpr (Pairs) return (r & 3) << 1;
        if constexpr (Columns == 64) return ((r >> 1) & 1) | ((r >> 2) & 2);
        return (r & 3) | ((r >> 1) & 4);
    }
    // Byte of column c, a multiple of 4, of row r.
    static __device__ __forceinline__ unsigned at(unsigned r, unsigned c) {
        return r * rowBytes + ((c / 16) ^ key(r)) * 32 + c % 16 * 2;
    }
    // Eight consecutive rows of a column: lane l has rows r0 + 8 * (l / 16) .. of column c0 + l % 16.
    static __device__ __forceinline__ bf16x8 column(const std::uint8_t* tile, unsigned r0, unsigned c0, unsigned lane) {
        const unsigned r = r0 + lane / 16 * 8 + lane % 16 / 4, c = c0 + lane % 4 * 4;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsColumn)(tile + at(r, c)));
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsColumn)(tile + at(r + 4, c)));
        return __builtin_bit_cast(bf16x8, s16x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w});
    }
};

struct Gradient {
    const void* dy;
    std::uint64_t dyStride;
    const std::uint8_t *x, *xe;
    float *dw, *db; // the splits' sums, or the results where there is one split
    std::uint64_t splitPitch;
    unsigned rows, outer, inner, codePitch, expPitch, tilesN, tilesK, rowsPerSplit;
};

// Tiles of BN columns of dy by BK of x, WN x WK waves, for any dy. A step's bytes are loaded to registers while the
// step before is multiplied; dy is split into its parts on the way to LDS, which has one stage, since its
// parts leave little room and several workgroups share a CU.
// Narrow: rows of dy of fewer than 8 elements.
// Measured, 4096 x 4096 x 4096: FP32 454 us and f16 332, 303 and 414 TFLOP/s (910 and 830 of the MFMA's), bound by the
// split into parts and by LDS, which each part passes through; bf16 of odd rows 210. 262,144 x 256 x 47 FP32 46 us,
// 2.5 TB/s, without columns of x (the bias gradient alone) 24, 2.1 TB/s of dy; 1,000,000 x 128 x 256 268.
template <typename T, unsigned BN, unsigned BK, unsigned WN, unsigned WK, bool Narrow>
__global__ __launch_bounds__(64 * WN * WK) __attribute__((amdgpu_waves_per_eu(2))) void sumRows(Gradient a) {
    constexpr unsigned P = Parts<T>::count, Threads = 64 * WN * WK, NT = BN / WN / 16, KT = BK / WK / 16;
    constexpr unsigned DyLoads = kStep * BN / 8 / Threads;
    constexpr unsigned XLoads = kStep * BK / 16 / Threads, BT = NT / WK; // BT: bias operands of a wave
    static_assert(BT >= 1 && XLoads >= 1 && DyLoads >= 1, "every thread and wave has its share");
    typedef typename T::Raw Raw;
    extern __shared__ __align__(1024) std::uint8_t lds[]; // dy's parts, then x
    const unsigned t = threadIdx.x, lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const unsigned tiles = a.tilesN * a.tilesK, tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
    const unsigned n0 = tile % a.tilesN * BN, k0 = tile / a.tilesN * BK;
    const unsigned first = split * a.rowsPerSplit, last = min(first + a.rowsPerSplit, a.rows);
    const Raw* dy = static_cast<const Raw*>(a.dy);

    typedef typename Group<T>::Vec Vec;
    Vec raw[DyLoads];
    u32x4 q[XLoads];
    unsigned e[XLoads];
    const auto buffer = [](const void* p, unsigned bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
    };
    // Rows of the step from `row` on; past the split's end there are none, and loads give zeros.
    const auto rowsOf = [&](unsigned row) {
        return __builtin_amdgcn_readfirstlane(min(row < last ? last - row : 0u, kStep));
    };
    // No load is conditional, since what a branch loads is waited for where it ends: rows past the split's end read
    // its last row, and a chunk over the row's end the row's last 8 elements, put right on the way to LDS. The parts
    // of a step are inlined by force: a call would take every register that they share through memory.
    const bool ragged = !Narrow && n0 + BN > a.outer && a.outer % 8 != 0;
    auto fetchDy = [&](unsigned row) __attribute__((always_inline)) {
#pragma unroll
        for (unsigned i = 0; i < DyLoads; ++i) {
            const unsigned chunk = t + i * Threads, r = min(row + chunk / (BN / 8), last - 1), c = n0 + chunk % (BN / 8) * 8;
            const Raw* p = dy + r * a.dyStride;
            if constexpr (Narrow) {
#pragma unroll
                for (unsigned j = 0; j < 8; ++j) raw[i][j] = p[min(c + j, a.outer - 1)];
            } else {
                raw[i] = *reinterpret_cast<const typename Group<T>::Loose*>(p + min(c, a.outer - 8));
            }
        }
    };
    auto stashDy = [&](unsigned row) __attribute__((always_inline)) {
#pragma unroll
        for (unsigned i = 0; i < DyLoads; ++i) {
            const unsigned chunk = t + i * Threads, r = chunk / (BN / 8), c = chunk % (BN / 8) * 8;
            std::uint8_t* to = lds + Tile<BN>::at(r, c);
            Vec v = raw[i];
            if (ragged) {
                const unsigned past = n0 + c - min(n0 + c, a.outer - 8);
#pragma unroll
                for (unsigned by = 4; by; by /= 2)
#pragma unroll
                    for (unsigned j = 0; j + by < 8; ++j) v[j] = past & by ? v[j + by] : v[j];
            }
            if (row + kStep > last)
#pragma unroll
                for (unsigned j = 0; j < 8; ++j) v[j] = row + r < last ? v[j] : Raw(0.0f);
            if constexpr (P == 1) {
                *reinterpret_cast<Vec*>(to) = v;
            } else {
                float rest[8];
#pragma unroll
                for (unsigned j = 0; j < 8; ++j) rest[j] = T::get(v[j]);
                const bool large = peakBits(rest) >= 0x7F7F8000u; // rounds to an infinity, or is one, or a NaN
#pragma unroll
                for (unsigned p = 0; p < P; ++p) {
                    bf16x8 part;
#pragma unroll
                    for (unsigned j = 0; j < 8; ++j) {
                        part[j] = __bf16(rest[j]);
                        if (p + 1 < P) rest[j] -= float(part[j]);
                    }
                    // An infinity or a NaN is its first part and leaves no rest; a finite number's first part is finite.
                    if (p == 0 && large) {
#pragma unroll
                        for (unsigned j = 0; j < 8; ++j) {
                            const float f = T::get(v[j]), cut = __uint_as_float(__float_as_uint(f) & 0xFFFF0000u);
                            const bool finite = __builtin_isfinite(f), over = !__builtin_isfinite(float(part[j]));
                            part[j] = finite && over ? __bf16(cut) : part[j];
                            rest[j] = !finite ? 0.0f : over ? f - cut : rest[j];
                        }
                    }
                    *reinterpret_cast<bf16x8*>(to + p * Tile<BN>::bytes) = part;
                }
            }
        }
    };
    auto fetchX = [&](unsigned row) __attribute__((always_inline)) {
        const unsigned rows = rowsOf(row);
        const auto codes = buffer(a.x + std::uint64_t(row) * a.codePitch, rows * a.codePitch);
        const auto exponents = buffer(a.xe + std::uint64_t(row) * a.expPitch, rows * a.expPitch);
#pragma unroll
        for (unsigned i = 0; i < XLoads; ++i) {
            const unsigned chunk = t + i * Threads, r = chunk / (BK / 16), c = chunk % (BK / 16) * 16;
            const bool in = k0 + c < a.codePitch;
            q[i] = __builtin_amdgcn_raw_buffer_load_b128(codes, in ? r * a.codePitch + k0 + c : 0x80000000u, 0, 0);
            e[i] = __builtin_amdgcn_raw_buffer_load_b8(exponents, in ? r * a.expPitch + (k0 + c) / kBlock : 0x80000000u, 0, 0);
        }
    };
    auto stashX = [&]() __attribute__((always_inline)) {
        std::uint8_t* to = lds + P * Tile<BN>::bytes;
#pragma unroll
        for (unsigned i = 0; i < XLoads; ++i) {
            const unsigned chunk = t + i * Threads, r = chunk / (BK / 16), c = chunk % (BK / 16) * 16;
            const float s = scaleOf(e[i]);
#pragma unroll
            for (unsigned h = 0; h < 2; ++h) {
                bf16x8 w;
#pragma unroll
                for (unsigned j = 0; j < 2; ++j) {
                    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i][2 * h + j], s, false);
                    const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i][2 * h + j], s, true);
                    w[4 * j] = lo.x, w[4 * j + 1] = lo.y, w[4 * j + 2] = hi.x, w[4 * j + 3] = hi.y;
                }
                *reinterpret_cast<bf16x8*>(to + Tile<BK>::at(r, c + 8 * h)) = w;
            }
        }
    };
    const unsigned wn = wave % WN * (BN / WN), wk = wave / WN, kk = wk * (BK / WK);
    const bool bias = a.db && k0 == 0;
    const bf16x8 ones = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
    f32x4 acc[NT][KT] = {}, sums[BT] = {};
    auto half = [&](unsigned r0, auto withBias) __attribute__((always_inline)) {
        const std::uint8_t* base = lds;
        bf16x8 xf[KT];
#pragma unroll
        for (unsigned k = 0; k < KT; ++k) xf[k] = Tile<BK>::column(base + P * Tile<BN>::bytes, r0, kk + 16 * k, lane);
#pragma unroll
        for (unsigned p = 0; p < P; ++p) {
            bf16x8 df[NT];
#pragma unroll
            for (unsigned n = 0; n < NT; ++n) df[n] = Tile<BN>::column(base + p * Tile<BN>::bytes, r0, wn + 16 * n, lane);
#pragma unroll
            for (unsigned n = 0; n < NT; ++n)
#pragma unroll
                for (unsigned k = 0; k < KT; ++k)
                    acc[n][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[k], df[n], acc[n][k], 0, 0, 0);
            // The WK waves of these columns share the bias operands.
            if constexpr (decltype(withBias)::value)
#pragma unroll
                for (unsigned b = 0; b < BT; ++b)
                    sums[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, Tile<BN>::column(base + p * Tile<BN>::bytes, r0,
                                                                      wn + 16 * (wk * BT + b), lane), sums[b], 0, 0, 0);
        }
    };
    auto walk = [&](auto withBias) __attribute__((always_inline)) {
        for (unsigned row = first; row < last; row += kStep) {
            fetchX(row + kStep);
            fetchDy(row + kStep);
            __builtin_amdgcn_sched_barrier(0); // the compiler would move the loads down to their use
            half(0, withBias);
            half(32, withBias);
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            stashX();
            stashDy(row + kStep);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
    };
    if (first < last) {
        fetchX(first);
        fetchDy(first);
        stashX();
        stashDy(first);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (bias)
            walk(std::true_type{});
        else
            walk(std::false_type{});
    }
    // x was the first operand: a lane has 4 consecutive columns of x for one of dy's.
    float* dw = a.dw + split * a.splitPitch;
    typedef f32x4 Loose4 __attribute__((aligned(4)));
#pragma unroll
    for (unsigned n = 0; n < NT; ++n) {
        const unsigned row = n0 + wn + 16 * n + lane % 16;
        if (row >= a.outer) continue;
#pragma unroll
        for (unsigned k = 0; k < KT; ++k) {
            const unsigned column = k0 + kk + 16 * k + lane / 16 * 4;
            float* to = dw + std::uint64_t(row) * a.inner + column;
            if (column + 4 <= a.inner) {
                *reinterpret_cast<Loose4*>(to) = acc[n][k];
            } else {
#pragma unroll
                for (unsigned i = 0; i < 4; ++i)
                    if (column + i < a.inner) to[i] = acc[n][k][i];
            }
        }
    }
    if (bias && lane < 16) {
        // Every row of a product with ones is the sum.
#pragma unroll
        for (unsigned b = 0; b < BT; ++b) {
            const unsigned column = n0 + wn + 16 * (wk * BT + b) + lane;
            if (column < a.outer) a.db[split * a.splitPitch + column] = sums[b][0];
        }
    }
}

// acc += a b in the accumulation registers, in place (the compiler moves accumulators that fill them about
// between MFMAs). It does not know this instruction's latency: whoever reads acc has to let it finish.
__device__ __forceinline__ void multiplyInPlace(f32x16& acc, bf16x8 a, bf16x8 b) {
    asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// dy of bf16 with aligned rows: tiles of 256 x 256, or 128 x 128 where a weight has few. Four waves of a quarter
// each; of the large tile one fills a SIMD's registers, of the small two share it. A step is four chunks of 16
// rows; while one is multiplied, the next one's operands are read from LDS to a second set of registers, a read
// behind each MFMA. The 32 x 32 MFMA leaves 32 cycles for what has to be issued beside it, the 16 x 16 one 16, which
// the reads, conversions and writes do not fit into.
// A step's bytes are loaded to registers two steps ahead, and written to the other stage while the step before
// is multiplied; one barrier a step, before its last chunk.
// Bias: the workgroup also sums dy's columns, from the registers that they pass through.
// Measured: 8192 x 4096 x 8192 537 us, 1.02 PFLOP/s, and 4096 x 4096 x 4096 129 (a library's product of bf16 matrices
// 372 and 96); the MFMAs' cycles are 58% of it, the rest is issuing conversions, LDS writes and transposing reads beside
// them. 2048 x 1024 x 4096 32 us in tiles of 128, one a unit.
template <unsigned B, bool Bias> __device__ __forceinline__ void sumTile(const Gradient& a, std::uint8_t* lds) {
    typedef Tile<B, true> In;
    constexpr unsigned Tiles = B / 64, Threads = 256, StageBytes = 2 * In::bytes;
    constexpr unsigned DyLoads = kStep * B / 8 / Threads, XLoads = kStep * B / 16 / Threads;
    const unsigned t = threadIdx.x, lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const unsigned tiles = a.tilesN * a.tilesK, tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
    const unsigned n0 = tile % a.tilesN * B, k0 = tile / a.tilesN * B;
    const unsigned first = split * a.rowsPerSplit, last = min(first + a.rowsPerSplit, a.rows);
    const __bf16* dy = static_cast<const __bf16*>(a.dy) + n0;
    // A thread's chunks: 8 columns of dy, 16 of x, of rows DyApart or XApart from each other, all with one key.
    constexpr unsigned DyApart = Threads * 8 / B, XApart = Threads * 16 / B;
    static_assert(DyApart % 4 == 0 && XApart % 4 == 0, "the key is the row's place among four");
    const unsigned dyRow = t / (B / 8), dyColumn = t % (B / 8) * 8, xRow = t / (B / 16), xColumn = t % (B / 16) * 16;
    const unsigned dyPitch = unsigned(a.dyStride * 2);
    const unsigned dyAt = n0 + dyColumn < a.outer ? dyRow * dyPitch + dyColumn * 2 : 0x80000000u;
    const unsigned xAt = k0 + xColumn < a.codePitch ? xRow * a.codePitch + k0 + xColumn : 0x80000000u;
    const unsigned eAt = k0 + xColumn < a.codePitch ? xRow * a.expPitch + (k0 + xColumn) / kBlock : 0x80000000u;
    const unsigned dyTo = In::at(dyRow, dyColumn), xTo = In::at(xRow, xColumn), xTo8 = In::at(xRow, xColumn + 8);
    u32x4 raw[2][DyLoads], q[2][XLoads]; // two steps' bytes
    unsigned e[2][XLoads];
    float sums[8] = {};
    // Load `i` of the step from `row` on, dy's, then x's; past the split's end zeros, from beyond the
    // buffers.
    auto fetch = [&](unsigned row, unsigned set, unsigned i) {
        const unsigned rows =
            __builtin_amdgcn_readfirstlane(min(row < last ? last - row : 0u, kStep));
        const auto buffer = [](const void* p, unsigned bytes) {
            return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
        };
        if (i < DyLoads) {
            const auto from = buffer(dy + row * a.dyStride, rows * dyPitch);
            raw[set][i] = __builtin_amdgcn_raw_buffer_load_b128(from, dyAt, i * DyApart * dyPitch, 0);
        } else {
            i -= DyLoads;
            const auto codes = buffer(a.x + std::uint64_t(row) * a.codePitch, rows * a.codePitch);
            const auto exponents = buffer(a.xe + std::uint64_t(row) * a.expPitch, rows * a.expPitch);
            q[set][i] = __builtin_amdgcn_raw_buffer_load_b128(codes, xAt, i * XApart * a.codePitch, 0);
            e[set][i] = __builtin_amdgcn_raw_buffer_load_b8(exponents, eAt, i * XApart * a.expPitch, 0);
        }
    };
    constexpr unsigned Loads = DyLoads + XLoads;
    // A step's parity is its stage and its set of registers.
    auto stashDy = [&](unsigned stage, unsigned i) {
        *reinterpret_cast<u32x4*>(lds + stage * StageBytes + dyTo + i * DyApart * In::rowBytes) = raw[stage][i];
        if constexpr (Bias) {
            const bf16x8 v = __builtin_bit_cast(bf16x8, raw[stage][i]);
#pragma unroll
            for (unsigned j = 0; j < 8; ++j) sums[j] += float(v[j]);
        }
    };
    // Half h of 16 codes.
    auto stashX = [&](unsigned stage, unsigned i, unsigned h) {
        const float s = scaleOf(e[stage][i]);
        bf16x8 w;
#pragma unroll
        for (unsigned j = 0; j < 2; ++j) {
            const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[stage][i][2 * h + j], s, false);
            const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[stage][i][2 * h + j], s, true);
            w[4 * j] = lo.x, w[4 * j + 1] = lo.y, w[4 * j + 2] = hi.x, w[4 * j + 3] = hi.y;
        }
        *reinterpret_cast<bf16x8*>(lds + stage * StageBytes + In::bytes + i * XApart * In::rowBytes +
                                   (h ? xTo8 : xTo)) = w;
    };
    const unsigned wn = wave % 2 * (B / 2), kk = wave / 2 * (B / 2);
    // Where a lane reads its 4 rows of column 32 i + lane % 32 of the wave's: rows 8 * (lane / 32) on, of chunk 0.
    // The keys of rows 4 or 16 further are the same.
    unsigned xRead[2][Tiles], dyRead[2][Tiles];
#pragma unroll
    for (unsigned s = 0; s < 2; ++s)
#pragma unroll
        for (unsigned i = 0; i < Tiles; ++i) {
            const unsigned r = lane / 32 * 8 + lane % 16 / 4, c = 32 * i + lane / 16 % 2 * 16 + lane % 4 * 4;
            xRead[s][i] = s * StageBytes + In::bytes + In::at(r, kk + c);
            dyRead[s][i] = s * StageBytes + In::at(r, wn + c);
            asm("" : "+v"(xRead[s][i]), "+v"(dyRead[s][i])); // kept, not computed again for every read
        }
    auto column = [&](unsigned at, unsigned chunk) {
        const std::uint8_t* p = lds + at + chunk * 16 * In::rowBytes;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsColumn)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsColumn)(p + 4 * In::rowBytes));
        return __builtin_bit_cast(bf16x8, s16x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w});
    };
    f32x16 acc[Tiles][Tiles] = {};
    bf16x8 xf[2][Tiles], df[2][Tiles];
    // Of `count` things spread over `slots`, those before slot m.
    constexpr auto share = [](unsigned m, unsigned count, unsigned slots) { return m * count / slots; };
    constexpr unsigned Slots = Tiles * Tiles, Pieces = DyLoads + 2 * XLoads;
    auto step = [&](unsigned row, auto sel) {
        constexpr unsigned S = decltype(sel)::value;
#pragma unroll
        for (unsigned c = 0; c < 4; ++c) {
            const unsigned set = c % 2;
            if (c == 3) { // the next step's stage from here on
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
#pragma unroll
            for (unsigned m = 0; m < Slots; ++m) {
                const unsigned n = m / Tiles, k = m % Tiles;
                // What goes beside MFMA m: the next chunk's operands; the next step's bytes, dy's, then x's, which are
                // converted; in the last chunk the loads of the step after the next two, into the registers that
                // are free by then.
#pragma unroll
                for (unsigned i = share(m, 2 * Tiles, Slots); i < share(m + 1, 2 * Tiles, Slots); ++i) {
                    const unsigned stage = c == 3 ? 1 - S : S, next = c == 3 ? 0 : c + 1;
                    if (i % 2 == 0)
                        xf[1 - set][i / 2] = column(xRead[stage][i / 2], next);
                    else
                        df[1 - set][i / 2] = column(dyRead[stage][i / 2], next);
                }
                if (c < 3) {
                    const unsigned at = c * Slots + m;
#pragma unroll
                    for (unsigned i = share(at, Pieces, 3 * Slots); i < share(at + 1, Pieces, 3 * Slots); ++i) {
                        if (i < DyLoads)
                            stashDy(1 - S, i);
                        else
                            stashX(1 - S, (i - DyLoads) / 2, (i - DyLoads) % 2);
                    }
                } else {
#pragma unroll
                    for (unsigned i = share(m, Loads, Slots); i < share(m + 1, Loads, Slots); ++i)
                        fetch(row + 3 * kStep, 1 - S, i);
                }
                __builtin_amdgcn_sched_barrier(0);
                multiplyInPlace(acc[n][k], xf[set][k], df[set][n]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // Where the loop ends the compiler copies the sums: the last MFMAs, of 8 passes, have to be done by then.
        if (S == 1) asm volatile("s_nop 15\n\ts_nop 3" : "+a"(acc[Tiles - 1][Tiles - 2]), "+a"(acc[Tiles - 1][Tiles - 1]));
    };
#pragma unroll
    for (unsigned i = 0; i < Loads; ++i) fetch(first, 0, i);
#pragma unroll
    for (unsigned i = 0; i < Loads; ++i) fetch(first + kStep, 1, i);
#pragma unroll
    for (unsigned i = 0; i < XLoads; ++i) stashX(0, i, 0), stashX(0, i, 1);
#pragma unroll
    for (unsigned i = 0; i < DyLoads; ++i) stashDy(0, i);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (unsigned i = 0; i < Loads; ++i) fetch(first + 2 * kStep, 0, i);
#pragma unroll
    for (unsigned i = 0; i < Tiles; ++i) xf[0][i] = column(xRead[0][i], 0), df[0][i] = column(dyRead[0][i], 0);
    for (unsigned row = first; row < last; row += 2 * kStep) {
        step(row, std::integral_constant<unsigned, 0>{});
        step(row + kStep, std::integral_constant<unsigned, 1>{});
    }
    float* dw = a.dw + split * a.splitPitch;
    typedef f32x4 Loose4 __attribute__((aligned(4)));
#pragma unroll
    for (unsigned n = 0; n < Tiles; ++n) {
        const unsigned row = n0 + wn + 32 * n + lane % 32;
        if (row >= a.outer) continue;
#pragma unroll
        for (unsigned k = 0; k < Tiles; ++k)
#pragma unroll
            for (unsigned j = 0; j < 4; ++j) {
                const unsigned column = k0 + kk + 32 * k + 8 * j + lane / 32 * 4;
                float* to = dw + std::uint64_t(row) * a.inner + column;
                if (column + 4 <= a.inner) {
                    *reinterpret_cast<Loose4*>(to) = f32x4{acc[n][k][4 * j], acc[n][k][4 * j + 1], acc[n][k][4 * j + 2],
                                                          acc[n][k][4 * j + 3]};
                } else {
#pragma unroll
                    for (unsigned i = 0; i < 4; ++i)
                        if (column + i < a.inner) to[i] = acc[n][k][4 * j + i];
                }
            }
    }
    if constexpr (Bias) {
        // The threads with the same columns add theirs through LDS, which nobody reads any more.
        __syncthreads();
        float* part = reinterpret_cast<float*>(lds);
#pragma unroll
        for (unsigned j = 0; j < 8; ++j) part[dyRow * B + dyColumn + j] = sums[j];
        __syncthreads();
        if (t < B && n0 + t < a.outer) {
            float s = 0.0f;
#pragma unroll
            for (unsigned r = 0; r < DyApart; ++r) s += part[r * B + t];
            a.db[split * a.splitPitch + n0 + t] = s;
        }
    }
}

// Two bodies, not a condition in one: accumulators that fill their registers leave no room to join paths.
template <unsigned B> __device__ __forceinline__ void sumTileWithBias(const Gradient& a, std::uint8_t* lds) {
    if (a.db && blockIdx.x % (a.tilesN * a.tilesK) < a.tilesN)
        sumTile<B, true>(a, lds);
    else
        sumTile<B, false>(a, lds);
}
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void sumRowsInPlace256(Gradient a) {
    extern __shared__ __align__(1024) std::uint8_t lds[]; // two stages of dy, then x
    sumTileWithBias<256>(a, lds);
}
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void sumRowsInPlace128(Gradient a) {
    extern __shared__ __align__(1024) std::uint8_t lds[];
    sumTileWithBias<128>(a, lds);
}

// dw and db from the splits' sums, added in a fixed order: Ways threads add every Ways-th split of four
// values, then their sums through LDS. A split's db follows its dw. 256 splits of 47 x 256 5.6 us, bound by latency.
template <unsigned Ways>
__global__ __launch_bounds__(64 * Ways) void addSplits(const float* __restrict__ parts, float* __restrict__ dw,
                                                        float* __restrict__ db, std::uint64_t size, std::uint64_t dbAt,
                                                        unsigned outer, std::uint64_t pitch, unsigned splits) {
    __shared__ f32x4 sums[Ways][64];
    const unsigned lane = threadIdx.x % 64, way = threadIdx.x / 64;
    const std::uint64_t at = (std::uint64_t(blockIdx.x) * 64 + lane) * 4;
    f32x4 s = {};
    if (at < pitch)
#pragma unroll 4
        for (unsigned k = way; k < splits; k += Ways) s += *reinterpret_cast<const f32x4*>(parts + k * pitch + at);
    sums[way][lane] = s;
    __syncthreads();
    if (way || at >= pitch) return;
#pragma unroll
    for (unsigned w = 1; w < Ways; ++w) s += sums[w][lane];
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
        if (at + i < size)
            dw[at + i] = s[i];
        else if (db && at >= dbAt && at + i - dbAt < outer)
            db[at + i - dbAt] = s[i];
    }
}

// ------------------------------------------------------------------------------------------------
// Host side

// Form of a call: tile, and how many splits of the rows.
struct Plan {
    unsigned bn, bk, splits, steps; // steps of a split
    bool aligned;
};

constexpr unsigned kUnits = 256; // compute units

bool alignedRows(const DenseMatrix& dy, std::uint32_t outer) {
    return dy.type == DenseType::bf16 && reinterpret_cast<std::uintptr_t>(dy.data) % 16 == 0 && dy.stride % 8 == 0 &&
           outer % 8 == 0 && dy.stride < (1u << 23);
}

// The bias gradient alone is a weight gradient of no columns, whose one column of tiles has nothing else to store.
unsigned tilesOf(std::uint32_t n, unsigned size) { return n ? (n + size - 1) / size : 1; }

std::uint64_t rounded4(std::uint64_t n) { return (n + 3) / 4 * 4; }
std::uint64_t pitchOf(std::uint32_t inner, std::uint32_t outer) {
    return rounded4(std::uint64_t(outer) * inner) + rounded4(outer);
}

// The splits with the least estimated time, in microseconds: rounds of workgroups on the chip times the steps of
// each, and the traffic of the partial sums, written once and read once. `alone` and `shared` are the time of
// a step of a workgroup that has its CU to itself and of one that shares it with perUnit - 1 others.
double planTime(Plan& p, std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, double alone, double shared,
                unsigned perUnit) {
    const std::uint64_t tiles = tilesOf(inner, p.bk) * std::uint64_t(tilesOf(outer, p.bn));
    const std::uint64_t steps = std::max<std::uint64_t>(1, (std::uint64_t(rows) + kStep - 1) / kStep);
    double best = 1e30;
    auto consider = [&](std::uint64_t splits) {
        splits = std::max<std::uint64_t>(1, std::min(splits, steps));
        const std::uint64_t each = (steps + splits - 1) / splits, used = (steps + each - 1) / each;
        const std::uint64_t rounds = (tiles * used + kUnits * perUnit - 1) / (kUnits * perUnit);
        double time = tiles * used <= kUnits ? 8.0 + double(each) * alone : double(rounds) * (8.0 + double(each) * shared);
        if (used > 1) time += 4.0 + double(used) * double(pitchOf(inner, outer)) * 8.0 / 4.0e6;
        if (time < best) best = time, p.splits = unsigned(used), p.steps = unsigned(each);
    };
    consider(1);
    consider(kUnits / tiles);
    for (unsigned rounds = 1; rounds <= 4; ++rounds) consider(std::uint64_t(rounds) * kUnits * perUnit / tiles);
    return best;
}

// Steps measured, in us: the large tile 2.0 (4096 x 4096 x 4096 135, 8192 x 4096 x 8192 545), the small one 0.75 alone
// (2048 x 1024 x 4096 32) and 1.15 shared (2048 x 2048 x 4096 46). Where dy is not bf16 in aligned rows: bf16 1.2 alone
// (2048 x 1024 x 4095 46) and 1.65 shared (4096 x 4096 x 4095 212), f16 2.0 (71) and 2.9 (4096 x 4096 x 4096 372), f32
// 2.75 (96; in two splits that share a CU 82) and 3.9 (514).
Plan planOf(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type, bool aligned) {
    Plan small = {outer <= 64 && !aligned ? 64u : 128u, 128, 1, 1, aligned}, large = {256, 256, 1, 1, aligned};
    if (!aligned) {
        const double alone = type == DenseType::f32 ? 2.75 : type == DenseType::f16 ? 2.0 : 1.2;
        const double shared = type == DenseType::f32 ? 3.9 : type == DenseType::f16 ? 2.9 : 1.65;
        planTime(small, rows, inner, outer, alone, shared, 2);
        return small;
    }
    const double smallTime = planTime(small, rows, inner, outer, 0.75, 1.15, 2);
    return planTime(large, rows, inner, outer, 2.0, 2.0, 1) < smallTime ? large : small;
}

template <typename T, unsigned BN, unsigned BK, unsigned WN, unsigned WK, bool Narrow>
void launchSum(const Gradient& a, std::uint64_t blocks, hipStream_t stream) {
    constexpr unsigned lds = Parts<T>::count * Tile<BN>::bytes + Tile<BK>::bytes;
    hipLaunchKernelGGL((sumRows<T, BN, BK, WN, WK, Narrow>), dim3(unsigned(blocks)), dim3(64 * WN * WK), lds, stream, a);
}

} // namespace

const char* weightGradBlocksForm(DenseMatrix dy, std::uint32_t rows, std::uint32_t inner, std::uint32_t outer,
                                 std::uint32_t* splits) {
    checkType("weight gradient", dy.type);
    checkColumns("weight gradient", outer);
    const Plan p = planOf(rows, inner, outer, dy.type, alignedRows(dy, outer));
    if (splits) *splits = p.splits;
    if (p.aligned) return p.bn == 256 ? "sumRowsInPlace256" : "sumRowsInPlace128";
    return outer < 8 ? "sumRowsNarrow" : p.bn == 64 ? "sumRows64" : "sumRows128";
}

std::size_t weightGradBlocksWorkspace(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type) {
    if (!rows || !outer) return 0;
    // The larger of the two forms' needs: which one runs depends on dy's alignment.
    std::uint64_t splits = planOf(rows, inner, outer, type, false).splits;
    if (type == DenseType::bf16) splits = std::max<std::uint64_t>(splits, planOf(rows, inner, outer, type, true).splits);
    return splits == 1 ? 0 : std::size_t(splits * pitchOf(inner, outer) * sizeof(float));
}

void weightGradBlocks(DenseMatrix dy, BlockRows x, float* dw, float* db, std::uint32_t rows, std::uint32_t inner,
                      std::uint32_t outer, void* workspace, std::size_t workspaceBytes, hipStream_t stream) {
    const char* where = "weight gradient";
    if (!dw && db) inner = 0, x = {nullptr, nullptr, BlockCodes::e4m3};
    if (dw) checkColumns(where, inner);
    checkColumns(where, outer);
    checkRows(where, rows);
    checkType(where, dy.type);
    if (x.type != BlockCodes::e4m3) reject(where, "x must have E4M3 codes");
    if (!dw && !db) reject(where, "null weight gradient");
    if (reinterpret_cast<std::uintptr_t>(dw) % 4 || reinterpret_cast<std::uintptr_t>(db) % 4)
        reject(where, "gradients must be float-aligned");
    if (rows) {
        checkDense(where, dy.data, dy.stride, dy.type, outer);
        if (dw) checkCodes(where, x.codes, x.exponents);
    }
    const std::size_t need = weightGradBlocksWorkspace(rows, inner, outer, dy.type);
    if (need > workspaceBytes || (need && !workspace)) reject(where, "workspace too small");
    if (reinterpret_cast<std::uintptr_t>(workspace) % 16) reject(where, "workspace must be 16-byte aligned");
    const Plan p = planOf(rows, inner, outer, dy.type, alignedRows(dy, outer));
    const std::uint64_t size = std::uint64_t(outer) * inner, pitch = pitchOf(inner, outer);
    auto* parts = static_cast<float*>(workspace);
    Gradient a = {};
    a.dy = dy.data, a.dyStride = dy.stride, a.x = x.codes, a.xe = x.exponents;
    a.rows = rows, a.outer = outer, a.inner = inner;
    a.codePitch = unsigned(blockCodePitch(inner)), a.expPitch = unsigned(blockExponentPitch(inner));
    a.tilesN = tilesOf(outer, p.bn), a.tilesK = tilesOf(inner, p.bk);
    a.rowsPerSplit = p.steps * kStep;
    a.dw = p.splits == 1 ? dw : parts;
    a.db = !db ? nullptr : p.splits == 1 ? db : parts + rounded4(size);
    a.splitPitch = p.splits == 1 ? 0 : pitch;
    const std::uint64_t blocks = std::uint64_t(a.tilesN) * a.tilesK * p.splits;
    checkGrid(where, blocks, 256);
    if (p.aligned) {
        if (p.bn == 256)
            hipLaunchKernelGGL(sumRowsInPlace256, dim3(unsigned(blocks)), dim3(256), 4 * Tile<256>::bytes, stream, a);
        else
            hipLaunchKernelGGL(sumRowsInPlace128, dim3(unsigned(blocks)), dim3(256), 4 * Tile<128>::bytes, stream, a);
    } else {
        withType(dy.type, [&](auto tag) {
            typedef decltype(tag) T;
            if (outer < 8)
                launchSum<T, 64, 128, 1, 4, true>(a, blocks, stream);
            else if (p.bn == 64)
                launchSum<T, 64, 128, 1, 4, false>(a, blocks, stream);
            else
                launchSum<T, 128, 128, 2, 2, false>(a, blocks, stream);
        });
    }
    checkHip(hipGetLastError());
    if (p.splits > 1) {
        const dim3 grid(unsigned((pitch / 4 + 63) / 64));
        // 16 ways where there are many splits of a small gradient (262,144 x 256 x 47, the call, 32 us : 35 with 4);
        // 4 where workgroups abound (100,000 x 256 x 256 35.0 : 35.7, 8192 x 1024 x 1024 38 : 45).
        if (p.splits >= 32 && grid.x <= 128)
            hipLaunchKernelGGL(addSplits<16>, grid, dim3(1024), 0, stream, parts, dw, db, size, rounded4(size), outer,
                               pitch, p.splits);
        else
            hipLaunchKernelGGL(addSplits<4>, grid, dim3(256), 0, stream, parts, dw, db, size, rounded4(size), outer,
                               pitch, p.splits);
        checkHip(hipGetLastError());
    }
}

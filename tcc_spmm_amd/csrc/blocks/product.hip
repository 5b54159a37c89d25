// The product of 8-bit blocks, y = x w^T + bias (include/blocks.h), and the linear layer on dense x.
#include "device_product.h"
#include "hip_support.h"

#include <algorithm>
#include <type_traits>

namespace {

using namespace blocks;

struct Product {
    const std::uint8_t *x, *xe; // null x: dense input
    const std::uint8_t *w, *we;
    const float* bias;
    void* y;
    std::uint64_t yStride;
    unsigned rows, outer, count, expPitch; // count: blocks of a row; code rows are 128 * count bytes
    unsigned inner, tilesM, tilesN;
    const void* dense;
    std::uint64_t denseStride;
    std::uint8_t *keep, *keepExp;
};

// ------------------------------------------------------------------------------------------------
// 16-bit outputs: the scaled 8-bit MFMA on tiles of BM x BN. Its sums, here and in the kernels below, are those that
// include/blocks.h states for 16-bit types: fewer bits than FP32's within eight products, at twice the bf16 MFMA's rate.
//
// A block of 128 along the inner axis is one step: 128 bytes of each of the tile's rows, loaded to LDS
// without passing registers, Stages deep. The 16-byte chunks of a row are stored in an order that
// depends on the row (its key), so that the rows an MFMA operand takes at once lie in different banks.
// The order of the inner axis inside a block is free, since both operands share it and each has one
// scale there: a lane takes chunks g and g + 4 of its row.
// The weight is the MFMA's first operand, whose rows become consecutive values of one lane: rows are
// dealt to pairs of MFMAs so that a lane ends with 8 consecutive outputs of one row of y.
//
// Groups of waves share a tile where there are few: each takes a run of the inner axis, with stages of its own,
// and the first adds the others' sums. A step costs its barrier and its LDS reads' latency, so half the
// steps are nearly half the time.
// Measured, bf16: 2048 x 1024 x 4096 16 us in tiles of 128 and 2048 x 4096 x 1024 18 in tiles of 64, bound by the LDS
// reads that follow each barrier (the MFMAs' cycles are a third); 24 x 4096 x 8192 6.8 us in tiles of 32, 4.9 TB/s of
// the weight, 777 x 1001 x 1437 6.7 in tiles of 64.
template <typename T, unsigned BM, unsigned BN, unsigned WM, unsigned WN, unsigned Stages, unsigned Groups>
__global__ __launch_bounds__(64 * WM * WN * Groups) void multiplyTiles(Product a) {
    constexpr unsigned Waves = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
    constexpr unsigned XL = BM / 8 / Waves, WL = BN / 8 / Waves;
    static_assert(Stages == 2 || Stages == 4, "the stage is a constant of the unrolled step");
    static_assert(BN / WN <= 128 && NT % 2 == 0, "a wave's columns share a weight tile");
    extern __shared__ __align__(1024) std::uint8_t shared[];
    const unsigned lane = threadIdx.x % kWave, allWaves = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned wave = allWaves % Waves, part = Groups == 1 ? 0 : allWaves / Waves;
    std::uint8_t* lds = shared + part * Stages * (BM + BN) * kBlock;
    // This group's blocks: `steps` of them from `first` on, those past the last being zeros.
    const unsigned steps = Groups == 1 ? a.count : (a.count + 4 * Groups - 1) / (4 * Groups) * 4, first = part * steps;
    const unsigned tile = tileOf(blockIdx.x, gridDim.x, a.tilesM, a.tilesN);
    const unsigned tm = tile % a.tilesM * BM, tn = tile / a.tilesM * BN;
    const unsigned pitch = a.count * kBlock;
    // Rows past the end are past the buffer and read as zeros; their results are not stored.
    const auto xr = rowsAt(a.x, pitch, tm, a.rows), wr = rowsAt(a.w, pitch, tn, a.outer);
    // A load fills 8 rows of LDS in order, 16 bytes a lane, so a lane fetches the chunk that belongs in its
    // place; a wave's loads are 8 * Waves rows apart, which leaves the rows' keys the same.
    static_assert(Waves % 2 == 0, "the weight's key takes bit 3 of the row");
    const unsigned r = wave * 8 + lane / 8;
    const unsigned xo = r * pitch + ((lane % 8) ^ (r & 7)) * 16;
    const unsigned wo = r * pitch + ((lane % 8) ^ ((r & 3) | ((r >> 1) & 4))) * 16;
    // Block k's bytes into stage s; past the last block zeros, from beyond the buffer, so that every wave has
    // the same number of loads outstanding.
    auto load = [&](unsigned k, unsigned s) {
        std::uint8_t* to = lds + s * (BM + BN) * kBlock + wave * 1024;
        const unsigned from = k < a.count ? k * kBlock : 0x7FFFFFFFu;
#pragma unroll
        for (unsigned j = 0; j < XL; ++j)
            loadToLds(xr, to + j * Waves * 1024, xo, from + j * Waves * 8 * pitch);
#pragma unroll
        for (unsigned j = 0; j < WL; ++j)
            loadToLds(wr, to + BM * kBlock + j * Waves * 1024, wo, from + j * Waves * 8 * pitch);
    };
    const unsigned wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
    const unsigned l16 = lane % 16, g = lane / 16;
    // Four steps' exponents a dword: of this lane's row of each X operand, and of the wave's weight tile.
    const std::uint8_t* we = a.we + std::uint64_t(min((tn + wn) / kBlock, (a.outer - 1) / kBlock)) * a.expPitch;
    const std::uint8_t* xe[MT];
    unsigned xs[MT], ws, xsNext[MT], wsNext;
#pragma unroll
    for (unsigned m = 0; m < MT; ++m)
        xe[m] = a.xe + std::uint64_t(min(tm + wm + m * 16 + l16, a.rows - 1)) * a.expPitch;
    auto loadExponents = [&](unsigned k4) {
#pragma unroll
        for (unsigned m = 0; m < MT; ++m) xsNext[m] = *reinterpret_cast<const unsigned*>(xe[m] + k4);
        wsNext = *reinterpret_cast<const unsigned*>(we + k4);
    };
    f32x4 acc[NT][MT] = {};
    loadExponents(min(first, (a.count - 1) / 4 * 4));
#pragma unroll
    for (unsigned s = 0; s + 1 < Stages; ++s) load(first + s, s);
    const unsigned xKey = l16 & 7, wKey = (l16 & 3) | (l16 & 4);
    const std::uint8_t* xRead = lds + (wm + l16) * kBlock;
    const std::uint8_t* wRead = lds + BM * kBlock + (wn + l16 / 4 * 8 + l16 % 4) * kBlock;
    auto step = [&](unsigned k, auto sel) {
        constexpr unsigned S = decltype(sel)::value;
        constexpr unsigned at = S % Stages * (BM + BN) * kBlock;
        waitBarrier<(Stages - 2) * (XL + WL)>();
        load(k + Stages - 1, (S + Stages - 1) % Stages);
        i32x8 xf[MT];
#pragma unroll
        for (unsigned m = 0; m < MT; ++m)
            xf[m] = join(*reinterpret_cast<const u32x4*>(xRead + at + m * 16 * kBlock + ((g ^ xKey) * 16)),
                         *reinterpret_cast<const u32x4*>(xRead + at + m * 16 * kBlock + (((g + 4) ^ xKey) * 16)));
#pragma unroll
        for (unsigned n = 0; n < NT; ++n) {
            const unsigned r = (n / 2 * 32 + n % 2 * 4) * kBlock;
            const i32x8 wf = join(*reinterpret_cast<const u32x4*>(wRead + at + r + ((g ^ wKey) * 16)),
                                  *reinterpret_cast<const u32x4*>(wRead + at + r + (((g + 4) ^ wKey) * 16)));
#pragma unroll
            for (unsigned m = 0; m < MT; ++m)
                acc[n][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf[m], acc[n][m], 0, 0, S, int(ws), S,
                                                                             int(xs[m]));
        }
    };
    auto nextExponents = [&](unsigned k4) {
        // Past the last block (of a group's steps) codes are zeros, and so that the products are, the exponents finite.
        const unsigned keep = Groups == 1 ? ~0u : finiteExponents(k4, a.count);
#pragma unroll
        for (unsigned m = 0; m < MT; ++m) xs[m] = (xsNext[m] & keep) | (0x7F7F7F7Fu & ~keep);
        ws = (wsNext & keep) | (0x7F7F7F7Fu & ~keep);
        loadExponents(min(k4 + 4, (a.count - 1) / 4 * 4));
    };
    unsigned k = first;
    for (; k + 4 <= first + steps; k += 4) {
        nextExponents(k);
        step(k, std::integral_constant<unsigned, 0>{});
        step(k + 1, std::integral_constant<unsigned, 1>{});
        step(k + 2, std::integral_constant<unsigned, 2>{});
        step(k + 3, std::integral_constant<unsigned, 3>{});
    }
    if (Groups == 1 && k < steps) {
        nextExponents(k);
        step(k, std::integral_constant<unsigned, 0>{});
        if (k + 1 < steps) step(k + 1, std::integral_constant<unsigned, 1>{});
        if (k + 2 < steps) step(k + 2, std::integral_constant<unsigned, 2>{});
    }
    // Loads to LDS past the last step have to land before the workgroup gives its LDS back.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (Groups > 1) {
        __syncthreads();
        f32x4* sums = reinterpret_cast<f32x4*>(shared) + wave * NT * MT * kWave + lane;
        if (part)
#pragma unroll
            for (unsigned i = 0; i < NT * MT; ++i)
                sums[((part - 1) * Waves * NT * MT + i) * kWave] = acc[i / MT][i % MT];
        __syncthreads();
        if (part) return;
#pragma unroll
        for (unsigned p = 0; p + 1 < Groups; ++p)
#pragma unroll
            for (unsigned i = 0; i < NT * MT; ++i) acc[i / MT][i % MT] += sums[(p * Waves * NT * MT + i) * kWave];
    }
    typename T::Raw* y = static_cast<typename T::Raw*>(a.y);
    auto store = [&](auto whole) {
        constexpr bool Whole = decltype(whole)::value;
#pragma unroll
        for (unsigned n = 0; n < NT; n += 2) {
            const unsigned column = tn + wn + n * 16 + g * 8;
            float b[8];
            bias8<Whole>(a.bias, column, a.outer, b);
#pragma unroll
            for (unsigned m = 0; m < MT; ++m) {
                const unsigned row = tm + wm + m * 16 + l16;
                float v[8];
#pragma unroll
                for (unsigned i = 0; i < 8; ++i) v[i] = acc[n + i / 4][m][i % 4];
                if (Whole || row < a.rows) put8<T, Whole>(y + row * a.yStride, column, a.outer, v, b);
            }
        }
    };
    if (tm + BM <= a.rows && tn + BN <= a.outer)
        store(std::true_type{});
    else
        store(std::false_type{});
}

// acc += a b with the operands' scales in byte S of `as` and `bs`, in the accumulation registers. Where
// accumulators fill them, the compiler moves them about between MFMAs; asm with one operand for both the
// sum and the result does not let it. The compiler does not know this instruction's latency: whoever
// reads acc has to let the last one finish.
template <unsigned S>
__device__ __forceinline__ void multiplyInPlace(f32x4& acc, i32x8 a, i32x8 b, unsigned as, unsigned bs) {
    static_assert(S < 2, "the bytes that the two forms below select");
    if constexpr (S == 0)
        asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]"
            : "+a"(acc) : "v"(a), "v"(b), "v"(as), "v"(bs));
    else
        asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0]"
            : "+a"(acc) : "v"(a), "v"(b), "v"(as), "v"(bs));
}

// The same on tiles of 256 x 256, for products with enough of them: a CU can then multiply twice as long on
// every byte it loads (a tile of 128 x 128 needs 64 bytes a clock, all that a CU can load).
// Four waves, one a SIMD, of 128 x 128 each, whose accumulators fill the accumulation registers. LDS holds two
// stages of a block. A block is multiplied in four quarters, a pair of the weight's operands with all of
// x's in each: in a quarter the next pair is read from LDS, and in the last one also, as each operand of
// x is used for the last time, its place is filled with the next block's. So no MFMA waits for LDS. The
// loads into LDS are spread over the quarters, each into a place that was read for the last time a
// quarter or more before, and each has at least a block's time to arrive:
//   quarter 0: pairs 2 and 3 of block k + 1;  1 and 2: x of block k + 2;  3: pairs 0 and 1 of block k + 2
// with a barrier before quarters 1 and 3.
// The 16 x 16 MFMA is the one to feed: on random codes the card's power holds the scaled 32 x 32 x 64 to 3.2
// PFLOP/s and the scaled 16 x 16 x 128 to 3.8 (on zeros both reach 4.7).
// Measured: 4096 x 4096 x 8192 bf16 114 us, 2.4 PFLOP/s (a library's product of plain 8-bit matrices, without scales
// of blocks, 93 us), 8192 x 8192 x 4096 245. The MFMAs' own cycles are 60% of it; waves wait for instructions to issue
// half of the time and for memory an eighth, and no LDS access conflicts.
template <typename T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void multiplyWide(Product a) {
    constexpr unsigned B = 256, Stage = 2 * B * kBlock, Tiles = 8;
    extern __shared__ __align__(1024) std::uint8_t lds[]; // two stages: 256 rows of x, 256 of w
    const unsigned lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned tile = tileOf(blockIdx.x, gridDim.x, a.tilesM, a.tilesN);
    const unsigned tm = tile % a.tilesM * B, tn = tile / a.tilesM * B;
    const unsigned pitch = a.count * kBlock;
    const auto xr = rowsAt(a.x, pitch, tm, a.rows), wr = rowsAt(a.w, pitch, tn, a.outer);
    // Chunks and rows are dealt as in multiplyTiles.
    auto keyX = [](unsigned r) { return r & 7; };
    auto keyW = [](unsigned r) { return (r & 3) | (r >> 1 & 4); };
    const unsigned fill = wave * 8 + lane / 8; // a wave's loads are 32 rows apart, with the same keys
    const unsigned xo = fill * pitch + ((lane % 8) ^ keyX(fill)) * 16;
    const unsigned wo = fill * pitch + ((lane % 8) ^ keyW(fill)) * 16;
    // An eighth of block k's rows of x or w into stage s; past the last block zeros, from beyond the buffer.
    auto from = [&](unsigned k) { return k < a.count ? k * kBlock : 0x7FFFFFFFu; };
    auto loadX = [&](unsigned k, unsigned s, unsigned part) {
        loadToLds(xr, lds + s * Stage + wave * 1024 + part * 4096, xo, from(k) + part * 32 * pitch);
    };
    auto loadW = [&](unsigned k, unsigned s, unsigned part) {
        loadToLds(wr, lds + s * Stage + B * kBlock + wave * 1024 + part * 4096, wo, from(k) + part * 32 * pitch);
    };
    const unsigned wm = wave % 2 * 128, wn = wave / 2 * 128, l16 = lane % 16, g = lane / 16;
    const unsigned wRow = l16 / 4 * 8 + l16 % 4;
    // A lane's two chunks of its row in either stage: bytes of LDS, which the loads' offsets reach a stage of.
    unsigned xRead[2][2], wRead[2][2];
#pragma unroll
    for (unsigned s = 0; s < 2; ++s)
#pragma unroll
        for (unsigned c = 0; c < 2; ++c) {
            xRead[s][c] = s * Stage + (wm + l16) * kBlock + ((g + 4 * c) ^ keyX(l16)) * 16;
            wRead[s][c] = s * Stage + (B + wn + wRow) * kBlock + ((g + 4 * c) ^ keyW(wRow)) * 16;
            asm("" : "+v"(xRead[s][c]), "+v"(wRead[s][c])); // kept, not computed again for every load
        }
    i32x8 xf[Tiles], wf[2][2];
    auto readX = [&](unsigned s, unsigned m) {
        const std::uint8_t* at = lds + m * 16 * kBlock;
        xf[m] = join(*reinterpret_cast<const u32x4*>(at + xRead[s][0]), *reinterpret_cast<const u32x4*>(at + xRead[s][1]));
    };
    auto readW = [&](unsigned s, unsigned n) {
        const std::uint8_t* at = lds + (n / 2 * 32 + n % 2 * 4) * kBlock;
        wf[n / 2 % 2][n % 2] =
            join(*reinterpret_cast<const u32x4*>(at + wRead[s][0]), *reinterpret_cast<const u32x4*>(at + wRead[s][1]));
    };
    const auto er = rowsAt(a.xe, a.expPitch, tm, a.rows);
    const std::uint8_t* we = a.we + std::uint64_t(min((tn + wn) / kBlock, (a.outer - 1) / kBlock)) * a.expPitch;
    // Two blocks' exponents at a time, a byte each.
    unsigned xs[Tiles], ws, xsNext[Tiles], wsNext;
    auto loadExponents = [&](unsigned block) {
        block = min(block, (a.count - 1) / 2 * 2);
#pragma unroll
        for (unsigned m = 0; m < Tiles; ++m)
            xsNext[m] = __builtin_amdgcn_raw_buffer_load_b16(er, (wm + l16) * a.expPitch, m * 16 * a.expPitch + block, 0);
        wsNext = *reinterpret_cast<const unsigned short*>(we + block);
    };
    f32x4 acc[Tiles][Tiles] = {};
    loadExponents(0);
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) loadX(0, 0, i), loadW(0, 0, i);
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) loadX(1, 1, i);
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) loadW(1, 1, i / 2 + i % 2 * 4);
    waitBarrier<12>();
#pragma unroll
    for (unsigned i = 0; i < 2; ++i) readW(0, i);
#pragma unroll
    for (unsigned i = 0; i < Tiles; ++i) readX(0, i);
    // Block S of the pair that the exponents are for. The fences keep the compiler from moving the reads and
    // loads between the MFMAs down to where their results are needed, which is where they would be
    // waited for.
    auto blockStep = [&](unsigned k, auto block) {
        constexpr unsigned S = decltype(block)::value;
        auto multiply = [&](unsigned m, unsigned n0) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (unsigned n = n0; n < n0 + 2; ++n)
                multiplyInPlace<S>(acc[n][m], wf[n / 2 % 2][n % 2], xf[m], ws, xs[m]);
            __builtin_amdgcn_sched_barrier(0);
        };
        // Pair p of the weight's operands lies in eighths p and p + 4: waves start at row 0 or 128.
#pragma unroll
        for (unsigned q = 0; q < 4; ++q) {
            // Before quarter 1 pairs 2 and 3 of this block have to be there, before 3 x and pair 0 of the next. What
            // was loaded since stays outstanding, and in a pair's first block the exponents.
            if (q == 1) waitBarrier<S == 0 ? 25 : 16>();
            if (q == 3) waitBarrier<S == 0 ? 21 : 12>();
#pragma unroll
            for (unsigned m = 0; m < Tiles; ++m) {
                if (m % 4 == 0) {
                    if (q < 3)
                        readW(S, 2 * q + 2 + m / 4);
                    else
                        readW(1 - S, m / 4);
                }
                if (m % 2 == 1) {
                    const unsigned i = m / 2, eighth = i / 2 + i % 2 * 4;
                    if (q == 0) loadW(k + S + 1, 1 - S, 2 + eighth);
                    if (q == 1) loadX(k + S + 2, S, i);
                    if (q == 2) loadX(k + S + 2, S, 4 + i);
                    if (q == 3) loadW(k + S + 2, S, eighth);
                }
                multiply(m, 2 * q);
                if (q == 3) readX(1 - S, m);
            }
        }
        // Where the loop ends the compiler copies the sums, without knowing that they come from an MFMA: the last
        // ones, of 8 passes, have to be done by then.
        if (S == 1)
            asm volatile("s_nop 15\n\ts_nop 3" : "+a"(acc[6][6]), "+a"(acc[7][6]), "+a"(acc[6][7]), "+a"(acc[7][7]));
    };
    for (unsigned k = 0; k < a.count; k += 2) {
        // A block past the last has codes of zeros, and has to have finite exponents.
        const unsigned keep = finiteExponents(k, a.count) & 0xFFFFu;
#pragma unroll
        for (unsigned m = 0; m < Tiles; ++m) xs[m] = (xsNext[m] & keep) | (0x7F7Fu & ~keep);
        ws = (wsNext & keep) | (0x7F7Fu & ~keep);
        loadExponents(k + 2);
        blockStep(k, std::integral_constant<unsigned, 0>{});
        blockStep(k, std::integral_constant<unsigned, 1>{});
    }
    // Loads to LDS past the last step have to land before the workgroup gives its LDS back.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    typename T::Raw* y = static_cast<typename T::Raw*>(a.y);
    auto store = [&](auto whole) {
        constexpr bool Whole = decltype(whole)::value;
#pragma unroll
        for (unsigned n = 0; n < Tiles; n += 2) {
            const unsigned column = tn + wn + n * 16 + g * 8;
            float b[8];
            bias8<Whole>(a.bias, column, a.outer, b);
#pragma unroll
            for (unsigned m = 0; m < Tiles; ++m) {
                const unsigned row = tm + wm + m * 16 + l16;
                float v[8];
#pragma unroll
                for (unsigned j = 0; j < 8; ++j) v[j] = acc[n + j / 4][m][j % 4];
                if (Whole || row < a.rows) put8<T, Whole>(y + row * a.yStride, column, a.outer, v, b);
            }
        }
    };
    if (tm + B <= a.rows && tn + B <= a.outer)
        store(std::true_type{});
    else
        store(std::false_type{});
}

// ------------------------------------------------------------------------------------------------
// FP32 outputs: the codes' values, exact in bf16 (values8), through the bf16 MFMA, whose sums are FP32's. Tiles of
// 128 x 128, steps of half a block: a row's 64 values are 128 bytes of LDS, stored in the chunk order of
// the 8-bit kernel. Codes pass through registers to be converted, in every tile anew, which with the bf16 MFMA's
// half rate bounds it: 4096 x 4096 x 8192 360 us, 0.76 PFLOP/s (a library's product in FP32 0.15). The 8-bit MFMA cuts
// products off 13 bits below the largest of eight, 1.2e-5 of the sum off on random numbers, which a 16-bit output's
// rounding is twenty times as large as and an FP32 one's far smaller.
__global__ __launch_bounds__(256) void multiplyTilesExact(Product a) {
    constexpr unsigned B = 128;
    __shared__ __align__(1024) std::uint8_t lds[2][2][B * 128];
    const unsigned t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    const unsigned tm = blockIdx.x % a.tilesM * B, tn = blockIdx.x / a.tilesM * B;
    const unsigned pitch = a.count * kBlock;
    const unsigned r = t / 4, part = t % 4; // 16 codes of rows r and r + 64 of each operand
    const std::uint8_t *xp[2], *wp[2], *xep[2];
#pragma unroll
    for (unsigned h = 0; h < 2; ++h) {
        const std::uint64_t xrow = min(tm + r + 64 * h, a.rows - 1);
        xp[h] = a.x + xrow * pitch + part * 16;
        xep[h] = a.xe + xrow * a.expPitch;
        wp[h] = a.w + std::uint64_t(min(tn + r + 64 * h, a.outer - 1)) * pitch + part * 16;
    }
    const std::uint8_t* wep = a.we + std::uint64_t(tn / kBlock) * a.expPitch;
    u32x4 xq[2], wq[2];
    unsigned xb[2], wb;
    auto fetch = [&](unsigned k) {
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
            xq[h] = *reinterpret_cast<const u32x4*>(xp[h] + k * 64);
            wq[h] = *reinterpret_cast<const u32x4*>(wp[h] + k * 64);
            xb[h] = xep[h][k / 2];
        }
        wb = wep[k / 2];
    };
    auto put = [&](std::uint8_t* to, unsigned row, u32x4 q, float scale) {
        *reinterpret_cast<bf16x8*>(to + row * 128 + ((2 * part) ^ (row & 7)) * 16) = values8(q.x, q.y, scale);
        *reinterpret_cast<bf16x8*>(to + row * 128 + ((2 * part + 1) ^ (row & 7)) * 16) = values8(q.z, q.w, scale);
    };
    auto stash = [&](unsigned s) {
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
            put(lds[s][0], r + 64 * h, xq[h], scaleOf(xb[h]));
            put(lds[s][1], r + 64 * h, wq[h], scaleOf(wb));
        }
    };
    const unsigned wm = wave % 2 * 64, wn = wave / 2 * 64, l16 = lane % 16, g = lane / 16;
    f32x4 acc[4][4] = {};
    const unsigned steps = 2 * a.count;
    fetch(0);
    stash(0);
    __syncthreads();
    for (unsigned k = 0; k < steps; ++k) {
        if (k + 1 < steps) fetch(k + 1);
        const std::uint8_t *bx = lds[k % 2][0], *bw = lds[k % 2][1];
#pragma unroll
        for (unsigned h = 0; h < 2; ++h) {
            bf16x8 xf[4];
#pragma unroll
            for (unsigned m = 0; m < 4; ++m) {
                const unsigned row = wm + m * 16 + l16;
                xf[m] = *reinterpret_cast<const bf16x8*>(bx + row * 128 + ((4 * h + g) ^ (row & 7)) * 16);
            }
#pragma unroll
            for (unsigned n = 0; n < 4; ++n) {
                const unsigned row = wn + n * 16 + l16;
                const bf16x8 wf = *reinterpret_cast<const bf16x8*>(bw + row * 128 + ((4 * h + g) ^ (row & 7)) * 16);
#pragma unroll
                for (unsigned m = 0; m < 4; ++m)
                    acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[m], acc[n][m], 0, 0, 0);
            }
        }
        if (k + 1 < steps) {
            stash((k + 1) % 2);
            __syncthreads();
        }
    }
    float* y = static_cast<float*>(a.y);
#pragma unroll
    for (unsigned n = 0; n < 4; ++n) {
        const unsigned column = tn + wn + n * 16 + g * 4;
        const f32x4 b = bias4(a.bias, column, a.outer);
#pragma unroll
        for (unsigned m = 0; m < 4; ++m) {
            const unsigned row = tm + wm + m * 16 + l16;
            if (row < a.rows) put4(y + row * a.yStride, column, a.outer, acc[n][m] + b);
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Many rows through a narrow layer (a graph's, after the sparse product): the weight fits in LDS. A workgroup
// takes it there once, as MFMA operands, and then each of its waves goes through rows of its own, 16 at a
// time, without a barrier: dense x is read once, quantized in the layout of an operand, kept if asked for, and
// multiplied with every column. Bound by HBM; what it saves against the tiles is writing and reading codes.
// Measured, FP32: 2,449,029 x 128 -> 256 804 us, 4.7 TB/s; 262,144 x 256 -> 47 with x kept 88 us, 4.4 TB/s;
// 262,144 x 47 -> 256 92, 3.4 TB/s, where rows of 188 bytes are read 16 at a time, 64 bytes of each. bf16: 1,000,000 x
// 128 -> 256 179, 4.3 TB/s; 300,000 x 512 -> 256 120, 3.8; f16, 1,000,000 x 100 -> 47 94, 3.1. Loads and stores
// are ordinary ones: a row's lines come and go in two or more accesses, and nontemporal loads took 3 to 10% longer
// (1,000,000 x 128 -> 128 255 us : 230), nontemporal stores up to 17% (1,000,000 x 128 -> 256 406 : 350).
//
// A lane reads 16 bytes of its row at a time, four lanes 64 bytes side by side. That gives it 32 elements of a
// block in an order of their own; the order along the inner axis is free as long as both operands share it,
// so the weight is laid out in the same order: element e of a block is in lane group e / 4 % 4 (FP32) or
// e / 8 % 4, after those of the groups before it in the block.
// swapGroups<16>: where bit 4 of the lane is set, a takes the b of the lane without it, which takes a in turn;
// swapGroups<32>: bit 5.
template <unsigned Lanes> __device__ __forceinline__ void swapGroups(unsigned& a, unsigned& b) {
    const auto r = Lanes == 16 ? __builtin_amdgcn_permlane16_swap(a, b, false, false)
                               : __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
}

template <typename T, unsigned Blocks>
__global__ __launch_bounds__(512) void multiplyRows(Product a) {
    constexpr bool Exact = std::is_same<T, F32>::value;
    constexpr unsigned Run = Exact ? 4 : 8, Image = Exact ? 256 : 128; // elements of a load; bytes of a weight block
    constexpr unsigned Together = 4, Fill = 4; // column tiles multiplied at a time; loads of the weight in flight
    typedef typename T::Raw Raw;
    typedef Raw RunVec __attribute__((ext_vector_type(Run)));
    typedef RunVec LooseRun __attribute__((aligned(alignof(Raw))));
    extern __shared__ __align__(1024) std::uint8_t lds[];
    const unsigned t = threadIdx.x, lane = t % kWave, wave = t / kWave, l16 = lane % 16, g = lane / 16;
    const unsigned tiles = (a.outer + 16 * Together - 1) / (16 * Together) * Together, slots = tiles * 16;
    // Column of slot s: a 16-bit y has 8 columns of two tiles in one lane.
    auto columnOf = [](unsigned s) {
        if constexpr (Exact) return s;
        return s / 32 * 32 + s % 16 / 4 * 8 + s / 16 % 2 * 4 + s % 4;
    };
    for (unsigned i0 = t; i0 < slots * Blocks * 8; i0 += 512 * Fill) {
        u32x4 q[Fill];
        unsigned e[Fill];
#pragma unroll
        for (unsigned f = 0; f < Fill; ++f) {
            const unsigned i = i0 + f * 512, part = i % 8, block = i / 8 % Blocks;
            const unsigned column = min(columnOf(i / 8 / Blocks), a.outer - 1);
            q[f] = *reinterpret_cast<const u32x4*>(a.w + (std::uint64_t(column) * Blocks + block) * kBlock + part * 16);
            e[f] = a.we[std::uint64_t(column / kBlock) * a.expPitch + block];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (unsigned f = 0; f < Fill; ++f) {
            const unsigned i = i0 + f * 512, part = i % 8, block = i / 8 % Blocks, slot = i / 8 / Blocks;
            if (slot >= slots) break;
            const bool in = columnOf(slot) < a.outer;
            std::uint8_t* to = lds + (block * slots + slot) * Image;
            if constexpr (Exact) {
                // 16-byte chunks of a 256-byte row: 4 * group + (element of the group) / 8.
                const float scale = in ? scaleOf(e[f]) : 0.0f;
#pragma unroll
                for (unsigned j = 0; j < 4; ++j) {
                    const unsigned c = in ? q[f][j] : 0;
                    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, false);
                    const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, true);
                    *reinterpret_cast<u32x2*>(to + ((4 * j + part / 2) ^ (slot & 15)) * 16 + part % 2 * 8) =
                        u32x2{__builtin_bit_cast(unsigned, lo), __builtin_bit_cast(unsigned, hi)};
                }
            } else {
#pragma unroll
                for (unsigned j = 0; j < 2; ++j) {
                    const unsigned at = (part % 2 * 2 + j) * 32 + part / 2 * 8;
                    *reinterpret_cast<u32x2*>(to + ((at / 16) ^ (slot & 7)) * 16 + at % 16) =
                        in ? u32x2{q[f][2 * j], q[f][2 * j + 1]} : u32x2{0, 0};
                }
            }
        }
    }
    __syncthreads();
    const unsigned groups = (a.rows + 15) / 16;
    for (unsigned group = blockIdx.x * 8 + wave; group < groups; group += gridDim.x * 8) {
        const unsigned row = group * 16 + l16;
        const Raw* x = static_cast<const Raw*>(a.dense) + min(row, a.rows - 1) * a.denseStride;
        RunVec raw[Blocks][32 / Run];
#pragma unroll
        for (unsigned b = 0; b < Blocks; ++b)
#pragma unroll
            for (unsigned i = 0; i < 32 / Run; ++i) {
                const unsigned at = min(b * kBlock + (i * 4 + g) * Run, a.inner - Run);
                raw[b][i] = RunVec{};
                if (b + 1 < Blocks || b * kBlock + i * 4 * Run < a.inner)
                    raw[b][i] = *reinterpret_cast<const LooseRun*>(x + at);
            }
        __builtin_amdgcn_sched_barrier(0);
        if (a.inner != Blocks * kBlock) {
            // The last block ends early: runs past the row read its last elements, which move to their places.
#pragma unroll
            for (unsigned i = 0; i < 32 / Run; ++i) {
                const unsigned at = (Blocks - 1) * kBlock + (i * 4 + g) * Run, past = at - min(at, a.inner - Run);
                RunVec& v = raw[Blocks - 1][i];
                if (a.inner % Run) {
#pragma unroll
                    for (unsigned by = Run / 2; by; by /= 2)
#pragma unroll
                        for (unsigned j = 0; j + by < Run; ++j) v[j] = past & by ? v[j + by] : v[j];
                }
#pragma unroll
                for (unsigned j = 0; j < Run; ++j) v[j] = past + j < Run ? v[j] : Raw(0.0f);
            }
        }
        u32x4 q[Blocks][2];
        unsigned xe[Blocks];
#pragma unroll
        for (unsigned b = 0; b < Blocks; ++b) {
            float v[4][8];
            unsigned peak = 0;
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) {
#pragma unroll
                for (unsigned j = 0; j < 8; ++j) v[i][j] = T::get(raw[b][(i * 8 + j) / Run][j % Run]);
                peak = max(peak, peakBits(v[i]));
            }
            peak = max(peak, unsigned(__shfl_xor(int(peak), 16)));
            peak = max(peak, unsigned(__shfl_xor(int(peak), 32)));
            xe[b] = exponentOf<BlockCodes::e4m3>(peak);
            const u32x2 q0 = encode8<BlockCodes::e4m3>(v[0], xe[b]), q1 = encode8<BlockCodes::e4m3>(v[1], xe[b]);
            const u32x2 q2 = encode8<BlockCodes::e4m3>(v[2], xe[b]), q3 = encode8<BlockCodes::e4m3>(v[3], xe[b]);
            q[b][0] = u32x4{q0.x, q0.y, q1.x, q1.y};
            q[b][1] = u32x4{q2.x, q2.y, q3.x, q3.y};
            if (a.keep) {
                // Lane groups exchange codes until each has 16 bytes side by side: four store 64 bytes of a row.
                std::uint8_t* to = a.keep + (std::uint64_t(row) * Blocks + b) * kBlock;
#pragma unroll
                for (unsigned h = 0; h < 2; ++h) {
                    unsigned c[4] = {q[b][h][0], q[b][h][1], q[b][h][2], q[b][h][3]};
                    if constexpr (Exact) {
                        swapGroups<16>(c[0], c[1]), swapGroups<16>(c[2], c[3]);
                        swapGroups<32>(c[0], c[2]), swapGroups<32>(c[1], c[3]);
                    } else {
                        swapGroups<16>(c[0], c[2]), swapGroups<16>(c[1], c[3]);
                    }
                    const unsigned at = h * 64 + (Exact ? g * 16 : g % 2 * 32 + g / 2 * 16);
                    if (row < a.rows) *reinterpret_cast<u32x4*>(to + at) = u32x4{c[0], c[1], c[2], c[3]};
                }
            }
        }
        if (a.keep && row < a.rows && g == 0) {
            unsigned exponents = 0x7F7F7F7Fu;
#pragma unroll
            for (unsigned b = 0; b < Blocks; ++b) exponents ^= (xe[b] ^ 0x7Fu) << 8 * b;
            reinterpret_cast<unsigned*>(a.keepExp)[row] = exponents;
        }
        Raw* y = static_cast<Raw*>(a.y) + row * a.yStride;
        for (unsigned tile = 0; tile < tiles; tile += Together) {
            f32x4 acc[Together] = {};
#pragma unroll
            for (unsigned b = 0; b < Blocks; ++b) {
                const std::uint8_t* w = lds + (b * slots + tile * 16 + l16) * Image;
                if constexpr (Exact) {
                    const float scale = scaleOf(xe[b]);
#pragma unroll
                    for (unsigned i = 0; i < 4; ++i) {
                        const bf16x8 xf = values8(q[b][i / 2][i % 2 * 2], q[b][i / 2][i % 2 * 2 + 1], scale);
#pragma unroll
                        for (unsigned n = 0; n < Together; ++n)
                            acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                *reinterpret_cast<const bf16x8*>(w + n * 16 * Image + ((4 * g + i) ^ l16) * 16), xf,
                                acc[n], 0, 0, 0);
                    }
                } else {
                    const unsigned we = a.we[std::uint64_t(tile * 16 / kBlock) * a.expPitch + b];
#pragma unroll
                    for (unsigned n = 0; n < Together; ++n) {
                        const u32x4* p = reinterpret_cast<const u32x4*>(w + n * 16 * Image);
                        acc[n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                            join(p[(2 * g) ^ (l16 & 7)], p[(2 * g + 1) ^ (l16 & 7)]), join(q[b][0], q[b][1]), acc[n], 0, 0,
                            0, int(we), 0, int(xe[b]));
                    }
                }
            }
            // The sums are needed here, by all lanes: left to itself the compiler moves the multiplication, with its reads
            // of LDS, to where only the lanes with a row run.
#pragma unroll
            for (unsigned n = 0; n < Together; ++n) asm volatile("" ::"v"(acc[n]));
            if (row >= a.rows) continue;
            if constexpr (Exact) {
#pragma unroll
                for (unsigned n = 0; n < Together; ++n) {
                    const unsigned column = (tile + n) * 16 + g * 4;
                    put4(y, column, a.outer, acc[n] + bias4(a.bias, column, a.outer));
                }
            } else {
#pragma unroll
                for (unsigned n = 0; n < Together; n += 2) {
                    const unsigned column = (tile + n) * 16 + g * 8;
                    float v[8], b[8];
#pragma unroll
                    for (unsigned i = 0; i < 8; ++i) v[i] = acc[n + i / 4][i % 4];
                    bias8<false>(a.bias, column, a.outer, b);
                    put8<T, false>(y, column, a.outer, v, b);
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Few rows (single tokens, small batches): a workgroup takes 16 columns of y for up to 64 rows; its eight waves
// share the blocks of the inner axis and add their sums through LDS in the waves' order. The weight's
// codes go from memory to the MFMA's registers, each byte read once on the chip, four blocks' loads at a
// time before the first is used: what bounds this is how many bytes are on their way. A lane takes 32
// consecutive codes of its row.
// Dense: up to kFusedRows rows of dense x, which every workgroup quantizes for itself into LDS while its
// first weights are on their way; more rows than that are cheaper to quantize once, in a launch of its own.
// Measured, 4096 x 4096 bf16: 1 row 5.3 us (6.2 among others), 3.2 TB/s, about 2 us of it the launch and the first
// load's way; 2 rows 7.3, 4 rows 8.9, where the two launches of 5 rows take 9.1. FP32 blocks: 16 rows 8.4, 64 rows 18.
constexpr unsigned kTokenWaves = 8, kFusedRows = 4;

template <typename T, unsigned MT, bool Dense>
__global__ __launch_bounds__(kWave* kTokenWaves) void multiplyTokens(Product a) {
    constexpr bool Exact = std::is_same<T, F32>::value;
    constexpr unsigned Ahead = 4; // blocks of a wave loaded at a time
    __shared__ f32x4 sums[kTokenWaves][MT][kWave];
    extern __shared__ __align__(16) std::uint8_t lds[]; // Dense: x's codes, then its exponents
    const unsigned t = threadIdx.x, lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const unsigned l16 = lane % 16, g = lane / 16, n0 = blockIdx.x * 16, pitch = a.count * kBlock;
    const unsigned m0 = Dense ? 0 : blockIdx.y * 16 * MT;
    const std::uint8_t* wp = a.w + min(n0 + l16, a.outer - 1) * std::uint64_t(pitch) + g * 32;
    const std::uint8_t* wep = a.we + std::uint64_t(n0 / kBlock) * a.expPitch;
    std::uint8_t* exponents = lds + a.rows * pitch;
    u32x4 w[Ahead][2];
    auto fetch = [&](unsigned k) {
#pragma unroll
        for (unsigned u = 0; u < Ahead; ++u) {
            const std::uint8_t* p = wp + std::uint64_t(min(k + u * kTokenWaves, a.count - 1)) * kBlock;
            w[u][0] = *reinterpret_cast<const u32x4*>(p);
            w[u][1] = *reinterpret_cast<const u32x4*>(p + 16);
        }
    };
    fetch(wave);
    if constexpr (Dense) {
        const unsigned sub = t % kBlockLanes;
        for (unsigned item = t / kBlockLanes; item < a.rows * a.count; item += kWave * kTokenWaves / kBlockLanes) {
            const unsigned row = item / a.count, block = item - row * a.count;
            float v[8];
            load8<T>(static_cast<const typename T::Raw*>(a.dense) + row * a.denseStride, block * kBlock + sub * 8, a.inner, v);
            const unsigned e = exponentOf<BlockCodes::e4m3>(rowMax(peakBits(v)));
            const u32x2 q = encode8<BlockCodes::e4m3>(v, e);
            *reinterpret_cast<u32x2*>(lds + row * pitch + block * kBlock + sub * 8) = q;
            if (sub == 0) exponents[item] = std::uint8_t(e);
            if (a.keep && blockIdx.x == 0) {
                *reinterpret_cast<u32x2*>(a.keep + row * std::uint64_t(pitch) + block * kBlock + sub * 8) = q;
                if (block + sub < (block + 1 == a.count ? a.expPitch : block + 1))
                    a.keepExp[row * std::uint64_t(a.expPitch) + block + sub] = std::uint8_t(sub ? 127u : e);
            }
        }
        __syncthreads();
    }
    f32x4 acc[MT] = {};
    for (unsigned k = wave; k < a.count; k += Ahead * kTokenWaves) {
        u32x4 x[Ahead][MT][2];
        unsigned xe[Ahead][MT];
#pragma unroll
        for (unsigned u = 0; u < Ahead; ++u) {
            const unsigned block = min(k + u * kTokenWaves, a.count - 1);
#pragma unroll
            for (unsigned m = 0; m < MT; ++m) {
                const unsigned row = min(m0 + m * 16 + l16, a.rows - 1);
                const std::uint8_t* p = Dense ? lds + row * pitch : a.x + row * std::uint64_t(pitch);
                x[u][m][0] = *reinterpret_cast<const u32x4*>(p + block * kBlock + g * 32);
                x[u][m][1] = *reinterpret_cast<const u32x4*>(p + block * kBlock + g * 32 + 16);
                xe[u][m] = Dense ? exponents[row * a.count + block] : a.xe[row * std::uint64_t(a.expPitch) + block];
            }
        }
        __builtin_amdgcn_sched_barrier(0); // the compiler would move the loads down to their use
#pragma unroll
        for (unsigned u = 0; u < Ahead; ++u) {
            if (k + u * kTokenWaves >= a.count) break;
            const unsigned we = wep[k + u * kTokenWaves];
#pragma unroll
            for (unsigned m = 0; m < MT; ++m) {
                if constexpr (Exact) {
                    const float xs = scaleOf(xe[u][m]), ws = scaleOf(we);
#pragma unroll
                    for (unsigned i = 0; i < 4; ++i) {
                        const u32x4 wq = w[u][i / 2], xq = x[u][m][i / 2];
                        acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            values8(wq[i % 2 * 2], wq[i % 2 * 2 + 1], ws), values8(xq[i % 2 * 2], xq[i % 2 * 2 + 1], xs),
                            acc[m], 0, 0, 0);
                    }
                } else {
                    acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(w[u][0], w[u][1]),
                                                                              join(x[u][m][0], x[u][m][1]), acc[m], 0, 0,
                                                                              0, int(we), 0, int(xe[u][m]));
                }
            }
        }
        if (k + Ahead * kTokenWaves < a.count) fetch(k + Ahead * kTokenWaves);
    }
#pragma unroll
    for (unsigned m = 0; m < MT; ++m) sums[wave][m][lane] = acc[m];
    __syncthreads();
    // Output i of 256 * MT: column fastest.
    typename T::Raw* y = static_cast<typename T::Raw*>(a.y);
    for (unsigned i = t; i < 256 * MT; i += kWave * kTokenWaves) {
        const unsigned column = i % 16, r = i / 16, row = m0 + r;
        if (n0 + column >= a.outer || row >= a.rows) continue;
        float s = 0.0f;
#pragma unroll
        for (unsigned v = 0; v < kTokenWaves; ++v) s += sums[v][r / 16][r % 16 + column / 4 * 16][column % 4];
        if (a.bias) s += a.bias[n0 + column];
        y[row * a.yStride + n0 + column] = T::put(s);
    }
}

// ------------------------------------------------------------------------------------------------
// Host side

// Whether multiplyTokens takes an FP32 product, by the least estimated time in microseconds: rounds of its
// workgroups, 64 rows by 16 columns, against rounds of tiles of 128. The constants fit these times (rows x inner x
// outer, this form : tiles): 64 x 4096 x 4096 18 : 58, 100 x 4096 x 4096 29 : 59, 256 x 4096 x 4096 61 : 69,
// 512 x 4096 x 4096 119 : 72, 512 x 8192 x 512 31 : 115, 256 x 1024 x 1024 12.9 : 18.9, 300 x 1000 x 1000 22 : 19,
// 1024 x 1024 x 1024 46 : 19, 256 x 512 x 8192 52 : 13, 4096 x 4096 x 4096 - : 178.
bool exactTokens(std::uint32_t rows, std::uint32_t outer, unsigned count) {
    const auto over = [](std::uint64_t n, std::uint64_t size) { return (n + size - 1) / size; };
    const std::uint64_t groups = over(rows, 64) * over(outer, 16), tiles = over(rows, 128) * over(outer, 128);
    const double tokens = double(over(groups, 256)) * (count <= 4 ? 6.0 : 14.5 * std::max(1.0, count / 32.0));
    const double exact = tiles <= 256 ? 5.0 + 1.7 * count : double(over(tiles, 512)) * (5.0 + 2.6 * count);
    return rows <= 64 || (over(rows, 64) < 65536 && tokens < exact);
}

void launchTokens(const Product& p, hipStream_t stream) {
    const dim3 threads(kWave * kTokenWaves);
    const unsigned across = (p.outer + 15) / 16;
    if (p.rows <= 16)
        hipLaunchKernelGGL((multiplyTokens<F32, 1, false>), dim3(across), threads, 0, stream, p);
    else if (p.rows <= 32)
        hipLaunchKernelGGL((multiplyTokens<F32, 2, false>), dim3(across), threads, 0, stream, p);
    else
        hipLaunchKernelGGL((multiplyTokens<F32, 4, false>), dim3(across, (p.rows + 63) / 64), threads, 0, stream, p);
    checkHip(hipGetLastError());
}

// LDS of x's codes and exponents in a fused product of few rows.
std::size_t fusedLds(std::uint32_t rows, unsigned count) { return (std::size_t(rows) * count * (kBlock + 1) + 15) / 16 * 16; }
bool fusedTokens(std::uint32_t rows, std::uint32_t inner) {
    return rows <= kFusedRows && fusedLds(rows, (inner + kBlock - 1) / kBlock) <= 48 * 1024;
}

template <typename T> void launchFusedTokens(const Product& p, hipStream_t stream) {
    hipLaunchKernelGGL((multiplyTokens<T, 1, true>), dim3((p.outer + 15) / 16), dim3(kWave * kTokenWaves),
                       fusedLds(p.rows, p.count), stream, p);
    checkHip(hipGetLastError());
}

// The tile of a 16-bit product: the least estimated time, in microseconds, rounds of workgroups on the chip
// times the blocks of the inner axis. A CU holds one workgroup of tiles of 256 or, with its four groups of
// waves, 32, two of 128 or 64. The constants fit these times (rows x inner x outer: 256, 128, 64, 32):
//   4096 x 4096 x 8192 122, 192, 269, -     2048 x 1024 x 4096 22, 15.2, 20, -    2048 x 4096 x 1024 49, 28.8, 17.7, 40
//   1024 x 4096 x 4096 51, 31.3, 31.0, 78   512 x 4096 x 4096 48, 26.9, 17.9, 40  16384 x 512 x 512 16, 10.9, 14.4, -
//   777 x 1001 x 1437 23, 9.9, 6.7, 16      300 x 2000 x 6000 31, 13.8, 9.5, 27   100000 x 256 x 256 29, 20.9, 30.7, -
//   128 x 4096 x 4096 48, 24, 8.9, 11.0     24 x 4096 x 8192 -, -, 9.7, 6.8       16 x 1024 x 4096 -, -, 4.2, 4.5
enum class Form { wide, middle, small, few };
Form formOf(std::uint32_t rows, std::uint32_t outer, unsigned count) {
    const auto tiles = [&](unsigned size) {
        return std::uint64_t((rows + size - 1) / size) * ((outer + size - 1) / size);
    };
    const auto rounds = [](std::uint64_t n, unsigned slots) { return double((n + slots - 1) / slots); };
    const std::uint64_t half = tiles(128), quarter = tiles(64);
    const double wide = rounds(tiles(256), 256) * (11.5 + 1.5 * count);
    double middle = half <= 256 ? 5.0 + 0.75 * count : rounds(half, 512) * (5.0 + 1.3 * count);
    double small = quarter <= 256 ? 2.9 + 0.18 * count : rounds(quarter, 512) * (1.5 + 0.5 * count);
    double few = rounds(tiles(32), 256) * (3.9 + 0.09 * count);
    // 2^27 rows and more can be too many tiles of these for a launch.
    if (!launchTakes(half, 512)) middle = wide + 1.0;
    if (!launchTakes(quarter, 256)) small = wide + 1.0;
    if (!launchTakes(tiles(32), 512)) few = wide + 1.0;
    const double least = std::min(std::min(wide, middle), std::min(small, few));
    return least == wide ? Form::wide : least == middle ? Form::middle : least == small ? Form::small : Form::few;
}

// The launch of a product, for calls to refuse before they launch anything, the coding of x among it. multiplyTokens is taken
// for no more rows than a launch takes.
void checkTiles(const char* where, std::uint32_t rows, std::uint32_t outer, unsigned count, DenseType type) {
    const auto check = [&](unsigned size, unsigned threads) {
        checkGrid(where, std::uint64_t((rows + size - 1) / size) * ((outer + size - 1) / size), threads);
    };
    if (type == DenseType::f32) {
        if (!exactTokens(rows, outer, count)) check(128, 256);
        return;
    }
    switch (formOf(rows, outer, count)) {
    case Form::wide: return check(256, 256);
    case Form::middle: return check(128, 512);
    case Form::small: return check(64, 256);
    case Form::few: return check(32, 512);
    }
}

template <typename T, unsigned BM, unsigned BN, unsigned WM, unsigned WN, unsigned Stages, unsigned Groups>
void launchTiles(Product p, hipStream_t stream) {
    p.tilesM = (p.rows + BM - 1) / BM, p.tilesN = (p.outer + BN - 1) / BN;
    const std::uint64_t tiles = std::uint64_t(p.tilesM) * p.tilesN;
    const std::size_t lds = Groups * Stages * (BM + BN) * kBlock;
    hipLaunchKernelGGL((multiplyTiles<T, BM, BN, WM, WN, Stages, Groups>), dim3(unsigned(tiles)),
                       dim3(64 * WM * WN * Groups), lds, stream, p);
    checkHip(hipGetLastError());
}

template <typename T> void launchWide(Product p, hipStream_t stream) {
    p.tilesM = (p.rows + 255) / 256, p.tilesN = (p.outer + 255) / 256;
    const std::uint64_t tiles = std::uint64_t(p.tilesM) * p.tilesN;
    hipLaunchKernelGGL((multiplyWide<T>), dim3(unsigned(tiles)), dim3(256), 2 * 2 * 256 * kBlock, stream, p);
    checkHip(hipGetLastError());
}

template <typename T> void launchProduct(Product p, hipStream_t stream) {
    if constexpr (std::is_same<T, F32>::value) {
        if (exactTokens(p.rows, p.outer, p.count)) return launchTokens(p, stream);
        p.tilesM = (p.rows + 127) / 128;
        const std::uint64_t tiles = std::uint64_t(p.tilesM) * ((p.outer + 127) / 128);
        hipLaunchKernelGGL(multiplyTilesExact, dim3(unsigned(tiles)), dim3(256), 0, stream, p);
        checkHip(hipGetLastError());
    } else {
        switch (formOf(p.rows, p.outer, p.count)) {
        case Form::wide: launchWide<T>(p, stream); break;
        case Form::middle: launchTiles<T, 128, 128, 4, 2, 2, 1>(p, stream); break;
        case Form::small: launchTiles<T, 64, 64, 2, 2, 4, 1>(p, stream); break;
        case Form::few: launchTiles<T, 32, 32, 2, 1, 4, 4>(p, stream); break;
        }
    }
}

void checkWeight(const char* where, const BlockWeightView& w, const float* bias) {
    checkCodes(where, w.codes, w.exponents);
    if (reinterpret_cast<std::uintptr_t>(bias) % 4) reject(where, "bias not float-aligned");
}

} // namespace

void matmulBlocks(BlockRows x, BlockWeightView w, const float* bias, void* y, DenseType type, std::uint64_t stride,
                  std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, hipStream_t stream) {
    const char* where = "matmul blocks";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkRows(where, rows);
    if (x.type != BlockCodes::e4m3) reject(where, "x must have E4M3 codes");
    checkType(where, type);
    if (!rows) return;
    checkCodes(where, x.codes, x.exponents);
    checkWeight(where, w, bias);
    checkDense(where, y, stride, type, outer);
    Product p = {};
    p.x = x.codes, p.xe = x.exponents, p.w = w.codes, p.we = w.exponents, p.bias = bias;
    p.y = y, p.yStride = stride, p.rows = rows, p.outer = outer, p.inner = inner;
    p.count = (inner + kBlock - 1) / kBlock;
    p.expPitch = unsigned(blockExponentPitch(inner));
    checkTiles(where, rows, outer, p.count, type);
    withType(type, [&](auto tag) { launchProduct<decltype(tag)>(p, stream); });
}

namespace {
// The weight's bytes in LDS if a narrow layer with many rows goes through multiplyRows, else 0. A group of 128 rows
// fills an image of its own, so the larger it is, the more rows it takes to pay. Measured in us, here against a
// launch that quantizes and tiles: f32 128 -> 128 (32 KiB) at 4096 rows 8.3 : 9.0, 8192 8.3 : 10.2; bf16 128 -> 256
// (32 KiB) at 4096 7.2 : 5.3, 8192 7.6 : 6.9, 20000 9.0 : 12.0; f32 128 -> 256 (64 KiB) at 8192 12.3 : 10.8, 20000
// 13.4 : 16.3; bf16 512 -> 256 (128 KiB) at 8192 15.5 : 10.7, 16384 18 : 18, 300000 129 : 172. Rows of fewer than 8
// elements cannot be read 8 at a time.
constexpr unsigned kRowsLds = 160 * 1024;
std::size_t rowsImage(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type) {
    const std::uint64_t count = (inner + kBlock - 1) / kBlock, slots = (std::uint64_t(outer) + 63) / 64 * 64;
    const std::uint64_t bytes = slots * count * (type == DenseType::f32 ? 256 : 128);
    const bool enough = inner >= 8 && rows >= (bytes <= 32 * 1024 ? 8192u : 16384u);
    return enough && count <= 4 && bytes <= kRowsLds ? std::size_t(bytes) : 0;
}

template <typename T> void launchRows(const Product& p, std::size_t lds, hipStream_t stream) {
    // Two workgroups a CU where their images fit; rows of at least one round of its waves for each.
    const unsigned grid = std::min((p.rows + 127) / 128, lds <= kRowsLds / 2 ? 512u : 256u);
    switch (p.count) {
    case 1: hipLaunchKernelGGL((multiplyRows<T, 1>), dim3(grid), dim3(512), lds, stream, p); break;
    case 2: hipLaunchKernelGGL((multiplyRows<T, 2>), dim3(grid), dim3(512), lds, stream, p); break;
    case 3: hipLaunchKernelGGL((multiplyRows<T, 3>), dim3(grid), dim3(512), lds, stream, p); break;
    case 4: hipLaunchKernelGGL((multiplyRows<T, 4>), dim3(grid), dim3(512), lds, stream, p); break;
    }
    checkHip(hipGetLastError());
}

std::size_t rounded(std::uint64_t bytes) { return std::size_t((bytes + 255) / 256 * 256); }
} // namespace

const char* matmulBlocksForm(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type) {
    checkColumns("matmul blocks", inner);
    checkColumns("matmul blocks", outer);
    checkType("matmul blocks", type);
    const unsigned count = (inner + kBlock - 1) / kBlock;
    if (type == DenseType::f32) return exactTokens(rows, outer, count) ? "multiplyTokens" : "multiplyTilesExact";
    switch (formOf(rows, outer, count)) {
    case Form::wide: return "multiplyWide";
    case Form::middle: return "multiplyTiles128";
    case Form::small: return "multiplyTiles64";
    default: return "multiplyTiles32";
    }
}

const char* linearBlocksForm(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type) {
    const char* product = matmulBlocksForm(rows, inner, outer, type);
    return rowsImage(rows, inner, outer, type) ? "multiplyRows" : fusedTokens(rows, inner) ? "multiplyTokensDense" : product;
}

std::size_t linearBlocksWorkspace(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type,
                                  bool keep) {
    if (keep || fusedTokens(rows, inner) || rowsImage(rows, inner, outer, type)) return 0;
    return rounded(rows * blockCodePitch(inner)) + rounded(rows * blockExponentPitch(inner));
}

void linearBlocks(DenseMatrix x, BlockWeightView w, const float* bias, void* y, std::uint64_t yStride, BlockRows keep,
                  std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, void* workspace,
                  std::size_t workspaceBytes, hipStream_t stream) {
    const char* where = "linear blocks";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkRows(where, rows);
    checkType(where, x.type);
    if (!keep.codes != !keep.exponents) reject(where, "kept codes and exponents come together");
    if (keep.codes && keep.type != BlockCodes::e4m3) reject(where, "kept blocks must have E4M3 codes");
    if (!rows) return;
    checkDense(where, x.data, x.stride, x.type, inner);
    checkDense(where, y, yStride, x.type, outer);
    checkWeight(where, w, bias);
    if (keep.codes) checkCodes(where, keep.codes, keep.exponents);
    const std::size_t need = linearBlocksWorkspace(rows, inner, outer, x.type, keep.codes);
    if (need > workspaceBytes || (need && !workspace)) reject(where, "workspace too small");
    if (reinterpret_cast<std::uintptr_t>(workspace) % 16) reject(where, "workspace must be 16-byte aligned");
    const std::size_t image = rowsImage(rows, inner, outer, x.type);
    if (fusedTokens(rows, inner) || image) {
        Product p = {};
        p.w = w.codes, p.we = w.exponents, p.bias = bias, p.y = y, p.yStride = yStride;
        p.rows = rows, p.outer = outer, p.inner = inner;
        p.count = (inner + kBlock - 1) / kBlock;
        p.expPitch = unsigned(blockExponentPitch(inner));
        p.dense = x.data, p.denseStride = x.stride, p.keep = keep.codes, p.keepExp = keep.exponents;
        withType(x.type, [&](auto tag) {
            if (image)
                launchRows<decltype(tag)>(p, image, stream);
            else
                launchFusedTokens<decltype(tag)>(p, stream);
        });
        return;
    }
    checkTiles(where, rows, outer, (inner + kBlock - 1) / kBlock, x.type);
    auto* spare = static_cast<std::uint8_t*>(workspace);
    if (!keep.codes) keep = {spare, spare + rounded(rows * blockCodePitch(inner)), BlockCodes::e4m3};
    quantizeBlocks(x, keep, rows, inner, stream);
    matmulBlocks(keep, w, bias, y, x.type, yStride, rows, inner, outer, stream);
}

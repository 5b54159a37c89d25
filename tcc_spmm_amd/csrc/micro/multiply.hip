// Products with weights in microscaled 4-bit blocks, y = x w^T + bias (include/micro.h), the linear layer on dense x, and
// the experts' products (include/experts.h).
//
// What the kernels share. The weight is the scaled MFMA's first operand, x its second; 16 rows of each by 128 elements of
// the inner axis, a step. Of a row in 4 bits a lane takes 32 elements in a row, 16 bytes, block g = lane / 16 of the
// step, and gives that block's scale; of a row in 8 bits it takes elements 16 g to 16 g + 15 and 64 more, which is how
// the instruction pairs them, and the row's one scale. A dword of exponents has four steps, a byte each, for
// either (include/micro.h), so that no kernel moves them about.
#include "blocks/device_product.h"
#include "experts.h"
#include "hip_support.h"
#include "micro/device_micro.h"

#include <algorithm>
#include <cmath>

namespace {

using namespace micro;

struct Product {
    const std::uint8_t *x, *xe;
    const std::uint8_t *w, *we;
    const float* bias;
    void* y;
    std::uint64_t yStride;
    unsigned rows, inner, outer, count; // count: steps of a row
    std::uint64_t xeRow, xeNext; // microWide: bytes from a row's exponents of x to the next row's, from four steps' to the next
    unsigned tilesM, tilesN;            // experts: tilesM is the most that their rows can make
    const void* dense;
    std::uint64_t denseStride;
    std::uint8_t *keep, *keepExp;
    // Experts: rows are the plan's choices.
    const std::int32_t *offsets, *order; // null order: x has a row for each
    unsigned experts, each;
};

// Bytes of rows of codes and of exponents.
template <bool X8> __device__ __forceinline__ unsigned xPitch(const Product& a) { return a.count * (X8 ? kStep : kStep / 2); }
template <bool X8> __device__ __forceinline__ unsigned xExpPitch(const Product& a) { return (a.count + 3) / 4 * (X8 ? 4 : 16); }
__device__ __forceinline__ unsigned wPitch(const Product& a) { return a.count * (kStep / 2); }
__device__ __forceinline__ unsigned wExpPitch(const Product& a) { return (a.count + 3) / 4 * 16; }

// Steps in which block g of the four holds elements of the row.
__device__ __forceinline__ unsigned stepsOfLane(const Product& a, unsigned g) {
    return ((a.inner + kMicroBlock - 1) / kMicroBlock + 3 - g) / 4;
}

// acc += w x of one step; ws and xs have the scales in byte S.
template <bool X8, unsigned S>
__device__ __forceinline__ f32x4 multiply(u32x4 w, u32x4 x0, u32x4 x1, f32x4 acc, unsigned ws, unsigned xs) {
    const u32x4 none = {};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(w, none), X8 ? join(x0, x1) : join(x0, none), acc, 4,
                                                            X8 ? 0 : 4, S, int(ws), S, int(xs));
}

// The values of 8 E2M1 codes as bf16. Exact but for the upper end: values of 2^128 and more, which exponents above 252 can
// give and quantizing does not, are infinite.
__device__ __forceinline__ bf16x8 microValues8(unsigned q, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
    return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// ------------------------------------------------------------------------------------------------
// Experts: which rows a workgroup multiplies with which weight.
//
// The row tiles of all experts, one expert after the other and at last the rows of none, are numbered; how many each has
// is known to the device alone. A wave counts them, 64 experts at a time, and finds the one that its number falls
// into. A launch has as many workgroups as any plan of these sizes can need; those past the last tile end at once.
// Tiles of no expert, whose outputs are zeros and which nothing is multiplied for, are dealt to the workgroups by themselves
// behind all others: in one run with them the last XCDs would have nothing to multiply. 8192 tokens to 4 of 32 experts, 2048 x
// 4096 in 4 bits, by the share of choices away: none 280 us, a tenth 264, half 195, all 44, the zeros at 6.1 TB/s.
struct Span {
    unsigned expert, first, end; // rows [first, end) of the tile's expert
};

__device__ __forceinline__ unsigned tilesOfLane(const Product& a, unsigned e, unsigned tile, unsigned& lo, unsigned& hi) {
    lo = e <= a.experts ? min(unsigned(a.offsets[e]), a.rows) : a.rows;
    hi = e < a.experts ? min(unsigned(a.offsets[e + 1]), a.rows) : a.rows;
    hi = max(lo, hi);
    return (hi - lo + tile - 1) / tile;
}

__device__ __forceinline__ unsigned scanWave(unsigned v, unsigned lane) {
#pragma unroll
    for (unsigned by = 1; by < kWave; by *= 2) {
        const unsigned up = unsigned(__shfl_up(int(v), by));
        v += lane >= by ? up : 0;
    }
    return v;
}

// Row tile `id` of `tile` rows each, `id` being any function of their number and that of the last ones, of no expert. False:
// there is no such tile.
template <typename F>
__device__ __forceinline__ bool spanOf(const Product& a, unsigned tile, unsigned lane, F idOf, Span& s) {
    unsigned lo, hi, n = tilesOfLane(a, lane, tile, lo, hi), upTo = scanWave(n, lane), before = 0;
    unsigned total = __builtin_amdgcn_readlane(upTo, kWave - 1), none = __builtin_amdgcn_readlane(n, a.experts % kWave);
    for (unsigned base = kWave; base <= a.experts; base += kWave) { // more experts than lanes: their tiles too
        unsigned l, h, m = tilesOfLane(a, base + lane, tile, l, h);
        none = __builtin_amdgcn_readlane(m, a.experts % kWave); // at last that of the run which they are in
#pragma unroll
        for (unsigned by = kWave / 2; by; by /= 2) m += unsigned(__shfl_xor(int(m), by));
        total += __builtin_amdgcn_readfirstlane(m);
    }
    const unsigned id = idOf(total, none);
    if (id >= total) return false;
    unsigned base = 0;
    while (base <= a.experts && id >= unsigned(__builtin_amdgcn_readlane(upTo, kWave - 1))) {
        before = __builtin_amdgcn_readlane(upTo, kWave - 1), base += kWave;
        n = tilesOfLane(a, base + lane, tile, lo, hi), upTo = scanWave(n, lane) + before;
    }
    const std::uint64_t past = __ballot(upTo > id);
    if (!past) return false; // lists that are no plan, whose tiles are more than 32 bits hold
    const unsigned at = unsigned(__builtin_ctzll(past)), start = __builtin_amdgcn_readlane(upTo - n, at);
    const unsigned first = unsigned(__builtin_amdgcn_readlane(lo, at)) + (id - start) * tile;
    s = {base + at, min(first, a.rows - 1), unsigned(__builtin_amdgcn_readlane(hi, at))};
    return true;
}

// The row of x that sorted row r takes.
__device__ __forceinline__ unsigned sourceOf(const Product& a, unsigned r) {
    r = min(r, a.rows - 1);
    return a.order ? min(unsigned(a.order[r]), a.rows - 1) / a.each : r;
}

// Zeros for rows of no expert.
template <typename T>
__device__ __forceinline__ void zeroTile(const Product& a, const Span& s, unsigned rows, unsigned tn, unsigned columns) {
    const unsigned end = min(s.end, s.first + rows);
    const float zeros[8] = {};
    for (unsigned i = threadIdx.x; i < rows * columns / 8; i += blockDim.x) {
        const unsigned row = s.first + i / (columns / 8), column = tn + i % (columns / 8) * 8;
        if (row < end && column < a.outer)
            put8<T, false>(static_cast<typename T::Raw*>(a.y) + row * a.yStride, column, a.outer, zeros, zeros);
    }
}

// Tile `id` of all: its row tile of `tilesM`, the last `none` of which are of no expert, and its first column. Past the
// last one: tilesM.
template <unsigned BN>
__device__ __forceinline__ unsigned expertTile(const Product& a, unsigned id, unsigned tilesM, unsigned none, unsigned& tn) {
    const unsigned used = tilesM - none, total = used * a.tilesN;
    if (id < total) {
        const unsigned tile = tileOf(id, total, used, a.tilesN);
        tn = tile / used * BN;
        return tile % used;
    }
    tn = (id - total) % a.tilesN * BN;
    return min(used + (id - total) / a.tilesN, tilesM);
}

// A workgroup's tile: rows [first, end) of an expert's and columns from tn on. False: it has nothing left to do.
struct Tile {
    unsigned expert, first, end, tn;
};
template <typename T, bool Experts, unsigned BM, unsigned BN>
__device__ __forceinline__ bool findTile(const Product& a, unsigned lane, Tile& t) {
    if constexpr (Experts) {
        Span s;
        const bool some = spanOf(a, BM, lane, [&](unsigned tilesM, unsigned none) {
            return expertTile<BN>(a, blockIdx.x, tilesM, none, t.tn);
        }, s);
        if (!some) return false;
        t = {s.expert, s.first, s.end, t.tn};
        if (s.expert < a.experts) return true;
        zeroTile<T>(a, s, BM, t.tn, BN);
        return false;
    } else {
        const unsigned tile = tileOf(blockIdx.x, gridDim.x, a.tilesM, a.tilesN);
        t = {0, tile % a.tilesM * BM, a.rows, tile / a.tilesM * BN};
        return true;
    }
}

// The expert's weight and bias. The tile is the same in all lanes, and said to be: the compiler does not see it behind
// spanOf's loop, and would read buffers lane by lane.
template <bool Experts> __device__ __forceinline__ void take(Product& a, Tile& t) {
    if constexpr (Experts) {
        t = {unsigned(__builtin_amdgcn_readfirstlane(t.expert)), unsigned(__builtin_amdgcn_readfirstlane(t.first)),
             unsigned(__builtin_amdgcn_readfirstlane(t.end)), unsigned(__builtin_amdgcn_readfirstlane(t.tn))};
        const std::uint64_t rows = std::uint64_t(t.expert) * a.outer;
        a.w += rows * wPitch(a), a.we += rows * wExpPitch(a);
        if (a.bias) a.bias += rows;
    }
}

// ------------------------------------------------------------------------------------------------
// Tiles of BM x BN. A step of the loop is 128 bytes of each of x's rows: 128 elements in 8 bits, 256 in 4, of which each
// half is an MFMA's. They and the weight's rows are loaded to LDS without passing registers, Stages deep. The
// 16-byte chunks of a row are stored in an order that depends on the row, so that the rows an MFMA operand takes at once
// lie in different banks. Rows of the weight are dealt to pairs of MFMAs so that a lane ends with 8
// consecutive outputs of one row of y. Groups of waves share a tile where there are few, each with a run of the inner axis
// and stages of its own; the first adds the others' sums.
// An FP32 y of E4M3 rows takes the codes' values, exact in bf16, through the bf16 MFMA, whose sums are FP32's: a wave converts
// the codes that it has read from LDS, four conversions for each MFMA of 16 cycles in tiles of 64.
// What bounds them is the chain of a step, a barrier and the LDS reads behind it, and for few rows the weight's way from
// memory. Measured, us: 48 x 4096 x 8191 with 8-bit rows 9.3 in tiles of 64 x 32 (11.5 in tiles of 64, twice the steps for half
// the CUs); 17 x 4096 x 4096 6.6 in tiles of 32; 24 tokens to 4 of 32 experts, 2048 x 4096, 25 in tiles of 64, 5.8 TB/s of the weights; 6002 rows of 8 experts, 2048 x 1000, 30
// in tiles of 128; FP32: 2001 x 1024 x 4097 32, 0.53 PFLOP/s, 2001 x 4097 x 1024 26, 0.64.
template <typename T, bool X8, bool Experts, unsigned BM, unsigned BN, unsigned WM, unsigned WN, unsigned Stages, unsigned Groups>
__global__ __launch_bounds__(64 * WM * WN * Groups) void microTiles(Product a) {
    constexpr unsigned Waves = WM * WN, MT = BM / WM / 16, NT = BN / WN / 16;
    constexpr bool Exact = X8 && std::is_same<T, F32>::value;
    constexpr unsigned Halves = X8 ? 1 : 2, Dword = 4 / Halves; // MFMAs of a step; steps of a dword of exponents
    constexpr unsigned WRow = Halves * 64, Stage = BM * 128 + BN * WRow; // bytes
    constexpr unsigned XL = BM / 8 / Waves, WL = BN * WRow / 1024 / Waves;
    static_assert(XL * Waves * 8 == BM && WL * Waves * 1024 == BN * WRow, "whole loads of a wave");
    static_assert((Stages == 2 || Stages == 4) && Dword % Halves == 0, "the stage is a constant of the unrolled step");
    static_assert(NT % 2 == 0 && Waves % 2 == 0, "pairs of operands; keys take bit 3 of the row");
    extern __shared__ __align__(1024) std::uint8_t shared[];
    const unsigned lane = threadIdx.x % kWave, allWaves = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned wave = allWaves % Waves, part = Groups == 1 ? 0 : allWaves / Waves;
    std::uint8_t* lds = shared + part * Stages * Stage;
    Tile found;
    if (!findTile<T, Experts, BM, BN>(a, lane, found)) return;
    take<Experts>(a, found);
    const unsigned tm = found.first, end = found.end, tn = found.tn;
    const unsigned all = (a.count + Halves - 1) / Halves; // steps; this group's are `steps` from `first` on
    const unsigned steps = Groups == 1 ? all : (all + Dword * Groups - 1) / (Dword * Groups) * Dword, first = part * steps;
    const unsigned pitch = xPitch<X8>(a), pitchW = wPitch(a);
    // Rows past the end are past the buffer and read as zeros, or another expert's; their results are not stored.
    const bool byToken = Experts && a.order;
    const auto xr = rowsAt(a.x, pitch, byToken ? 0 : tm, byToken ? a.rows / a.each : a.rows);
    const auto wr = rowsAt(a.w, pitchW, tn, a.outer);
    const unsigned fill = wave * 8 + lane / 8, chunk = (lane % 8) ^ (fill & 7);
    unsigned xo[XL];
#pragma unroll
    for (unsigned j = 0; j < XL; ++j) {
        const unsigned r = fill + j * Waves * 8;
        xo[j] = (byToken ? sourceOf(a, tm + r) : r) * pitch + chunk * 16;
    }
    const unsigned fillW = X8 ? wave * 16 + lane / 4 : fill;
    auto keyW = [](unsigned r) { return X8 ? (r >> 1 & 1) | (r >> 2 & 2) : (r & 3) | (r >> 1 & 4); };
    const unsigned chunkW = X8 ? (lane % 4) ^ keyW(fillW) : (lane % 8) ^ keyW(fillW);
    const unsigned wo = fillW * pitchW + chunkW * 16;
    // An odd number of steps of 128 ends in the middle of the last 256: the weight's second half is zeros there, and x's,
    // finite codes of the next row, count nothing.
    const unsigned woLast = a.count % Halves && chunkW >= 4 ? 0x7FFFFFFFu : wo;
    // Step k's bytes into stage s; past the last zeros, from beyond the buffer, so that every wave has the same number
    // of loads outstanding.
    auto load = [&](unsigned k, unsigned s) {
        std::uint8_t* to = lds + s * Stage + wave * 1024;
        const unsigned w = k + 1 == all ? woLast : wo, fromX = k < all ? k * 128 : 0x7FFFFFFFu;
        const unsigned fromW = k < all ? k * WRow : 0x7FFFFFFFu;
#pragma unroll
        for (unsigned j = 0; j < XL; ++j) loadToLds(xr, to + j * Waves * 1024, xo[j], fromX);
#pragma unroll
        for (unsigned j = 0; j < WL; ++j)
            loadToLds(wr, to + BM * 128 + j * Waves * 1024, w, fromW + j * Waves * (1024 / WRow) * pitchW);
    };
    const unsigned wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
    const unsigned l16 = lane % 16, g = lane / 16, wRow = l16 / 4 * 8 + l16 % 4;
    // Exponents of four MFMAs a dword: of this lane's row of each operand.
    const std::uint8_t *xe[MT], *we[NT];
    unsigned xs[MT], ws[NT], xsNext[MT], wsNext[NT];
#pragma unroll
    for (unsigned m = 0; m < MT; ++m) {
        const unsigned r = min(tm + wm + m * 16 + l16, a.rows - 1);
        xe[m] = a.xe + std::uint64_t(byToken ? sourceOf(a, r) : r) * xExpPitch<X8>(a) + (X8 ? 0 : 4 * g);
    }
#pragma unroll
    for (unsigned n = 0; n < NT; ++n)
        we[n] = a.we + std::uint64_t(min(tn + wn + n / 2 * 32 + n % 2 * 4 + wRow, a.outer - 1)) * wExpPitch(a) + 4 * g;
    const unsigned lastDword = (a.count - 1) / 4, mine = stepsOfLane(a, g);
    auto loadExponents = [&](unsigned dword) {
        dword = min(dword, lastDword);
#pragma unroll
        for (unsigned m = 0; m < MT; ++m) xsNext[m] = *reinterpret_cast<const unsigned*>(xe[m] + dword * (X8 ? 4 : 16));
#pragma unroll
        for (unsigned n = 0; n < NT; ++n) wsNext[n] = *reinterpret_cast<const unsigned*>(we[n] + dword * 16);
    };
    f32x4 acc[NT][MT] = {};
    loadExponents(first / Dword);
#pragma unroll
    for (unsigned s = 0; s + 1 < Stages; ++s) load(first + s, s);
    const unsigned xKey = l16 & 7, wKey = keyW(wRow);
    const std::uint8_t* xRead = lds + (wm + l16) * 128;
    const std::uint8_t* wRead = lds + BM * 128 + (wn + wRow) * WRow;
    auto step = [&](unsigned k, auto sel) {
        constexpr unsigned S = decltype(sel)::value;
        constexpr unsigned at = S % Stages * Stage;
        waitBarrier<(Stages - 2) * (XL + WL)>();
        load(k + Stages - 1, (S + Stages - 1) % Stages);
        u32x4 xf[MT][2];
#pragma unroll
        for (unsigned m = 0; m < MT; ++m)
#pragma unroll
            for (unsigned c = 0; c < 2; ++c)
                xf[m][c] = *reinterpret_cast<const u32x4*>(xRead + at + m * 16 * 128 +
                                                           (((Exact ? 2 * g + c : g + 4 * c) ^ xKey) * 16));
        if constexpr (Exact) {
            // The bf16 MFMA on the values: a lane has elements 32 g to 32 g + 31 of both rows, 8 a time.
            bf16x8 xv[MT][4];
#pragma unroll
            for (unsigned m = 0; m < MT; ++m)
#pragma unroll
                for (unsigned i = 0; i < 4; ++i)
                    xv[m][i] = values8(xf[m][i / 2][i % 2 * 2], xf[m][i / 2][i % 2 * 2 + 1], scaleOf(xs[m] >> 8 * S & 255));
#pragma unroll
            for (unsigned n = 0; n < NT; ++n) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(wRead + at + (n / 2 * 32 + n % 2 * 4) * WRow + ((g ^ wKey) * 16));
                const float scale = scaleOf(ws[n] >> 8 * S & 255);
#pragma unroll
                for (unsigned i = 0; i < 4; ++i) {
                    const bf16x8 wv = microValues8(w[i], scale);
#pragma unroll
                    for (unsigned m = 0; m < MT; ++m)
                        acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[m][i], acc[n][m], 0, 0, 0);
                }
            }
            return;
        }
#pragma unroll
        for (unsigned n = 0; n < NT; ++n) {
            const std::uint8_t* r = wRead + at + (n / 2 * 32 + n % 2 * 4) * WRow;
            const u32x4 w0 = *reinterpret_cast<const u32x4*>(r + ((g ^ wKey) * 16));
#pragma unroll
            for (unsigned m = 0; m < MT; ++m)
                acc[n][m] = multiply<X8, S * Halves % 4>(w0, xf[m][0], xf[m][1], acc[n][m], ws[n], xs[m]);
            if constexpr (!X8) {
                const u32x4 w1 = *reinterpret_cast<const u32x4*>(r + (((g + 4) ^ wKey) * 16));
#pragma unroll
                for (unsigned m = 0; m < MT; ++m)
                    acc[n][m] = multiply<X8, (S * Halves + 1) % 4>(w1, xf[m][1], xf[m][1], acc[n][m], ws[n], xs[m]);
            }
        }
    };
    auto nextExponents = [&](unsigned k) {
        // Past the last block codes are zeros, and so that the products are, the exponents finite.
        const unsigned keepW = finiteExponents(k * Halves, mine), keepX = X8 ? finiteExponents(k * Halves, a.count) : keepW;
#pragma unroll
        for (unsigned m = 0; m < MT; ++m) xs[m] = (xsNext[m] & keepX) | (0x7F7F7F7Fu & ~keepX);
#pragma unroll
        for (unsigned n = 0; n < NT; ++n) ws[n] = (wsNext[n] & keepW) | (0x7F7F7F7Fu & ~keepW);
        loadExponents(k / Dword + 1);
    };
    // Steps in runs of four, whose stages are constants, of one or two dwords of exponents.
    unsigned k = first;
    for (; k + 4 <= first + steps; k += 4) {
        nextExponents(k);
        step(k, std::integral_constant<unsigned, 0>{});
        step(k + 1, std::integral_constant<unsigned, 1>{});
        if constexpr (Dword == 2) nextExponents(k + 2);
        step(k + 2, std::integral_constant<unsigned, 2>{});
        step(k + 3, std::integral_constant<unsigned, 3>{});
    }
    // Of several groups each has whole dwords of steps.
    if ((Groups == 1 || Dword == 2) && k < first + steps) {
        nextExponents(k);
        step(k, std::integral_constant<unsigned, 0>{});
        if (k + 1 < first + steps) step(k + 1, std::integral_constant<unsigned, 1>{});
        if (Groups == 1 && k + 2 < first + steps) {
            if constexpr (Dword == 2) nextExponents(k + 2);
            step(k + 2, std::integral_constant<unsigned, 2>{});
        }
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
                if (Whole || row < end) put8<T, Whole>(y + row * a.yStride, column, a.outer, v, b);
            }
        }
    };
    if (tm + BM <= end && tn + BN <= a.outer)
        store(std::true_type{});
    else
        store(std::false_type{});
}

// acc += w x of one step, with the scales in byte S of ws and xs, in the accumulation registers: asm with one operand for
// both the sum and the result, since the compiler moves accumulators that fill the register file about. It does not
// know this instruction's latency: whoever reads acc has to let the last one finish.
template <bool X8, unsigned S>
__device__ __forceinline__ void multiplyInPlace(f32x4& acc, u32x4 w, u32x4 x0, u32x4 x1, unsigned ws, unsigned xs) {
    const i32x8 x = join(x0, x1);
    if constexpr (X8) {
        if constexpr (S == 0)
            asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4"
                : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
        else
            asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4"
                : "+a"(acc) : "v"(w), "v"(x), "v"(ws), "v"(xs));
    } else {
        if constexpr (S == 0)
            asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                : "+a"(acc) : "v"(w), "v"(x0), "v"(ws), "v"(xs));
        else if constexpr (S == 1)
            asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                : "+a"(acc) : "v"(w), "v"(x0), "v"(ws), "v"(xs));
        else if constexpr (S == 2)
            asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0] cbsz:4 blgp:4"
                : "+a"(acc) : "v"(w), "v"(x0), "v"(ws), "v"(xs));
        else
            asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0] cbsz:4 blgp:4"
                : "+a"(acc) : "v"(w), "v"(x0), "v"(ws), "v"(xs));
    }
}

// The same on tiles of 256 x 256, for products with enough of them: four waves, one a SIMD, of 128 x 128 each, whose
// accumulators fill the accumulation registers. LDS holds two stages. A step is multiplied in four quarters, a pair of
// the weight's operands with all of x's in each, first half by half where x is in 4 bits: in a quarter the next pair is read
// from LDS, and in the last one also, as each operand of x is used for the last time, its place is filled with the next
// step's. So no MFMA waits for LDS. The loads into LDS are spread over the quarters, each into a place that was read
// for the last time a quarter or more before, and each has at least a step's time to arrive:
//   quarter 0: pairs 2 and 3 of step k + 1;  1 and 2: x of step k + 2;  3: pairs 0 and 1 of step k + 2
// with a barrier before quarters 1 and 3.
// Measured: 4096 x 4096 x 8192 with 8-bit rows, bf16, 116 us, 2.4 PFLOP/s; 8192 x 4096 x 8192 in 4 bits 148, 3.7 PFLOP/s; 8192
// tokens to 4 of 32 experts, 2048 x 4096 in 4 bits, 271, 2.0. A step in 4 bits, 256 elements, is 1.8 us on all CUs at once, 4.7
// PFLOP/s, where this card's power lets registers alone multiply random codes at 5.8 (zeros 6.7); one in 8 bits, 128 elements,
// 1.5 us, 2.9 PFLOP/s of 4.1. What remains is a tile's beginning and end, 8 us: all CUs store at once (5 us at HBM's rate), and
// its first loads. MFMAs are busy 43% of all cycles, 58% with 8-bit rows, and no LDS access conflicts.
// The tiles that a workgroup goes through, one after the other, a grid apart: in the last pair of a tile's steps the loads are
// those of the next tile's first, so that it begins as the sums of this one are stored (8192 x 512 x 8192 52 us : 45, 8 even
// rounds of experts 238 : 232, nine uneven ones 297 : 271). For experts the tiles and the rows' sources are looked up in front
// of all, into LDS: looked up by every lane for itself in each tile they cost 3 us a tile.
constexpr unsigned kWideGroups = 256, kWideTiles = 16; // workgroups, one a CU; the most tiles of one, for experts

struct WideTile {
    unsigned expert, first, end, tn;
};

// `bytes` from p on.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bytesAt(const std::uint8_t* p, std::uint64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<std::uint8_t*>(p), 0,
                                             unsigned(min(bytes, std::uint64_t(0x7FFFFFFF))), 0x00020000);
}

// What the loads of a tile go by.
struct WideRows {
    __amdgpu_buffer_rsrc_t x, w, xe, we;
};

template <typename T, bool X8, bool Experts> __device__ __forceinline__ void wideTiles(const Product& a) {
    constexpr unsigned B = 256, Tiles = 8, Halves = X8 ? 1 : 2, WRow = Halves * 64, Stage = B * (128 + WRow);
    constexpr unsigned WL = B * WRow / 1024 / 4, WRows = 4096 / WRow; // a wave's loads of a step's weight; rows of all four's
    constexpr unsigned Exps = 2 * Tiles;                               // loads of exponents, for two steps
    extern __shared__ __align__(1024) std::uint8_t lds[]; // two stages: 256 rows of x, 256 of w; experts: tiles, sources
    const unsigned lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const unsigned all = (a.count + Halves - 1) / Halves, pairs = (all + 1) / 2 * 2;
    const unsigned pitch = xPitch<X8>(a), pitchW = wPitch(a), pitchXe = unsigned(a.xeRow), pitchWe = wExpPitch(a);
    const bool byToken = Experts && a.order;
    WideTile* const list = reinterpret_cast<WideTile*>(lds + 2 * Stage);
    unsigned* const sources = reinterpret_cast<unsigned*>(lds + 2 * Stage + kWideTiles * sizeof(WideTile));
    unsigned tiles = 0; // of this workgroup; rows of no expert are zeros at once and none of them
    if constexpr (Experts) {
        for (unsigned turn = 0; turn < kWideTiles; ++turn) {
            Span s;
            unsigned tn = 0;
            const bool some = spanOf(a, B, lane, [&](unsigned tilesM, unsigned none) {
                return expertTile<B>(a, blockIdx.x + turn * gridDim.x, tilesM, none, tn);
            }, s);
            if (!some) break;
            if (s.expert >= a.experts) {
                zeroTile<T>(a, s, B, tn, B);
                continue;
            }
            if (threadIdx.x == 0) list[tiles] = {s.expert, s.first, s.end, tn};
            sources[tiles * B + threadIdx.x] = byToken ? sourceOf(a, s.first + threadIdx.x) : threadIdx.x;
            ++tiles;
        }
        tiles = __builtin_amdgcn_readfirstlane(tiles);
        __syncthreads();
    } else {
        const unsigned total = a.tilesM * a.tilesN;
        tiles = blockIdx.x < total ? (total - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
    }
    // Tile i of this workgroup.
    auto tileAt = [&](unsigned i) {
        if constexpr (Experts) {
            const WideTile t = list[i];
            return WideTile{unsigned(__builtin_amdgcn_readfirstlane(t.expert)), unsigned(__builtin_amdgcn_readfirstlane(t.first)),
                            unsigned(__builtin_amdgcn_readfirstlane(t.end)), unsigned(__builtin_amdgcn_readfirstlane(t.tn))};
        } else {
            const unsigned tile = tileOf(blockIdx.x + i * gridDim.x, a.tilesM * a.tilesN, a.tilesM, a.tilesN);
            return WideTile{0, tile % a.tilesM * B, a.rows, tile / a.tilesM * B};
        }
    };
    // A tile's operands from its first rows on; by token all of x. `some` false: nothing, every load gives zeros.
    auto rowsOf = [&](const WideTile& t, bool some) {
        const std::uint64_t before = std::uint64_t(t.expert) * a.outer;
        const unsigned xFirst = byToken ? 0 : t.first, xRows = !some ? xFirst : byToken ? a.rows / a.each : a.rows;
        const unsigned wRows = some ? a.outer : t.tn;
        // Exponents behind the last row's may be any there are: no results of those rows are stored.
        const std::uint64_t xBytes = std::uint64_t(byToken ? a.rows / a.each : a.rows) * xExpPitch<X8>(a);
        return WideRows{rowsAt(a.x, pitch, xFirst, xRows), rowsAt(a.w + before * pitchW, pitchW, t.tn, wRows),
                        bytesAt(a.xe + xFirst * a.xeRow, xBytes - xFirst * a.xeRow),
                        rowsAt(a.we + before * pitchWe, pitchWe, t.tn, wRows)};
    };
    if (!tiles) return;
    // Chunks and rows are dealt as in microTiles.
    auto keyX = [](unsigned r) { return r & 7; };
    auto keyW = [](unsigned r) { return X8 ? (r >> 1 & 1) | (r >> 2 & 2) : (r & 3) | (r >> 1 & 4); };
    const unsigned fill = wave * 8 + lane / 8, fillW = X8 ? wave * 16 + lane / 4 : fill;
    const unsigned chunk = (lane % 8) ^ keyX(fill), chunkW = X8 ? (lane % 4) ^ keyW(fillW) : (lane % 8) ^ keyW(fillW);
    const unsigned wm = wave % 2 * 128, wn = wave / 2 * 128, l16 = lane % 16, g = lane / 16;
    const unsigned wRow = l16 / 4 * 8 + l16 % 4, mine = stepsOfLane(a, g);
    // A wave's loads are 32 rows of x apart, with the same keys; a token's rows may lie anywhere.
    unsigned xo[Experts ? 8 : 1], xeo[Experts ? Tiles : 1];
    auto place = [&](unsigned i) {
#pragma unroll
        for (unsigned j = 0; j < (Experts ? 8 : 1); ++j) {
            xo[j] = (Experts ? sources[i * B + fill + j * 32] : fill) * pitch + chunk * 16;
            xeo[j] = (Experts ? sources[i * B + wm + j * 16 + l16] : wm + l16) * pitchXe + (X8 ? 0 : 4 * g);
        }
    };
    const unsigned wo = fillW * pitchW + chunkW * 16, weo = (wn + wRow) * pitchWe + 4 * g;
    const unsigned woLast = a.count % Halves && chunkW >= 4 ? 0x7FFFFFFFu : wo; // the half of a step that is not there
    // Step k's rows of x or w into stage s; past the last zeros, from beyond the buffer.
    auto loadX = [&](const WideRows& r, unsigned k, unsigned s, unsigned part) {
        const unsigned from = k < all ? k * 128 : 0x7FFFFFFFu;
        std::uint8_t* to = lds + s * Stage + wave * 1024 + part * 4096;
        if constexpr (Experts)
            loadToLds(r.x, to, xo[part], from);
        else
            loadToLds(r.x, to, xo[0], from + part * 32 * pitch);
    };
    auto loadW = [&](const WideRows& r, unsigned k, unsigned s, unsigned part) {
        const unsigned from = k < all ? k * WRow : 0x7FFFFFFFu;
        loadToLds(r.w, lds + s * Stage + B * 128 + wave * 1024 + part * 4096, k + 1 == all ? woLast : wo,
                  from + part * WRows * pitchW);
    };
    // Load i of the first or the last two pairs of both halves of the waves.
    auto partW = [](unsigned last, unsigned i) { return X8 ? i * 2 + last : i / 2 + i % 2 * 4 + last * 2; };
    // A lane's chunks of its row in either stage: bytes of LDS, which the loads' offsets reach a stage of.
    unsigned xRead[2][2], wRead[2][Halves];
#pragma unroll
    for (unsigned s = 0; s < 2; ++s) {
#pragma unroll
        for (unsigned c = 0; c < 2; ++c) {
            xRead[s][c] = s * Stage + (wm + l16) * 128 + ((g + 4 * c) ^ keyX(l16)) * 16;
            asm("" : "+v"(xRead[s][c])); // kept, not computed again for every load
        }
#pragma unroll
        for (unsigned c = 0; c < Halves; ++c) {
            wRead[s][c] = s * Stage + B * 128 + (wn + wRow) * WRow + ((g + 4 * c) ^ keyW(wRow)) * 16;
            asm("" : "+v"(wRead[s][c]));
        }
    }
    u32x4 xf[Tiles][2], wf[2][2][Halves];
    auto readX = [&](unsigned s, unsigned m, unsigned c) {
        xf[m][c] = *reinterpret_cast<const u32x4*>(lds + m * 16 * 128 + xRead[s][c]);
    };
    auto readW = [&](unsigned s, unsigned n) {
#pragma unroll
        for (unsigned c = 0; c < Halves; ++c)
            wf[n / 2 % 2][n % 2][c] = *reinterpret_cast<const u32x4*>(lds + (n / 2 * 32 + n % 2 * 4) * WRow + wRead[s][c]);
    };
    // Two steps' exponents at a time, of this lane's row of each operand: a byte for each MFMA.
    unsigned xs[Tiles], ws[Tiles], xsNext[Tiles], wsNext[Tiles];
    auto loadExponents = [&](const WideRows& r, unsigned k) { // of steps k and k + 1, k even
        const unsigned dword = X8 ? k / 4 : k / 2, in = X8 ? k % 4 : 0;
        const unsigned fromX = dword * unsigned(a.xeNext) + in, fromW = dword * 16 + in;
#pragma unroll
        for (unsigned m = 0; m < Tiles; ++m) {
            const unsigned at = Experts ? xeo[m] : xeo[0], from = fromX + (Experts ? 0 : m * 16 * pitchXe);
            const unsigned fromN = fromW + (m / 2 * 32 + m % 2 * 4) * pitchWe;
            if constexpr (X8) {
                xsNext[m] = __builtin_amdgcn_raw_buffer_load_b16(r.xe, at, from, 0);
                wsNext[m] = __builtin_amdgcn_raw_buffer_load_b16(r.we, weo, fromN, 0);
            } else {
                xsNext[m] = __builtin_amdgcn_raw_buffer_load_b32(r.xe, at, from, 0);
                wsNext[m] = __builtin_amdgcn_raw_buffer_load_b32(r.we, weo, fromN, 0);
            }
        }
    };
    f32x4 acc[Tiles][Tiles];
    WideTile tile = tileAt(0);
    WideRows rows = rowsOf(tile, true), ahead = rows; // of this tile, and of the steps that are loaded now
    place(0);
    loadExponents(ahead, 0);
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) loadX(ahead, 0, 0, i);
#pragma unroll
    for (unsigned i = 0; i < WL; ++i) loadW(ahead, 0, 0, i);
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) loadX(ahead, 1, 1, i);
#pragma unroll
    for (unsigned i = 0; i < WL / 2; ++i) loadW(ahead, 1, 1, partW(0, i));
    waitBarrier<8 + WL / 2>();
#pragma unroll
    for (unsigned i = 0; i < 2; ++i) readW(0, i);
#pragma unroll
    for (unsigned i = 0; i < Tiles; ++i) readX(0, i, 0), readX(0, i, 1);
    // Step S of the pair that the exponents are for; the pair behind it begins at step f of `ahead`. The fences keep the
    // compiler from moving the reads and loads between the MFMAs down to where their results are needed, which is where
    // they would be waited for.
    auto blockStep = [&](unsigned k, unsigned f, auto block) {
        constexpr unsigned S = decltype(block)::value;
#pragma unroll
        for (unsigned q = 0; q < 4; ++q) {
            // Before quarter 1 pairs 2 and 3 of this step have to be there, before 3 x and pairs 0 and 1 of the next. What
            // was loaded since stays outstanding, and in a pair's first step the exponents.
            if (q == 1) waitBarrier<8 + WL + (S == 0 ? Exps : 0)>();
            if (q == 3) waitBarrier<8 + WL / 2 + (S == 0 ? Exps : 0)>();
#pragma unroll
            for (unsigned h = 0; h < Halves; ++h)
#pragma unroll
                for (unsigned m = 0; m < Tiles; ++m) {
                    const unsigned i = h * Tiles + m, turns = Halves * Tiles; // of a quarter
                    if (i % (turns / 2) == 0) {
                        if (q < 3)
                            readW(S, 2 * q + 2 + i / (turns / 2));
                        else
                            readW(1 - S, i / (turns / 2));
                    }
                    if (i % (turns / 4) == turns / 4 - 1) {
                        const unsigned j = i / (turns / 4);
                        if (q == 0 && j < WL / 2) S == 0 ? loadW(rows, k + 1, 1, partW(1, j)) : loadW(ahead, f, 0, partW(1, j));
                        if (q == 1) loadX(ahead, f + S, S, j);
                        if (q == 2) loadX(ahead, f + S, S, 4 + j);
                        if (q == 3 && j < WL / 2) loadW(ahead, f + S, S, partW(0, j));
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    auto multiply = [&](unsigned n, auto byte) {
                        multiplyInPlace<X8, decltype(byte)::value>(acc[n][m], wf[n / 2 % 2][n % 2][h], xf[m][h], xf[m][1],
                                                                   ws[n], xs[m]);
                    };
#pragma unroll
                    for (unsigned n = 2 * q; n < 2 * q + 2; ++n) {
                        if (h == 0)
                            multiply(n, std::integral_constant<unsigned, S * Halves>{});
                        else
                            multiply(n, std::integral_constant<unsigned, S * Halves + Halves - 1>{});
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if (q == 3) {
                        readX(1 - S, m, h);
                        if constexpr (X8) readX(1 - S, m, 1);
                    }
                }
        }
        // Where the loop ends the sums are read, by who does not know that they come from an MFMA: the last ones, of up to
        // 8 passes, have to be done by then.
        if (S == 1)
            asm volatile("s_nop 15\n\ts_nop 3" : "+a"(acc[6][6]), "+a"(acc[7][6]), "+a"(acc[6][7]), "+a"(acc[7][7]));
    };
    for (unsigned i = 0; i < tiles; ++i) {
#pragma unroll
        for (unsigned n = 0; n < Tiles; ++n)
#pragma unroll
            for (unsigned m = 0; m < Tiles; ++m) acc[n][m] = f32x4{};
        const bool more = i + 1 < tiles;
        const WideTile next = more ? tileAt(i + 1) : tile;
        for (unsigned k = 0; k < pairs; k += 2) {
            // Past the last block codes are zeros, and have to have finite exponents.
            const unsigned keepW = finiteExponents(k * Halves, mine), keepX = X8 ? finiteExponents(k, a.count) : keepW;
#pragma unroll
            for (unsigned m = 0; m < Tiles; ++m) {
                xs[m] = (xsNext[m] & keepX) | (0x7F7F7F7Fu & ~keepX);
                ws[m] = (wsNext[m] & keepW) | (0x7F7F7F7Fu & ~keepW);
            }
            const bool last = k + 2 >= pairs;
            const unsigned f = last ? 0 : k + 2;
            if (last) {
                ahead = rowsOf(next, more);
                if constexpr (Experts) place(i + more);
            }
            loadExponents(ahead, f);
            blockStep(k, f, std::integral_constant<unsigned, 0>{});
            blockStep(k, f, std::integral_constant<unsigned, 1>{});
        }
        typename T::Raw* y = static_cast<typename T::Raw*>(a.y);
        const float* bias = a.bias ? a.bias + std::uint64_t(tile.expert) * a.outer : nullptr;
        auto store = [&](auto whole) {
            constexpr bool Whole = decltype(whole)::value;
#pragma unroll
            for (unsigned n = 0; n < Tiles; n += 2) {
                const unsigned column = tile.tn + wn + n * 16 + g * 8;
                float b[8];
                bias8<Whole>(bias, column, a.outer, b);
#pragma unroll
                for (unsigned m = 0; m < Tiles; ++m) {
                    const unsigned row = tile.first + wm + m * 16 + l16;
                    float v[8];
#pragma unroll
                    for (unsigned j = 0; j < 8; ++j) // one by one: the compiler would move all sums at once, and spill
                        asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[j]) : "a"(acc[n + j / 4][m][j % 4]));
                    if (Whole || row < tile.end) put8<T, Whole>(y + row * a.yStride, column, a.outer, v, b);
                }
            }
        };
        if (tile.first + B <= tile.end && tile.tn + B <= a.outer)
            store(std::true_type{});
        else
            store(std::false_type{});
        tile = next, rows = ahead;
    }
    // Loads to LDS past the last step have to land before the workgroup gives its LDS back.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <typename T, bool Experts>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void microWide8(Product a) {
    wideTiles<T, true, Experts>(a);
}
template <typename T, bool Experts>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void microWide4(Product a) {
    wideTiles<T, false, Experts>(a);
}

// ------------------------------------------------------------------------------------------------
// Up to kFusedRows rows of dense x (single tokens), in one launch: a workgroup takes 16 columns of y; its eight waves share the
// inner axis, a run of steps each, and add their sums through LDS in the waves' order. The weight's codes go from memory to
// the MFMA's registers, each byte read once on the chip, four steps' loads at a time before the first is used; every
// workgroup codes x for itself into LDS while its first weights are on their way. Measured: 1 x 4096 x 4096 bf16 4.9 us, 1.8 TB/s
// of the weight, most of it the launch and two loads' ways, which the same layer in 8 bits takes 4.9 to 5.3 for as well: what 4
// bits save here is memory. A row more is 0.5 us, the coding in every workgroup.
constexpr unsigned kTokenWaves = 8, kFusedRows = 16; // the rows of an MFMA

template <typename T, bool X8> __global__ __launch_bounds__(kWave* kTokenWaves) void microTokens(Product a) {
    constexpr bool Exact = X8 && std::is_same<T, F32>::value;
    constexpr unsigned Ahead = 4; // steps of a wave loaded at a time
    __shared__ f32x4 sums[kTokenWaves][kWave];
    extern __shared__ __align__(16) std::uint8_t lds[]; // x's codes, then its exponents
    const unsigned t = threadIdx.x, lane = t % kWave, wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const unsigned l16 = lane % 16, g = lane / 16, n0 = blockIdx.x * 16;
    const unsigned pitch = xPitch<X8>(a), each = (a.count + kTokenWaves - 1) / kTokenWaves;
    const unsigned from = wave * each, to = min(from + each, a.count);
    const std::uint64_t wrow = min(n0 + l16, a.outer - 1);
    const std::uint8_t* wp = a.w + wrow * wPitch(a) + g * 16;
    const std::uint8_t* wep = a.we + wrow * wExpPitch(a) + g * 4;
    const unsigned mine = stepsOfLane(a, g);
    u32x4 w[Ahead];
    unsigned ws[Ahead];
    auto fetch = [&](unsigned k) {
#pragma unroll
        for (unsigned u = 0; u < Ahead; ++u) {
            const unsigned at = min(k + u, a.count - 1);
            w[u] = *reinterpret_cast<const u32x4*>(wp + std::uint64_t(at) * 64);
            ws[u] = at < mine ? wep[at / 4 * 16 + at % 4] : 127u;
        }
    };
    fetch(from);
    std::uint8_t* exponents = lds + a.rows * pitch; // a byte a block: [row][step] or [row][step][4]
    const unsigned sub = t % kBlockLanes;
    for (unsigned item = t / kBlockLanes; item < a.rows * a.count; item += kWave * kTokenWaves / kBlockLanes) {
        const unsigned row = item / a.count, step = item - row * a.count;
        float v[8];
        load8<T>(static_cast<const typename T::Raw*>(a.dense) + row * a.denseStride, step * kStep + sub * 8, a.inner, v);
        if constexpr (X8) {
            const unsigned e = exponentOf<BlockCodes::e4m3>(rowMax(peakBits(v)));
            const u32x2 q = encode8<BlockCodes::e4m3>(v, e);
            *reinterpret_cast<u32x2*>(lds + row * pitch + step * kStep + sub * 8) = q;
            if (sub == 0) exponents[item] = std::uint8_t(e);
            if (a.keep && blockIdx.x == 0) {
                *reinterpret_cast<u32x2*>(a.keep + row * std::uint64_t(pitch) + step * kStep + sub * 8) = q;
                if (step + sub < (step + 1 == a.count ? xExpPitch<true>(a) : step + 1))
                    a.keepExp[row * std::uint64_t(xExpPitch<true>(a)) + step + sub] = std::uint8_t(sub ? 127u : e);
            }
        } else {
            const unsigned e = microExponent(max4(peakBits(v)));
            *reinterpret_cast<unsigned*>(lds + row * pitch + step * (kStep / 2) + sub * 4) = microEncode<8>(v, e);
            if (sub % 4 == 0) exponents[item * 4 + sub / 4] = std::uint8_t(e);
        }
    }
    __syncthreads();
    const unsigned row = min(l16, a.rows - 1);
    const std::uint8_t* xp = lds + row * pitch + (Exact ? g * 32 : g * 16);
    const std::uint8_t* xep = exponents + row * a.count * (X8 ? 1 : 4) + (X8 ? 0 : g);
    f32x4 acc = {};
    for (unsigned k = from; k < to; k += Ahead) {
        u32x4 x[Ahead][2];
        unsigned xs[Ahead];
#pragma unroll
        for (unsigned u = 0; u < Ahead; ++u) {
            const unsigned at = min(k + u, a.count - 1);
            x[u][0] = x[u][1] = *reinterpret_cast<const u32x4*>(xp + at * (X8 ? kStep : kStep / 2));
            if constexpr (X8) x[u][1] = *reinterpret_cast<const u32x4*>(xp + at * kStep + (Exact ? 16 : 64));
            xs[u] = xep[at * (X8 ? 1 : 4)];
        }
        __builtin_amdgcn_sched_barrier(0); // the compiler would move the loads down to their use
#pragma unroll
        for (unsigned u = 0; u < Ahead; ++u) {
            if (k + u >= to) break;
            if constexpr (Exact) {
                // A lane has elements 32 g to 32 g + 31 of both rows.
                const float wScale = scaleOf(ws[u]), xScale = scaleOf(xs[u]);
#pragma unroll
                for (unsigned i = 0; i < 4; ++i)
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        microValues8(w[u][i], wScale), values8(x[u][i / 2][i % 2 * 2], x[u][i / 2][i % 2 * 2 + 1], xScale),
                        acc, 0, 0, 0);
            } else {
                acc = multiply<X8, 0>(w[u], x[u][0], x[u][1], acc, ws[u], xs[u]);
            }
        }
        if (k + Ahead < to) fetch(k + Ahead);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    // Output t: column fastest.
    const unsigned column = n0 + t % 16, r = t / 16;
    if (r >= a.rows || column >= a.outer) return;
    float s = 0.0f;
#pragma unroll
    for (unsigned v = 0; v < kTokenWaves; ++v) s += sums[v][r + t % 16 / 4 * 16][t % 4];
    if (a.bias) s += a.bias[column];
    static_cast<typename T::Raw*>(a.y)[r * a.yStride + column] = T::put(s);
}

// ------------------------------------------------------------------------------------------------
// Host side

enum class Form { wide, middle, small, half, few };
const char* formName(Form f) {
    switch (f) {
    case Form::wide: return "microWide";
    case Form::middle: return "microTiles128";
    case Form::small: return "microTiles64";
    case Form::half: return "microTiles64x32";
    default: return "microTiles32";
    }
}

// Rows and columns of a form's tile, and the threads that take one.
struct TileSize {
    unsigned up, across, threads;
};
constexpr TileSize tileSize(Form f) {
    switch (f) {
    case Form::wide: return {256, 256, 256};
    case Form::middle: return {128, 128, 512};
    case Form::small: return {64, 64, 256};
    case Form::half: return {64, 32, 256};
    default: return {32, 32, 256};
    }
}

std::uint64_t over(std::uint64_t n, std::uint64_t size) { return (n + size - 1) / size; }

// The most row tiles that `rows` sorted rows of `experts` experts and of none can make.
std::uint64_t mostTiles(std::uint64_t rows, std::uint64_t experts, unsigned tile) {
    return std::min(rows, rows / tile + experts + 1);
}

// The tile of a product: the least estimated time, in microseconds. A CU holds one workgroup of tiles of 256, two of 128, two or
// three of 64 and of those whose two groups of waves share the inner axis, 64 x 32 and 32; while tiles are at most one a CU, each
// step is quicker. tilesOf says how many row tiles of a size there are, launched how many workgroups a launch of it has. The
// constants fit these times (rows x inner x outer: 256, 128, 64, 64 x 32, 32; 8-bit rows in bf16, 4-bit rows, 8-bit rows in FP32):
//   17 x 4096 x 4096   - 24 9.8 7.7 6.6, - 23 7.8 6.4 5.6, - - 16 11 8.3     48 x 4096 x 8191  47 26 12 9.3 10, 29 24 9.5 7.7 9.1, - - 16 12 12
//   200 x 1024 x 1024  21 8.6 4.2 3.9 3.5, 18 9.1 4.4 3.9 3.4, - - 6.2 5.1 4.3   512 x 4096 x 1024 - 27 11 8.9 9.9, - 23 8.6 6.8 8.6, - - 16 11 12
//   777 x 1001 x 1437  23 10 7.0 8.7 8.7, 20 11 7.3 9.5 9.0, - 15 9.3 10 10   2048 x 512 x 2048 14 7.4 8.2 - -, 12 7.5 9.0 - -, - 13 12 - -
//   1024 x 8192 x 2048 108 58 35 - -, 63 49 28 - -, - 96 49 - -          4096 x 2048 x 4096 36 48 61 - -, 27 46 61 - -, - 105 92 - -
//   100000 x 256 x 256 25 21 26 - -, 26 29 41 - -, - 39 36 - -           3000 x 2000 x 3000 34 37 38 - -, 26 35 36 - -, - 77 53 - -
template <typename Tiles, typename Launched>
Form leastOf(std::uint32_t inner, std::uint32_t outer, DenseType type, RowFormat format, bool few, Tiles tilesOf, Launched launched) {
    const double k = double(over(inner, kStep));
    const bool x8 = format == RowFormat::e4m3, exact = x8 && type == DenseType::f32;
    const auto tiles = [&](unsigned up, unsigned across) { return tilesOf(up) * double(over(outer, across)); };
    const auto rounds = [](double n, unsigned slots) { return std::ceil(n / slots); };
    const auto takes = [&](Form f) {
        return launchTakes(launched(tileSize(f).up) * over(outer, tileSize(f).across), tileSize(f).threads);
    };
    const auto by = [&](double n, double one, double oneStep, double some, double slots, double step) {
        return n <= 256 ? one + oneStep * k : some + n / 512 * (slots + step * k);
    };
    constexpr double never = 1e300;
    const double half = tiles(128, 128);
    double wide = rounds(tiles(256, 256), 256) * (x8 ? 9.0 + 1.56 * k : 11.0 + 0.84 * k);
    double middle = half <= 256 ? (x8 ? 3.5 + 0.8 * k : 4.5 + 0.68 * k) : rounds(half, 512) * (x8 ? 2.7 + 1.32 * k : 5.2 + 1.1 * k);
    double small = exact ? by(tiles(64, 64), 2.6, 0.42, 2.2, 2.2, 0.66)
                   : x8  ? by(tiles(64, 64), 2.2, 0.26, 2.2, 1.1, 0.44)
                         : by(tiles(64, 64), 2.8, 0.18, 2.2, 2.2, 0.38);
    double narrow = exact ? by(tiles(64, 32), 2.9, 0.255, 2.0, 3.5, 0.55)
                    : x8  ? by(tiles(64, 32), 2.5, 0.195, 1.5, 3.0, 0.36)
                          : by(tiles(64, 32), 3.0, 0.13, 2.0, 4.0, 0.35);
    double fewest = exact ? by(tiles(32, 32), 2.8, 0.18, 1.5, 2.8, 0.25)
                    : x8  ? by(tiles(32, 32), 2.4, 0.14, 1.5, 2.0, 0.21)
                          : by(tiles(32, 32), 2.6, 0.1, 1.5, 2.6, 0.16);
    if (exact) wide = middle = never; // of no size the quickest: half the wave's conversions are of operands that others have too
    if (!takes(Form::middle)) middle = never;
    if (!takes(Form::small)) small = never;
    if (!few || !takes(Form::half)) narrow = never;
    if (!few || !takes(Form::few)) fewest = never;
    const double least = std::min({wide, middle, small, narrow, fewest});
    if (least == never) return Form::small; // more tiles than a launch takes, which checkTiles refuses
    return least == small    ? Form::small
           : least == narrow ? Form::half
           : least == fewest ? Form::few
           : least == middle ? Form::middle
                             : Form::wide;
}

Form formOf(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type, RowFormat format) {
    const auto up = [&](unsigned size) { return over(rows, size); };
    return leastOf(inner, outer, type, format, true, [&](unsigned size) { return double(up(size)); }, up);
}

// The same for experts, of whose rows only the mean is known: each of those that can have any makes whole tiles and, by the
// spread of their numbers, three quarters of one more. (24 tokens to 4 of 32, 2048 x 4096: 57, 39, 23 in tiles of 64; 1024 tokens
// 111, 91, 89; 8192 in 4 bits 297, 423, 571.) Tiles of 32 were the quickest for none.
Form expertFormOf(const ExpertPlan& plan, std::uint32_t inner, std::uint32_t outer, DenseType type, RowFormat format) {
    const double used = std::min(plan.choices, plan.experts);
    const auto tiles = [&](unsigned size) { return std::max(used, plan.choices / double(size) + 0.75 * used); };
    return leastOf(inner, outer, type, format, false, tiles,
                   [&](unsigned size) { return mostTiles(plan.choices, plan.experts, size); });
}

// A form's tiles, for calls to refuse before they launch anything, the coding of x among it.
void checkTiles(const char* where, Form form, std::uint64_t up, std::uint32_t outer) {
    checkGrid(where, up * over(outer, tileSize(form).across), tileSize(form).threads);
}
Form checkedForm(const char* where, std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type, RowFormat format) {
    const Form form = formOf(rows, inner, outer, type, format);
    checkTiles(where, form, over(rows, tileSize(form).up), outer);
    return form;
}
Form checkedForm(const char* where, const ExpertPlan& plan, std::uint32_t inner, std::uint32_t outer, DenseType type,
                 RowFormat format) {
    const Form form = expertFormOf(plan, inner, outer, type, format);
    checkTiles(where, form, mostTiles(plan.choices, plan.experts, tileSize(form).up), outer);
    return form;
}

template <typename T, bool X8, bool Experts, unsigned BM, unsigned BN, unsigned WM, unsigned WN, unsigned Stages, unsigned Groups>
void launchTiles(Product p, hipStream_t stream) {
    const std::uint64_t up = Experts ? mostTiles(p.rows, p.experts, BM) : over(p.rows, BM);
    p.tilesM = unsigned(up), p.tilesN = unsigned(over(p.outer, BN));
    const std::uint64_t tiles = up * p.tilesN;
    constexpr unsigned lds = Groups * Stages * (BM * 128 + BN * (X8 ? 64 : 128));
    hipLaunchKernelGGL((microTiles<T, X8, Experts, BM, BN, WM, WN, Stages, Groups>), dim3(unsigned(tiles)),
                       dim3(64 * WM * WN * Groups), lds, stream, p);
    checkHip(hipGetLastError());
}

template <typename T, bool X8, bool Experts> void launchWide(Product p, hipStream_t stream) {
    const std::uint64_t up = Experts ? mostTiles(p.rows, p.experts, 256) : over(p.rows, 256);
    p.tilesM = unsigned(up), p.tilesN = unsigned(over(p.outer, 256));
    const std::uint64_t tiles = up * p.tilesN, least = Experts ? over(tiles, 8 * kWideTiles) * 8 : 0;
    // A multiple of the XCDs, so that a workgroup's tiles stay with one.
    const dim3 grid(unsigned(std::min<std::uint64_t>(tiles, std::max<std::uint64_t>(kWideGroups, least)))), threads(256);
    constexpr unsigned lds = 2 * 256 * (X8 ? 192 : 256) + (Experts ? kWideTiles * (sizeof(WideTile) + 256 * 4) : 0);
    if constexpr (X8)
        hipLaunchKernelGGL((microWide8<T, Experts>), grid, threads, lds, stream, p);
    else
        hipLaunchKernelGGL((microWide4<T, Experts>), grid, threads, lds, stream, p);
    checkHip(hipGetLastError());
}

template <typename T, bool X8, bool Experts> void launchForm(Form form, Product p, hipStream_t stream) {
    constexpr bool exact = X8 && std::is_same<T, F32>::value;
    if (form == Form::small) return launchTiles<T, X8, Experts, 64, 64, 2, 2, 4, 1>(p, stream);
    if constexpr (!Experts)
        if (form == Form::few) return launchTiles<T, X8, false, 32, 32, 2, 1, 4, 2>(p, stream);
    if constexpr (!Experts)
        if (form == Form::half) return launchTiles<T, X8, false, 64, 32, 2, 1, 4, 2>(p, stream);
    if constexpr (!exact) {
        if (form == Form::middle) return launchTiles<T, X8, Experts, 128, 128, 4, 2, 2, 1>(p, stream);
        launchWide<T, X8, Experts>(p, stream);
    }
}

// Calls f with the element type's tag and whether rows are in 8 bits.
template <typename F> void withRows(DenseType type, RowFormat format, F f) {
    withType(type, [&](auto tag) {
        if (format == RowFormat::e4m3)
            f(tag, std::true_type{});
        else
            f(tag, std::false_type{});
    });
}

void checkRowCodes(const char* where, const CodedRows& x) {
    if (x.format == RowFormat::e4m3)
        checkCodes(where, x.codes, x.exponents);
    else
        checkMicro(where, {x.codes, x.exponents});
}

std::uint64_t codePitch(std::uint32_t inner, RowFormat f) {
    return f == RowFormat::e4m3 ? blockCodePitch(inner) : microCodePitch(inner);
}
std::uint64_t exponentPitch(std::uint32_t inner, RowFormat f) {
    return f == RowFormat::e4m3 ? blockExponentPitch(inner) : microExponentPitch(inner);
}
std::size_t rounded(std::uint64_t bytes) { return std::size_t((bytes + 255) / 256 * 256); }

// x's exponents by fours of steps, all rows' side by side, as microWide is quickest to read them: what it wants of a row at a
// time lies in a line of its own else. Rows in 4 bits are coded so, those in 8 bits have theirs copied into that order (of
// 4096 x 4096 4.8 us, of 6002 x 1000 2.3).
// For fewer than 2^31 bytes of them. (4096 x 4096 x 8192, 8-bit rows 136 us : 115, 4-bit 84 : 78; the weight's, 83.)
__global__ __launch_bounds__(256) void packExponents(const unsigned* __restrict__ from, unsigned* __restrict__ to, unsigned rows,
                                                     unsigned groups) {
    const unsigned row = blockIdx.x * 256 + threadIdx.x;
    if (row < rows) to[std::uint64_t(blockIdx.y) * rows + row] = from[std::uint64_t(row) * groups + blockIdx.y];
}

bool packs(Form form, std::uint64_t xRows, std::uint32_t inner, RowFormat format) {
    return form == Form::wide && xRows * exponentPitch(inner, format) < std::uint64_t(1) << 31;
}

// Where microWide finds x's exponents.
void setExponents(Product& p, RowFormat format, bool packed, std::uint64_t xRows) {
    const std::uint64_t part = format == RowFormat::e4m3 ? 4 : 16;
    p.xeRow = packed ? part : over(p.count, 4) * part, p.xeNext = packed ? xRows * part : part;
}

// Bytes of dense rows' codes and exponents, and of the packed copy of 8-bit ones'; `keep`: the first two are the caller's.
std::size_t codedBytes(std::uint64_t rows, std::uint32_t inner, RowFormat format, bool packed, bool keep) {
    const std::size_t exponents = rounded(rows * exponentPitch(inner, format));
    return (keep ? 0 : rounded(rows * codePitch(inner, format)) + exponents) +
           (packed && format == RowFormat::e4m3 ? exponents : 0);
}

// Codes dense rows into `space`, or what is kept of them, and lets p read them.
void encode(Product& p, DenseMatrix x, RowFormat format, BlockRows keep, bool packed, std::uint32_t rows, std::uint32_t inner,
            std::uint8_t* space, hipStream_t stream) {
    CodedRows out = {keep.codes, keep.exponents, format};
    if (!keep.codes) {
        out.codes = space, out.exponents = space + rounded(rows * codePitch(inner, format));
        space = out.exponents + rounded(rows * exponentPitch(inner, format));
    }
    p.x = out.codes, p.xe = out.exponents;
    setExponents(p, format, packed, rows);
    if (format == RowFormat::e2m1) return quantizeMicroRowsTo(x, {out.codes, out.exponents}, packed, rows, inner, stream);
    quantizeBlocks(x, {out.codes, out.exponents, BlockCodes::e4m3}, rows, inner, stream);
    if (!packed) return;
    const unsigned groups = unsigned(over(p.count, 4));
    hipLaunchKernelGGL(packExponents, dim3(unsigned(over(rows, 256)), groups), dim3(256), 0, stream,
                       reinterpret_cast<const unsigned*>(out.exponents), reinterpret_cast<unsigned*>(space), rows, groups);
    checkHip(hipGetLastError());
    p.xe = space;
}

// LDS of x's codes and exponents in a fused product of few rows.
std::size_t fusedLds(std::uint32_t rows, std::uint32_t inner, RowFormat f) {
    const std::size_t count = over(inner, kStep);
    return (rows * count * (f == RowFormat::e4m3 ? kStep + 1 : kStep / 2 + 4) + 15) / 16 * 16;
}
// Whether the layer takes microTokens: by its estimated time on the GPU against coding and product in launches of their own, of
// which one more costs the caller 4 us and the GPU one of them. The constants fit these (rows x inner x outer, bf16, 8-bit
// rows, this : two): 2 x 4096 x 4096 5.1 : 8.0, 8 x 4096 x 4096 8.1 : 8.1, 16 x 2048 x 4096 8.4 : 6.9, 16 x 512 x 4096 4.8 : 5.7,
// 6 x 2048 x 8192 8.3 : 7.0, 8 x 4096 x 8192 11.5 : 8.0; the call's time 8 x 4096 x 4096 7.9 : 12.0, 16 x 2048 x 4096 8.2 : 11.9.
// Beyond 4096 x 8192 neither side has been measured, and the estimates have no term for a weight that comes from HBM.
bool fusedTokens(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, RowFormat f) {
    const double count = double(over(inner, kStep)), more = double(over(outer, 4096)) - 1.0;
    const double fused = 4.0 + more + 0.0165 * rows * count * (1.0 + 0.5 * more), two = 5.3 + 0.085 * count;
    return rows <= kFusedRows && fusedLds(rows, inner, f) <= 48 * 1024 && fused <= two + 1.5;
}

Product productOf(MicroRows w, const float* bias, void* y, std::uint64_t stride, std::uint32_t rows, std::uint32_t inner,
                  std::uint32_t outer) {
    Product p = {};
    p.w = w.codes, p.we = w.exponents, p.bias = bias, p.y = y, p.yStride = stride;
    p.rows = rows, p.inner = inner, p.outer = outer, p.count = unsigned(over(inner, kStep));
    return p;
}

void checkWeight(const char* where, const MicroRows& w, const float* bias) {
    checkMicro(where, w);
    if (reinterpret_cast<std::uintptr_t>(bias) % 4) reject(where, "bias not float-aligned");
}

} // namespace

const char* matmulMicroForm(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type, RowFormat format) {
    const char* where = "matmul micro";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkType(where, type);
    checkFormat(where, format);
    return formName(formOf(rows, inner, outer, type, format));
}

const char* linearMicroForm(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type, RowFormat format) {
    const char* product = matmulMicroForm(rows, inner, outer, type, format);
    return fusedTokens(rows, inner, outer, format) ? "microTokens" : product;
}

void matmulMicro(CodedRows x, MicroRows w, const float* bias, void* y, DenseType type, std::uint64_t stride,
                 std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, hipStream_t stream) {
    const char* where = "matmul micro";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkRows(where, rows);
    checkType(where, type);
    checkFormat(where, x.format);
    if (!rows) return;
    checkRowCodes(where, x);
    checkWeight(where, w, bias);
    checkDense(where, y, stride, type, outer);
    Product p = productOf(w, bias, y, stride, rows, inner, outer);
    p.x = x.codes, p.xe = x.exponents;
    setExponents(p, x.format, false, rows);
    const Form form = checkedForm(where, rows, inner, outer, type, x.format);
    withRows(type, x.format, [&](auto tag, auto x8) {
        launchForm<decltype(tag), decltype(x8)::value, false>(form, p, stream);
    });
}

std::size_t linearMicroWorkspace(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type,
                                 RowFormat format, bool keep) {
    if (!rows || fusedTokens(rows, inner, outer, format)) return 0;
    return codedBytes(rows, inner, format, packs(formOf(rows, inner, outer, type, format), rows, inner, format), keep);
}

void linearMicro(DenseMatrix x, RowFormat format, MicroRows w, const float* bias, void* y, std::uint64_t yStride,
                 BlockRows keep, std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, void* workspace,
                 std::size_t workspaceBytes, hipStream_t stream) {
    const char* where = "linear micro";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkRows(where, rows);
    checkType(where, x.type);
    checkFormat(where, format);
    if (!keep.codes != !keep.exponents) reject(where, "kept codes and exponents come together");
    if (keep.codes && (format != RowFormat::e4m3 || keep.type != BlockCodes::e4m3))
        reject(where, "kept blocks must have E4M3 codes");
    if (!rows) return;
    checkDense(where, x.data, x.stride, x.type, inner);
    checkDense(where, y, yStride, x.type, outer);
    checkWeight(where, w, bias);
    if (keep.codes) checkCodes(where, keep.codes, keep.exponents);
    const std::size_t need = linearMicroWorkspace(rows, inner, outer, x.type, format, keep.codes);
    if (need > workspaceBytes || (need && !workspace)) reject(where, "workspace too small");
    if (reinterpret_cast<std::uintptr_t>(workspace) % 16) reject(where, "workspace must be 16-byte aligned");
    if (fusedTokens(rows, inner, outer, format)) {
        Product p = productOf(w, bias, y, yStride, rows, inner, outer);
        p.dense = x.data, p.denseStride = x.stride, p.keep = keep.codes, p.keepExp = keep.exponents;
        withRows(x.type, format, [&](auto tag, auto x8) {
            hipLaunchKernelGGL((microTokens<decltype(tag), decltype(x8)::value>), dim3(unsigned(over(outer, 16))),
                               dim3(kWave * kTokenWaves), fusedLds(rows, inner, format), stream, p);
        });
        return checkHip(hipGetLastError());
    }
    const Form form = checkedForm(where, rows, inner, outer, x.type, format);
    Product p = productOf(w, bias, y, yStride, rows, inner, outer);
    encode(p, x, format, keep, packs(form, rows, inner, format), rows, inner, static_cast<std::uint8_t*>(workspace), stream);
    withRows(x.type, format, [&](auto tag, auto x8) {
        launchForm<decltype(tag), decltype(x8)::value, false>(form, p, stream);
    });
}

namespace {
void checkExperts(const char* where, const ExpertPlan& plan) {
    if (!plan.experts || plan.experts > kMaxExperts) reject(where, "experts must be 1 to 1024");
    if (!plan.each || plan.each > kMaxEach) reject(where, "choices of a token must be 1 to 1024");
    if (plan.choices >> 31) reject(where, "2^31 choices or more");
    if (plan.choices % plan.each) reject(where, "choices are not whole tokens'");
    if (!plan.choices) return;
    if (!plan.offsets || !plan.order) reject(where, "null plan");
    if (reinterpret_cast<std::uintptr_t>(plan.offsets) % 4 || reinterpret_cast<std::uintptr_t>(plan.order) % 4)
        reject(where, "plan not aligned to its elements");
}
} // namespace

const char* matmulExpertsForm(ExpertPlan plan, std::uint32_t inner, std::uint32_t outer, DenseType type, RowFormat format) {
    const char* where = "matmul experts";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkType(where, type);
    checkFormat(where, format);
    if (!plan.experts || plan.experts > kMaxExperts) reject(where, "experts must be 1 to 1024");
    return formName(expertFormOf(plan, inner, outer, type, format));
}

namespace {
Product expertsProduct(bool byToken, MicroRows w, const float* bias, void* y, std::uint64_t stride, const ExpertPlan& plan,
                       std::uint32_t inner, std::uint32_t outer) {
    Product p = productOf(w, bias, y, stride, plan.choices, inner, outer);
    p.offsets = plan.offsets, p.order = byToken ? plan.order : nullptr;
    p.experts = plan.experts, p.each = plan.each;
    return p;
}

std::uint32_t rowsOf(const ExpertPlan& plan, bool byToken) {
    return byToken && plan.each ? plan.choices / plan.each : plan.choices;
}
bool packs(const ExpertPlan& plan, bool byToken, std::uint32_t inner, std::uint32_t outer, DenseType type, RowFormat format) {
    return packs(expertFormOf(plan, inner, outer, type, format), rowsOf(plan, byToken), inner, format);
}

// Codes of tokens are reached by 32 bits.
void checkTokens(const char* where, const ExpertPlan& plan, bool byToken, std::uint32_t inner, RowFormat format) {
    if (byToken && rowsOf(plan, true) * codePitch(inner, format) >> 31)
        reject(where, "codes of tokens of 2^31 bytes or more: gather them");
}
} // namespace

void matmulExperts(CodedRows x, bool byToken, MicroRows w, const float* bias, void* y, DenseType type, std::uint64_t stride,
                   ExpertPlan plan, std::uint32_t inner, std::uint32_t outer, hipStream_t stream) {
    const char* where = "matmul experts";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkType(where, type);
    checkFormat(where, x.format);
    checkExperts(where, plan);
    if (!plan.choices) return;
    checkRowCodes(where, x);
    checkWeight(where, w, bias);
    checkDense(where, y, stride, type, outer);
    checkTokens(where, plan, byToken, inner, x.format);
    Product p = expertsProduct(byToken, w, bias, y, stride, plan, inner, outer);
    p.x = x.codes, p.xe = x.exponents;
    setExponents(p, x.format, false, plan.choices);
    const Form form = checkedForm(where, plan, inner, outer, type, x.format);
    withRows(type, x.format, [&](auto tag, auto x8) {
        launchForm<decltype(tag), decltype(x8)::value, true>(form, p, stream);
    });
}

std::size_t linearExpertsWorkspace(ExpertPlan plan, bool byToken, std::uint32_t inner, std::uint32_t outer, DenseType type,
                                   RowFormat format) {
    const std::uint64_t rows = rowsOf(plan, byToken);
    if (!rows || !plan.experts) return 0;
    return codedBytes(rows, inner, format, packs(plan, byToken, inner, outer, type, format), false);
}

void linearExperts(DenseMatrix x, RowFormat format, bool byToken, MicroRows w, const float* bias, void* y,
                   std::uint64_t yStride, ExpertPlan plan, std::uint32_t inner, std::uint32_t outer, void* workspace,
                   std::size_t workspaceBytes, hipStream_t stream) {
    const char* where = "linear experts";
    checkColumns(where, inner);
    checkColumns(where, outer);
    checkType(where, x.type);
    checkFormat(where, format);
    checkExperts(where, plan);
    if (!plan.choices) return;
    const std::uint32_t rows = rowsOf(plan, byToken);
    checkDense(where, x.data, x.stride, x.type, inner);
    checkDense(where, y, yStride, x.type, outer);
    checkWeight(where, w, bias);
    const std::size_t need = linearExpertsWorkspace(plan, byToken, inner, outer, x.type, format);
    if (need > workspaceBytes || !workspace) reject(where, "workspace too small");
    if (reinterpret_cast<std::uintptr_t>(workspace) % 16) reject(where, "workspace must be 16-byte aligned");
    checkTokens(where, plan, byToken, inner, format);
    const Form form = checkedForm(where, plan, inner, outer, x.type, format);
    Product p = expertsProduct(byToken, w, bias, y, yStride, plan, inner, outer);
    encode(p, x, format, {}, packs(plan, byToken, inner, outer, x.type, format), rows, inner,
           static_cast<std::uint8_t*>(workspace), stream);
    withRows(x.type, format, [&](auto tag, auto x8) {
        launchForm<decltype(tag), decltype(x8)::value, true>(form, p, stream);
    });
}

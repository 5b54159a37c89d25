// Device helpers of the 8-bit block format (include/blocks.h) and of dense matrices of three types.
#pragma once

#include "blocks.h"

#include <hip/hip_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>

namespace blocks {

constexpr unsigned kWave = 64;
// A block of 128 elements is held by 16 lanes, 8 consecutive elements each: one DPP row, so that the
// block's maximum is four DPP steps, and 16 bytes a lane of a 16-bit type.
constexpr unsigned kBlockLanes = 16; // of eight elements each

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Element types as the kernels see them.
struct F32 {
    typedef float Raw;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
struct BF16 {
    typedef __bf16 Raw;
    static __device__ __forceinline__ float get(__bf16 v) { return float(v); }
    static __device__ __forceinline__ __bf16 put(float v) { return __bf16(v); }
};
struct F16 {
    typedef _Float16 Raw;
    static __device__ __forceinline__ float get(_Float16 v) { return float(v); }
    static __device__ __forceinline__ _Float16 put(float v) { return _Float16(v); }
};

// Dense rows start at any element (odd widths, slices), so vectors of elements are moved with their
// element's alignment; the hardware takes unaligned 16-byte accesses.
template <typename T> struct Group {
    typedef typename T::Raw Raw;
    typedef Raw Vec __attribute__((ext_vector_type(8)));
    typedef Vec Loose __attribute__((aligned(alignof(Raw))));
};

// Elements [at, at + 8) of a row of n, zero past its end.
template <typename T>
__device__ __forceinline__ void load8(const typename T::Raw* row, unsigned at, unsigned n, float (&v)[8]) {
    if (at + 8 <= n) {
        const typename Group<T>::Vec g =
            __builtin_nontemporal_load(reinterpret_cast<const typename Group<T>::Loose*>(row + at));
#pragma unroll
        for (unsigned i = 0; i < 8; ++i) v[i] = T::get(g[i]);
    } else {
#pragma unroll
        for (unsigned i = 0; i < 8; ++i) v[i] = at + i < n ? T::get(row[at + i]) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(typename T::Raw* row, unsigned at, unsigned n, const float (&v)[8]) {
    if (at + 8 <= n) {
        typename Group<T>::Vec g;
#pragma unroll
        for (unsigned i = 0; i < 8; ++i) g[i] = T::put(v[i]);
        __builtin_nontemporal_store(g, reinterpret_cast<typename Group<T>::Loose*>(row + at));
    } else {
#pragma unroll
        for (unsigned i = 0; i < 8; ++i)
            if (at + i < n) row[at + i] = T::put(v[i]);
    }
}

// A lane's eight elements of the block that starts at column `at` of a row of n, with the codes of the same
// elements. Of FP32 they are four of each half, so that every access of a block's lanes is 256 bytes side by side:
// with eight in a row, 16 bytes of each 32, a nontemporal store wrote at half the rate (dequantizing 1,000,000 x 256,
// 407 us to 204).
template <typename T>
__device__ __forceinline__ void loadBlock(const typename T::Raw* row, unsigned at, unsigned lane, unsigned n, float (&v)[8]) {
    if constexpr (!std::is_same<T, F32>::value) {
        load8<T>(row, at + lane * 8, n, v);
    } else {
        typedef f32x4 Loose __attribute__((aligned(4)));
#pragma unroll
        for (unsigned h = 0; h < 8; h += 4) {
            const unsigned c = at + h * (kBlock / 8) + lane * 4;
            if (c + 4 <= n) {
                const f32x4 g = __builtin_nontemporal_load(reinterpret_cast<const Loose*>(row + c));
#pragma unroll
                for (unsigned i = 0; i < 4; ++i) v[h + i] = g[i];
            } else {
#pragma unroll
                for (unsigned i = 0; i < 4; ++i) v[h + i] = c + i < n ? row[c + i] : 0.0f;
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ void storeBlock(typename T::Raw* row, unsigned at, unsigned lane, unsigned n, const float (&v)[8]) {
    if constexpr (!std::is_same<T, F32>::value) {
        store8<T>(row, at + lane * 8, n, v);
    } else {
        typedef f32x4 Loose __attribute__((aligned(4)));
#pragma unroll
        for (unsigned h = 0; h < 8; h += 4) {
            const unsigned c = at + h * (kBlock / 8) + lane * 4;
            if (c + 4 <= n) {
                __builtin_nontemporal_store(f32x4{v[h], v[h + 1], v[h + 2], v[h + 3]}, reinterpret_cast<Loose*>(row + c));
            } else {
#pragma unroll
                for (unsigned i = 0; i < 4; ++i)
                    if (c + i < n) row[c + i] = v[h + i];
            }
        }
    }
}

template <typename T> __device__ __forceinline__ u32x2 loadCodes(const std::uint8_t* block, unsigned lane) {
    if constexpr (!std::is_same<T, F32>::value)
        return *reinterpret_cast<const u32x2*>(block + lane * 8);
    else
        return u32x2{*reinterpret_cast<const unsigned*>(block + lane * 4),
                     *reinterpret_cast<const unsigned*>(block + kBlock / 2 + lane * 4)};
}

template <typename T> __device__ __forceinline__ void storeCodes(std::uint8_t* block, unsigned lane, u32x2 q) {
    if constexpr (!std::is_same<T, F32>::value) {
        *reinterpret_cast<u32x2*>(block + lane * 8) = q;
    } else {
        *reinterpret_cast<unsigned*>(block + lane * 4) = q.x;
        *reinterpret_cast<unsigned*>(block + kBlock / 2 + lane * 4) = q.y;
    }
}

// Bits of the largest magnitude of v; an infinity or a NaN gives at least 0x7F800000.
__device__ __forceinline__ unsigned peakBits(const float (&v)[8]) {
    unsigned m = 0;
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

// Maximum over the 16 lanes of a DPP row, in all of them: rotations by 8, 4, 2 and 1.
__device__ __forceinline__ unsigned rowMax(unsigned m) {
    m = max(m, unsigned(__builtin_amdgcn_mov_dpp(int(m), 0x128, 0xF, 0xF, false)));
    m = max(m, unsigned(__builtin_amdgcn_mov_dpp(int(m), 0x124, 0xF, 0xF, false)));
    m = max(m, unsigned(__builtin_amdgcn_mov_dpp(int(m), 0x122, 0xF, 0xF, false)));
    return max(m, unsigned(__builtin_amdgcn_mov_dpp(int(m), 0x121, 0xF, 0xF, false)));
}

// The exponent byte of a block from its peak's bits. 448 = 1.75 * 2^8 and 127 = 1.984375 * 2^6: the
// power is the peak's own less 8 or 6, one more where the peak's mantissa is above the limit's.
template <BlockCodes C> __device__ __forceinline__ unsigned exponentOf(unsigned peak) {
    constexpr int lead = C == BlockCodes::e4m3 ? 8 : 6;
    constexpr unsigned past = C == BlockCodes::e4m3 ? 0x600000u : 0x7E0000u;
    if (peak >= 0x7F800000u) return 255;
    const int e = int(peak >> 23) - lead + ((peak & 0x7FFFFFu) > past ? 1 : 0);
    return peak == 0 ? 127u : unsigned(e < 1 ? 1 : e);
}

// 2^(127 - e) for 1 <= e <= 253, which covers every finite block; a NaN block's codes are made of zeros.
__device__ __forceinline__ float inverseScale(unsigned e) { return __uint_as_float((254u - e) << 23); }

// 2^(e - 127); NaN for 255, the subnormal 2^-127 for 0.
__device__ __forceinline__ float scaleOf(unsigned e) {
    return __uint_as_float(e == 255 ? 0x7FC00000u : e == 0 ? 0x00400000u : e << 23);
}

// Codes of v * s, rounded half to even.
template <BlockCodes C> __device__ __forceinline__ u32x2 packCodes(const float (&v)[8], float s) {
    u32x2 q;
#pragma unroll
    for (unsigned h = 0; h < 2; ++h) {
        if constexpr (C == BlockCodes::e4m3) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * s, v[4 * h + 1] * s, 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * s, v[4 * h + 3] * s, w, true);
            q[h] = unsigned(w);
        } else {
            // Adding 1.5 * 2^23 leaves the rounded integer in the low bits of the sum.
            unsigned b[4];
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) b[i] = __float_as_uint(fmaf(v[4 * h + i], s, 12582912.0f));
            const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u);
            const unsigned hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000C0Cu);
            q[h] = lo | hi;
        }
    }
    return q;
}

// Codes of 8 elements. `e` is the block's exponent.
template <BlockCodes C> __device__ __forceinline__ u32x2 encode8(const float (&v)[8], unsigned e) {
    if (e == 255) return u32x2{0u, 0u};
    const float s = inverseScale(e);
    // At this exponent the largest elements would round to 2^128, which FP32 reads as an infinity.
    if (e == (C == BlockCodes::e4m3 ? 247u : 249u)) {
        constexpr float most = C == BlockCodes::e4m3 ? 240.0f : 63.0f;
        float c[8];
#pragma unroll
        for (unsigned i = 0; i < 8; ++i) c[i] = fminf(fmaxf(v[i] * s, -most), most);
        return packCodes<C>(c, 1.0f);
    }
    return packCodes<C>(v, s);
}

// The values of 8 codes.
template <BlockCodes C> __device__ __forceinline__ void decode8(u32x2 q, float scale, float (&v)[8]) {
#pragma unroll
    for (unsigned h = 0; h < 2; ++h) {
        if constexpr (C == BlockCodes::e4m3) {
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(int(q[h]), false);
            const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(int(q[h]), true);
            v[4 * h] = a.x * scale, v[4 * h + 1] = a.y * scale;
            v[4 * h + 2] = b.x * scale, v[4 * h + 3] = b.y * scale;
        } else {
#pragma unroll
            for (unsigned i = 0; i < 4; ++i)
                v[4 * h + i] = float(int(q[h] << (24 - 8 * i)) >> 24) * scale;
        }
    }
}

// Workgroups of a walk over the blocks of all rows, 256 threads each: a launch takes fewer than 2^32 threads a
// dimension, so from kGridRow on they are dealt to rows of a second one.
constexpr unsigned kGridRow = 1u << 23;
__device__ __forceinline__ unsigned flatGroup() { return blockIdx.y * kGridRow + blockIdx.x; }

// item / count for a flat index over rows of `count` blocks: magic = ceil(2^32 / count) makes the high
// word at most one too large.
__device__ __forceinline__ unsigned rowOf(unsigned item, unsigned count, unsigned magic) {
    if (count == 1) return item;
    const unsigned r = __umulhi(item, magic);
    return r - (r * count > item ? 1u : 0u);
}

} // namespace blocks

// Host side: checks shared by the entry points.
namespace blocks {

inline unsigned rowMagic(unsigned count) {
    return unsigned(((std::uint64_t(1) << 32) + count - 1) / count);
}

inline dim3 flatGrid(unsigned groups) {
    return groups <= kGridRow ? dim3(groups) : dim3(kGridRow, (groups + kGridRow - 1) / kGridRow);
}

inline void reject(const char* where, const char* what) {
    throw std::invalid_argument(std::string(where) + ": " + what);
}

// Whether a launch takes that many workgroups: it has fewer than 2^32 threads.
constexpr bool launchTakes(std::uint64_t groups, unsigned threads) {
    return groups < (std::uint64_t(1) << 32) / threads;
}
inline void checkGrid(const char* where, std::uint64_t groups, unsigned threads) {
    if (!launchTakes(groups, threads)) reject(where, "more tiles than a launch takes");
}

inline std::size_t elementBytes(DenseType t) { return t == DenseType::f32 ? 4 : 2; }

inline void checkType(const char* where, DenseType t) {
    if (unsigned(t) > 2) reject(where, "unknown element type");
}

inline void checkDense(const char* where, const void* data, std::uint64_t stride, DenseType type,
                       std::uint64_t columns) {
    checkType(where, type);
    if (!data) reject(where, "null dense matrix");
    if (stride < columns) reject(where, "row stride shorter than a row");
    if (reinterpret_cast<std::uintptr_t>(data) % elementBytes(type)) reject(where, "dense matrix not aligned to its elements");
}

inline void checkCodes(const char* where, const std::uint8_t* codes, const std::uint8_t* exponents) {
    if (!codes || !exponents) reject(where, "null codes or exponents");
    if (reinterpret_cast<std::uintptr_t>(codes) % 16) reject(where, "codes must be 16-byte aligned");
    if (reinterpret_cast<std::uintptr_t>(exponents) % 4) reject(where, "exponents must be 4-byte aligned");
}

// Widths up to 2^22 keep every offset inside a tile of rows below 2^31.
constexpr std::uint32_t kMaxColumns = 1u << 22;
inline void checkColumns(const char* where, std::uint32_t columns) {
    if (!columns) reject(where, "rows of zero elements");
    if (columns > kMaxColumns) reject(where, "rows of more than 4,194,304 elements");
}

inline void checkRows(const char* where, std::uint32_t rows) {
    if (rows >> 31) reject(where, "2^31 rows or more");
}

// Calls f with the type's tag.
template <typename F> void withType(DenseType t, F f) {
    switch (t) {
    case DenseType::f32: f(F32{}); break;
    case DenseType::bf16: f(BF16{}); break;
    case DenseType::f16: f(F16{}); break;
    }
}

// Calls f with the code type as a constant.
template <typename F> void withCodes(BlockCodes c, F f) {
    if (c == BlockCodes::e4m3)
        f(std::integral_constant<BlockCodes, BlockCodes::e4m3>{});
    else
        f(std::integral_constant<BlockCodes, BlockCodes::int8>{});
}

} // namespace blocks

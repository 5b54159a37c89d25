// Device helpers of the microscaled 4-bit format (include/micro.h).
#pragma once

#include "blocks/device_blocks.h"
#include "micro.h"

namespace micro {

using namespace blocks;

constexpr unsigned kStep = 128; // elements of a scaled MFMA along the inner axis: four blocks

// The exponent byte of a block from its peak's bits. 6 = 1.5 * 2^2: the power is the peak's own less 2, one more where
// the peak's mantissa is above a half.
__device__ __forceinline__ unsigned microExponent(unsigned peak) {
    if (peak >= 0x7F800000u) return 255;
    const int e = int(peak >> 23) - 2 + ((peak & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    return peak == 0 ? 127u : unsigned(e < 1 ? 1 : e);
}

// E2M1 codes of N elements (a multiple of 2, at most 8), the first in the lowest half byte.
template <unsigned N> __device__ __forceinline__ unsigned microEncode(const float* v, unsigned e) {
    if (e == 255) return 0;
    const float s = inverseScale(e);
    float c[N];
#pragma unroll
    for (unsigned i = 0; i < N; ++i) c[i] = v[i] * s;
    // At this exponent the largest elements would round to 2^128, which FP32 reads as an infinity.
    if (e == 253) {
#pragma unroll
        for (unsigned i = 0; i < N; ++i) c[i] = fminf(fmaxf(c[i], -3.0f), 3.0f);
    }
    unsigned q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, c[0], c[1], 1.0f, 0);
    if constexpr (N > 2) q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, c[2], c[3], 1.0f, 1);
    if constexpr (N > 4) q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, c[4], c[5], 1.0f, 2);
    if constexpr (N > 6) q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, c[6], c[7], 1.0f, 3);
    return q;
}

// The values of four codes in the low half of q.
__device__ __forceinline__ void microDecode4(unsigned q, float scale, float* v) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
    v[0] = a.x * scale, v[1] = a.y * scale, v[2] = b.x * scale, v[3] = b.y * scale;
}

// The largest over the 4 or 8 lanes that hold a block, in all of them.
__device__ __forceinline__ unsigned max4(unsigned m) {
    m = max(m, unsigned(__builtin_amdgcn_mov_dpp(int(m), 0xB1, 0xF, 0xF, false))); // quad_perm 1 0 3 2
    return max(m, unsigned(__builtin_amdgcn_mov_dpp(int(m), 0x4E, 0xF, 0xF, false))); // quad_perm 2 3 0 1
}
__device__ __forceinline__ unsigned max8(unsigned m) {
    m = max4(m);
    return max(m, unsigned(__builtin_amdgcn_mov_dpp(int(m), 0x141, 0xF, 0xF, false))); // the other way round in 8 lanes
}

// Where block 4 * step + i of a row lies in its exponents.
__device__ __forceinline__ unsigned exponentAt(unsigned step, unsigned i) { return step / 4 * 16 + i * 4 + step % 4; }

} // namespace micro

// quantizeMicro, or with the exponents in the products' own order: 16 bytes of each row side by side, [fours of steps][rows].
void quantizeMicroRowsTo(DenseMatrix x, MicroRows out, bool packed, std::uint32_t rows, std::uint32_t columns,
                         hipStream_t stream);

namespace micro {
inline void checkMicro(const char* where, const MicroRows& r) {
    if (!r.codes || !r.exponents) reject(where, "null codes or exponents");
    if (reinterpret_cast<std::uintptr_t>(r.codes) % 16) reject(where, "codes must be 16-byte aligned");
    if (reinterpret_cast<std::uintptr_t>(r.exponents) % 16) reject(where, "exponents must be 16-byte aligned");
}
inline void checkFormat(const char* where, RowFormat f) {
    if (unsigned(f) > 1) reject(where, "unknown row format");
}
} // namespace micro

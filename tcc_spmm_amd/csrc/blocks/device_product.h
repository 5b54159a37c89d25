// Device helpers of the products of coded rows: loads into LDS, waits, the order of tiles, and the outputs.
#pragma once

#include "blocks/device_blocks.h"

namespace blocks {

typedef __attribute__((address_space(3))) void* LdsPtr;

__device__ __forceinline__ i32x8 join(u32x4 p, u32x4 q) {
    return i32x8{int(p.x), int(p.y), int(p.z), int(p.w), int(q.x), int(q.y), int(q.z), int(q.w)};
}

// The values of 8 E4M3 codes as bf16: the conversion multiplies by the scale's power of two. Exact but for the ends of
// the range: multiples of 2^-134 and less (exponents below 3) are rounded, values of 2^128 and more infinite.
__device__ __forceinline__ bf16x8 values8(unsigned lo, unsigned hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// 16 bytes a lane from `rsrc`, at `lane + uniform`, to LDS at `to` + 16 * lane, past the registers.
__device__ __forceinline__ void loadToLds(__amdgpu_buffer_rsrc_t rsrc, std::uint8_t* to, unsigned lane, unsigned uniform) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LdsPtr)to, 16, lane, uniform, 0, 0);
}

// Eight consecutive outputs, columns [at, at + 8) of a row of n, with the bias added. Plain stores: the
// L2 puts the lines together that several stores of a wave fill.
template <typename T, bool Whole>
__device__ __forceinline__ void put8(typename T::Raw* row, unsigned at, unsigned n, const float (&v)[8], const float (&b)[8]) {
    typename Group<T>::Vec g;
#pragma unroll
    for (unsigned i = 0; i < 8; ++i) g[i] = T::put(v[i] + b[i]);
    if (Whole || at + 8 <= n) {
        *reinterpret_cast<typename Group<T>::Loose*>(row + at) = g;
    } else {
#pragma unroll
        for (unsigned i = 0; i < 8; ++i)
            if (at + i < n) row[at + i] = g[i];
    }
}

// bias[at .. at + 8), or zeros without one or past its end.
template <bool Whole> __device__ __forceinline__ void bias8(const float* bias, unsigned at, unsigned n, float (&b)[8]) {
    typedef f32x4 Loose4 __attribute__((aligned(4)));
    if (!bias) {
#pragma unroll
        for (unsigned i = 0; i < 8; ++i) b[i] = 0.0f;
    } else if (Whole || at + 8 <= n) {
        const f32x4 lo = *reinterpret_cast<const Loose4*>(bias + at), hi = *reinterpret_cast<const Loose4*>(bias + at + 4);
#pragma unroll
        for (unsigned i = 0; i < 4; ++i) b[i] = lo[i], b[4 + i] = hi[i];
    } else {
#pragma unroll
        for (unsigned i = 0; i < 8; ++i) b[i] = at + i < n ? bias[at + i] : 0.0f;
    }
}

// The same for four FP32 outputs.
typedef f32x4 LooseF32x4 __attribute__((aligned(4)));
__device__ __forceinline__ f32x4 bias4(const float* bias, unsigned at, unsigned n) {
    f32x4 b = {};
    if (!bias) return b;
    if (at + 4 <= n) return *reinterpret_cast<const LooseF32x4*>(bias + at);
#pragma unroll
    for (unsigned i = 0; i < 4; ++i)
        if (at + i < n) b[i] = bias[at + i];
    return b;
}
__device__ __forceinline__ void put4(float* row, unsigned at, unsigned n, f32x4 v) {
    if (at + 4 <= n) {
        *reinterpret_cast<LooseF32x4*>(row + at) = v;
    } else {
#pragma unroll
        for (unsigned i = 0; i < 4; ++i)
            if (at + i < n) row[at + i] = v[i];
    }
}

// Waits until at most N of this wave's memory loads are outstanding and its LDS reads are done, then
// for the workgroup. One asm block with a memory clobber, so that no access moves across it.
template <unsigned N> __device__ __forceinline__ void waitBarrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The bytes of a dword of exponents, of blocks k to k + 3, that belong to blocks before `count`.
__device__ __forceinline__ unsigned finiteExponents(unsigned k, unsigned count) {
    return k + 4 <= count ? ~0u : k >= count ? 0u : (1u << 8 * (count - k)) - 1;
}

// Rows from `first` on of a matrix of `rows` rows of `pitch` bytes.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rowsAt(const std::uint8_t* p, unsigned pitch, unsigned first, unsigned rows) {
    const std::uint64_t bytes = std::uint64_t(rows - first) * pitch;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<std::uint8_t*>(p) + std::uint64_t(first) * pitch, 0,
                                             unsigned(min(bytes, std::uint64_t(0x7FFFFFFF))), 0x00020000);
}

// The tile of a workgroup, as (row tile) + tilesM * (column tile). Workgroups go round the eight XCDs, each
// with an L2 of its own: an XCD gets a run of tiles that walks bands of eight row tiles, so that the tiles
// it works on at once share rows of both operands.
__device__ __forceinline__ unsigned tileOf(unsigned id, unsigned total, unsigned tilesM, unsigned tilesN) {
    const unsigned xcd = id % 8, each = total / 8, more = total % 8;
    const unsigned i = xcd * each + min(xcd, more) + id / 8;
    const unsigned band = i / (8 * tilesN), in = i - band * 8 * tilesN;
    const unsigned high = min(8u, tilesM - 8 * band);
    return 8 * band + in % high + tilesM * (in / high);
}

} // namespace blocks

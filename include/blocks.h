// Dense layers in 8-bit blocks: the format, the linear layer and its gradients, and activations whose
// input is kept in 8 bits for the backward pass. No counterpart in the reference, whose only 8-bit
// features are INT8 with one FP32 scale per row (format/int8_features.h).
//
// Format. 128 consecutive elements of a row are a block; a weight's block is a tile of 128 x 128. A block
// has one scale, a power of two held as a byte e that stands for 2^(e - 127): the smallest, and at least
// 2^-126, that brings the block's largest magnitude to at most 448 (E4M3 codes) or 127 (INT8 codes); a
// block of zeros has e = 127. A code is its element times 2^(127 - e), rounded half to even: the
// product is exact in FP32, so that is the only rounding. (An element that would round to 2^128 takes the
// code below, so that every value is finite in FP32.) A block with an infinity or a NaN has e = 255
// and codes 0 and stands for NaNs; 255 stands for NaN in given exponents too.
// Codes are [rows][128 * ceil(columns / 128)] bytes, zero past the row's end. Exponents are
// [rows][4 * ceil(blocks / 4)] bytes (a weight's: [ceil(rows / 128)][..]), 127 past the row's end.
//
// Every function is asynchronous on `stream` and allocates nothing. Sizes of zero rows return without a
// launch. Errors are thrown before any launch: std::invalid_argument for null or misaligned buffers,
// sizes and strides out of range and workspaces that are too small, std::runtime_error for the
// runtime's. Rows may be up to 2^31 - 1, their elements up to 2^22, and a product's or weight's tiles fewer than 2^24
// (of 256 x 256 for a 16-bit y, 128 x 128 otherwise), which is what a launch takes. Codes must be 16-byte aligned and
// exponents 4-byte aligned (anything from hipMalloc or torch); dense matrices need only their element's alignment, with
// any row stride of at least a row.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

enum class DenseType : std::uint32_t { f32 = 0, bf16 = 1, f16 = 2 };
enum class BlockCodes : std::uint32_t { e4m3 = 0, int8 = 1 };
enum class BlockActivation : std::uint32_t { silu = 0, gelu = 1, geluTanh = 2 };

constexpr std::uint32_t kBlock = 128;

// Bytes of a row of codes, and of a row of exponents.
constexpr std::uint64_t blockCodePitch(std::uint32_t columns) {
    return (std::uint64_t(columns) + kBlock - 1) / kBlock * kBlock;
}
constexpr std::uint64_t blockExponentPitch(std::uint32_t columns) {
    return (blockCodePitch(columns) / kBlock + 3) / 4 * 4;
}

// A dense row-major matrix; stride in elements.
struct DenseMatrix {
    const void* data;
    std::uint64_t stride;
    DenseType type;
};

// Codes and exponents of `rows` rows of `columns` elements, in blocks along the row.
struct BlockRows {
    std::uint8_t* codes;
    std::uint8_t* exponents;
    BlockCodes type;
};

// E4M3 codes and exponents of a weight [outer][inner] in tiles, and of its transpose [inner][outer]
// (null where nothing reads them: only the input gradient does).
struct BlockWeightView {
    std::uint8_t* codes;
    std::uint8_t* exponents;
    std::uint8_t* codesT;
    std::uint8_t* exponentsT;
};

void quantizeBlocks(DenseMatrix x, BlockRows out, std::uint32_t rows, std::uint32_t columns,
                    hipStream_t stream = nullptr);

// The values that codes stand for.
void dequantizeBlocks(BlockRows x, void* out, DenseType type, std::uint64_t stride, std::uint32_t rows,
                      std::uint32_t columns, hipStream_t stream = nullptr);

// Tiles of a weight, with the transposed copy if out.codesT and out.exponentsT are given, in one pass.
void quantizeWeightBlocks(DenseMatrix w, BlockWeightView out, std::uint32_t outer, std::uint32_t inner,
                          hipStream_t stream = nullptr);

// y = x w^T + bias for x in E4M3 blocks [rows][inner] and w in E4M3 tiles [outer][inner]; bias null or
// FP32 [outer]. Called with the transposed weight it gives the input gradient from the output
// gradient's blocks. An FP32 y has its sums in FP32, through the bf16 MFMA on the codes' values. Those are exact for
// exponents of 3 to 246; below, a value is rounded to a multiple of 2^-133, bf16's last, and one of 2^128 or more, which
// FP32 rows never give, is infinite (as in dequantizeBlocks). For 16-bit types products of codes are exact at every
// exponent, and the sums are the 8-bit MFMA's: of 8 consecutive products each is cut off, towards
// zero, 13 bits below the power of two of the largest, and from there on sums are FP32's. So a sum is at most
// 7 * 2^-13 of its terms' magnitudes off; on random numbers 1.2e-5 of the sums' norm, a twentieth of an f16
// rounding, which shows as a last place here and there. Who needs FP32 sums in 16 bits takes an FP32 y and rounds it.
void matmulBlocks(BlockRows x, BlockWeightView w, const float* bias, void* y, DenseType type,
                  std::uint64_t stride, std::uint32_t rows, std::uint32_t inner, std::uint32_t outer,
                  hipStream_t stream = nullptr);

// The linear layer on dense x: quantizeBlocks and matmulBlocks with y's type that of x, in one launch
// where that is faster. `keep` with null codes keeps nothing; else it receives x's blocks, the backward
// pass's checkpoint. workspaceBytes must be at least linearBlocksWorkspace(..) for the same sizes and type.
std::size_t linearBlocksWorkspace(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type,
                                  bool keep);
void linearBlocks(DenseMatrix x, BlockWeightView w, const float* bias, void* y, std::uint64_t yStride,
                  BlockRows keep, std::uint32_t rows, std::uint32_t inner, std::uint32_t outer,
                  void* workspace, std::size_t workspaceBytes, hipStream_t stream = nullptr);

// The kernel that a call of these sizes takes, by name, for tests and measurements; its splits of the rows for a gradient.
// matmulBlocks and linearBlocks; linearBlocks calls matmulBlocks where the names are the same.
const char* matmulBlocksForm(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type);
const char* linearBlocksForm(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer, DenseType type);

// dw = dy^T x for dense dy [rows][outer] and x's E4M3 blocks [rows][inner], FP32 [outer][inner]
// contiguous, and, if db is not null, db = the sums of dy's columns. All sums in FP32, of x's values as in an FP32 y of
// matmulBlocks; a dy of f16 or f32 goes through the bf16 MFMA as two or three bf16 parts, which together hold it exactly
// (FP32: to 2^-25 of it, or 2^-134 where that is more).
// Repeated calls give the same bits. Zero rows give zero gradients. A null dw asks for db alone: neither x nor inner is
// read, and the workspace is that of inner = 0.
std::size_t weightGradBlocksWorkspace(std::uint32_t rows, std::uint32_t inner, std::uint32_t outer,
                                      DenseType type);
void weightGradBlocks(DenseMatrix dy, BlockRows x, float* dw, float* db, std::uint32_t rows,
                      std::uint32_t inner, std::uint32_t outer, void* workspace, std::size_t workspaceBytes,
                      hipStream_t stream = nullptr);

const char* weightGradBlocksForm(DenseMatrix dy, std::uint32_t rows, std::uint32_t inner, std::uint32_t outer,
                                 std::uint32_t* splits);

// y = f(x) for x [rows][width], or, gated, y = f(g) u for x = [g | u] of [rows][2 * width]; y has x's
// type. `keep` receives x's blocks for the backward pass (null codes: nothing is kept): rows of `width`,
// gated two for each row of x, the gate's and the factor's.
void activationBlocks(DenseMatrix x, BlockActivation f, bool gated, void* y, std::uint64_t yStride,
                      BlockRows keep, std::uint32_t rows, std::uint32_t width, hipStream_t stream = nullptr);

// dx from dy [rows][width] and the kept blocks; dx has dy's type and x's shape.
void activationBlocksBackward(DenseMatrix dy, BlockRows kept, BlockActivation f, bool gated, void* dx,
                              std::uint64_t dxStride, std::uint32_t rows, std::uint32_t width,
                              hipStream_t stream = nullptr);

// Layers of many experts: tokens sorted by expert and back, and the experts' products with weights in microscaled 4-bit
// blocks (micro.h). No counterpart in the reference; the way back is its sparse product's kind of sum, with one entry of
// the matrix for each choice of a token.
//
// A router gives each of `tokens` tokens `each` choices, numbers of experts. A choice outside [0, experts) is for an
// expert that is not here. The plan of a set of choices, three arrays of int32 in device memory:
//   order[choices]       the choices sorted by expert, those of one expert in their own order, those for no expert
//                        here last. Row r of the sorted rows belongs to choice order[r], of token order[r] / each.
//   places[choices]      the row of each choice: order[places[c]] == c
//   offsets[experts + 1] expert e's rows are [offsets[e], offsets[e + 1]); those from offsets[experts] on have none
//
// Every function is asynchronous on `stream` and allocates nothing. Without choices they return without a launch
// (sortExperts still writes the offsets). Errors are thrown before any launch, as in blocks.h. Choices may be up to
// 2^31 - 1, of up to 1024 each, and experts 1 to 1024; tokens of rows of more than 1024 elements fewer than 2^24 in a gather
// or a combine, which is what a launch takes (of shorter rows a workgroup takes several). Kernels hold what they read of a
// plan to the sizes given, so that a plan of other sizes gives wrong rows, never an access out of range.
#pragma once

#include "micro.h"

constexpr std::uint32_t kMaxExperts = 1024;
constexpr std::uint32_t kMaxEach = 1024;

struct ExpertPlan {
    std::int32_t* offsets;
    std::int32_t* order;
    std::int32_t* places;
    std::uint32_t choices; // tokens * each
    std::uint32_t each;
    std::uint32_t experts;
};

// The plan of choices given as int32 or int64 (idBytes 4 or 8). Repeated calls give the same plan.
std::size_t sortExpertsWorkspace(std::uint32_t choices, std::uint32_t experts);
void sortExperts(const void* ids, std::uint32_t idBytes, ExpertPlan plan, void* workspace, std::size_t workspaceBytes,
                 hipStream_t stream = nullptr);

// rows[r] = x[order[r] / each], of x's type; rows of no expert are zeros.
void gatherExperts(DenseMatrix x, ExpertPlan plan, void* rows, std::uint64_t stride, std::uint32_t width,
                   hipStream_t stream = nullptr);

// y[t] = the sum over t's choices c of weights[c] * rows[places[c]], in FP32 and in the choices' order, rounded once to
// the rows' type; null weights are ones, and choices for no expert here add nothing. Without weights it is the gradient
// of gatherExperts.
void combineExperts(DenseMatrix rows, ExpertPlan plan, const void* weights, DenseType weightType, void* y,
                    std::uint64_t stride, std::uint32_t width, hipStream_t stream = nullptr);

// The gradients of combineExperts from dy [tokens][width]: drows[places[c]] = weights[c] * dy[t], of dy's type, zeros for
// rows of no expert, and dweights[c] = dy[t] . rows[places[c]], summed in FP32, of weightType, zero for choices of no
// expert here. Either may be null; without dweights rows are not read. rows has dy's type.
void combineExpertsBackward(DenseMatrix dy, DenseMatrix rows, ExpertPlan plan, const void* weights, DenseType weightType,
                            void* drows, std::uint64_t stride, void* dweights, std::uint32_t width,
                            hipStream_t stream = nullptr);

// y[r] = x[row] w[e]^T + bias[e] for each sorted row r of expert e, with the sums of matmulMicro; zeros for rows of no
// expert. x has a row for each sorted row, or, byToken, for each token, and row r takes that of its token; codes of
// tokens are then at most 2^31 - 1 bytes (of more: gatherExperts moves codes and exponents as 16-bit matrices of half as many
// columns as they are). w is a stack of [experts][outer] rows of `inner` elements; bias null or FP32
// [experts][outer]. With the transposed stack it gives the rows' input gradient.
void matmulExperts(CodedRows x, bool byToken, MicroRows w, const float* bias, void* y, DenseType type, std::uint64_t stride,
                   ExpertPlan plan, std::uint32_t inner, std::uint32_t outer, hipStream_t stream = nullptr);

// The same on dense x, in `format`, with y's type that of x.
std::size_t linearExpertsWorkspace(ExpertPlan plan, bool byToken, std::uint32_t inner, std::uint32_t outer, DenseType type,
                                   RowFormat format);
void linearExperts(DenseMatrix x, RowFormat format, bool byToken, MicroRows w, const float* bias, void* y,
                   std::uint64_t yStride, ExpertPlan plan, std::uint32_t inner, std::uint32_t outer, void* workspace,
                   std::size_t workspaceBytes, hipStream_t stream = nullptr);

// The kernel that a call of these sizes takes, by name, for tests and measurements.
const char* matmulExpertsForm(ExpertPlan plan, std::uint32_t inner, std::uint32_t outer, DenseType type, RowFormat format);

// Shared types of the linear cross entropy (linear_ce.hip): operand layouts,
// the element types' splitting into matrix-core operands, and the plan of a
// call's workspace.
//
//   logits l[n, v] = sum_d x[n, d] w[v, d]          (never stored)
//   lse_n = log sum_v exp l[n, v],  loss_n = lse_n - l[n, t_n] + z lse_n^2
//   G[n, v] = a_n exp(l[n, v] - lse_n) + b_n [v == t_n],
//       a_n = g_n (1 + 2 z lse_n), b_n = -g_n
//   dx = G w, dw = G^T x
//
// Rows whose target is ignore_index are taken out before any product: the
// kernels run over the live rows only, in their order.
#pragma once

#include "lse_common.hpp"

namespace fl {
namespace lce {

enum DType { kF32 = 0, kF16 = 1, kBF16 = 2 };

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// The matrix cores take 16-bit operands.  fp16 and bf16 go in as they are.  An
// fp32 value is the sum of three bf16 parts of 8 bits each (truncated, so
// that the first part of a large value does not overflow), and a product of
// two is the six partial products whose parts' indices add up to at most 2;
// the ones left out are below 2^-21 of the product together.  The bf16 matrix
// rate is 16 times the fp32 one, so six products cost 0.375 of one fp32
// product.
constexpr int kTerms = 6;
__device__ constexpr int kTermA[kTerms] = {0, 0, 1, 1, 0, 2};
__device__ constexpr int kTermB[kTerms] = {0, 1, 0, 1, 2, 0};

__device__ __forceinline__ void split3(float v, uint16_t (&o)[3]) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    o[0] = (uint16_t)(u >> 16);
    const float r1 = v - __builtin_bit_cast(float, u & 0xFFFF0000u);
    // a part that is inf or NaN has no rest
    const bool fin = __builtin_isfinite(v);
    const uint32_t u1 = fin ? __builtin_bit_cast(uint32_t, r1) : 0u;
    o[1] = (uint16_t)(u1 >> 16);
    const float r2 = __builtin_bit_cast(float, u1) - __builtin_bit_cast(float, u1 & 0xFFFF0000u);
    o[2] = (uint16_t)(__builtin_bit_cast(uint32_t, r2) >> 16);
}

// One product's operand: 16-bit rows `ld` elements apart, in `parts` copies
// `part` elements apart, `cols` (a multiple of 8) of a row's elements readable.
// What a tile reaches beyond the rows and columns is read as the last row and
// the last 8 columns.
struct Operand {
    const uint16_t* p;
    int64_t ld;
    int64_t part;
    int rows;
    int64_t cols;
};

}  // namespace lce
}  // namespace fl

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

// The matrix cores take 16-bit operands.  fp16 and bf16 go in as they are; fp32
// goes in as parts, whose products' parts' indices add up to less than their
// number.
//
// Logits: two fp16 parts of 11 bits, taken after a power of two that brings the
// row's largest finite magnitude to [2^14, 2^15).  An element is then exact to
// 2^-23 of itself or 2^-39 of its row's largest, whichever is more; three partial
// products, the one left out below 2^-22 of the product.  A scale a row, so that
// no row's result depends on another row's size.
//
// dx and dw: three bf16 parts of 8 bits, to nearest: exact down to 2^-126, which
// G, whose entries reach from 1 down to nothing, needs and fp16's exponents do
// not give (values within 2^-9 of the largest fp32 count as infinite, and
// infinite ones make NaN).  Six partial products; those left out
// are below 2^-24 of the product together.
//
// The 16-bit matrix rate is 16 times the fp32 one, so three products cost 0.19
// and six 0.375 of one fp32 product.
__host__ __device__ constexpr int terms(int parts) { return parts == 1 ? 1 : parts == 2 ? 3 : 6; }
// parts of term t: 00 01 10 | 11 02 20
__device__ constexpr int term_a(int t) { return t == 2 || t == 3 ? 1 : t == 5 ? 2 : 0; }
__device__ constexpr int term_b(int t) { return t == 1 || t == 3 ? 1 : t == 4 ? 2 : 0; }

__device__ __forceinline__ void split2(float v, uint16_t (&o)[2]) {
    const _Float16 hi = (_Float16)v;
    // an infinite part has no rest
    const _Float16 lo = __builtin_isfinite(v) ? (_Float16)(v - (float)hi) : (_Float16)0.0f;
    o[0] = __builtin_bit_cast(uint16_t, hi);
    o[1] = __builtin_bit_cast(uint16_t, lo);
}
__device__ __forceinline__ uint16_t bf16_bits(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ void split3(float v, uint16_t (&o)[3]) {
    o[0] = bf16_bits(v);
    const float r1 = v - __builtin_bit_cast(float, (uint32_t)o[0] << 16);  // NaN of an infinite v
    o[1] = bf16_bits(r1);
    o[2] = bf16_bits(r1 - __builtin_bit_cast(float, (uint32_t)o[1] << 16));
}

// Exponent e of the power of two that brings a magnitude m to [2^(to - 1),
// 2^to), within what fp32 holds; 0 for nothing, inf and NaN.
__device__ __forceinline__ int scale_exp(float m, int to) {
    if (!(m > 0.0f) || !__builtin_isfinite(m)) return 0;
    const int e = to - __builtin_amdgcn_frexp_expf(m);
    return e < -126 ? -126 : e > 126 ? 126 : e;
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

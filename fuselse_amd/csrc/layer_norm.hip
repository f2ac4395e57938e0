// Layer norm over the last dimension, forward and backward, on gfx950.
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   dx = r (a - mean a - h mean(a h)) with a = g w;  dw = sum_rows g h, db = sum_rows g
//
// A row is held in registers by some lanes of a wave or a block, or read again from
// the caches, so that memory sees each operand once; only the backward of rows of
// more than 1024 vectors reads x and g twice, since a block's registers do not hold
// sums for as many columns.  The mean is kept as two numbers: m0, the rounded sum
// over D, and m1, the mean of the differences to it.  x - m0 - m1 then keeps its
// digits when the row has a large value in common, which one fp32 mean would take
// from it.  Lanes meet the same columns in every row and sum dw and db in registers;
// the blocks' sums are joined in an order that their number alone decides.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/fuselse_amd.h"
#include "fl_status.hpp"
#include "row_vec.hpp"

// The rounded m0 is subtracted in both directions: a product contracted into the
// subtraction would give the forward another m0 than the backward's.
#pragma clang fp contract(off)

namespace fl {
namespace layer_norm {
namespace {

struct Args {
    const void* x;
    int64_t ldx;
    int64_t rows, D;
    const void* w;  // NULL: 1
    const void* b;  // NULL: 0
    bool params_f32;
    float eps;
    void* y;       // forward: y; backward: dx (NULL: not wanted)
    f32x4* stats;  // [rows]: m0, -m1 r, r
    const void* g;
    int64_t ldg;
    float* part;  // [blocks][2][D]: sums of g h and of g
    int blocks;
};

// Columns c, c + 1, .. of a parameter, widened.
template <typename T>
__device__ __forceinline__ void load_param_at(const Args& p, const void* a, int64_t c, float (&v)[Elem<T>::kVec]) {
    if (p.params_f32) {
#pragma unroll
        for (int k = 0; k < Elem<T>::kVec; k += 4) {
            float f[4];
            load_vec_any<float>(static_cast<const float*>(a) + c + k, f);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[k + i] = f[i];
        }
    } else {
        load_vec_any<T>(static_cast<const T*>(a) + c, v);
    }
}

// Sums over a row's lanes: LANES up to a wave within it, more across the block.
template <int LANES, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*sh)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (LANES >= 2) v[i] += reduce_partner<1>(v[i]);
        if constexpr (LANES >= 4) v[i] += reduce_partner<2>(v[i]);
        if constexpr (LANES >= 8) v[i] += reduce_partner<4>(v[i]);
        if constexpr (LANES >= 16) v[i] += reduce_partner<8>(v[i]);
        if constexpr (LANES >= 32) v[i] += reduce_partner<16>(v[i]);
        if constexpr (LANES >= 64) v[i] += reduce_partner<32>(v[i]);
    }
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) sh[threadIdx.x >> 6][i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < LANES / 64; ++w) s += sh[w][i];
            v[i] = s;
        }
    }
}

// What the backward needs of a row: m0, -m1 r and r, so that h is two operations:
// (x - m0) r - m1 r.  m1 and the mean square are of the differences times f, a power of two.
__device__ __forceinline__ f32x4 row_stats(float m0, float m1, float mean_square, float eps, float f = 1.0f) {
    const float var = mean_square - m1 * m1;
    const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps * f * f);
    return f32x4{m0, -m1 * rstd, rstd * f, 0.0f};
}

// Sums over a row may leave fp32 where its elements do not.  That of the elements is then
// made of elements scaled down (row_mean_wide).  That of the squared differences to m0
// may too, and where the elements are equal, or all but, these differences are m0's
// rounding alone, of which no variance is left.  Such a row is summed again: m0 moves by
// the differences' mean, so that equal elements come to differ by 0 exactly; unscaled
// differences are then in range where only m0 was off; and scaled down they are whatever
// they are.  sums(m0, f, d) gives d, the row's sums of f (x - m0) and of its squares, and
// move(m0, to) what it keeps of x - m0.  The tests that find such rows cost other rows
// nothing that shows: (65536, 4096) in bf16 186 us with and without them, (16384, 16384)
// 192 and 190.
__device__ __forceinline__ bool finite(float v) { return __builtin_fabsf(v) < kInf; }
constexpr float kDown = 0x1p-26f;  // of 2^24 elements
template <typename Sum>
__device__ __forceinline__ float row_mean_wide(float inv, Sum sum) {
    return sum(kDown) * inv * (1.0f / kDown);
}

__device__ __forceinline__ bool row_stats_hold(const float (&d)[2], float inv) {
    const float m1 = d[0] * inv, mean_square = d[1] * inv;
    return mean_square < kInf && mean_square - m1 * m1 >= mean_square * 0x1p-10f;
}
constexpr float kWide = 0x1p-80f;  // squares of 2^24 elements that it scales down are in range
template <typename Sums, typename Move>
__device__ __forceinline__ f32x4 row_stats_wide(float m0, float inv, float eps, float (&d)[2], Sums sums, Move move) {
    float f = finite(d[0]) ? 1.0f : kWide;
    if (f != 1.0f) sums(m0, f, d);
    const float to = m0 + d[0] * inv * (1.0f / f);
    move(m0, to);
#pragma unroll 1
    for (f = 1.0f;; f = kWide) {
        sums(to, f, d);
        if (f != 1.0f || d[1] < kInf) break;
    }
    return row_stats(to, d[0] * inv, d[1] * inv, eps, f);
}

// How a block is laid out for rows of LANES * NV vectors at most.
template <int LANES>
struct Shape {
    static constexpr int kThreads = LANES > 256 ? LANES : 256;
    static constexpr int kRows = kThreads / LANES;
};

// Lane `sub` holds vectors sub, sub + LANES, .. of a row.  Where rows are no whole
// vectors (!WHOLE) the last vector is moved back to end with the row, so that all
// loads and stores are whole; the elements that it shares with the one before
// count once, there.
template <typename T, int LANES, int NV, bool WHOLE>
struct Columns {
    using Type = T;
    static constexpr int VE = Elem<T>::kVec;
    int at[NV];    // the vector's first column
    int skip[NV];  // its elements that do not count: VE, or those shared
    __device__ __forceinline__ Columns(int D, int sub) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (sub + j * LANES) * VE;
            at[j] = WHOLE ? c : c < D - VE ? c : D - VE;
            skip[j] = c >= D ? VE : WHOLE ? 0 : c - at[j];
        }
    }
    __device__ __forceinline__ bool any(int j) const { return skip[j] < VE; }
    __device__ __forceinline__ bool counts(int j, int k) const { return WHOLE ? skip[j] == 0 : k >= skip[j]; }
};

template <typename T, int NV, typename C>
__device__ __forceinline__ void load_row(const C& col, const T* row, u32x4 (&v)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = col.any(j) ? load_raw_stream(row + col.at[j]) : u32x4{0, 0, 0, 0};
}

// Vector j's columns of a parameter, or `fill` where there is none.
template <typename C, int VE>
__device__ __forceinline__ void load_param(const Args& p, const C& col, int j, const void* a, float fill,
                                           float (&v)[VE]) {
#pragma unroll
    for (int k = 0; k < VE; ++k) v[k] = fill;
    if (a && col.any(j)) load_param_at<typename C::Type>(p, a, col.at[j], v);
}

template <typename T, typename C>
__device__ __forceinline__ void store_vec(const C& col, int j, T* row, const float (&v)[Elem<T>::kVec]) {
    if (col.any(j)) __builtin_nontemporal_store(pack_vec<T>(v), reinterpret_cast<u32x4_any*>(row + col.at[j]));
}

// Adds a vector's elements to s, two an instruction where they are 16-bit.
template <typename T>
__device__ __forceinline__ void add_vec(u32x4 r, float& s) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t e = r[k];
        if constexpr (sizeof(T) == 4) s += __builtin_bit_cast(float, e);
        else if constexpr (__is_same(T, _Float16))
            s = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, e), f16x2{(_Float16)1.0f, (_Float16)1.0f}, s, false);
        else
            s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, e), bf16x2{(__bf16)1.0f, (__bf16)1.0f}, s,
                                                false);
    }
}

// A row's loads are issued before the row before it is reduced, and the parameters
// stay in registers, but for rows of more than 2048 vectors, whose block is alone on
// its CU and has too few.
template <typename T, int LANES, int NV, bool WHOLE>
__global__ __launch_bounds__(Shape<LANES>::kThreads) void fwd_kernel(Args p) {
    constexpr int VE = Elem<T>::kVec;
    __shared__ float sh1[Shape<LANES>::kThreads / 64][1], sh2[Shape<LANES>::kThreads / 64][2];
    const int sub = (int)threadIdx.x % LANES;
    const Columns<T, LANES, NV, WHOLE> col((int)p.D, sub);
    const float inv = 1.0f / (float)p.D;
    const int64_t step = (int64_t)p.blocks * Shape<LANES>::kRows;
    int64_t r = (int64_t)blockIdx.x * Shape<LANES>::kRows + (int)threadIdx.x / LANES;
    constexpr bool HOLD = LANES <= 256 || NV <= 2;
    u32x4 next[NV];
    if (r < p.rows) load_row<T>(col, static_cast<const T*>(p.x) + r * p.ldx, next);
    float w[HOLD ? NV : 1][VE], b[HOLD ? NV : 1][VE];
    if constexpr (HOLD) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            load_param(p, col, j, p.w, 1.0f, w[j]);
            load_param(p, col, j, p.b, 0.0f, b[j]);
        }
    }
    for (; r < p.rows; r += step) {
        float x[NV][VE];
        float s[1] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            Elem<T>::cvt(next[j], x[j]);
            if constexpr (WHOLE) {
                add_vec<T>(next[j], s[0]);
            } else {
#pragma unroll
                for (int k = 0; k < VE; ++k)
                    if (col.counts(j, k)) s[0] += x[j][k];
            }
        }
        if (r + step < p.rows) load_row<T>(col, static_cast<const T*>(p.x) + (r + step) * p.ldx, next);
        row_sum<LANES>(s, sh1);
        float m0 = s[0] * inv;
        if (!finite(m0))
            m0 = row_mean_wide(inv, [&](float f) {
                float o[1] = {};
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int k = 0; k < VE; ++k)
                        if (col.counts(j, k)) o[0] += x[j][k] * f;
                row_sum<LANES>(o, sh1);
                return o[0];
            });
        float d[2] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                x[j][k] -= m0;
                if (col.counts(j, k)) {
                    d[0] += x[j][k];
                    d[1] = __builtin_fmaf(x[j][k], x[j][k], d[1]);
                }
            }
        row_sum<LANES>(d, sh2);
        f32x4 st = row_stats(m0, d[0] * inv, d[1] * inv, p.eps);
        if (!row_stats_hold(d, inv))
            st = row_stats_wide(
                m0, inv, p.eps, d,
                [&](float, float f, float (&o)[2]) {
                    o[0] = o[1] = 0.0f;
#pragma unroll
                    for (int j = 0; j < NV; ++j)
#pragma unroll
                        for (int k = 0; k < VE; ++k)
                            if (col.counts(j, k)) {
                                const float c = x[j][k] * f;
                                o[0] += c;
                                o[1] = __builtin_fmaf(c, c, o[1]);
                            }
                    row_sum<LANES>(o, sh2);
                },
                [&](float from, float to) {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
#pragma unroll
                        for (int k = 0; k < VE; ++k) x[j][k] = x[j][k] + from - to;
                });
        if (p.stats && sub == 0) p.stats[r] = st;
        T* y = static_cast<T*>(p.y) + r * p.D;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            constexpr int ONE = HOLD ? 1 : 0;
            if constexpr (!HOLD) {
                load_param(p, col, j, p.w, 1.0f, w[0]);
                load_param(p, col, j, p.b, 0.0f, b[0]);
            }
#pragma unroll
            for (int k = 0; k < VE; ++k)
                x[j][k] = __builtin_fmaf(__builtin_fmaf(x[j][k], st[2], st[1]), w[j * ONE][k], b[j * ONE][k]);
            store_vec<T>(col, j, y, x[j]);
        }
    }
}

// With more than 256 lanes a row it gives dx alone.
template <typename T, int LANES, int NV, bool WHOLE>
__global__ __launch_bounds__(Shape<LANES>::kThreads) void bwd_kernel(Args p) {
    constexpr int VE = Elem<T>::kVec;
    constexpr int ROWS = Shape<LANES>::kRows;
    __shared__ float sh2[2][Shape<LANES>::kThreads / 64][2];
    const int sub = (int)threadIdx.x % LANES;
    const Columns<T, LANES, NV, WHOLE> col((int)p.D, sub);
    const float inv = 1.0f / (float)p.D;
    const int64_t step = (int64_t)p.blocks * ROWS;
    int64_t r = (int64_t)blockIdx.x * ROWS + (int)threadIdx.x / LANES;
    u32x4 next_x[NV], next_g[NV];
    f32x4 next_st{0, 0, 0, 0};
    if (r < p.rows) {
        load_row<T>(col, static_cast<const T*>(p.x) + r * p.ldx, next_x);
        load_row<T>(col, static_cast<const T*>(p.g) + r * p.ldg, next_g);
        next_st = p.stats[r];
    }
    constexpr bool SUMS = LANES <= 256, HOLD = SUMS || NV <= 2;
    constexpr int ONE = HOLD ? 1 : 0;
    float w[HOLD ? NV : 1][VE], dw[SUMS ? NV : 1][VE] = {}, db[SUMS ? NV : 1][VE] = {};
    if constexpr (HOLD) {
#pragma unroll
        for (int j = 0; j < NV; ++j) load_param(p, col, j, p.w, 1.0f, w[j]);
    }
    for (int turn = 0; r < p.rows; r += step, turn ^= 1) {
        const float m0 = next_st[0], shift = next_st[1], rstd = next_st[2];
        float h[NV][VE], g[NV][VE];
        float s[2] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            Elem<T>::cvt(next_x[j], h[j]);
            Elem<T>::cvt(next_g[j], g[j]);
            if constexpr (!HOLD) load_param(p, col, j, p.w, 1.0f, w[0]);
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                h[j][k] = __builtin_fmaf(h[j][k] - m0, rstd, shift);
                if constexpr (SUMS) {
                    dw[j][k] = __builtin_fmaf(g[j][k], h[j][k], dw[j][k]);
                    db[j][k] += g[j][k];
                }
                g[j][k] *= w[j * ONE][k];
                if (col.counts(j, k)) {
                    s[0] += g[j][k];
                    s[1] = __builtin_fmaf(g[j][k], h[j][k], s[1]);
                }
            }
        }
        if (r + step < p.rows) {
            load_row<T>(col, static_cast<const T*>(p.x) + (r + step) * p.ldx, next_x);
            load_row<T>(col, static_cast<const T*>(p.g) + (r + step) * p.ldg, next_g);
            next_st = p.stats[r + step];
        }
        if (!p.y) continue;
        row_sum<LANES>(s, sh2[turn]);
        const float c0 = -rstd * (s[0] * inv), c1 = -rstd * (s[1] * inv);
        T* dx = static_cast<T*>(p.y) + r * p.D;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
#pragma unroll
            for (int k = 0; k < VE; ++k)
                g[j][k] = __builtin_fmaf(h[j][k], c1, __builtin_fmaf(g[j][k], rstd, c0));
            store_vec<T>(col, j, dx, g[j]);
        }
    }
    if (!SUMS || !p.part) return;
    // the block's rows, joined over its groups of lanes in their order
    float* part = p.part + (int64_t)blockIdx.x * 2 * p.D;
    if constexpr (!SUMS) {
    } else if constexpr (ROWS == 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k)
                if (col.counts(j, k)) {
                    part[col.at[j] + k] = dw[j][k];
                    part[p.D + col.at[j] + k] = db[j][k];
                }
    } else {
        constexpr int W = LANES * NV * VE;
        __shared__ float sum[2][W];
        for (int q = 0; q < ROWS; ++q) {
            if ((int)threadIdx.x / LANES == q) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int k = 0; k < VE; ++k)
                        if (col.counts(j, k)) {
                            const int c = col.at[j] + k;
                            sum[0][c] = q ? sum[0][c] + dw[j][k] : dw[j][k];
                            sum[1][c] = q ? sum[1][c] + db[j][k] : db[j][k];
                        }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < (int)p.D; c += Shape<LANES>::kThreads) {
            part[c] = sum[0][c];
            part[p.D + c] = sum[1][c];
        }
    }
}

// Rows of one vector or less, one a thread; shorter ones go element by element in
// memory, with zeros behind them in registers.  (1048576, 7) in bf16: 17 us forward
// and 23 backward, 10.7 and 11.0 ms by a block a row; (1048576, 8) 11 and 17, by eight
// lanes a row 32 and 58.
constexpr int kShort = 256;

template <typename T>
__device__ __forceinline__ void load_short(const T* row, int64_t D, float (&x)[Elem<T>::kVec]) {
    Elem<T>::cvt(row_load(row, D, 0), x);
}
template <typename T>
__device__ __forceinline__ void load_param_short(const Args& p, const void* a, float fill, float (&v)[Elem<T>::kVec]) {
#pragma unroll
    for (int k = 0; k < Elem<T>::kVec; ++k) {
        v[k] = fill;
        if (a && k < p.D)
            v[k] = p.params_f32 ? static_cast<const float*>(a)[k] : Elem<T>::scalar(static_cast<const T*>(a) + k);
    }
}

template <typename T>
__global__ __launch_bounds__(kShort) void fwd_short(Args p) {
    constexpr int VE = Elem<T>::kVec;
    const float inv = 1.0f / (float)p.D;
    float w[VE], b[VE];
    load_param_short<T>(p, p.w, 1.0f, w);
    load_param_short<T>(p, p.b, 0.0f, b);
    for (int64_t r = (int64_t)blockIdx.x * kShort + threadIdx.x; r < p.rows; r += (int64_t)p.blocks * kShort) {
        float x[VE], s = 0.0f, d[2] = {};
        load_short(static_cast<const T*>(p.x) + r * p.ldx, p.D, x);
#pragma unroll
        for (int k = 0; k < VE; ++k)
            if (k < p.D) s += x[k];
        float m0 = s * inv;
        if (!finite(m0))
            m0 = row_mean_wide(inv, [&](float f) {
                float o = 0.0f;
#pragma unroll
                for (int k = 0; k < VE; ++k)
                    if (k < p.D) o += x[k] * f;
                return o;
            });
#pragma unroll
        for (int k = 0; k < VE; ++k) {
            x[k] -= m0;
            if (k < p.D) {
                d[0] += x[k];
                d[1] = __builtin_fmaf(x[k], x[k], d[1]);
            }
        }
        f32x4 st = row_stats(m0, d[0] * inv, d[1] * inv, p.eps);
        if (!row_stats_hold(d, inv))
            st = row_stats_wide(
                m0, inv, p.eps, d,
                [&](float, float f, float (&o)[2]) {
                    o[0] = o[1] = 0.0f;
#pragma unroll
                    for (int k = 0; k < VE; ++k)
                        if (k < p.D) {
                            const float c = x[k] * f;
                            o[0] += c;
                            o[1] = __builtin_fmaf(c, c, o[1]);
                        }
                },
                [&](float from, float to) {
#pragma unroll
                    for (int k = 0; k < VE; ++k) x[k] = x[k] + from - to;
                });
        if (p.stats) p.stats[r] = st;
#pragma unroll
        for (int k = 0; k < VE; ++k) x[k] = __builtin_fmaf(__builtin_fmaf(x[k], st[2], st[1]), w[k], b[k]);
        row_store(static_cast<T*>(p.y) + r * p.D, p.D, 0, pack_vec<T>(x));
    }
}

template <typename T>
__global__ __launch_bounds__(kShort) void bwd_short(Args p) {
    constexpr int VE = Elem<T>::kVec;
    __shared__ float sh[kShort / 64][2 * VE];
    const float inv = 1.0f / (float)p.D;
    float w[VE], sums[2 * VE] = {};  // of g h, of g
    load_param_short<T>(p, p.w, 1.0f, w);
    for (int64_t r = (int64_t)blockIdx.x * kShort + threadIdx.x; r < p.rows; r += (int64_t)p.blocks * kShort) {
        float h[VE], g[VE], s0 = 0.0f, s1 = 0.0f;
        load_short(static_cast<const T*>(p.x) + r * p.ldx, p.D, h);
        load_short(static_cast<const T*>(p.g) + r * p.ldg, p.D, g);
        const f32x4 st = p.stats[r];
#pragma unroll
        for (int k = 0; k < VE; ++k) {
            h[k] = __builtin_fmaf(h[k] - st[0], st[2], st[1]);
            sums[k] = __builtin_fmaf(g[k], h[k], sums[k]);
            sums[VE + k] += g[k];
            g[k] *= w[k];
            if (k < p.D) {
                s0 += g[k];
                s1 = __builtin_fmaf(g[k], h[k], s1);
            }
        }
        if (!p.y) continue;
        const float c0 = -st[2] * (s0 * inv), c1 = -st[2] * (s1 * inv);
#pragma unroll
        for (int k = 0; k < VE; ++k) g[k] = __builtin_fmaf(h[k], c1, __builtin_fmaf(g[k], st[2], c0));
        row_store(static_cast<T*>(p.y) + r * p.D, p.D, 0, pack_vec<T>(g));
    }
    if (!p.part) return;
    row_sum<kShort>(sums, sh);
    if (threadIdx.x > 0) return;
    float* part = p.part + (int64_t)blockIdx.x * 2 * p.D;
#pragma unroll
    for (int k = 0; k < VE; ++k)
        if (k < p.D) {
            part[k] = sums[k];
            part[p.D + k] = sums[VE + k];
        }
}

// Rows too long for registers, by a block that reads them again from the caches for
// each step.
constexpr int kLong = 1024;

// Vector v of a row, the elements that another vector has too marked by skip.
template <typename T>
struct LongVec {
    int64_t at;
    int skip;
    __device__ __forceinline__ LongVec(int64_t D, int v) {
        at = row_vec_at<T>(D, v);
        skip = (int)((int64_t)v * Elem<T>::kVec - at);
    }
    __device__ __forceinline__ bool counts(int k) const { return k >= skip; }
};
template <typename T>
__device__ __forceinline__ void load_long(const T* row, int64_t D, int v, float (&x)[Elem<T>::kVec]) {
    Elem<T>::cvt(row_load(row, D, v), x);
}
template <typename T>
__device__ __forceinline__ void load_param_long(const Args& p, const void* a, float fill, int64_t at,
                                                float (&v)[Elem<T>::kVec]) {
#pragma unroll
    for (int k = 0; k < Elem<T>::kVec; ++k) v[k] = fill;
    if (a) load_param_at<T>(p, a, at, v);
}

template <typename T>
__global__ __launch_bounds__(kLong) void fwd_long(Args p) {
    constexpr int VE = Elem<T>::kVec;
    __builtin_assume(p.D >= VE);  // more than 1024 vectors
    __shared__ float sh1[kLong / 64][1], sh2[kLong / 64][2];
    const float inv = 1.0f / (float)p.D;
    const int nvec = row_vectors<T>(p.D);
    for (int64_t r = blockIdx.x; r < p.rows; r += p.blocks) {
        const T* row = static_cast<const T*>(p.x) + r * p.ldx;
        float d[2], x[VE], w[VE], b[VE];
        const auto sum = [&](float f) {
            float o[1] = {};
            for (int v = threadIdx.x; v < nvec; v += kLong) {
                const LongVec<T> at(p.D, v);
                load_long(row, p.D, v, x);
#pragma unroll
                for (int k = 0; k < VE; ++k)
                    if (at.counts(k)) o[0] += x[k] * f;
            }
            row_sum<kLong>(o, sh1);
            return o[0];
        };
        const auto sums = [&](float m0, float f, float (&o)[2]) {
            o[0] = o[1] = 0.0f;
            for (int v = threadIdx.x; v < nvec; v += kLong) {
                const LongVec<T> at(p.D, v);
                load_long(row, p.D, v, x);
#pragma unroll
                for (int k = 0; k < VE; ++k)
                    if (at.counts(k)) {
                        const float c = (x[k] - m0) * f;
                        o[0] += c;
                        o[1] = __builtin_fmaf(c, c, o[1]);
                    }
            }
            row_sum<kLong>(o, sh2);
        };
        float m0 = sum(1.0f) * inv;
        if (!finite(m0)) m0 = row_mean_wide(inv, sum);
        sums(m0, 1.0f, d);
        f32x4 st = row_stats(m0, d[0] * inv, d[1] * inv, p.eps);
        if (!row_stats_hold(d, inv)) st = row_stats_wide(m0, inv, p.eps, d, sums, [](float, float) {});
        if (p.stats && threadIdx.x == 0) p.stats[r] = st;
        for (int v = threadIdx.x; v < nvec; v += kLong) {
            const LongVec<T> at(p.D, v);
            load_long(row, p.D, v, x);
            load_param_long<T>(p, p.w, 1.0f, at.at, w);
            load_param_long<T>(p, p.b, 0.0f, at.at, b);
#pragma unroll
            for (int k = 0; k < VE; ++k) x[k] = __builtin_fmaf(__builtin_fmaf(x[k] - st[0], st[2], st[1]), w[k], b[k]);
            row_store(static_cast<T*>(p.y) + r * p.D, p.D, v, pack_vec<T>(x));
        }
    }
}

// dx of such rows; their dw and db take another kernel, columns at a time.
template <typename T>
__global__ __launch_bounds__(kLong) void dx_long(Args p) {
    constexpr int VE = Elem<T>::kVec;
    __builtin_assume(p.D >= VE);  // more than 1024 vectors
    __shared__ float sh2[kLong / 64][2];
    const float inv = 1.0f / (float)p.D;
    const int nvec = row_vectors<T>(p.D);
    for (int64_t r = blockIdx.x; r < p.rows; r += p.blocks) {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx;
        const T* g = static_cast<const T*>(p.g) + r * p.ldg;
        const f32x4 st = p.stats[r];
        float s[2] = {}, h[VE], a[VE], w[VE];
        for (int v = threadIdx.x; v < nvec; v += kLong) {
            const LongVec<T> at(p.D, v);
            load_long(x, p.D, v, h);
            load_long(g, p.D, v, a);
            load_param_long<T>(p, p.w, 1.0f, at.at, w);
#pragma unroll
            for (int k = 0; k < VE; ++k)
                if (at.counts(k)) {
                    s[0] = __builtin_fmaf(a[k], w[k], s[0]);
                    s[1] = __builtin_fmaf(a[k] * w[k], __builtin_fmaf(h[k] - st[0], st[2], st[1]), s[1]);
                }
        }
        row_sum<kLong>(s, sh2);
        const float c0 = -st[2] * (s[0] * inv), c1 = -st[2] * (s[1] * inv);
        for (int v = threadIdx.x; v < nvec; v += kLong) {
            const LongVec<T> at(p.D, v);
            load_long(x, p.D, v, h);
            load_long(g, p.D, v, a);
            load_param_long<T>(p, p.w, 1.0f, at.at, w);
#pragma unroll
            for (int k = 0; k < VE; ++k)
                a[k] = __builtin_fmaf(__builtin_fmaf(h[k] - st[0], st[2], st[1]), c1,
                                      __builtin_fmaf(a[k] * w[k], st[2], c0));
            row_store(static_cast<T*>(p.y) + r * p.D, p.D, v, pack_vec<T>(a));
        }
    }
}

// A group's rows of 64 vectors of columns: sums of g h and of g, over the waves; the
// groups' are joined as blocks' are.  A wave has one row's loads in flight, as the
// others fill the memory: (16384, 16384) in bf16 184 us, 218 with two or more.
template <typename T>
__global__ __launch_bounds__(256) void columns_long(Args p) {
    constexpr int VE = Elem<T>::kVec;
    __builtin_assume(p.D >= VE);  // more than 1024 vectors
    __shared__ float sh[2][4][64 * VE];
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int v = (int)blockIdx.x * 64 + lane;
    const bool live = v < row_vectors<T>(p.D);
    const LongVec<T> at(p.D, live ? v : 0);
    float dw[VE] = {}, db[VE] = {};
    if (live) {
#pragma unroll 1
        for (int64_t r = (int64_t)blockIdx.y * 4 + wave; r < p.rows; r += (int64_t)gridDim.y * 4) {
            float x[VE], g[VE];
            load_long(static_cast<const T*>(p.x) + r * p.ldx, p.D, v, x);
            load_long(static_cast<const T*>(p.g) + r * p.ldg, p.D, v, g);
            const f32x4 st = p.stats[r];
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                dw[k] = __builtin_fmaf(g[k], __builtin_fmaf(x[k] - st[0], st[2], st[1]), dw[k]);
                db[k] += g[k];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < VE; ++k) {
        sh[0][wave][lane * VE + k] = dw[k];
        sh[1][wave][lane * VE + k] = db[k];
    }
    __syncthreads();
    if (wave > 1 || !live) return;
    float* part = p.part + ((int64_t)blockIdx.y * 2 + wave) * p.D + at.at;
#pragma unroll
    for (int k = 0; k < VE; ++k) {
        float s = sh[wave][0][lane * VE + k];
#pragma unroll
        for (int q = 1; q < 4; ++q) s += sh[wave][q][lane * VE + k];
        if (at.counts(k)) part[k] = s;
    }
}

// Joins the blocks' sums: 32 columns a block, 32 runs of blocks each.
constexpr int kJoinCols = 32, kJoinRuns = 32;
template <typename T>
__global__ __launch_bounds__(kJoinCols * kJoinRuns) void join_kernel(const float* part, int blocks, int64_t D,
                                                                    void* dw, void* db, bool f32) {
    __shared__ float sh[kJoinRuns][kJoinCols];
    const int col = (int)threadIdx.x % kJoinCols, run = (int)threadIdx.x / kJoinCols;
    const int64_t c = (int64_t)blockIdx.x * kJoinCols + col;
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    float s = 0.0f;
    if (c < D)
#pragma unroll 8
        for (int b = run; b < blocks; b += kJoinRuns) s += part[((int64_t)b * 2 + blockIdx.y) * D + c];
    sh[run][col] = s;
    __syncthreads();
    if (run == 0 && c < D) {
#pragma unroll
        for (int k = 1; k < kJoinRuns; ++k) s += sh[k][col];
        if (f32) static_cast<float*>(out)[c] = s;
        else Elem<T>::put(static_cast<T*>(out) + c, s);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check(const char* name, int64_t rows, int64_t D, int64_t ldx, int dtype) {
    FL_CHECK(rows >= 0 && D >= 1, "%s: bad shape (rows=%lld, D=%lld)", name, (long long)rows, (long long)D);
    FL_CHECK(dtype >= 0 && dtype <= 2, "%s: dtype %d", name, dtype);
    FL_CHECK(ldx >= D, "%s: rows of x overlap", name);
    if (rows > ((int64_t)1 << 31) - 1 || D > (1 << 24))
        return set_error(FL_ERANGE, "%s: at most 2^31 - 1 rows and 2^24 columns", name);
    return ok();
}

bool aligned(const void* p, int size) { return (reinterpret_cast<uintptr_t>(p) & (unsigned)(size - 1)) == 0; }
int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

// Lanes a row and vectors a lane, the fewest lanes that hold it in four vectors each;
// lanes 1: the row is one vector or less, 0: longer than a block holds.
struct Plan {
    int lanes, nv, rows;  // rows a block at once
};
Plan plan(int64_t D, int dtype) {
    const int64_t vecs = (D * elem_size(dtype) + 15) / 16;
    if (D * elem_size(dtype) <= 16) return {1, 1, kShort};
    if (vecs <= 8) return {8, 1, 32};
    if (vecs <= 16) return {16, 1, 16};
    if (vecs <= 32) return {32, 1, 8};
    if (vecs <= 64) return {64, 1, 4};
    if (vecs <= 128) return {64, 2, 4};
    if (vecs <= 256) return {64, 4, 4};
    if (vecs <= 512) return {256, 2, 1};
    if (vecs <= 1024) return {256, 4, 1};
    if (vecs <= 2048) return {1024, 2, 1};
    if (vecs <= 4096) return {1024, 4, 1};
    return {0, 0, 1};
}
int block_count(int64_t rows, const Plan& q, int most) {
    const int64_t want = (rows + q.rows - 1) / q.rows;
    return (int)(want < most ? want : most);
}
// Blocks of a forward: with ever more, short-lived ones memory is walked in order,
// which takes less time until a block's parameters cost as much as its rows: (65536,
// 4096) in bf16 209 us with 1024 blocks, 190 with 8192, 246 with one a row.
int fwd_blocks(int64_t rows, const Plan& q) { return block_count(rows, q, q.lanes > 256 ? 1024 : 8192); }
// Blocks of a backward, each with its sums to join: as many as are at work at
// once.  With four vectors a lane that is one a CU: (32768, 4096) in fp32 269 us for
// 276 with two, but (65536, 4096) in bf16, two vectors, 314 for 281.
int bwd_blocks(int64_t rows, const Plan& q) { return block_count(rows, q, q.nv >= 4 ? 256 : 512); }

// Rows too long for the backward's registers: groups of rows whose columns a block
// sums, about four blocks a CU in all.
int column_tiles(int64_t D, int dtype) { return (int)((D * elem_size(dtype) + 1023) / 1024); }
int row_groups(int64_t rows, int64_t D, int dtype) {
    const int64_t most = (rows + 15) / 16, want = (1024 + column_tiles(D, dtype) - 1) / column_tiles(D, dtype);
    return (int)(want < most ? want : most);
}
// Rows of more than 256 lanes: a block of 1024 threads holds no sums beside them
// ((16384, 16384) in bf16 950 us, spilling, for 448), and past 16 columns a lane not
// even the rows ((8192, 20000) 375 us for dx, 233 where they are read again).
bool bwd_long_rows(const Plan& q) { return q.lanes == 0 || q.lanes > 256; }
constexpr int kBwdColumns = 16384;
int bwd_columns(const Plan& q, int dtype) { return q.lanes * q.nv * 16 / elem_size(dtype); }

template <typename T, bool WHOLE, typename F>
void by_plan(const Plan& q, F f) {
#define FL_CASE(L, N) \
    if (q.lanes == L && q.nv == N) \
    return f(T{}, std::integral_constant<int, L>{}, std::integral_constant<int, N>{}, std::bool_constant<WHOLE>{})
    FL_CASE(8, 1);
    FL_CASE(16, 1);
    FL_CASE(32, 1);
    FL_CASE(64, 1);
    FL_CASE(64, 2);
    FL_CASE(64, 4);
    FL_CASE(256, 2);
    FL_CASE(256, 4);
    FL_CASE(1024, 2);
    FL_CASE(1024, 4);
#undef FL_CASE
}
template <typename F>
void by_type(int dtype, F f) {
    if (dtype == 0) f(float{});
    else if (dtype == 1) f(_Float16{});
    else f(bf16_t{});
}
template <typename F>
void by_shape(const Plan& q, int64_t D, int dtype, F f) {
    by_type(dtype, [&](auto t) {
        if (D % (16 / elem_size(dtype)) == 0) by_plan<decltype(t), true>(q, f);
        else by_plan<decltype(t), false>(q, f);
    });
}

}  // namespace
}  // namespace layer_norm
}  // namespace fl

using namespace fl;
using namespace fl::layer_norm;

extern "C" int fl_layer_norm_fwd(const void* x, int64_t row_stride, int64_t rows, int64_t D, int dtype,
                                 const void* weight, const void* bias, int params_dtype, float eps, void* y,
                                 float* stats, void* stream) {
    const char* name = "fl_layer_norm_fwd";
    const int rc = check(name, rows, D, row_stride, dtype);
    if (rc != FL_OK || rows == 0) return rc;
    FL_CHECK(eps >= 0.0f, "%s: eps has to be at least 0", name);
    FL_CHECK(params_dtype == 0 || params_dtype == dtype, "%s: parameters' dtype %d", name, params_dtype);
    FL_CHECK(x && y, "%s: NULL pointer argument", name);
    const int ps = elem_size(params_dtype), es = elem_size(dtype);
    FL_CHECK(aligned(x, es) && aligned(y, es) && aligned(weight, ps) && aligned(bias, ps) && aligned(stats, 16),
             "%s: pointers are not element-aligned, or stats not 16-byte aligned", name);
    const Plan q = plan(D, dtype);
    Args a{};
    a.x = x;
    a.ldx = row_stride;
    a.rows = rows;
    a.D = D;
    a.w = weight;
    a.b = bias;
    a.params_f32 = params_dtype == 0;
    a.eps = eps;
    a.y = y;
    a.stats = reinterpret_cast<f32x4*>(stats);
    a.blocks = fwd_blocks(rows, q);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (q.lanes == 0) {
        by_type(dtype, [&](auto t) { fwd_long<decltype(t)><<<(unsigned)a.blocks, kLong, 0, s>>>(a); });
        return launch_status(name);
    }
    if (q.lanes == 1) {
        by_type(dtype, [&](auto t) { fwd_short<decltype(t)><<<(unsigned)a.blocks, kShort, 0, s>>>(a); });
        return launch_status(name);
    }
    by_shape(q, D, dtype, [&](auto t, auto lanes, auto nv, auto whole) {
        constexpr int L = decltype(lanes)::value;
        fwd_kernel<decltype(t), L, decltype(nv)::value, decltype(whole)::value>
            <<<(unsigned)a.blocks, Shape<L>::kThreads, 0, s>>>(a);
    });
    return launch_status(name);
}

extern "C" size_t fl_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t D, int dtype) {
    if (rows < 0 || D < 1 || D > (1 << 24) || dtype < 0 || dtype > 2) return 0;
    const Plan q = plan(D, dtype);
    return (size_t)(bwd_long_rows(q) ? row_groups(rows, D, dtype) : bwd_blocks(rows, q)) * 2 * (size_t)D * 4;
}

extern "C" int fl_layer_norm_bwd(const void* grad, int64_t grad_stride, const void* x, int64_t row_stride, int64_t rows,
                                 int64_t D, int dtype, const void* weight, int params_dtype, const float* stats,
                                 void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    const char* name = "fl_layer_norm_bwd";
    const int rc = check(name, rows, D, row_stride, dtype);
    if (rc != FL_OK) return rc;
    FL_CHECK(grad_stride >= D, "%s: rows of grad overlap", name);
    FL_CHECK(params_dtype == 0 || params_dtype == dtype, "%s: parameters' dtype %d", name, params_dtype);
    FL_CHECK(rows == 0 || (grad && x && stats), "%s: NULL pointer argument", name);
    const int ps = elem_size(params_dtype), es = elem_size(dtype);
    FL_CHECK(aligned(x, es) && aligned(grad, es) && aligned(dx, es) && aligned(weight, ps) && aligned(dweight, ps) &&
                 aligned(dbias, ps) && aligned(stats, 16),
             "%s: pointers are not element-aligned, or stats not 16-byte aligned", name);
    const bool params = dweight || dbias;
    const size_t need = params ? fl_layer_norm_bwd_workspace_bytes(rows, D, dtype) : 0;
    FL_CHECK(workspace_bytes >= need, "%s: workspace of %llu bytes, %llu needed", name,
             (unsigned long long)workspace_bytes, (unsigned long long)need);
    FL_CHECK(need == 0 || (workspace && aligned(workspace, 4)), "%s: workspace is not 4-byte aligned", name);
    if (!dx && !params) return ok();
    const Plan q = plan(D, dtype);
    Args a{};
    a.x = x;
    a.ldx = row_stride;
    a.rows = rows;
    a.D = D;
    a.w = weight;
    a.params_f32 = params_dtype == 0;
    a.y = dx;
    a.stats = const_cast<f32x4*>(reinterpret_cast<const f32x4*>(stats));
    a.g = grad;
    a.ldg = grad_stride;
    a.part = params ? static_cast<float*>(workspace) : nullptr;
    const bool lng = bwd_long_rows(q);
    const int groups = row_groups(rows, D, dtype);
    a.blocks = lng ? block_count(rows, q, 1024) : bwd_blocks(rows, q);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (rows > 0 && (q.lanes == 0 || bwd_columns(q, dtype) > kBwdColumns)) {
        if (dx) by_type(dtype, [&](auto t) { dx_long<decltype(t)><<<(unsigned)a.blocks, kLong, 0, s>>>(a); });
    } else if (rows > 0 && q.lanes == 1) {
        by_type(dtype, [&](auto t) { bwd_short<decltype(t)><<<(unsigned)a.blocks, kShort, 0, s>>>(a); });
    } else if (rows > 0 && (dx || !lng)) {
        by_shape(q, D, dtype, [&](auto t, auto lanes, auto nv, auto whole) {
            constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value;
            if constexpr (L * NV * Elem<decltype(t)>::kVec <= kBwdColumns)
                bwd_kernel<decltype(t), L, NV, decltype(whole)::value>
                    <<<(unsigned)a.blocks, Shape<L>::kThreads, 0, s>>>(a);
        });
    }
    if (rows > 0 && lng && params)
        by_type(dtype, [&](auto t) {
            columns_long<decltype(t)><<<dim3((unsigned)column_tiles(D, dtype), (unsigned)groups), 256, 0, s>>>(a);
        });
    if (params)
        by_type(dtype, [&](auto t) {
            join_kernel<decltype(t)><<<dim3((unsigned)((D + kJoinCols - 1) / kJoinCols), 2), kJoinCols * kJoinRuns, 0, s>>>(
                a.part, lng ? groups : a.blocks, D, dweight, dbias, a.params_f32);
        });
    return launch_status(name);
}

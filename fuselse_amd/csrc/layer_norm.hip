// Layer norm over the last dimension, forward and backward, on gfx950.
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   dx = r (a - mean a - h mean(a h)) with a = g w;  dw = sum_rows g h, db = sum_rows g
//
// A row is held in registers by some lanes of a wave, a block, or, past 4096
// vectors, read again from the caches, so memory sees each operand once.  The
// mean is kept as two numbers: m0, the rounded sum over D, and m1, the mean of
// the differences to it.  x - m0 - m1 then keeps its digits when the row has a
// large value in common, which one fp32 mean would take from it.  Lanes meet the
// same columns in every row and sum dw and db in registers; the blocks' sums are
// joined in their order.
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
    f32x4* stats;  // [rows]: m0, m1, r
    const void* g;
    int64_t ldg;
    float* part;  // [blocks][2][D]: sums of g h and of g
    int blocks;
};

template <typename T>
__device__ __forceinline__ float param(const Args& p, const void* a, int64_t c) {
    return p.params_f32 ? static_cast<const float*>(a)[c] : Elem<T>::scalar(static_cast<const T*>(a) + c);
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

// How a block is laid out for rows of LANES * NV vectors at most.
template <int LANES>
struct Shape {
    static constexpr int kThreads = LANES > 256 ? LANES : 256;
    static constexpr int kRows = kThreads / LANES;
};

// Lane `sub` holds vectors sub, sub + LANES, ..; elements past the row are 0.
template <typename T, int LANES, int NV, bool WHOLE>
__device__ __forceinline__ void load_row(const T* row, int D, int sub, float (&v)[NV][Elem<T>::kVec]) {
    constexpr int VE = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (sub + j * LANES) * VE;
        if constexpr (WHOLE) {
            u32x4 r{0, 0, 0, 0};
            if (c < D) r = load_raw_stream(row + c);
            Elem<T>::cvt(r, v[j]);
        } else {
            load_vec_part<T>(row + c, D - c, 0.0f, v[j]);
        }
    }
}

template <typename T, int LANES, int NV>
__device__ __forceinline__ void load_params(const Args& p, const void* a, float fill, int sub,
                                            float (&v)[NV][Elem<T>::kVec]) {
    constexpr int VE = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) {
            const int c = (sub + j * LANES) * VE + k;
            v[j][k] = a && c < p.D ? param<T>(p, a, c) : fill;
        }
}

template <typename T, int LANES, int NV, bool WHOLE>
__device__ __forceinline__ void store_row(T* row, int D, int sub, const float (&v)[NV][Elem<T>::kVec]) {
    constexpr int VE = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (sub + j * LANES) * VE;
        if (WHOLE ? c < D : c + VE <= D) {
            __builtin_nontemporal_store(pack_vec<T>(v[j]), reinterpret_cast<u32x4_any*>(row + c));
        } else if constexpr (!WHOLE) {
#pragma unroll
            for (int k = 0; k < VE; ++k)
                if (c + k < D) Elem<T>::put(row + c + k, v[j][k]);
        }
    }
}

template <typename T, int LANES, int NV, bool WHOLE>
__global__ __launch_bounds__(Shape<LANES>::kThreads) void fwd_kernel(Args p) {
    constexpr int VE = Elem<T>::kVec;
    __shared__ float sh1[Shape<LANES>::kThreads / 64][1], sh2[Shape<LANES>::kThreads / 64][2];
    const int sub = (int)threadIdx.x % LANES, D = (int)p.D;
    const float inv = 1.0f / (float)D;
    float w[NV][VE], b[NV][VE];
    load_params<T, LANES, NV>(p, p.w, 1.0f, sub, w);
    load_params<T, LANES, NV>(p, p.b, 0.0f, sub, b);
    for (int64_t r = (int64_t)blockIdx.x * Shape<LANES>::kRows + (int)threadIdx.x / LANES; r < p.rows;
         r += (int64_t)p.blocks * Shape<LANES>::kRows) {
        float x[NV][VE];
        load_row<T, LANES, NV, WHOLE>(static_cast<const T*>(p.x) + r * p.ldx, D, sub, x);
        float s[1] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) s[0] += x[j][k];
        row_sum<LANES>(s, sh1);
        const float m0 = s[0] * inv;
        float d[2] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                x[j][k] -= m0;
                if ((sub + j * LANES) * VE + (WHOLE ? 0 : k) < D) {
                    d[0] += x[j][k];
                    d[1] = __builtin_fmaf(x[j][k], x[j][k], d[1]);
                }
            }
        row_sum<LANES>(d, sh2);
        const float m1 = d[0] * inv;
        const float var = d[1] * inv - m1 * m1;
        const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + p.eps);
        if (p.stats && sub == 0) p.stats[r] = f32x4{m0, m1, rstd, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) x[j][k] = __builtin_fmaf((x[j][k] - m1) * rstd, w[j][k], b[j][k]);
        store_row<T, LANES, NV, WHOLE>(static_cast<T*>(p.y) + r * p.D, D, sub, x);
    }
}

template <typename T, int LANES, int NV, bool WHOLE>
__global__ __launch_bounds__(Shape<LANES>::kThreads) void bwd_kernel(Args p) {
    constexpr int VE = Elem<T>::kVec;
    constexpr int ROWS = Shape<LANES>::kRows;
    __shared__ float sh2[Shape<LANES>::kThreads / 64][2];
    const int sub = (int)threadIdx.x % LANES, D = (int)p.D;
    const float inv = 1.0f / (float)D;
    float w[NV][VE], dw[NV][VE] = {}, db[NV][VE] = {};
    load_params<T, LANES, NV>(p, p.w, 1.0f, sub, w);
    for (int64_t r = (int64_t)blockIdx.x * ROWS + (int)threadIdx.x / LANES; r < p.rows;
         r += (int64_t)p.blocks * ROWS) {
        float x[NV][VE], g[NV][VE];
        load_row<T, LANES, NV, WHOLE>(static_cast<const T*>(p.x) + r * p.ldx, D, sub, x);
        load_row<T, LANES, NV, WHOLE>(static_cast<const T*>(p.g) + r * p.ldg, D, sub, g);
        const f32x4 st = p.stats[r];
        const float m0 = st[0], m1 = st[1], rstd = st[2];
        float s[2] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                const float h = (x[j][k] - m0 - m1) * rstd;
                x[j][k] = h;
                if ((sub + j * LANES) * VE + (WHOLE ? 0 : k) < D) {
                    dw[j][k] = __builtin_fmaf(g[j][k], h, dw[j][k]);
                    db[j][k] += g[j][k];
                    g[j][k] *= w[j][k];
                    s[0] += g[j][k];
                    s[1] = __builtin_fmaf(g[j][k], h, s[1]);
                }
            }
        if (!p.y) continue;
        row_sum<LANES>(s, sh2);
        const float c0 = s[0] * inv, c1 = s[1] * inv;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) g[j][k] = rstd * (g[j][k] - c0 - x[j][k] * c1);
        store_row<T, LANES, NV, WHOLE>(static_cast<T*>(p.y) + r * p.D, D, sub, g);
    }
    if (!p.part) return;
    // the block's rows, joined over its groups of lanes in their order
    float* part = p.part + (int64_t)blockIdx.x * 2 * p.D;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                const int c = (sub + j * LANES) * VE + k;
                if (c < D) {
                    part[c] = dw[j][k];
                    part[p.D + c] = db[j][k];
                }
            }
    } else {
        constexpr int W = LANES * NV * VE;
        __shared__ float sum[2][W];
        for (int q = 0; q < ROWS; ++q) {
            if ((int)threadIdx.x / LANES == q) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int k = 0; k < VE; ++k) {
                        const int c = (sub + j * LANES) * VE + k;
                        sum[0][c] = q ? sum[0][c] + dw[j][k] : dw[j][k];
                        sum[1][c] = q ? sum[1][c] + db[j][k] : db[j][k];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < D; c += Shape<LANES>::kThreads) {
            part[c] = sum[0][c];
            part[p.D + c] = sum[1][c];
        }
    }
}

// Rows too long for a block's registers: a block reads the row again from the
// caches for each step.
constexpr int kLong = 1024;
template <typename T>
__global__ __launch_bounds__(kLong) void fwd_long(Args p) {
    __shared__ float sh1[kLong / 64][1], sh2[kLong / 64][2];
    const float inv = 1.0f / (float)p.D;
    for (int64_t r = blockIdx.x; r < p.rows; r += p.blocks) {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx;
        T* y = static_cast<T*>(p.y) + r * p.D;
        float s[1] = {}, d[2] = {};
        for (int64_t c = threadIdx.x; c < p.D; c += kLong) s[0] += Elem<T>::scalar(x + c);
        row_sum<kLong>(s, sh1);
        const float m0 = s[0] * inv;
        for (int64_t c = threadIdx.x; c < p.D; c += kLong) {
            const float v = Elem<T>::scalar(x + c) - m0;
            d[0] += v;
            d[1] = __builtin_fmaf(v, v, d[1]);
        }
        row_sum<kLong>(d, sh2);
        const float m1 = d[0] * inv;
        const float var = d[1] * inv - m1 * m1;
        const float rstd = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + p.eps);
        if (p.stats && threadIdx.x == 0) p.stats[r] = f32x4{m0, m1, rstd, 0.0f};
        for (int64_t c = threadIdx.x; c < p.D; c += kLong) {
            const float w = p.w ? param<T>(p, p.w, c) : 1.0f, b = p.b ? param<T>(p, p.b, c) : 0.0f;
            Elem<T>::put(y + c, __builtin_fmaf((Elem<T>::scalar(x + c) - m0 - m1) * rstd, w, b));
        }
    }
}
template <typename T>
__global__ __launch_bounds__(kLong) void bwd_long(Args p) {
    __shared__ float sh2[kLong / 64][2];
    const float inv = 1.0f / (float)p.D;
    float* part = p.part ? p.part + (int64_t)blockIdx.x * 2 * p.D : nullptr;
    bool first = true;
    for (int64_t r = blockIdx.x; r < p.rows; r += p.blocks, first = false) {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx;
        const T* g = static_cast<const T*>(p.g) + r * p.ldg;
        const f32x4 st = p.stats[r];
        const float m0 = st[0], m1 = st[1], rstd = st[2];
        float s[2] = {};
        for (int64_t c = threadIdx.x; c < p.D; c += kLong) {
            const float h = (Elem<T>::scalar(x + c) - m0 - m1) * rstd, gv = Elem<T>::scalar(g + c);
            if (part) {  // this thread alone meets column c
                part[c] = first ? gv * h : __builtin_fmaf(gv, h, part[c]);
                part[p.D + c] = first ? gv : part[p.D + c] + gv;
            }
            const float a = gv * (p.w ? param<T>(p, p.w, c) : 1.0f);
            s[0] += a;
            s[1] = __builtin_fmaf(a, h, s[1]);
        }
        if (!p.y) continue;
        row_sum<kLong>(s, sh2);
        const float c0 = s[0] * inv, c1 = s[1] * inv;
        T* dx = static_cast<T*>(p.y) + r * p.D;
        for (int64_t c = threadIdx.x; c < p.D; c += kLong) {
            const float h = (Elem<T>::scalar(x + c) - m0 - m1) * rstd;
            const float a = Elem<T>::scalar(g + c) * (p.w ? param<T>(p, p.w, c) : 1.0f);
            Elem<T>::put(dx + c, rstd * (a - c0 - h * c1));
        }
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

// Lanes a row and vectors a lane; lanes 0: the row is longer than a block holds.
struct Plan {
    int lanes, nv, rows;  // rows a block at once
};
Plan plan(int64_t D, int dtype) {
    const int64_t vecs = (D * elem_size(dtype) + 15) / 16;
    if (vecs <= 16) return {16, 1, 16};
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
int fwd_blocks(int64_t rows, const Plan& q) { return block_count(rows, q, 2048); }
int bwd_blocks(int64_t rows, const Plan& q) { return block_count(rows, q, 512); }

template <typename T, bool WHOLE, typename F>
void by_plan(const Plan& q, F f) {
#define FL_CASE(L, N) \
    if (q.lanes == L && q.nv == N) \
    return f(T{}, std::integral_constant<int, L>{}, std::integral_constant<int, N>{}, std::bool_constant<WHOLE>{})
    FL_CASE(16, 1);
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
    by_shape(q, D, dtype, [&](auto t, auto lanes, auto nv, auto whole) {
        constexpr int L = decltype(lanes)::value;
        fwd_kernel<decltype(t), L, decltype(nv)::value, decltype(whole)::value>
            <<<(unsigned)a.blocks, Shape<L>::kThreads, 0, s>>>(a);
    });
    return launch_status(name);
}

extern "C" size_t fl_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t D, int dtype) {
    if (rows < 0 || D < 1 || D > (1 << 24) || dtype < 0 || dtype > 2) return 0;
    return (size_t)bwd_blocks(rows, plan(D, dtype)) * 2 * (size_t)D * 4;
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
    a.blocks = bwd_blocks(rows, q);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (rows > 0) {
        if (q.lanes == 0) {
            by_type(dtype, [&](auto t) { bwd_long<decltype(t)><<<(unsigned)a.blocks, kLong, 0, s>>>(a); });
        } else {
            by_shape(q, D, dtype, [&](auto t, auto lanes, auto nv, auto whole) {
                constexpr int L = decltype(lanes)::value;
                bwd_kernel<decltype(t), L, decltype(nv)::value, decltype(whole)::value>
                    <<<(unsigned)a.blocks, Shape<L>::kThreads, 0, s>>>(a);
            });
        }
    }
    if (params)
        by_type(dtype, [&](auto t) {
            join_kernel<decltype(t)><<<dim3((unsigned)((D + kJoinCols - 1) / kJoinCols), 2), kJoinCols * kJoinRuns, 0, s>>>(
                a.part, a.blocks, D, dweight, dbias, a.params_f32);
        });
    return launch_status(name);
}

// Linear cross entropy on gfx950: the softmax cross entropy of hidden states
// against a vocabulary projection, forward and backward, in pieces of the
// vocabulary and without the logits in memory (formulas: linear_ce.hpp).
//
// Forward: a plan kernel lists the live rows, a packing kernel lays their
// hidden states out, the logits product reduces each of its tiles to a (max,
// sum) pair per row and keeps the target's logit, and a finishing kernel joins
// the pairs.  Backward, per piece of the vocabulary: the logits again, turned
// into G in 16 bits; dx += G w in fp32; dw = G^T x.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/fuselse_amd.h"
#include "fl_status.hpp"
#include "linear_ce.hpp"

namespace fl {
namespace lce {
namespace {

// ---------------------------------------------------------------------------
// Element types
// ---------------------------------------------------------------------------
template <int DT> struct Io;
template <> struct Io<kF32> {
    typedef float T;
    static constexpr int kParts = 3;
    static constexpr bool kHalf = false;
};
template <> struct Io<kF16> {
    typedef _Float16 T;
    static constexpr int kParts = 1;
    static constexpr bool kHalf = true;
};
template <> struct Io<kBF16> {
    typedef bf16_t T;
    static constexpr int kParts = 1;
    static constexpr bool kHalf = false;
};

// A value as its 16-bit matrix operands: exact for x and w; G, computed in
// fp32, is rounded to nearest even in fp16 and bf16 (its share of the error of
// dx and dw is that of one rounding of a term of their sums) and exact in fp32.
template <int DT>
__device__ __forceinline__ void to_parts(float v, uint16_t (&o)[Io<DT>::kParts]) {
    if constexpr (DT == kF32) split3(v, o);
    else if constexpr (DT == kF16) o[0] = __builtin_bit_cast(uint16_t, (_Float16)v);
    else o[0] = __builtin_bit_cast(uint16_t, (__bf16)v);
}

template <bool HALF>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// What the host lays out in the workspace for one call
// ---------------------------------------------------------------------------
struct Head {          // at the workspace's start, written by the plan kernel
    int live;          // rows whose target is not ignore_index
    int pad;
    float inv_scale;   // undoes the power of two that a and b carry
    float pad2;
};

// ---------------------------------------------------------------------------
// Plan: one block lists the live rows in order, and for the backward their
// coefficients a and b, scaled by a power of two that brings the largest to
// [2^9, 2^10): G in fp16 then loses nothing to its smallest values that a sum
// of its row would show.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int block_scan_excl(int v, int* sh, int* total) {
    const int t = threadIdx.x;
    sh[t] = v;
    __syncthreads();
    for (int d = 1; d < kPlanThreads; d <<= 1) {
        const int add = t >= d ? sh[t - d] : 0;
        __syncthreads();
        sh[t] += add;
        __syncthreads();
    }
    *total = sh[kPlanThreads - 1];
    const int r = sh[t] - v;
    __syncthreads();
    return r;
}

struct PlanArgs {
    const int64_t* target;
    int64_t n, v, ignore;
    Head* head;
    int* rows;    // live row -> row
    int* pos;     // row -> live row, -1 for an ignored one
    int* tgt;     // live row -> target, -1 for one outside [0, v)
    // forward: ignored rows' results
    float* loss_rows;
    float* lse_out;
    // backward
    const float* grad;
    int grad_stride;
    const float* lse_in;
    float z;
    int mean;
    float* a;
    float* b;
    float* lse;
};

template <bool BWD>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs p) {
    __shared__ int sh[kPlanThreads];
    const int64_t per = (p.n + kPlanThreads - 1) / kPlanThreads;
    const int64_t r0 = (int64_t)threadIdx.x * per;
    const int64_t r1 = r0 + per < p.n ? r0 + per : p.n;
    int mine = 0;
    for (int64_t r = r0; r < r1; ++r) mine += p.target[r] != p.ignore;
    int live;
    int at = block_scan_excl(mine, sh, &live);
    float big = 0.0f;
    const float mean = p.mean ? 1.0f / (float)(live > 0 ? live : 1) : 1.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const int64_t t = p.target[r];
        if (t == p.ignore) {
            p.pos[r] = -1;
            if constexpr (!BWD) {
                p.loss_rows[r] = 0.0f;
                p.lse_out[r] = 0.0f;
            }
            continue;
        }
        const bool in = t >= 0 && t < p.v;
        p.rows[at] = (int)r;
        p.pos[r] = at;
        p.tgt[at] = in ? (int)t : -1;
        if constexpr (BWD) {
            const float g = p.grad[r * p.grad_stride] * mean;
            const float l = p.lse_in[r];
            const float a = in ? g * (1.0f + 2.0f * p.z * l) : __builtin_nanf("");
            const float b = in ? -g : __builtin_nanf("");
            p.a[at] = a;
            p.b[at] = b;
            p.lse[at] = l;
            big = fmaxf(big, fmaxf(__builtin_fabsf(a), __builtin_fabsf(b)));
        }
        ++at;
    }
    if constexpr (BWD) {
        float* shf = reinterpret_cast<float*>(sh);
        shf[threadIdx.x] = big;
        __syncthreads();
        for (int d = kPlanThreads / 2; d > 0; d >>= 1) {
            if ((int)threadIdx.x < d) shf[threadIdx.x] = fmaxf(shf[threadIdx.x], shf[threadIdx.x + d]);
            __syncthreads();
        }
        big = shf[0];
        int e = 0;
        if (big > 0.0f && __builtin_isfinite(big)) {
            e = 10 - (__builtin_amdgcn_frexp_expf(big));
            e = e < -100 ? -100 : e > 100 ? 100 : e;
        }
        const float scale = __builtin_ldexpf(1.0f, e);
        if (threadIdx.x == 0) p.head->inv_scale = __builtin_ldexpf(1.0f, -e);
        at = at - mine;
        for (int k = 0; k < mine; ++k) {
            p.a[at + k] *= scale;
            p.b[at + k] *= scale;
        }
    }
    if (threadIdx.x == 0) p.head->live = live;
}

// ---------------------------------------------------------------------------
// Packing: rows of x (the live ones) or w as 16-bit operands of ldp elements,
// zero beyond D, and transposed with rows up to a multiple of 64 (zero beyond
// the last).
// ---------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ float load1(const typename Io<DT>::T* p) {
    return Elem<typename Io<DT>::T>::scalar(p);
}

template <int DT>
__global__ __launch_bounds__(256) void pack_rows(const typename Io<DT>::T* src, int64_t lds_, int64_t d, const int* rows,
                                                 const int* live, int64_t n, uint16_t* dst, int64_t ldp,
                                                 int64_t part) {
    const int64_t total = live ? *live : n;
    const int64_t r = blockIdx.x;
    if (r >= total) return;
    const typename Io<DT>::T* s = src + (rows ? (int64_t)rows[r] : r) * lds_;
    for (int64_t c = threadIdx.x; c < ldp; c += 256) {
        uint16_t o[Io<DT>::kParts];
        to_parts<DT>(c < d ? load1<DT>(s + c) : 0.0f, o);
#pragma unroll
        for (int k = 0; k < Io<DT>::kParts; ++k) dst[k * part + r * ldp + c] = o[k];
    }
}

// dst[c][r] for rows r of src, r up to ldp (zero past the last row)
template <int DT>
__global__ __launch_bounds__(256) void pack_cols(const typename Io<DT>::T* src, int64_t lds_, int64_t d, const int* rows,
                                                 const int* live, int64_t n, uint16_t* dst, int64_t ldp,
                                                 int64_t part) {
    __shared__ float tile[64][65];
    const int64_t total = live ? *live : n;
    const int64_t rb = (int64_t)blockIdx.x * 64, cb = (int64_t)blockIdx.y * 64;
    if (rb >= ((total + 63) & ~(int64_t)63)) return;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int i = ty; i < 64; i += 4) {
        const int64_t r = rb + i, c = cb + tx;
        tile[i][tx] = r < total && c < d ? load1<DT>(src + (rows ? (int64_t)rows[r] : r) * lds_ + c) : 0.0f;
    }
    __syncthreads();
    for (int i = ty; i < 64; i += 4) {
        const int64_t c = cb + i, r = rb + tx;
        if (c < d && r < ldp) {
            uint16_t o[Io<DT>::kParts];
            to_parts<DT>(tile[tx][i], o);
#pragma unroll
            for (int k = 0; k < Io<DT>::kParts; ++k) dst[k * part + c * ldp + r] = o[k];
        }
    }
}

// ---------------------------------------------------------------------------
// The product: C[m][n] = sum_k A[m][k] B[n][k] for a 128 x 128 tile in four
// waves of 64 x 64, K in steps of 32 through LDS.
// ---------------------------------------------------------------------------
constexpr int kTile = 128;
constexpr int kStep = 32;
constexpr int kThreads = 256;
constexpr int kLdsRow = kStep + 8;  // 16-bit elements a row, off the banks' period

struct Tile {
    f32x4 acc[4][4];
};

template <bool HALF, int PARTS>
__device__ __forceinline__ void tile_product(const Operand& A, const Operand& B, int64_t m0, int64_t n0, int64_t k0,
                                             int64_t k1, Tile& t, uint16_t (*sa)[kLdsRow], uint16_t (*sb)[kLdsRow]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) t.acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int lr = threadIdx.x >> 2, lc = (threadIdx.x & 3) * 8;
    for (int term = 0; term < (PARTS == 3 ? kTerms : 1); ++term) {
        const uint16_t* pa = A.p + (PARTS == 3 ? kTermA[term] * A.part : 0);
        const uint16_t* pb = B.p + (PARTS == 3 ? kTermB[term] * B.part : 0);
        for (int64_t k = k0; k < k1; k += kStep) {
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = lr + h * 64;
                const int64_t ra = m0 + r < A.rows ? m0 + r : A.rows - 1;
                const int64_t rb = n0 + r < B.rows ? n0 + r : B.rows - 1;
                *reinterpret_cast<u32x4*>(&sa[r][lc]) = *reinterpret_cast<const u32x4*>(pa + ra * A.ld + k + lc);
                *reinterpret_cast<u32x4*>(&sb[r][lc]) = *reinterpret_cast<const u32x4*>(pb + rb * B.ld + k + lc);
            }
            __syncthreads();
            u32x4 fa[4], fb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                fa[i] = *reinterpret_cast<const u32x4*>(&sa[wm + i * 16 + (lane & 15)][(lane >> 4) * 8]);
                fb[i] = *reinterpret_cast<const u32x4*>(&sb[wn + i * 16 + (lane & 15)][(lane >> 4) * 8]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) t.acc[i][j] = mfma<HALF>(fa[i], fb[j], t.acc[i][j]);
        }
    }
}

// acc[i][j][q] of a lane is C[m0 + wm + 16 i + 4 (lane / 16) + q][n0 + wn + 16 j + lane % 16].

struct StatArgs {
    Operand w, x;      // M: vocabulary rows, N: live rows
    int64_t k;
    const Head* head;
    const int* tgt;
    int64_t v0, v;     // the piece's first row, and its rows
    int64_t tiles_n;
    float2* part;      // [live row][parts]: (max, sum)
    int64_t parts;
    float* at_target;  // [live row]
};

template <int DT>
__global__ __launch_bounds__(kThreads) void logits_stats(StatArgs p) {
    __shared__ uint16_t sa[kTile][kLdsRow], sb[kTile][kLdsRow];
    const int live = p.head->live;
    const int64_t n0 = (blockIdx.x % p.tiles_n) * kTile, m0 = (blockIdx.x / p.tiles_n) * kTile;
    if (n0 >= live) return;
    p.x.rows = live;
    Tile t;
    tile_product<Io<DT>::kHalf, Io<DT>::kParts>(p.w, p.x, m0, n0, 0, p.k, t, sa, sb);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t mw = m0 + (wave & 1) * 64, nw = n0 + (wave >> 1) * 64;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t n = nw + j * 16 + (lane & 15);
        const int target = n < live ? p.tgt[n] : -1;
        float v[16];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t m = mw + i * 16 + (lane >> 4) * 4 + q;
                v[i * 4 + q] = m < p.v ? t.acc[i][j][q] : -kInf;
                if (p.v0 + m == target && m < p.v) p.at_target[n] = t.acc[i][j][q];
            }
        float m = -kInf, s = 0.0f;
        lse_fold<true>(m, s, v);
        lse_merge(m, s, exact_xor<16>(m), exact_xor<16>(s));
        lse_merge(m, s, exact_xor<32>(m), exact_xor<32>(s));
        if (lane < 16 && n < live && mw < p.v) p.part[n * p.parts + mw / 64] = make_float2(m, s);
    }
}

// Joins a live row's pairs; one wave a row.
__global__ __launch_bounds__(256) void finish_rows(const Head* head, const int* rows, const int* tgt,
                                                   const float2* part, int64_t parts, const float* at_target, float z,
                                                   float* loss_rows, float* lse_out) {
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= head->live) return;
    const int lane = threadIdx.x & 63;
    float m = -kInf, s = 0.0f;
    for (int64_t k = lane; k < parts; k += 64) {
        const float2 q = part[r * parts + k];
        lse_merge(m, s, q.x, q.y);
    }
    group_merge<64>(m, s);
    if (lane == 0) {
        const float lse = lse_finish<true>(m, s);
        const int row = rows[r];
        lse_out[row] = lse;
        loss_rows[row] = tgt[r] >= 0 ? lse - at_target[r] + z * lse * lse : __builtin_nanf("");
    }
}

// Sum of the rows' losses in a fixed order, over the live rows' number for the mean.
__global__ __launch_bounds__(1024) void reduce_rows(const Head* head, const float* rows, int64_t n, int mean,
                                                    float* out) {
    __shared__ double sh[1024];
    double s = 0.0;
    for (int64_t r = threadIdx.x; r < n; r += 1024) s += rows[r];
    sh[threadIdx.x] = s;
    __syncthreads();
    for (int d = 512; d > 0; d >>= 1) {
        if ((int)threadIdx.x < d) sh[threadIdx.x] += sh[threadIdx.x + d];
        __syncthreads();
    }
    if (threadIdx.x == 0) *out = (float)(mean ? sh[0] / (head->live > 0 ? head->live : 1) : sh[0]);
}

struct GradArgs {
    Operand w, x;
    int64_t k;
    const Head* head;
    const int* tgt;
    const float *a, *b, *lse;
    int64_t v0, v;       // the piece: vocabulary rows v0 .. v - 1 are w's rows 0 ..
    int64_t tiles_n;
    uint16_t* g;         // [live row][ldg]
    int64_t ldg, g_part;
    uint16_t* gt;        // [piece row][ldt]
    int64_t ldt, gt_part;
};

template <int DT>
__global__ __launch_bounds__(kThreads) void logits_grad(GradArgs p) {
    __shared__ uint16_t sa[kTile][kLdsRow], sb[kTile][kLdsRow];
    constexpr int P = Io<DT>::kParts;
    const int live = p.head->live;
    const int64_t n0 = (blockIdx.x % p.tiles_n) * kTile, m0 = (blockIdx.x / p.tiles_n) * kTile;
    if (n0 >= live) return;
    p.x.rows = live;
    Tile t;
    tile_product<Io<DT>::kHalf, P>(p.w, p.x, m0, n0, 0, p.k, t, sa, sb);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t mw = m0 + (wave & 1) * 64, nw = n0 + (wave >> 1) * 64;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t n = nw + j * 16 + (lane & 15);
        const bool in = n < live;
        const int target = in ? p.tgt[n] : -1;
        const float a = in ? p.a[n] : 0.0f, b = in ? p.b[n] : 0.0f, lse = in ? p.lse[n] : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = mw + i * 16 + (lane >> 4) * 4;
            uint16_t o[4][P];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float g = a * fexp2((t.acc[i][j][q] - lse) * kLog2e);
                if (p.v0 + m + q == target) g += b;
                to_parts<DT>(in && p.v0 + m + q < p.v ? g : 0.0f, o[q]);
            }
#pragma unroll
            for (int k = 0; k < P; ++k) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (n < p.ldt && m + q < p.v - p.v0) p.gt[k * p.gt_part + (m + q) * p.ldt + n] = o[q][k];
                }
                if (in && m < p.ldg) {
                    uint2 u;
                    u.x = o[0][k] | (uint32_t)o[1][k] << 16;
                    u.y = o[2][k] | (uint32_t)o[3][k] << 16;
                    *reinterpret_cast<uint2*>(p.g + k * p.g_part + n * p.ldg + m) = u;
                }
            }
        }
    }
}

struct ProductArgs {
    Operand a, b;       // M and N rows
    const Head* head;
    int64_t k;          // depth; with `live_k`, the live rows up to a multiple of 32
    int live_k, live_n;
    int64_t m, n, tiles_m;
    int splits;
    float* acc;         // [split][n][ldc] fp32 sums, added to when `add`
    int64_t ldc, split_stride;
    int add;
    void* out;          // [n][ldc] results
};

template <int DT, bool FINAL>
__global__ __launch_bounds__(kThreads) void product(ProductArgs p) {
    __shared__ uint16_t sa[kTile][kLdsRow], sb[kTile][kLdsRow];
    const int live = p.head->live;
    const int64_t m0 = (blockIdx.x % p.tiles_m) * kTile, n0 = (blockIdx.x / p.tiles_m) * kTile;
    const int split = blockIdx.y;
    const int64_t n_end = p.live_n ? live : p.n;
    if (n0 >= n_end) return;
    if (p.live_n) p.b.rows = live;
    const int64_t depth = p.live_k ? (int64_t)((live + kStep - 1) & ~(kStep - 1)) : p.k;
    const int64_t per = ((depth + p.splits - 1) / p.splits + kStep - 1) & ~(int64_t)(kStep - 1);
    const int64_t k0 = split * per;
    const int64_t k1 = k0 + per < depth ? k0 + per : depth;
    Tile t;
    tile_product<Io<DT>::kHalf, Io<DT>::kParts>(p.a, p.b, m0, n0, k0, k1, t, sa, sb);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t mw = m0 + (wave & 1) * 64, nw = n0 + (wave >> 1) * 64;
    typedef typename Io<DT>::T T;
    const float inv = p.head->inv_scale;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t n = nw + j * 16 + (lane & 15);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int64_t m = mw + i * 16 + (lane >> 4) * 4 + q;
                if (m < p.m && n < n_end) {
                    if constexpr (FINAL) {
                        Elem<T>::put(static_cast<T*>(p.out) + n * p.ldc + m, t.acc[i][j][q] * inv);
                    } else {
                        float* c = p.acc + split * p.split_stride + n * p.ldc + m;
                        *c = p.add ? *c + t.acc[i][j][q] : t.acc[i][j][q];
                    }
                }
            }
        }
}

// dx rows from the splits' sums; ignored rows are zero.
template <int DT>
__global__ __launch_bounds__(256) void finish_dx(const Head* head, const int* pos, const float* acc, int splits,
                                                 int64_t split_stride, int64_t d, void* dx) {
    typedef typename Io<DT>::T T;
    const int64_t r = blockIdx.x;
    const int at = pos[r];
    const float inv = head->inv_scale;
    for (int64_t c = threadIdx.x; c < d; c += 256) {
        float s = 0.0f;
        if (at >= 0) {
            for (int k = 0; k < splits; ++k) s += acc[k * split_stride + at * d + c];
            s *= inv;
        }
        Elem<T>::put(static_cast<T*>(dx) + r * d + c, s);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
constexpr int64_t div_up(int64_t v, int64_t by) { return (v + by - 1) / by; }

struct Layout {
    int64_t piece;       // vocabulary rows of a piece
    int64_t ldx;         // packed row of x and w
    int64_t ldn;         // transposed rows: live rows
    int64_t ldv;         // transposed rows: piece rows
    int splits;
    int64_t head, rows, pos, tgt, at_target, loss_rows, part, parts, a, b, lse, xp, xt, wp, wt, g, gt, acc, bytes;
};

int parts_of(int dtype) { return dtype == kF32 ? 3 : 1; }

Layout layout(int64_t N, int64_t V, int64_t D, int dtype, bool bwd) {
    Layout l{};
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    const int64_t parts = parts_of(dtype);
    l.piece = V < 16384 ? round_up(V, 64) : 16384;
    l.ldx = round_up(D, 64);
    l.ldn = round_up(N, 64);
    l.ldv = l.piece;
    l.head = take(sizeof(Head));
    l.rows = take(4 * N);
    l.pos = take(4 * N);
    l.tgt = take(4 * N);
    l.xp = take(2 * parts * N * l.ldx);
    l.wp = take(2 * parts * l.piece * l.ldx);
    if (!bwd) {
        l.parts = div_up(V, 64);
        l.at_target = take(4 * N);
        l.loss_rows = take(4 * N);
        l.part = take(8 * N * l.parts);
    } else {
        l.a = take(4 * N);
        l.b = take(4 * N);
        l.lse = take(4 * N);
        l.splits = 4;
        l.xt = take(2 * parts * D * l.ldn);
        l.wt = take(2 * parts * D * l.ldv);
        l.g = take(2 * parts * N * l.ldv);
        l.gt = take(2 * parts * l.piece * l.ldn);
        l.acc = take(4 * l.splits * N * D);
    }
    l.bytes = at;
    return l;
}

struct Call {
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t ldw;
    const int64_t* target;
    int64_t N, V, D;
    int64_t ignore;
    float z;
    int reduction;
    char* ws;
    hipStream_t s;
};

template <typename P>
P* at(const Call& c, int64_t off) {
    return reinterpret_cast<P*>(c.ws + off);
}

template <int DT>
Operand pack_w(const Call& c, const Layout& l, int64_t v0, int64_t rows) {
    typedef typename Io<DT>::T T;
    const int64_t part = l.piece * l.ldx;
    pack_rows<DT><<<dim3((unsigned)rows), 256, 0, c.s>>>(static_cast<const T*>(c.w) + v0 * c.ldw, c.ldw, c.D, nullptr,
                                                         nullptr, rows, at<uint16_t>(c, l.wp), l.ldx, part);
    return Operand{at<uint16_t>(c, l.wp), l.ldx, part, (int)rows};
}

template <int DT>
Operand pack_x(const Call& c, const Layout& l) {
    typedef typename Io<DT>::T T;
    const Head* head = at<Head>(c, l.head);
    const int64_t part = c.N * l.ldx;
    pack_rows<DT><<<dim3((unsigned)c.N), 256, 0, c.s>>>(static_cast<const T*>(c.x), c.ldx, c.D, at<int>(c, l.rows),
                                                        &head->live, c.N, at<uint16_t>(c, l.xp), l.ldx, part);
    return Operand{at<uint16_t>(c, l.xp), l.ldx, part, (int)c.N};
}

PlanArgs plan_args(const Call& c, const Layout& l) {
    PlanArgs p{};
    p.target = c.target;
    p.n = c.N;
    p.v = c.V;
    p.ignore = c.ignore;
    p.head = at<Head>(c, l.head);
    p.rows = at<int>(c, l.rows);
    p.pos = at<int>(c, l.pos);
    p.tgt = at<int>(c, l.tgt);
    p.z = c.z;
    p.mean = c.reduction == 2;
    return p;
}

template <int DT>
void run_fwd(const Call& c, float* loss, float* lse) {
    const Layout l = layout(c.N, c.V, c.D, DT, false);
    PlanArgs p = plan_args(c, l);
    p.loss_rows = c.reduction == 0 ? loss : at<float>(c, l.loss_rows);
    p.lse_out = lse;
    plan_kernel<false><<<1, kPlanThreads, 0, c.s>>>(p);
    const Operand x = pack_x<DT>(c, l);
    const int64_t tiles_n = div_up(c.N, kTile);
    for (int64_t v0 = 0; v0 < c.V; v0 += l.piece) {
        const int64_t rows = c.V - v0 < l.piece ? c.V - v0 : l.piece;
        StatArgs a{};
        a.w = pack_w<DT>(c, l, v0, rows);
        a.x = x;
        a.k = l.ldx;
        a.head = p.head;
        a.tgt = p.tgt;
        a.v0 = v0;
        a.v = rows;
        a.tiles_n = tiles_n;
        a.part = at<float2>(c, l.part) + v0 / 64;
        a.parts = l.parts;
        a.at_target = at<float>(c, l.at_target);
        logits_stats<DT><<<dim3((unsigned)(tiles_n * div_up(rows, kTile))), kThreads, 0, c.s>>>(a);
    }
    finish_rows<<<dim3((unsigned)div_up(c.N, 4)), 256, 0, c.s>>>(p.head, p.rows, p.tgt, at<float2>(c, l.part), l.parts,
                                                                 at<float>(c, l.at_target), c.z, p.loss_rows, lse);
    if (c.reduction != 0) reduce_rows<<<1, 1024, 0, c.s>>>(p.head, p.loss_rows, c.N, p.mean, loss);
}

template <int DT>
void run_bwd(const Call& c, const float* grad, const float* lse, void* dx, void* dw) {
    typedef typename Io<DT>::T T;
    const Layout l = layout(c.N, c.V, c.D, DT, true);
    PlanArgs p = plan_args(c, l);
    p.grad = grad;
    p.grad_stride = c.reduction == 0 ? 1 : 0;
    p.lse_in = lse;
    p.a = at<float>(c, l.a);
    p.b = at<float>(c, l.b);
    p.lse = at<float>(c, l.lse);
    plan_kernel<true><<<1, kPlanThreads, 0, c.s>>>(p);
    const Operand x = pack_x<DT>(c, l);
    Operand xt{at<uint16_t>(c, l.xt), l.ldn, c.D * l.ldn, (int)c.D};
    pack_cols<DT><<<dim3((unsigned)(l.ldn / 64), (unsigned)div_up(c.D, 64)), 256, 0, c.s>>>(
        static_cast<const T*>(c.x), c.ldx, c.D, p.rows, &p.head->live, c.N, at<uint16_t>(c, l.xt), l.ldn,
        c.D * l.ldn);
    const int64_t tiles_n = div_up(c.N, kTile), tiles_d = div_up(c.D, kTile);
    for (int64_t v0 = 0; v0 < c.V; v0 += l.piece) {
        const int64_t rows = c.V - v0 < l.piece ? c.V - v0 : l.piece;
        const int64_t depth = round_up(rows, 64);
        const T* w = static_cast<const T*>(c.w) + v0 * c.ldw;
        GradArgs g{};
        g.w = pack_w<DT>(c, l, v0, rows);
        g.x = x;
        g.k = l.ldx;
        g.head = p.head;
        g.tgt = p.tgt;
        g.a = p.a;
        g.b = p.b;
        g.lse = p.lse;
        g.v0 = v0;
        g.v = v0 + rows;
        g.tiles_n = tiles_n;
        g.g = at<uint16_t>(c, l.g);
        g.ldg = l.ldv;
        g.g_part = c.N * l.ldv;
        g.gt = at<uint16_t>(c, l.gt);
        g.ldt = l.ldn;
        g.gt_part = l.piece * l.ldn;
        logits_grad<DT><<<dim3((unsigned)(tiles_n * div_up(depth, kTile))), kThreads, 0, c.s>>>(g);
        if (dx) {
            pack_cols<DT><<<dim3((unsigned)(depth / 64), (unsigned)div_up(c.D, 64)), 256, 0, c.s>>>(
                w, c.ldw, c.D, nullptr, nullptr, rows, at<uint16_t>(c, l.wt), l.ldv, c.D * l.ldv);
            ProductArgs a{};
            a.a = Operand{at<uint16_t>(c, l.wt), l.ldv, c.D * l.ldv, (int)c.D};
            a.b = Operand{g.g, l.ldv, g.g_part, (int)c.N};
            a.head = p.head;
            a.k = depth;
            a.live_n = 1;
            a.m = c.D;
            a.n = c.N;
            a.tiles_m = tiles_d;
            a.splits = l.splits;
            a.acc = at<float>(c, l.acc);
            a.ldc = c.D;
            a.split_stride = c.N * c.D;
            a.add = v0 > 0;
            product<DT, false><<<dim3((unsigned)(tiles_d * tiles_n), (unsigned)l.splits), kThreads, 0, c.s>>>(a);
        }
        if (dw) {
            ProductArgs a{};
            a.a = xt;
            a.b = Operand{g.gt, l.ldn, g.gt_part, (int)rows};
            a.head = p.head;
            a.live_k = 1;
            a.m = c.D;
            a.n = rows;
            a.tiles_m = tiles_d;
            a.splits = 1;
            a.ldc = c.D;
            a.out = static_cast<T*>(dw) + v0 * c.D;
            product<DT, true><<<dim3((unsigned)(tiles_d * div_up(rows, kTile)), 1), kThreads, 0, c.s>>>(a);
        }
    }
    if (dx)
        finish_dx<DT><<<dim3((unsigned)c.N), 256, 0, c.s>>>(p.head, p.pos, at<float>(c, l.acc), l.splits, c.N * c.D, c.D,
                                                            dx);
}

int check(const char* name, const Call& c, int dtype, size_t ws_bytes, bool bwd) {
    FL_CHECK(c.N >= 0 && c.V >= 1 && c.D >= 1, "%s: bad shape (N=%lld, V=%lld, D=%lld)", name, (long long)c.N,
             (long long)c.V, (long long)c.D);
    FL_CHECK(dtype >= 0 && dtype <= 2, "%s: dtype %d", name, dtype);
    FL_CHECK(c.reduction >= 0 && c.reduction <= 2, "%s: reduction %d", name, c.reduction);
    FL_CHECK(c.ldx >= c.D && c.ldw >= c.D, "%s: rows of x or w overlap", name);
    if (c.N > (1 << 23) || c.V > (1 << 28) || c.D > (1 << 20))
        return set_error(FL_ERANGE, "%s: at most 2^23 rows, 2^28 vocabulary entries and 2^20 columns", name);
    if (c.N == 0) return ok();
    const int64_t size = dtype == kF32 ? 4 : 2;
    FL_CHECK(c.x && c.w && c.target, "%s: NULL pointer argument", name);
    FL_CHECK(reinterpret_cast<uintptr_t>(c.x) % size == 0 && reinterpret_cast<uintptr_t>(c.w) % size == 0,
             "%s: x or w is not element-aligned", name);
    const int64_t need = layout(c.N, c.V, c.D, dtype, bwd).bytes;
    FL_CHECK((int64_t)ws_bytes >= need, "%s: workspace of %llu bytes, %lld needed", name, (unsigned long long)ws_bytes,
             (long long)need);
    FL_CHECK(c.ws && (reinterpret_cast<uintptr_t>(c.ws) & 255u) == 0, "%s: workspace is not 256-byte aligned", name);
    return ok();
}

}  // namespace
}  // namespace lce
}  // namespace fl

using namespace fl::lce;

extern "C" size_t fl_linear_ce_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype, int backward) {
    if (N < 1 || V < 1 || D < 1 || dtype < 0 || dtype > 2 || N > (1 << 23) || V > (1 << 28) || D > (1 << 20)) return 0;
    return (size_t)layout(N, V, D, dtype, backward != 0).bytes;
}

extern "C" int fl_linear_ce_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* target,
                                int64_t N, int64_t V, int64_t D, int dtype, int64_t ignore_index, float z_loss,
                                int reduction, float* loss, float* lse, void* workspace, size_t workspace_bytes,
                                void* stream) {
    const Call c{x,      ldx, w, ldw, target, N, V, D, ignore_index, z_loss, reduction, static_cast<char*>(workspace),
                 static_cast<hipStream_t>(stream)};
    const int rc = check("fl_linear_ce_fwd", c, dtype, workspace_bytes, false);
    if (rc != FL_OK || N == 0) return rc;
    FL_CHECK(loss && lse, "fl_linear_ce_fwd: NULL pointer argument");
    if (dtype == kF32) run_fwd<kF32>(c, loss, lse);
    else if (dtype == kF16) run_fwd<kF16>(c, loss, lse);
    else run_fwd<kBF16>(c, loss, lse);
    return fl::launch_status("fl_linear_ce_fwd");
}

extern "C" int fl_linear_ce_bwd(const float* grad, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                const int64_t* target, const float* lse, int64_t N, int64_t V, int64_t D, int dtype,
                                int64_t ignore_index, float z_loss, int reduction, void* dx, void* dw,
                                void* workspace, size_t workspace_bytes, void* stream) {
    const Call c{x,      ldx, w, ldw, target, N, V, D, ignore_index, z_loss, reduction, static_cast<char*>(workspace),
                 static_cast<hipStream_t>(stream)};
    const int rc = check("fl_linear_ce_bwd", c, dtype, workspace_bytes, true);
    if (rc != FL_OK || N == 0) return rc;
    FL_CHECK(grad && lse, "fl_linear_ce_bwd: NULL pointer argument");
    if (!dx && !dw) return fl::ok();
    if (dtype == kF32) run_bwd<kF32>(c, grad, lse, dx, dw);
    else if (dtype == kF16) run_bwd<kF16>(c, grad, lse, dx, dw);
    else run_bwd<kBF16>(c, grad, lse, dx, dw);
    return fl::launch_status("fl_linear_ce_bwd");
}

// Balance loss, z loss and per-expert counts of a mixture-of-experts router on
// gfx950.
//
//   over the n tokens the mask keeps: p = softmax(l_t), lse_t = log sum exp l_t,
//   counts_e = how often e is among the tokens' k choices, f_e = counts_e / (n k),
//   balance = E sum_e f_e mean_t p_te,   z = mean_t lse_t^2,
//   dl_te = p_te (gb E / n (f_e - sum_j p_tj f_j) + gz 2 lse_t / n).
//
// A group of lanes holds a token's logits in registers; a lane meets the same
// experts in every token and sums their probabilities in registers, joined per
// block and then over blocks in a fixed order, so results do not depend on the
// order of the blocks.  Both directions read the logits once and are bound by
// memory, or by the launches where the batch is small.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/fuselse_amd.h"
#include "fl_status.hpp"
#include "row_stream.hpp"

namespace fl {
namespace router {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxExperts = 1024;

struct Args {
    const void* x;
    int64_t ldx;
    int64_t tokens;
    int experts;
    const int64_t* index;
    int top;
    const uint8_t* mask;  // NULL: every token counts
    float* lse;
    // per block
    float* sum_p;   // [blocks][experts]
    int* count;     // [blocks][experts]
    double* sum_z;  // [blocks]
    int* live;      // [blocks]
    int blocks;
    // results
    float* balance;
    float* z;
    int64_t* counts;
    float* coef;    // [experts + 1]: E f_e / n, and 2 / n
    // backward
    const float* gb;
    const float* gz;
    void* dx;
};

// A token's logits: NV vectors a lane, lane `sub` of G holding vectors
// sub, sub + G, ..; past the row -inf.  Returns its (max, sum) joined.
template <typename T, int G, int NV>
__device__ __forceinline__ void load_token(const T* x, int experts, int sub, float (&v)[NV][Elem<T>::kVec]) {
    constexpr int VE = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int e = (sub + j * G) * VE;
        load_vec_part<T>(x + e, experts - e, -kInf, v[j]);
    }
}

template <int G, int NV, int VE>
__device__ __forceinline__ float token_lse(const float (&v)[NV][VE]) {
    float m = -kInf, s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) lse_fold<true>(m, s, v[j]);
    group_merge<G>(m, s);
    return lse_finish<true>(m, s);
}

// Joins the blocks' sums and writes the results; one block.
__device__ __forceinline__ void finish(const Args& p) {
    __shared__ double sh[kThreads];
    __shared__ int shn;
    int n = 0;
    double z = 0.0;
    for (int b = threadIdx.x; b < p.blocks; b += kThreads) {
        n += p.live[b];
        z += p.sum_z[b];
    }
    if (threadIdx.x == 0) shn = 0;
    sh[threadIdx.x] = z;
    __syncthreads();
    atomicAdd(&shn, n);
    for (int d = kThreads / 2; d > 0; d >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < d) sh[threadIdx.x] += sh[threadIdx.x + d];
    }
    __syncthreads();
    n = shn;
    z = sh[0];
    __syncthreads();
    const double inv = n > 0 ? 1.0 / n : 0.0;
    double bal = 0.0;
    for (int e = threadIdx.x; e < p.experts; e += kThreads) {
        double sp = 0.0;
        int64_t c = 0;
        for (int b = 0; b < p.blocks; ++b) {
            sp += p.sum_p[(int64_t)b * p.experts + e];
            c += p.count[(int64_t)b * p.experts + e];
        }
        const double f = p.top > 0 ? c * inv / p.top : 0.0;
        p.counts[e] = c;
        p.coef[e] = (float)(p.experts * f * inv);
        bal += f * sp * inv;
    }
    sh[threadIdx.x] = bal;
    for (int d = kThreads / 2; d > 0; d >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < d) sh[threadIdx.x] += sh[threadIdx.x + d];
    }
    if (threadIdx.x == 0) {
        *p.balance = (float)(p.experts * sh[0]);
        *p.z = (float)(z * inv);
        p.coef[p.experts] = (float)(2.0 * inv);
    }
}

template <typename T, int G, int NV>
__global__ __launch_bounds__(kThreads) void fwd_tokens(Args p) {
    constexpr int VE = Elem<T>::kVec;
    constexpr int GROUPS = kThreads / G;
    constexpr int W = G * NV * VE;  // experts the lanes hold
    __shared__ float shp[GROUPS < 16 ? GROUPS : 16][W];
    __shared__ int shc[W];
    __shared__ double shz[kThreads];
    __shared__ int shl;
    const int group = threadIdx.x / G, sub = threadIdx.x % G;
    for (int e = threadIdx.x; e < W; e += kThreads) shc[e] = 0;
    if (threadIdx.x == 0) shl = 0;
    __syncthreads();
    float sum[NV][VE] = {};
    double z = 0.0;
    int live = 0;
    for (int64_t t = (int64_t)blockIdx.x * GROUPS + group; t < p.tokens; t += (int64_t)p.blocks * GROUPS) {
        if (p.mask && !p.mask[t]) {
            if (sub == 0) p.lse[t] = 0.0f;
            continue;
        }
        float v[NV][VE];
        load_token<T, G, NV>(static_cast<const T*>(p.x) + t * p.ldx, p.experts, sub, v);
        const float lse = token_lse<G, NV, VE>(v);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) sum[j][k] += fexp2((v[j][k] - lse) * kLog2e);
        if (sub == 0) {
            p.lse[t] = lse;
            z += (double)lse * lse;
            ++live;
        }
        for (int k = sub; k < p.top; k += G) {
            const int64_t e = p.index[t * p.top + k];
            if (e >= 0 && e < p.experts) atomicAdd(&shc[e], 1);
        }
    }
    if (sub == 0 && live) atomicAdd(&shl, live);
    // sums over the block's groups in order: at most 16 at a time
    float total[(W + kThreads - 1) / kThreads] = {};
    for (int g0 = 0; g0 < GROUPS; g0 += 16) {
        __syncthreads();
        if (group >= g0 && group < g0 + 16) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < VE; ++k) shp[group - g0][(sub + j * G) * VE + k] = sum[j][k];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < (W + kThreads - 1) / kThreads; ++i) {
            const int e = threadIdx.x + i * kThreads;
            if (e < W)
                for (int g = 0; g < (GROUPS < 16 ? GROUPS : 16); ++g) total[i] += shp[g][e];
        }
    }
    shz[threadIdx.x] = sub == 0 ? z : 0.0;
    for (int d = kThreads / 2; d > 0; d >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < d) shz[threadIdx.x] += shz[threadIdx.x + d];
    }
    const int64_t b = blockIdx.x;
#pragma unroll
    for (int i = 0; i < (W + kThreads - 1) / kThreads; ++i) {
        const int e = threadIdx.x + i * kThreads;
        if (e < p.experts) {
            p.sum_p[b * p.experts + e] = total[i];
            p.count[b * p.experts + e] = shc[e];
        }
    }
    if (threadIdx.x == 0) {
        p.sum_z[b] = shz[0];
        p.live[b] = shl;
    }
}

__global__ __launch_bounds__(kThreads) void fwd_finish(Args p) { finish(p); }

template <typename T, int G, int NV>
__global__ __launch_bounds__(kThreads) void bwd_tokens(Args p) {
    constexpr int VE = Elem<T>::kVec;
    constexpr int GROUPS = kThreads / G;
    const int group = threadIdx.x / G, sub = threadIdx.x % G;
    const float gb = p.gb ? *p.gb : 0.0f, gz = p.gz ? *p.gz * p.coef[p.experts] : 0.0f;
    float c[NV][VE];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) {
            const int e = (sub + j * G) * VE + k;
            c[j][k] = e < p.experts ? p.coef[e] : 0.0f;
        }
    for (int64_t t = (int64_t)blockIdx.x * GROUPS + group; t < p.tokens; t += (int64_t)p.blocks * GROUPS) {
        T* dx = static_cast<T*>(p.dx) + t * p.experts;
        float v[NV][VE];
        if (p.mask && !p.mask[t]) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < VE; ++k) v[j][k] = 0.0f;
        } else {
            load_token<T, G, NV>(static_cast<const T*>(p.x) + t * p.ldx, p.experts, sub, v);
            const float lse = p.lse[t];
            float dot = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < VE; ++k) {
                    v[j][k] = fexp2((v[j][k] - lse) * kLog2e);
                    dot += v[j][k] * c[j][k];
                }
            if constexpr (G >= 2) dot += reduce_partner<1>(dot);
            if constexpr (G >= 4) dot += reduce_partner<2>(dot);
            if constexpr (G >= 8) dot += reduce_partner<4>(dot);
            if constexpr (G >= 16) dot += reduce_partner<8>(dot);
            if constexpr (G >= 32) dot += reduce_partner<16>(dot);
            if constexpr (G >= 64) dot += reduce_partner<32>(dot);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < VE; ++k) v[j][k] *= gb * (c[j][k] - dot) + gz * lse;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) {
                const int e = (sub + j * G) * VE + k;
                if (e < p.experts) Elem<T>::put(dx + e, v[j][k]);
            }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

// Lanes a token: the smallest power of two whose vectors cover the experts.
int lanes(int experts, int dtype) {
    const int vecs = (experts * elem_size(dtype) + 15) / 16;
    int g = 1;
    while (g < vecs && g < 64) g *= 2;
    return g;
}

int block_count(int64_t tokens, int experts, int dtype) {
    const int groups = kThreads / lanes(experts, dtype);
    const int64_t want = (tokens + groups - 1) / groups;
    return (int)(want < 256 ? (want < 1 ? 1 : want) : 256);
}

struct Ws {
    int64_t sum_p, count, sum_z, live, bytes;
};
Ws ws_layout(int64_t tokens, int experts, int dtype) {
    const int64_t blocks = block_count(tokens, experts, dtype);
    Ws w{};
    w.sum_z = 0;
    w.live = blocks * 8;
    w.sum_p = w.live + blocks * 4;
    w.count = w.sum_p + blocks * experts * 4;
    w.bytes = w.count + blocks * experts * 4;
    return w;
}

// Calls f(T{}, lanes, vectors) with the last two as integral constants.
template <typename T, typename F>
void by_lanes(int experts, int dtype, F f) {
    const int g = lanes(experts, dtype);
    const int vecs = (experts * elem_size(dtype) + 15) / 16;
#define FL_CASE(G) \
    case G: f(T{}, std::integral_constant<int, G>{}, std::integral_constant<int, 1>{}); break
    switch (g) {
        FL_CASE(1);
        FL_CASE(2);
        FL_CASE(4);
        FL_CASE(8);
        FL_CASE(16);
        FL_CASE(32);
        default:
            if (vecs <= 64) f(T{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
            else if (vecs <= 128 || sizeof(T) == 2)  // 1024 halves are 128 vectors
                f(T{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
            else f(T{}, std::integral_constant<int, 64>{}, std::integral_constant<int, sizeof(T) == 2 ? 2 : 4>{});
    }
#undef FL_CASE
}
template <typename F>
void by_type(int experts, int dtype, F f) {
    if (dtype == 0) by_lanes<float>(experts, dtype, f);
    else if (dtype == 1) by_lanes<_Float16>(experts, dtype, f);
    else by_lanes<bf16_t>(experts, dtype, f);
}

int check(const char* name, int64_t tokens, int64_t ldx, int64_t experts, int dtype, int64_t top) {
    FL_CHECK(tokens >= 0 && experts >= 1 && top >= 0, "%s: bad shape (tokens=%lld, experts=%lld, top=%lld)", name,
             (long long)tokens, (long long)experts, (long long)top);
    FL_CHECK(dtype >= 0 && dtype <= 2, "%s: dtype %d", name, dtype);
    FL_CHECK(ldx >= experts, "%s: rows of logits overlap", name);
    if (experts > kMaxExperts) return set_error(FL_ERANGE, "%s: at most %d experts", name, kMaxExperts);
    if (top > 1024 || tokens > (1 << 30) || tokens * top >= ((int64_t)1 << 31))
        return set_error(FL_ERANGE, "%s: at most 2^30 tokens, 1024 choices each and 2^31 - 1 choices", name);
    return ok();
}

}  // namespace
}  // namespace router
}  // namespace fl

using namespace fl;
using namespace fl::router;

extern "C" size_t fl_router_workspace_bytes(int64_t tokens, int64_t experts, int dtype) {
    if (tokens < 0 || experts < 1 || experts > kMaxExperts) return 0;
    return (size_t)ws_layout(tokens, (int)experts, dtype).bytes;
}

extern "C" int fl_router_balance_fwd(const void* logits, int64_t row_stride, int64_t tokens, int64_t experts,
                                     int dtype, const int64_t* index, int64_t top, const uint8_t* mask,
                                     float* balance, float* z, int64_t* counts, float* lse, float* coef,
                                     void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "fl_router_balance_fwd";
    const int rc = check(name, tokens, row_stride, experts, dtype, top);
    if (rc != FL_OK) return rc;
    FL_CHECK(balance && z && counts && coef && (tokens == 0 || (logits && lse)) && (tokens * top == 0 || index),
             "%s: NULL pointer argument", name);
    const Ws w = ws_layout(tokens, (int)experts, dtype);
    FL_CHECK((int64_t)workspace_bytes >= w.bytes, "%s: workspace of %llu bytes, %lld needed", name,
             (unsigned long long)workspace_bytes, (long long)w.bytes);
    FL_CHECK(workspace && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, "%s: workspace is not 8-byte aligned",
             name);
    char* ws = static_cast<char*>(workspace);
    Args a{};
    a.x = logits;
    a.ldx = row_stride;
    a.tokens = tokens;
    a.experts = (int)experts;
    a.index = index;
    a.top = (int)top;
    a.mask = mask;
    a.lse = lse;
    a.sum_p = reinterpret_cast<float*>(ws + w.sum_p);
    a.count = reinterpret_cast<int*>(ws + w.count);
    a.sum_z = reinterpret_cast<double*>(ws + w.sum_z);
    a.live = reinterpret_cast<int*>(ws + w.live);
    a.blocks = block_count(tokens, (int)experts, dtype);
    a.balance = balance;
    a.z = z;
    a.counts = counts;
    a.coef = coef;
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type((int)experts, dtype, [&](auto t, auto g, auto nv) {
        fwd_tokens<decltype(t), decltype(g)::value, decltype(nv)::value><<<dim3((unsigned)a.blocks), kThreads, 0, s>>>(a);
    });
    fwd_finish<<<1, kThreads, 0, s>>>(a);
    return launch_status(name);
}

extern "C" int fl_router_balance_bwd(const float* grad_balance, const float* grad_z, const void* logits,
                                     int64_t row_stride, int64_t tokens, int64_t experts, int dtype,
                                     const uint8_t* mask, const float* lse, const float* coef, void* grad_logits,
                                     void* stream) {
    const char* name = "fl_router_balance_bwd";
    const int rc = check(name, tokens, row_stride, experts, dtype, 0);
    if (rc != FL_OK || tokens == 0) return rc;
    FL_CHECK(logits && lse && coef && grad_logits, "%s: NULL pointer argument", name);
    Args a{};
    a.x = logits;
    a.ldx = row_stride;
    a.tokens = tokens;
    a.experts = (int)experts;
    a.mask = mask;
    a.lse = const_cast<float*>(lse);
    a.coef = const_cast<float*>(coef);
    a.gb = grad_balance;
    a.gz = grad_z;
    a.dx = grad_logits;
    const int groups = kThreads / lanes((int)experts, dtype);
    const int64_t want = (tokens + groups - 1) / groups;
    a.blocks = (int)(want < 4096 ? want : 4096);
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type((int)experts, dtype, [&](auto t, auto g, auto nv) {
        bwd_tokens<decltype(t), decltype(g)::value, decltype(nv)::value><<<dim3((unsigned)a.blocks), kThreads, 0, s>>>(a);
    });
    return launch_status(name);
}

// Balance loss, z loss and per-expert counts of a mixture-of-experts router on
// gfx950.
//
//   over the n tokens the mask keeps: p = softmax(l_t), lse_t = log sum exp l_t,
//   counts_e = how often e is among the tokens' k choices, f_e = counts_e / (n k),
//   balance = E sum_e f_e mean_t p_te,   z = mean_t lse_t^2,
//   dl_te = p_te (gb E / n (f_e - sum_j p_tj f_j) + gz 2 lse_t / n).
//
// A group of lanes holds a token's logits in registers, up to four 16-byte
// vectors a lane, so that a wave has several tokens' loads in flight and few
// steps of a reduction to wait for.  A lane meets the same experts in every
// token and sums their probabilities in registers, joined per wave, per block
// and then over blocks in a fixed order, so results do not depend on the order
// of the blocks.  Both directions read the logits once and are bound by memory,
// or by the launches where the batch is small: one block then does it all.
// (131072, 256) in fp32 with 8 choices: forward 24.6 us (5.8 TB/s) and 9.5 for the
// join, backward 42 us (6.4 TB/s); (16383, 64) in bf16 with 6: 7.0 + 6.0 and 5.2 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/fuselse_amd.h"
#include "fl_status.hpp"
#include "row_stream.hpp"

namespace fl {
namespace router {
namespace {

constexpr int kThreads = 512;
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
    int2* part;     // [blocks][experts]: the probabilities' sum (fp32 bits), the choices
    double* sum_z;  // [blocks]
    int* live;      // [blocks]
    double* shares; // [finishing blocks]: of the balance
    int* arrived;   // finishing blocks that are done; cleared by the first kernel
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
    bool whole;  // rows of dx are whole 16-byte vectors
};

// A token's logits: NV vectors a lane, lane `sub` of G holding vectors
// sub, sub + G, ..; past the row -inf.
template <typename T, int G, int NV>
__device__ __forceinline__ void load_token(const T* x, int experts, int sub, float (&v)[NV][Elem<T>::kVec]) {
    constexpr int VE = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int e = (sub + j * G) * VE;
        load_vec_part<T>(x + e, experts - e, -kInf, v[j]);
    }
}

// Sum over a group's lanes of values that all of them get.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
    if constexpr (G >= 2) v += reduce_partner<1>(v);
    if constexpr (G >= 4) v += reduce_partner<2>(v);
    if constexpr (G >= 8) v += reduce_partner<4>(v);
    if constexpr (G >= 16) v += reduce_partner<8>(v);
    if constexpr (G >= 32) v += reduce_partner<16>(v);
    if constexpr (G >= 64) v += reduce_partner<32>(v);
    return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
    if constexpr (G >= 2) v = fmaxf(v, reduce_partner<1>(v));
    if constexpr (G >= 4) v = fmaxf(v, reduce_partner<2>(v));
    if constexpr (G >= 8) v = fmaxf(v, reduce_partner<4>(v));
    if constexpr (G >= 16) v = fmaxf(v, reduce_partner<8>(v));
    if constexpr (G >= 32) v = fmaxf(v, reduce_partner<16>(v));
    if constexpr (G >= 64) v = fmaxf(v, reduce_partner<32>(v));
    return v;
}

// Turns a token's logits into its probabilities and returns its log-sum-exp.  The
// probabilities come from differences to the maximum, not from the log-sum-exp,
// whose rounding in fp32 counts with the logits' own size (2e-5 around 1000).
template <int G, int NV, int VE>
__device__ __forceinline__ float token_softmax(float (&v)[NV][VE]) {
    float m = -kInf, s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) m = fmaxf(m, v[j][k]);
    const float b = lse_base(group_max<G>(m));
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) {
            v[j][k] = fexp2((v[j][k] - b) * kLog2e);
            s += v[j][k];
        }
    s = group_sum<G>(s);
    const float inv = 1.0f / s;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) v[j][k] *= inv;
    return b + flog2(s) * kLn2;
}

__device__ __forceinline__ double wave_sum(double v) {
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
    return v;
}
// Sum of v over the block, in a fixed order; all threads get it.
template <int THREADS = kThreads>
__device__ __forceinline__ double block_sum(double v, double* sh) {
    v = wave_sum(v);
    __syncthreads();
    if (lane_id() == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < THREADS / 64; ++w) v += sh[w];
    return v;
}

// Results from the sums over blocks of expert e's probabilities and choices (sp,
// c; of this thread's expert, e < experts), of z and of tokens.
__device__ __forceinline__ void results(const Args& p, int e, double sp, int64_t c, double z, int n, double& bal) {
    const double inv = n > 0 ? 1.0 / n : 0.0;
    const double f = p.top > 0 ? c * inv / p.top : 0.0;
    p.counts[e] = c;
    p.coef[e] = (float)(p.experts * f * inv);
    bal += f * sp * inv;
    if (e == 0) {
        *p.z = (float)(z * inv);
        p.coef[p.experts] = (float)(2.0 * inv);
    }
}

// Joins the blocks' sums, eight experts a block: the parts lie in other XCDs'
// memory, of which one CU reads no more than about 12 GB/s (256 blocks of 256
// experts: 42 us in one block).  The balance is the sum of the blocks' shares,
// added up in their order by the last block to arrive.
constexpr int kFinish = 256, kFinishExperts = 8, kRuns = kFinish / kFinishExperts;
__global__ __launch_bounds__(kFinish) void fwd_finish(Args p) {
    __shared__ double sh[kFinish / 64], shp[kRuns][kFinishExperts];
    __shared__ int shc[kRuns][kFinishExperts];
    double zs = 0.0, ns = 0.0;
    for (int b = threadIdx.x; b < p.blocks; b += kFinish) {
        zs += p.sum_z[b];
        ns += p.live[b];
    }
    const double z = block_sum<kFinish>(zs, sh);
    const int n = (int)block_sum<kFinish>(ns, sh);
    const int run = (int)threadIdx.x / kFinishExperts, ee = (int)threadIdx.x % kFinishExperts;
    const int e = (int)blockIdx.x * kFinishExperts + ee;
    double sp = 0.0, bal = 0.0;
    int c = 0;
    if (e < p.experts) {
        for (int b = run; b < p.blocks; b += kRuns) {
            const int2 v = p.part[(int64_t)b * p.experts + e];
            sp += __builtin_bit_cast(float, v.x);
            c += v.y;
        }
    }
    shp[run][ee] = sp;
    shc[run][ee] = c;
    __syncthreads();
    if (run == 0 && e < p.experts) {
        for (int k = 1; k < kRuns; ++k) {
            sp += shp[k][ee];
            c += shc[k][ee];
        }
        results(p, e, sp, c, z, n, bal);
    }
    bal = block_sum<kFinish>(bal, sh);
    if (threadIdx.x == 0) {
        __hip_atomic_store(&p.shares[blockIdx.x], bal, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int before = __hip_atomic_fetch_add(p.arrived, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        if (before == (int)gridDim.x - 1) {
            double all = 0.0;
            for (int b = 0; b < (int)gridDim.x; ++b)
                all += __hip_atomic_load(&p.shares[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *p.balance = (float)(p.experts * all);
        }
    }
}

template <typename T, int G, int NV>
__global__ __launch_bounds__(kThreads) void fwd_tokens(Args p) {
    constexpr int VE = Elem<T>::kVec;
    constexpr int GROUPS = kThreads / G, WAVES = kThreads / 64;
    constexpr int W = G * NV * VE;  // experts the lanes hold
    __shared__ float shp[WAVES][W];
    __shared__ int shc[W];
    __shared__ double sh[WAVES];
    const int group = threadIdx.x / G, sub = threadIdx.x % G, wave = threadIdx.x >> 6;
    for (int e = threadIdx.x; e < W; e += kThreads) shc[e] = 0;
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
        for (int k = sub; k < p.top; k += G) {
            const int64_t e = p.index[t * p.top + k];
            if (e >= 0 && e < p.experts) atomicAdd(&shc[e], 1);
        }
        const float lse = token_softmax<G, NV, VE>(v);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int k = 0; k < VE; ++k) sum[j][k] += v[j][k];
        if (sub == 0) {
            p.lse[t] = lse;
            z += (double)lse * lse;
            ++live;
        }
    }
    // over the wave's groups (lanes of the same sub), then over the waves
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int k = 0; k < VE; ++k) {
            float s = sum[j][k];
            for (int d = G; d < 64; d *= 2) s += __shfl_xor(s, d, 64);
            if ((threadIdx.x & 63) < G) shp[wave][(sub + j * G) * VE + k] = s;
        }
    const double zs = block_sum(z, sh);
    const int n = (int)block_sum((double)live, sh);
    const int64_t b = blockIdx.x;
    double bal = 0.0;
    for (int e = threadIdx.x; e < p.experts; e += kThreads) {
        float s = shp[0][e];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) s += shp[w][e];
        if (p.blocks == 1) {
            results(p, e, s, shc[e], zs, n, bal);
        } else {
            p.part[b * p.experts + e] = make_int2(__builtin_bit_cast(int, s), shc[e]);
        }
    }
    if (p.blocks == 1) {
        bal = block_sum(bal, sh);
        if (threadIdx.x == 0) *p.balance = (float)(p.experts * bal);
    } else if (threadIdx.x == 0) {
        p.sum_z[b] = zs;
        p.live[b] = n;
        if (b == 0) *p.arrived = 0;
    }
}

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
            token_softmax<G, NV, VE>(v);
            float dot = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < VE; ++k) dot += v[j][k] * c[j][k];
            dot = group_sum<G>(dot);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < VE; ++k) v[j][k] *= gb * (c[j][k] - dot) + gz * lse;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = (sub + j * G) * VE;
            if (p.whole) {
                if (e < p.experts) Elem<T>::put_vec(dx + e, v[j]);
            } else {
#pragma unroll
                for (int k = 0; k < VE; ++k)
                    if (e + k < p.experts) Elem<T>::put(dx + e + k, v[j][k]);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

// Lanes a token and vectors a lane: as few lanes as hold the experts in four
// vectors each, and one vector while up to four lanes do.  A wave then works on
// up to 16 tokens, and reads 4 KB at a time.
int vectors(int experts, int dtype) { return (experts * elem_size(dtype) + 15) / 16; }
void shape(int experts, int dtype, int& g, int& nv) {
    const int vecs = vectors(experts, dtype);
    nv = vecs <= 4 ? 1 : vecs <= 16 ? 2 : 4;
    g = 1;
    while (g * nv < vecs) g *= 2;
}

// Elements one block takes by itself, results and all, rather than a second
// launch: (256, 64) 6.1 us for 9.2, but (1024, 64) 13.2 for 9.6.
constexpr int64_t kAlone = 16384;

int block_count(int64_t tokens, int experts, int dtype) {
    int g, nv;
    shape(experts, dtype, g, nv);
    const int groups = kThreads / g;
    if (tokens * experts <= kAlone) return 1;
    // one block a CU: (131072, 256) 34.0 us in all, with half as many 44.0, with
    // twice as many, whose parts take longer to join, 37.2
    const int64_t want = (tokens + groups - 1) / groups;
    return (int)(want < 256 ? (want < 1 ? 1 : want) : 256);
}

struct Ws {
    int64_t sum_z, shares, part, live, arrived, bytes;
};
Ws ws_layout(int64_t tokens, int experts, int dtype) {
    const int64_t blocks = block_count(tokens, experts, dtype);
    Ws w{};
    w.sum_z = 0;
    w.shares = blocks * 8;
    w.part = w.shares + (experts + kFinishExperts - 1) / kFinishExperts * 8;
    w.live = w.part + blocks * experts * 8;
    w.arrived = w.live + blocks * 4;
    w.bytes = w.arrived + 4;
    return w;
}

// Calls f(T{}, lanes, vectors) with the last two as integral constants.
template <typename T, typename F>
void by_lanes(int experts, int dtype, F f) {
    int g, nv;
    shape(experts, dtype, g, nv);
#define FL_CASE(G, NV) \
    if (g == G && nv == NV) return f(T{}, std::integral_constant<int, G>{}, std::integral_constant<int, NV>{})
    FL_CASE(1, 1);
    FL_CASE(2, 1);
    FL_CASE(4, 1);
    FL_CASE(4, 2);
    FL_CASE(8, 2);
    FL_CASE(8, 4);
    FL_CASE(16, 4);
    FL_CASE(32, 4);
    if constexpr (sizeof(T) == 4) FL_CASE(64, 4);  // 1024 halves are 128 vectors
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
    a.part = reinterpret_cast<int2*>(ws + w.part);
    a.shares = reinterpret_cast<double*>(ws + w.shares);
    a.arrived = reinterpret_cast<int*>(ws + w.arrived);
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
    if (a.blocks > 1) fwd_finish<<<dim3((unsigned)((experts + kFinishExperts - 1) / kFinishExperts)), kFinish, 0, s>>>(a);
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
    a.whole = experts * elem_size(dtype) % 16 == 0 && (reinterpret_cast<uintptr_t>(grad_logits) & 15) == 0;
    int g, nv;
    shape((int)experts, dtype, g, nv);
    const int groups = kThreads / g;
    const int64_t want = (tokens + groups - 1) / groups;
    a.blocks = (int)(want < 2048 ? want : 2048);
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type((int)experts, dtype, [&](auto t, auto g, auto nv) {
        bwd_tokens<decltype(t), decltype(g)::value, decltype(nv)::value><<<dim3((unsigned)a.blocks), kThreads, 0, s>>>(a);
    });
    return launch_status(name);
}

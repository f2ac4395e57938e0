// Distillation from a teacher's top logits on gfx950.
//
//   p_k = softmax over the K teacher logits t_k / T of a row,
//   q_v = softmax over the V student logits s_v / T,
//   loss = T^2 sum_k p_k (log p_k - log q_{i_k}),
//   ds_v = g T (q_v - sum_{k: i_k = v} p_k).
//
// Forward: one pass over the student's row (running maximum and sum), K
// gathers.  Backward: one read and one write of the row.  Both are bound by
// memory; no product, no matrix cores.  (4092, 128256) in bf16 with 64 entries:
// forward 169 us, 6.2 TB/s, backward 314 us, 6.7 TB/s; (1533, 50257) in fp32 with
// 20: 53 us, 5.9 TB/s, and 99 us, 6.2 TB/s (a copy: 6.8).
//
// Entries whose teacher logit is -inf are unused, whatever their index; a row
// without any other has loss and gradient 0.  A used index outside [0, V) makes
// the row's loss and gradient NaN.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/fuselse_amd.h"
#include "fl_status.hpp"
#include "row_stream.hpp"

namespace fl {
namespace distill {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 1024;

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
struct FwdArgs {
    const void* x;
    RowMap map;
    const void* t;
    const int64_t* index;
    int64_t rows, v;
    int k;
    float inv_t, t2;
    int segs;
    int64_t seg_len;   // a multiple of the vector's elements
    float2* part;      // [row][segs] when segs > 1
    float* loss;
    float* lse;
    float* tlse;
    f32x4* pairs;      // NULL: not wanted
};

// The state (m, s) of v / T: m is the maximum of v itself and s the sum of exponentials
// of (v - m) c, c = log2 e / T in the exponent, so that no rounding counts with the
// values' own size (rows of 4096 around 1000 lost 2e-5 of their sum to it).
__device__ __forceinline__ float rescale(float from, float to, float c) {
    return from == -kInf ? 0.0f : fexp2((lse_base(from) - lse_base(to)) * c);
}

template <int K>
__device__ __forceinline__ void fold_scaled(float& m, float& s, const float (&v)[K], float c) {
    float mn = m;
#pragma unroll
    for (int k = 0; k < K; ++k) mn = fmaxf(mn, v[k]);
    const float b = lse_base(mn);
    s *= rescale(m, mn, c);
    m = mn;
    const float nb = -b * c;
    float acc = 0.0f;
    if (lse_fused_exp_ok(nb)) {
#pragma unroll
        for (int k = 0; k < K; ++k) acc += fexp2(__builtin_fmaf(v[k], c, nb));
        // nb's rounding is in every exponent, and is taken out again
        acc *= fexp2(-__builtin_fmaf(b, c, nb));
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) acc += fexp2((v[k] - b) * c);
    }
    s += acc;
}

__device__ __forceinline__ void merge_scaled(float& m, float& s, float m2, float s2, float c) {
    const float mn = fmaxf(m, m2);
    s = s * rescale(m, mn, c) + s2 * rescale(m2, mn, c);
    m = mn;
}

__device__ __forceinline__ float wave_sum(float v) {
    v += reduce_partner<1>(v);
    v += reduce_partner<2>(v);
    v += reduce_partner<4>(v);
    v += reduce_partner<8>(v);
    v += reduce_partner<16>(v);
    return v + reduce_partner<32>(v);
}

// Over the wave: the maximum, each lane's sum moved to it, the sum.
__device__ __forceinline__ void wave_merge(float& m, float& s, float c) {
    float mm = fmaxf(m, reduce_partner<1>(m));
    mm = fmaxf(mm, reduce_partner<2>(mm));
    mm = fmaxf(mm, reduce_partner<4>(mm));
    mm = fmaxf(mm, reduce_partner<8>(mm));
    mm = fmaxf(mm, reduce_partner<16>(mm));
    mm = fmaxf(mm, reduce_partner<32>(mm));
    s = wave_sum(s * rescale(m, mm, c));
    m = mm;
}

// A teacher's entry; one that 1 / T takes to -inf counts as that.
template <typename TT>
__device__ __forceinline__ float teacher_logit(const TT* t, float inv_t) {
    const float v = Elem<TT>::scalar(t);
    return v * inv_t == -kInf ? -kInf : v;
}

// Joins the teacher's side of a row, in one wave: its log-sum-exp over
// t_k / T and the loss.  Writes tlse: -inf for a row without a used entry,
// NaN where a used index is out of range; and for the backward both sides'
// maxima and logs of sums, the teacher's with the same marks.
template <typename T, typename TT>
__device__ __forceinline__ void finish_row(const FwdArgs& p, int64_t r, float sm, float ss) {
    const int lane = lane_id();
    const float c = p.inv_t * kLog2e;
    // log q = (x - maximum) / T - log of the sum: the log-sum-exp's own rounding, of
    // the maximum's size, stays out
    const float base = lse_base(sm), rest = flog2(ss) * kLn2;
    const TT* t = static_cast<const TT*>(p.t) + r * p.k;
    const int64_t* index = p.index + r * p.k;
    const T* x = static_cast<const T*>(p.x) + p.map.offset(r);
    float m = -kInf, s = 0.0f;
    for (int k = lane; k < p.k; k += 64) {
        const float v = teacher_logit(t + k, p.inv_t), mn = fmaxf(m, v);
        s = s * rescale(m, mn, c) + fexp2((v - lse_base(mn)) * c);
        m = mn;
    }
    wave_merge(m, s, c);
    const float tbase = lse_base(m);
    float trest = flog2(s) * kLn2, tlse = tbase * p.inv_t + trest;
    if (tlse == kInf) tlse = __builtin_nanf("");  // a softmax of +inf
    if (tlse != tlse) trest = tlse;
    float loss = 0.0f;
    if (m != -kInf || s != 0.0f) {  // a NaN never enters m, but makes s NaN
        bool bad = false;
        for (int k = lane; k < p.k; k += 64) {
            const float tv = teacher_logit(t + k, p.inv_t);
            if (tv == -kInf) continue;
            const int64_t i = index[k];
            if (i < 0 || i >= p.v) {
                bad = true;
                continue;
            }
            const float logp = (tv - tbase) * p.inv_t - trest;
            const float prob = fexp2(logp * kLog2e);
            // a probability that underflows to 0 contributes 0
            if (prob != 0.0f) loss += prob * (logp - ((Elem<T>::scalar(x + i) - base) * p.inv_t - rest));
        }
        loss = wave_sum(loss) * p.t2;
        if (__ballot(bad)) loss = tlse = trest = __builtin_nanf("");
    }
    if (lane == 0) {
        p.loss[r] = loss;
        p.lse[r] = base * p.inv_t + rest;
        p.tlse[r] = tlse;
        if (p.pairs) p.pairs[r] = f32x4{base, rest, tbase, trest};
    }
}

template <typename T, typename TT>
__global__ __launch_bounds__(kThreads) void fwd_rows(FwdArgs p) {
    constexpr int VE = Elem<T>::kVec, U = 4;
    const int64_t r = blockIdx.x / p.segs;
    const int seg = blockIdx.x % p.segs;
    const T* x = static_cast<const T*>(p.x) + p.map.offset(r);
    const int64_t e0 = seg * p.seg_len;
    const int64_t e1 = e0 + p.seg_len < p.v ? e0 + p.seg_len : p.v;
    float m = -kInf, s = 0.0f;
    int64_t e = e0 + (int64_t)threadIdx.x * VE;
    constexpr int64_t step = (int64_t)kThreads * VE;
    const float scale = p.inv_t * kLog2e;
    auto fold = [&](const u32x4 (&raw)[U]) {
        float v[U * VE];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float t[VE];
            Elem<T>::cvt(raw[u], t);
#pragma unroll
            for (int k = 0; k < VE; ++k) v[u * VE + k] = t[k];
        }
        fold_scaled(m, s, v, scale);
    };
    // U vectors are folded, under one rescale, while the next U are in flight (a
    // rescale each: 6% more time in bf16, whose vectors hold 8 elements)
    const int64_t full = U * step + VE - step;  // elements from e on that U vectors span
    u32x4 now[U], next[U];
    bool more = e + full <= e1;
    if (more) {
#pragma unroll
        for (int u = 0; u < U; ++u) now[u] = load_raw_stream<T>(x + e + u * step);
        e += U * step;
    }
    while (more) {
        const bool again = e + full <= e1;
        if (again) {
#pragma unroll
            for (int u = 0; u < U; ++u) next[u] = load_raw_stream<T>(x + e + u * step);
            e += U * step;
        }
        fold(now);
#pragma unroll
        for (int u = 0; u < U; ++u) now[u] = next[u];
        more = again;
    }
    for (; e < e1; e += step) {
        float v[VE];
        load_vec_part<T>(x + e, e1 - e, -kInf, v);
        fold_scaled(m, s, v, scale);
    }
    wave_merge(m, s, scale);
    __shared__ float sm[kThreads / 64], ss[kThreads / 64];
    if (lane_id() == 0) {
        sm[threadIdx.x >> 6] = m;
        ss[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    m = sm[0];
    s = ss[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) merge_scaled(m, s, sm[w], ss[w], scale);
    if (p.segs == 1) {
        finish_row<T, TT>(p, r, m, s);
    } else if (threadIdx.x == 0) {
        p.part[r * p.segs + seg] = make_float2(m, s);
    }
}

template <typename T, typename TT>
__global__ __launch_bounds__(64) void fwd_finish(FwdArgs p) {
    const int64_t r = blockIdx.x;
    const float c = p.inv_t * kLog2e;
    float m = -kInf, s = 0.0f;
    for (int k = threadIdx.x; k < p.segs; k += 64) {
        const float2 q = p.part[r * p.segs + k];
        merge_scaled(m, s, q.x, q.y, c);
    }
    wave_merge(m, s, c);
    finish_row<T, TT>(p, r, m, s);
}

// Sum of the rows' losses in a fixed order; the mean is over the rows that
// have a teacher.  norm receives what the backward multiplies by.
__global__ __launch_bounds__(1024) void reduce_rows(const float* rows, const float* tlse, int64_t n, int mean,
                                                    float* out, float* norm) {
    __shared__ double sh[1024];
    __shared__ int shn[1024];
    double s = 0.0;
    int live = 0;
    for (int64_t r = threadIdx.x; r < n; r += 1024) {
        s += rows[r];
        live += tlse[r] != -kInf;
    }
    sh[threadIdx.x] = s;
    shn[threadIdx.x] = live;
    __syncthreads();
    for (int d = 512; d > 0; d >>= 1) {
        if ((int)threadIdx.x < d) {
            sh[threadIdx.x] += sh[threadIdx.x + d];
            shn[threadIdx.x] += shn[threadIdx.x + d];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double by = mean ? 1.0 / (shn[0] > 0 ? shn[0] : 1) : 1.0;
        *out = (float)(sh[0] * by);
        *norm = (float)by;
    }
}

// ---------------------------------------------------------------------------
// Backward: a block per chunk of a row.
// ---------------------------------------------------------------------------
struct BwdArgs {
    const float* grad;
    int grad_stride;
    const float* norm;
    const void* x;
    RowMap map;
    const void* t;
    const int64_t* index;
    const float* lse;
    const float* tlse;
    const f32x4* pairs;  // NULL: lse and tlse in their place
    int64_t rows, v;
    int k;
    float inv_t, temp;
    int chunks;
    int64_t block0;
    void* dx;
};

constexpr int kBwdVecs = 2;  // vectors a thread

// A block takes kBwdVecs vectors a thread of a row of the result, from the
// result's first 128-byte line on, so that a wave stores whole lines; the input,
// whose rows may lie in another phase, is read at any alignment.  The elements
// before the first line and after the last vector belong to the first and the
// last chunk.
template <typename T, typename TT>
__global__ __launch_bounds__(kThreads) void bwd_rows(BwdArgs p) {
    constexpr int VE = Elem<T>::kVec;
    constexpr int kChunk = kThreads * kBwdVecs;  // vectors
    // of the chunk's entries, read four at a time: index, probability, element, thread
    __shared__ __attribute__((aligned(16))) int li[kMaxTop + 4], lo[kMaxTop + 4];
    __shared__ __attribute__((aligned(16))) float lp[kMaxTop + 4];
    __shared__ float lv[kMaxTop];
    __shared__ int ln;
    const int64_t block = p.block0 + blockIdx.x;
    const int64_t r = block / p.chunks;
    const int c = (int)(block % p.chunks), tid = threadIdx.x;
    const T* x = static_cast<const T*>(p.x) + p.map.offset(r);
    T* dx = static_cast<T*>(p.dx) + r * p.v;
    // the row's vectors, and this chunk's elements [e0, e1)
    int head = (int)(((128 - (reinterpret_cast<uintptr_t>(dx) & 127)) & 127) / sizeof(T));
    if (head > p.v) head = (int)p.v;
    const int vecs = (int)((p.v - head) / VE);
    const int v0 = c * kChunk, v1 = vecs - v0 < kChunk ? vecs : v0 + kChunk;
    const bool last = c == p.chunks - 1;
    const int body = head + v0 * VE;  // the chunk's first whole vector
    const int tail = head + vecs * VE;
    // the last chunk may have no vector, and begin behind the tail
    const int e0 = c == 0 ? 0 : body < tail ? body : tail, e1 = last ? (int)p.v : head + v1 * VE;

    // exponents are (x - maximum) / T - log of the sum: with the pairs no rounding
    // counts with the logits' own size
    const f32x4 of = p.pairs ? p.pairs[r] : f32x4{0.0f, p.lse[r], 0.0f, p.tlse[r]};
    const float base = of[0], rest = of[1], tbase = of[2], trest = of[3];
    const bool dead = trest == -kInf;
    u32x4 raw[kBwdVecs] = {};
    if (!dead && vecs > 0) {
#pragma unroll
        for (int u = 0; u < kBwdVecs; ++u) {
            // past the last vector: the last one, so that no load has a branch of its own
            const int v = v0 + u * kThreads + tid;
            raw[u] = load_raw_stream<T>(x + head + (int64_t)(v < vecs ? v : vecs - 1) * VE);
        }
    }
    const float g = dead ? 0.0f : p.grad[r * p.grad_stride] * p.temp * (p.norm ? *p.norm : 1.0f);
    // the teacher's entries of this chunk, in order, found by one wave
    if (tid < 64) {
        int n = 0;
        constexpr int U = 4;  // entries a lane whose loads are in flight
        for (int k0 = 0; !dead && k0 < p.k; k0 += 64 * U) {
            int64_t i[U];
            float tv[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = k0 + u * 64 + tid;
                i[u] = k < p.k ? p.index[r * p.k + k] : -1;
                tv[u] = k < p.k ? teacher_logit(static_cast<const TT*>(p.t) + r * p.k + k, p.inv_t) : -kInf;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool mine = tv[u] != -kInf && i[u] >= e0 && i[u] < e1;
                const uint64_t b = __ballot(mine);
                if (mine) {
                    const int at = n + __popcll(b & ((1ull << tid) - 1));
                    li[at] = (int)i[u];
                    lp[at] = g * fexp2(((tv[u] - tbase) * p.inv_t - trest) * kLog2e);
                }
                n += __popcll(b);
            }
        }
        if (tid < 4) {
            li[n + tid] = -1;
            lp[n + tid] = 0.0f;
        }
        if (tid == 0) ln = n;
    }
    __syncthreads();
    const float gq = trest != trest ? __builtin_nanf("") : g;
    auto grad = [&](float v) { return dead ? 0.0f : gq * fexp2(((v - base) * p.inv_t - rest) * kLog2e); };
    // The entries' elements, each with the sum of all entries of its index, a thread
    // an entry.  (9880, 527) in fp32 with 108 entries: 60 us, for 1224 by the elements'
    // own threads one entry after another; with 8 entries 26.
    const int n = ln;
    for (int j = tid; j < n + 3; j += kThreads) {
        const int i = li[j];  // past the last: -1, no thread
        lo[j] = i < 0 ? -1 : i < head ? i : i >= tail ? i - tail : (i - head) / VE % kThreads;
        if (i < 0) continue;
        const float q = grad(Elem<T>::scalar(x + i));
        float take = 0.0f;
        for (int k = 0; k < n; k += 4) {
            const int4 same = *reinterpret_cast<const int4*>(li + k);
            const f32x4 prob = *reinterpret_cast<const f32x4*>(lp + k);
            take += same.x == i ? prob[0] : 0.0f;
            take += same.y == i ? prob[1] : 0.0f;
            take += same.z == i ? prob[2] : 0.0f;
            take += same.w == i ? prob[3] : 0.0f;
        }
        lv[j] = q - take;
    }
    // the elements off the grid: one a thread
    if (c == 0 && tid < head) Elem<T>::put(dx + tid, grad(dead ? 0.0f : Elem<T>::scalar(x + tid)));
    if (last && tid < p.v - tail) Elem<T>::put(dx + tail + tid, grad(dead ? 0.0f : Elem<T>::scalar(x + tail + tid)));
    // stores past the chunk's vectors fall outside the resource and are dropped
    const __amdgpu_buffer_rsrc_t to =
        __builtin_amdgcn_make_buffer_rsrc(dx + body, 0, v1 > v0 ? (v1 - v0) * 16 : 0, 0x00020000);
#pragma unroll
    for (int u = 0; u < kBwdVecs; ++u) {
        float o[VE];
        Elem<T>::cvt(raw[u], o);
#pragma unroll
        for (int k = 0; k < VE; ++k) o[k] = grad(o[k]);
        Elem<T>::put_vec_buf(to, (u * kThreads + tid) * 16, o);
    }
    // An entry's element is written again by the thread that wrote it before: one
    // thread's stores to an address keep their order.
    if (n == 0) return;
    __syncthreads();
    for (int j = 0; j < n; j += 4) {
        const int4 owner = *reinterpret_cast<const int4*>(lo + j);
        if (owner.x == tid) Elem<T>::put(dx + li[j], lv[j]);
        if (owner.y == tid) Elem<T>::put(dx + li[j + 1], lv[j + 1]);
        if (owner.z == tid) Elem<T>::put(dx + li[j + 2], lv[j + 2]);
        if (owner.w == tid) Elem<T>::put(dx + li[j + 3], lv[j + 3]);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

// Segments a row is cut into in the forward: enough blocks for the chip, none
// shorter than 16 KB.  (16, 128256) in bf16: 16 segments 8.8 us, whole rows 22.1,
// 64 KB at least 13.1; more blocks than 1024 or shorter segments gain nothing.
int segments(int64_t rows, int64_t v, int dtype) {
    const int64_t most = v * elem_size(dtype) / 16384;
    int64_t want = rows > 0 ? (1024 + rows - 1) / rows : 1;
    if (want > most) want = most;
    if (want > 64) want = 64;
    return want < 1 ? 1 : (int)want;
}

struct Ws {
    int64_t part, rows, bytes;
};
Ws ws_layout(int64_t rows, int64_t v, int dtype) {
    Ws w{};
    const int segs = segments(rows, v, dtype);
    w.part = 0;
    w.rows = segs > 1 ? (rows * segs * 8 + 255) / 256 * 256 : 0;
    w.bytes = w.rows + rows * 4;
    return w;
}

template <typename T, typename TT>
void launch_fwd(const FwdArgs& a, hipStream_t s) {
    fwd_rows<T, TT><<<dim3((unsigned)(a.rows * a.segs)), kThreads, 0, s>>>(a);
    if (a.segs > 1) fwd_finish<T, TT><<<dim3((unsigned)a.rows), 64, 0, s>>>(a);
}

template <typename T, typename TT>
void launch_bwd(const BwdArgs& a, hipStream_t s) {
    BwdArgs b = a;
    // a row has at most this many whole vectors; with none its few elements
    // still take a chunk
    constexpr int64_t chunk = (int64_t)kThreads * kBwdVecs;
    b.chunks = (int)((a.v / Elem<T>::kVec + chunk - 1) / chunk);
    if (b.chunks < 1) b.chunks = 1;
    for_grid_chunks(a.rows * b.chunks, kThreads, [&](int64_t first, int64_t count) {
        b.block0 = first;
        bwd_rows<T, TT><<<dim3((unsigned)count), kThreads, 0, s>>>(b);
    });
}

// Calls f(T{}, TT{}) for the student's and the teacher's element types.
template <typename F>
void by_types(int dtype, int tdtype, F f) {
    auto inner = [&](auto t) {
        if (tdtype == 0) f(t, float{});
        else if (tdtype == 1) f(t, _Float16{});
        else f(t, bf16_t{});
    };
    if (dtype == 0) inner(float{});
    else if (dtype == 1) inner(_Float16{});
    else inner(bf16_t{});
}

int check(const char* name, int64_t rows, int64_t n1, int64_t v, int64_t k, int dtype, int tdtype, float temp) {
    FL_CHECK(rows >= 0 && v >= 1 && k >= 0 && n1 >= 1, "%s: bad shape (rows=%lld, V=%lld, K=%lld)", name,
             (long long)rows, (long long)v, (long long)k);
    FL_CHECK(dtype >= 0 && dtype <= 2 && tdtype >= 0 && tdtype <= 2, "%s: dtype %d, %d", name, dtype, tdtype);
    // the loss carries the square
    const float square = temp * temp;
    FL_CHECK(temp > 0.0f && __builtin_isnormal(square) && __builtin_isnormal(1.0f / square),
             "%s: temperature must be positive, its square and the square's inverse normal fp32 numbers", name);
    if (k > kMaxTop) return set_error(FL_ERANGE, "%s: at most %d teacher logits a row", name, kMaxTop);
    if (rows > (1 << 22) || v > (1 << 28)) return set_error(FL_ERANGE, "%s: at most 2^22 rows of 2^28 columns", name);
    return ok();
}

}  // namespace
}  // namespace distill
}  // namespace fl

using namespace fl;
using namespace fl::distill;

extern "C" size_t fl_distill_workspace_bytes(int64_t rows, int64_t V, int dtype) {
    if (rows < 1 || V < 1) return 0;
    return (size_t)ws_layout(rows, V, dtype).bytes;
}

namespace {

int forward(const char* name, const void* logits, int64_t rows, int64_t slice_rows, int64_t slice_stride,
            int64_t row_stride, int64_t V, int dtype, const void* teacher, int teacher_dtype, const int64_t* index,
            int64_t K, float temperature, int reduction, float* loss, float* lse, float* teacher_lse, float* pairs,
            float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check(name, rows, slice_rows, V, K, dtype, teacher_dtype, temperature);
    if (rc != FL_OK || rows == 0) return rc;
    FL_CHECK(reduction >= 0 && reduction <= 2, "%s: reduction %d", name, reduction);
    FL_CHECK(logits && loss && lse && teacher_lse && (K == 0 || (teacher && index)) && (reduction == 0 || norm),
             "%s: NULL pointer argument", name);
    FL_CHECK((reinterpret_cast<uintptr_t>(pairs) & 15u) == 0, "%s: pairs is not 16-byte aligned", name);
    const Ws w = ws_layout(rows, V, dtype);
    FL_CHECK((int64_t)workspace_bytes >= w.bytes, "%s: workspace of %llu bytes, %lld needed", name,
             (unsigned long long)workspace_bytes, (long long)w.bytes);
    FL_CHECK(workspace && (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, "%s: workspace is not 8-byte aligned",
             name);
    char* ws = static_cast<char*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    FwdArgs a{};
    a.x = logits;
    a.map = RowMap{slice_rows, slice_stride, row_stride};
    a.t = teacher;
    a.index = index;
    a.rows = rows;
    a.v = V;
    a.k = (int)K;
    a.inv_t = 1.0f / temperature;
    a.t2 = temperature * temperature;
    a.segs = segments(rows, V, dtype);
    const int64_t ve = 16 / elem_size(dtype);
    a.seg_len = ((V + a.segs - 1) / a.segs + ve - 1) / ve * ve;
    a.part = reinterpret_cast<float2*>(ws + w.part);
    a.loss = reduction == 0 ? loss : reinterpret_cast<float*>(ws + w.rows);
    a.lse = lse;
    a.tlse = teacher_lse;
    a.pairs = reinterpret_cast<f32x4*>(pairs);
    by_types(dtype, teacher_dtype, [&](auto t, auto tt) { launch_fwd<decltype(t), decltype(tt)>(a, s); });
    if (reduction != 0) reduce_rows<<<1, 1024, 0, s>>>(a.loss, teacher_lse, rows, reduction == 2, loss, norm);
    return launch_status(name);
}

// The gradient from both sides' pairs, or where there are none from their
// log-sum-exps.
int backward(const char* name, const float* grad, int grad_stride, const float* norm, const void* logits, int64_t rows,
             int64_t slice_rows, int64_t slice_stride, int64_t row_stride, int64_t V, int dtype, const void* teacher,
             int teacher_dtype, const int64_t* index, int64_t K, float temperature, const float* lse,
             const float* teacher_lse, const float* pairs, void* grad_logits, void* stream) {
    const int rc = check(name, rows, slice_rows, V, K, dtype, teacher_dtype, temperature);
    if (rc != FL_OK || rows == 0) return rc;
    FL_CHECK(grad_stride == 0 || grad_stride == 1, "%s: grad_stride %d", name, grad_stride);
    FL_CHECK(grad && logits && (pairs || (lse && teacher_lse)) && grad_logits && (K == 0 || (teacher && index)),
             "%s: NULL pointer argument", name);
    FL_CHECK((reinterpret_cast<uintptr_t>(pairs) & 15u) == 0, "%s: pairs is not 16-byte aligned", name);
    BwdArgs a{};
    a.grad = grad;
    a.grad_stride = grad_stride;
    a.norm = norm;
    a.x = logits;
    a.map = RowMap{slice_rows, slice_stride, row_stride};
    a.t = teacher;
    a.index = index;
    a.lse = lse;
    a.tlse = teacher_lse;
    a.pairs = reinterpret_cast<const f32x4*>(pairs);
    a.rows = rows;
    a.v = V;
    a.k = (int)K;
    a.inv_t = 1.0f / temperature;
    a.temp = temperature;
    a.dx = grad_logits;
    by_types(dtype, teacher_dtype,
             [&](auto t, auto tt) { launch_bwd<decltype(t), decltype(tt)>(a, static_cast<hipStream_t>(stream)); });
    return launch_status(name);
}

}  // namespace

extern "C" int fl_distill_fwd(const void* logits, int64_t rows, int64_t slice_rows, int64_t slice_stride,
                              int64_t row_stride, int64_t V, int dtype, const void* teacher, int teacher_dtype,
                              const int64_t* index, int64_t K, float temperature, int reduction, float* loss,
                              float* lse, float* teacher_lse, float* norm, void* workspace, size_t workspace_bytes,
                              void* stream) {
    return forward("fl_distill_fwd", logits, rows, slice_rows, slice_stride, row_stride, V, dtype, teacher,
                   teacher_dtype, index, K, temperature, reduction, loss, lse, teacher_lse, nullptr, norm, workspace,
                   workspace_bytes, stream);
}

extern "C" int fl_distill_fwd_pairs(const void* logits, int64_t rows, int64_t slice_rows, int64_t slice_stride,
                                    int64_t row_stride, int64_t V, int dtype, const void* teacher, int teacher_dtype,
                                    const int64_t* index, int64_t K, float temperature, int reduction, float* loss,
                                    float* lse, float* teacher_lse, float* pairs, float* norm, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (rows != 0) FL_CHECK(pairs, "fl_distill_fwd_pairs: NULL pointer argument");
    return forward("fl_distill_fwd_pairs", logits, rows, slice_rows, slice_stride, row_stride, V, dtype, teacher,
                   teacher_dtype, index, K, temperature, reduction, loss, lse, teacher_lse, pairs, norm, workspace,
                   workspace_bytes, stream);
}

extern "C" int fl_distill_bwd(const float* grad, int grad_stride, const float* norm, const void* logits, int64_t rows,
                              int64_t slice_rows, int64_t slice_stride, int64_t row_stride, int64_t V, int dtype,
                              const void* teacher, int teacher_dtype, const int64_t* index, int64_t K,
                              float temperature, const float* lse, const float* teacher_lse, void* grad_logits,
                              void* stream) {
    return backward("fl_distill_bwd", grad, grad_stride, norm, logits, rows, slice_rows, slice_stride, row_stride, V,
                    dtype, teacher, teacher_dtype, index, K, temperature, lse, teacher_lse, nullptr, grad_logits,
                    stream);
}

extern "C" int fl_distill_bwd_pairs(const float* grad, int grad_stride, const float* norm, const void* logits,
                                    int64_t rows, int64_t slice_rows, int64_t slice_stride, int64_t row_stride,
                                    int64_t V, int dtype, const void* teacher, int teacher_dtype, const int64_t* index,
                                    int64_t K, float temperature, const float* pairs, void* grad_logits, void* stream) {
    return backward("fl_distill_bwd_pairs", grad, grad_stride, norm, logits, rows, slice_rows, slice_stride, row_stride,
                    V, dtype, teacher, teacher_dtype, index, K, temperature, nullptr, nullptr, pairs, grad_logits,
                    stream);
}

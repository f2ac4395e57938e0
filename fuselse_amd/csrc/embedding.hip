// Embedding lookup with scaling, and the gradient of its matrix, on gfx950.
//
//   out[i] = scale W[id_i];   dW[v] = scale sum_{i: id_i = v} g_i
//
// The lookup copies rows and is bound by memory.  The gradient sorts the token
// ids (stably, so sums always run in the tokens' order and take no atomics), sums
// runs of equal ids in fp32 and rounds a row once.  A sorted run is cut where it
// crosses a border of 32 entries, so a token that comes often is summed by many
// waves; the pieces are joined in their order.  Rows that no token takes are
// zeroed by other blocks of the same launch: most of the gradient's time, where
// the vocabulary is large, is writing them.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/fuselse_amd.h"
#include "fl_status.hpp"
#include "key_sort.hpp"
#include "row_vec.hpp"

namespace fl {
namespace embedding {
namespace {

constexpr int kThreads = 256;

struct LookupArgs {
    const void* w;
    int64_t ldw, V, D;
    const int64_t* index;
    int64_t n;
    float scale;
    void* out;
    int lanes, steps;
    int64_t items;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_kernel(LookupArgs p) {
    constexpr int VE = Elem<T>::kVec;
    const int nvec = row_vectors<T>(p.D);
    const int sub = (int)threadIdx.x % p.lanes, per = kThreads / p.lanes;
    for (int64_t it = (int64_t)blockIdx.x * per + (int)threadIdx.x / p.lanes; it < p.items;
         it += (int64_t)gridDim.x * per) {
        const int64_t i = it / p.steps;
        const int v = (int)(it % p.steps) * 64 + sub;
        if (v >= nvec) continue;
        const int64_t id = p.index[i];
        const bool inside = id >= 0 && id < p.V;
        u32x4 r = row_load(static_cast<const T*>(p.w) + (inside ? id : 0) * p.ldw, p.D, v);
        if (!inside || p.scale != 1.0f) {
            float f[VE];
            Elem<T>::cvt(r, f);
#pragma unroll
            for (int k = 0; k < VE; ++k) f[k] = inside ? f[k] * p.scale : __builtin_nanf("");
            r = pack_vec<T>(f);
        }
        row_store(static_cast<T*>(p.out) + i * p.D, p.D, v, r);
    }
}

// ---------------------------------------------------------------------------
// The gradient
// ---------------------------------------------------------------------------
struct Entry {
    uint32_t id, at;  // id: V for tokens that give no gradient
};

// Entries as the caller has them, and their first digit.
struct FirstKey {
    const int64_t* index;
    int64_t V, padding;
    int mask;
    __device__ __forceinline__ uint32_t id(int64_t i) const {
        const int64_t v = index[i];
        return (uint32_t)(v >= 0 && v < V && v != padding ? v : V);
    }
    __device__ __forceinline__ Entry entry(int64_t i) const { return Entry{id(i), (uint32_t)i}; }
    __device__ __forceinline__ int operator()(int64_t i) const { return (int)(id(i) & (uint32_t)mask); }
};
// Entries in the order of their lower digits, and the next one.
struct NextKey {
    const Entry* e;
    int shift, mask;
    __device__ __forceinline__ Entry entry(int64_t i) const { return e[i]; }
    __device__ __forceinline__ int operator()(int64_t i) const { return (int)(e[i].id >> shift) & mask; }
};

template <typename Key>
__global__ __launch_bounds__(key_sort::kThreads) void place_kernel(Key key, int64_t n, int bits, const int* hist,
                                                                   const int* total, Entry* to) {
    __shared__ key_sort::Shared sh;
    const int64_t first = (int64_t)blockIdx.x * key_sort::kChunk;
    const int m = (int)(n - first < key_sort::kChunk ? n - first : key_sort::kChunk);
    const int bins = 1 << bits;
    int k[key_sort::kRounds], place[key_sort::kRounds], all[2], start[2];
#pragma unroll
    for (int j = 0; j < key_sort::kRounds; ++j)
        k[j] = key_sort::entry(j) < m ? key(first + key_sort::entry(j)) : 0;
    key_sort::rank(sh, k, m, bins, bits, place, all);
    key_sort::block_starts(sh, hist, total, gridDim.x, bins, all, start);
#pragma unroll
    for (int j = 0; j < key_sort::kRounds; ++j)
        if (key_sort::entry(j) < m)
            to[key_sort::placed(sh, k[j], place[j], bins)] = key.entry(first + key_sort::entry(j));
}

// Up to 4096 entries: one block sorts them by all digits, in shared memory.
__global__ __launch_bounds__(key_sort::kThreads) void sort_alone(FirstKey src, int n, int bits, int passes, Entry* to) {
    __shared__ key_sort::Shared sh;
    __shared__ Entry e[key_sort::kChunk];
    Entry mine[key_sort::kRounds];
#pragma unroll
    for (int j = 0; j < key_sort::kRounds; ++j)
        mine[j] = key_sort::entry(j) < n ? src.entry(key_sort::entry(j)) : Entry{0, 0};
    const int bins = 1 << bits;
    for (int pass = 0; pass < passes; ++pass) {
        int k[key_sort::kRounds], place[key_sort::kRounds], total[2], start[2];
#pragma unroll
        for (int j = 0; j < key_sort::kRounds; ++j) k[j] = (int)(mine[j].id >> (pass * bits)) & (bins - 1);
        key_sort::rank(sh, k, n, bins, bits, place, total);
        key_sort::starts(sh, total, bins, start);
        if ((int)threadIdx.x < bins) sh.start[threadIdx.x] = start[0];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < key_sort::kRounds; ++j)
            if (key_sort::entry(j) < n) e[key_sort::placed(sh, k[j], place[j], bins)] = mine[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < key_sort::kRounds; ++j)
            if (key_sort::entry(j) < n) mine[j] = e[key_sort::entry(j)];
    }
#pragma unroll
    for (int j = 0; j < key_sort::kRounds; ++j)
        if (key_sort::entry(j) < n) to[key_sort::entry(j)] = mine[j];
}

constexpr int kRun = 32;       // sorted entries a wave sums
constexpr int kAhead = 8;      // rows whose loads are in flight
constexpr int kFillRows = 64;  // rows of dW that a block looks through

struct GradArgs {
    const void* g;
    int64_t ldg;
    const Entry* e;
    int64_t n, V, D;
    float scale;
    void* dw;
    float* part;  // [runs][2][D]: a run's first and last pieces where they go on beyond it
    int64_t runs;
    int steps;
    int64_t sum_blocks;
};

// Sums of the sorted entries [32 run, 32 run + 32) of equal ids, 64 vectors of
// columns a wave.
template <typename T>
__device__ __forceinline__ void sum_run(const GradArgs& p, int64_t run, int step) {
    constexpr int VE = Elem<T>::kVec;
    const int lane = (int)threadIdx.x & 63, v = step * 64 + lane;
    const int nvec = row_vectors<T>(p.D);
    const int64_t first = run * kRun;
    const int m = (int)(p.n - first < kRun ? p.n - first : kRun);
    // lane l: entry l of the run; lane 32 the one behind it, lane 33 the one before
    Entry mine{0xFFFFFFFFu, 0};
    if (lane < m || (lane == kRun && first + m < p.n)) mine = p.e[first + (lane < m ? lane : m)];
    if (lane == kRun + 1 && run > 0) mine = p.e[first - 1];
    const uint32_t behind = (uint32_t)__builtin_amdgcn_readlane((int)mine.id, kRun);
    const uint32_t ahead = (uint32_t)__builtin_amdgcn_readlane((int)mine.id, kRun + 1);
    float acc[VE] = {};
    bool head = (uint32_t)__builtin_amdgcn_readfirstlane((int)mine.id) == ahead;  // the piece began before
    for (int i0 = 0; i0 < m; i0 += kAhead) {
        u32x4 raw[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u;
            const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)mine.id, i);
            const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)mine.at, i);
            if (i < m && id < p.V && v < nvec) raw[u] = row_load(static_cast<const T*>(p.g) + at * p.ldg, p.D, v);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u;
            if (i >= m) break;
            const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)mine.id, i);
            if (id >= p.V) return;  // nothing but such tokens from here on
            const uint32_t next = i + 1 < m ? (uint32_t)__builtin_amdgcn_readlane((int)mine.id, i + 1) : behind;
            if (v < nvec) {
                float f[VE];
                Elem<T>::cvt(raw[u], f);
#pragma unroll
                for (int k = 0; k < VE; ++k) acc[k] += f[k];
            }
            if (next != id || i + 1 == m) {
                const bool tail = next == id;  // the piece goes on behind the run
                if (v < nvec) {
                    if (head || tail) {
                        float* to = p.part + (run * 2 + (head ? 0 : 1)) * p.D;
#pragma unroll
                        for (int k = 0; k < VE; k += 4) {
                            float q[4] = {acc[k], acc[k + 1], acc[k + 2], acc[k + 3]};
                            if (p.D >= VE) {
                                __builtin_memcpy(to + row_vec_at<T>(p.D, v) + k, q, 16);
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    if (k + j < p.D) to[k + j] = q[j];
                            }
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < VE; ++k) acc[k] *= p.scale;
                        row_store(static_cast<T*>(p.dw) + id * p.D, p.D, v, pack_vec<T>(acc));
                    }
                }
#pragma unroll
                for (int k = 0; k < VE; ++k) acc[k] = 0.0f;
                head = false;
            }
        }
    }
}

// Zeros in those of the block's rows that no token takes: a lane a row searches
// the sorted ids for it.
template <typename T>
__device__ __forceinline__ void fill_rows(const GradArgs& p, int64_t block) {
    __shared__ int taken[kFillRows];
    const int64_t first = block * kFillRows;
    if (threadIdx.x < kFillRows) {
        const int64_t id = first + threadIdx.x;
        int64_t lo = 0, hi = p.n;  // the first entry that is not below id
        while (lo < hi) {
            const int64_t mid = (lo + hi) / 2;
            if ((int64_t)p.e[mid].id < id) lo = mid + 1;
            else hi = mid;
        }
        taken[threadIdx.x] = id >= p.V || (lo < p.n && (int64_t)p.e[lo].id == id);
    }
    __syncthreads();
    const int nvec = row_vectors<T>(p.D);
    for (int r = 0; r < kFillRows; ++r) {
        if (taken[r]) continue;
        T* row = static_cast<T*>(p.dw) + (first + r) * p.D;
        for (int v = threadIdx.x; v < nvec; v += kThreads) row_store(row, p.D, v, u32x4{0, 0, 0, 0});
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void grad_kernel(GradArgs p) {
    if ((int64_t)blockIdx.x >= p.sum_blocks) {
        fill_rows<T>(p, (int64_t)blockIdx.x - p.sum_blocks);
        return;
    }
    const int64_t it = (int64_t)blockIdx.x * (kThreads / 64) + (int)(threadIdx.x >> 6);
    if (it < p.runs * p.steps) sum_run<T>(p, it / p.steps, (int)(it % p.steps));
}

// Rows whose entries lie in several runs: the run they begin in finds their end
// and adds the pieces, a wave each 16th of them.
constexpr int kJoin = 1024;
template <typename T>
__global__ __launch_bounds__(kJoin) void join_kernel(GradArgs p) {
    constexpr int VE = Elem<T>::kVec, WAVES = kJoin / 64;
    __shared__ float sh[WAVES][64 * VE];
    const int64_t run = (int64_t)blockIdx.x / p.steps;
    const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    const int v = (int)((int64_t)blockIdx.x % p.steps) * 64 + lane;
    const int64_t last = run * kRun + kRun - 1;
    if (last + 1 >= p.n) return;
    const uint32_t id = p.e[last].id;
    if (id >= p.V || p.e[last + 1].id != id) return;
    if (p.e[run * kRun].id == id && run > 0 && p.e[run * kRun - 1].id == id) return;  // began before
    int64_t lo = last + 1, hi = p.n;  // the first entry past the row's
    while (lo < hi) {
        const int64_t mid = (lo + hi) / 2;
        if (p.e[mid].id <= id) lo = mid + 1;
        else hi = mid;
    }
    const int64_t pieces = (lo - 1) / kRun - run + 1;
    const int nvec = row_vectors<T>(p.D);
    float acc[VE] = {};
    if (v < nvec) {
        const int64_t at = p.D >= VE ? row_vec_at<T>(p.D, v) : 0;
        const int n = p.D >= VE ? VE : (int)p.D;
        for (int64_t k = wave; k < pieces; k += WAVES) {
            const float* from = p.part + ((run + k) * 2 + (k == 0 ? 1 : 0)) * p.D + at;
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (j < n) acc[j] += from[j];
        }
    }
#pragma unroll
    for (int j = 0; j < VE; ++j) sh[wave][lane * VE + j] = acc[j];
    __syncthreads();
    if (wave == 0 && v < nvec) {
        for (int w = 1; w < WAVES; ++w)
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[j] += sh[w][lane * VE + j];
#pragma unroll
        for (int j = 0; j < VE; ++j) acc[j] *= p.scale;
        row_store(static_cast<T*>(p.dw) + id * p.D, p.D, v, pack_vec<T>(acc));
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check(const char* name, int64_t n, int64_t V, int64_t D, int dtype) {
    FL_CHECK(n >= 0 && V >= 1 && D >= 1, "%s: bad shape (N=%lld, V=%lld, D=%lld)", name, (long long)n, (long long)V,
             (long long)D);
    FL_CHECK(dtype >= 0 && dtype <= 2, "%s: dtype %d", name, dtype);
    if (n > (1 << 30) || V > (1 << 30) || D > (1 << 20))
        return set_error(FL_ERANGE, "%s: at most 2^30 tokens, 2^30 vocabulary entries and 2^20 columns", name);
    return ok();
}

bool aligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == 0 ? 3u : 1u)) == 0; }

template <typename F>
void by_type(int dtype, F f) {
    if (dtype == 0) f(float{});
    else if (dtype == 1) f(_Float16{});
    else f(bf16_t{});
}

int vectors(int64_t D, int dtype) { return dtype == 0 ? row_vectors<float>(D) : row_vectors<_Float16>(D); }

// Digits that the ids 0 .. V (V: no gradient) are sorted by, of ten bits at most.
void digits(int64_t V, int& passes, int& bits) {
    int all = 1;
    while (((int64_t)1 << all) <= V) ++all;
    passes = (all + 9) / 10;
    bits = (all + passes - 1) / passes;
}

int64_t align256(int64_t v) { return (v + 255) & ~(int64_t)255; }

struct Ws {
    int64_t a, b, hist, total, part, bytes;
};
Ws ws_layout(int64_t n, int64_t V, int64_t D) {
    int passes, bits;
    digits(V, passes, bits);
    Ws w{};
    const bool alone = n <= key_sort::kChunk;
    w.a = 0;
    w.b = align256(8 * n);
    w.hist = w.b + (alone || passes == 1 ? 0 : align256(8 * n));
    w.total = w.hist + (alone ? 0 : align256(4 * (key_sort::chunks(n) << bits)));
    w.part = w.total + (alone ? 0 : align256((int64_t)4 << bits));
    w.bytes = w.part + (n <= kRun ? 0 : 8 * D * ((n + kRun - 1) / kRun));
    return w;
}

}  // namespace
}  // namespace embedding
}  // namespace fl

using namespace fl;
using namespace fl::embedding;

extern "C" int fl_embedding_fwd(const void* weight, int64_t row_stride, int64_t V, int64_t D, int dtype,
                                const int64_t* index, int64_t N, float scale, void* out, void* stream) {
    const char* name = "fl_embedding_fwd";
    const int rc = check(name, N, V, D, dtype);
    if (rc != FL_OK || N == 0) return rc;
    FL_CHECK(row_stride >= D, "%s: rows of the matrix overlap", name);
    FL_CHECK(weight && index && out, "%s: NULL pointer argument", name);
    FL_CHECK(aligned(weight, dtype) && aligned(out, dtype), "%s: pointers are not element-aligned", name);
    LookupArgs a{weight, row_stride, V, D, index, N, scale, out, 0, 0, 0};
    const int nvec = vectors(D, dtype);
    a.lanes = row_lanes(nvec);
    a.steps = row_steps(nvec);
    a.items = N * a.steps;
    const int per = kThreads / a.lanes;
    const int64_t want = (a.items + per - 1) / per;
    const unsigned blocks = (unsigned)(want < (1 << 22) ? want : (1 << 22));
    by_type(dtype, [&](auto t) {
        lookup_kernel<decltype(t)><<<blocks, kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
    });
    return launch_status(name);
}

extern "C" size_t fl_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t D) {
    if (N < 0 || V < 1 || D < 1 || N > (1 << 30) || V > (1 << 30) || D > (1 << 20)) return 0;
    return (size_t)ws_layout(N, V, D).bytes;
}

extern "C" int fl_embedding_bwd(const void* grad, int64_t grad_stride, const int64_t* index, int64_t N, int64_t V,
                                int64_t D, int dtype, float scale, int64_t padding, void* grad_weight, void* workspace,
                                size_t workspace_bytes, void* stream) {
    const char* name = "fl_embedding_bwd";
    const int rc = check(name, N, V, D, dtype);
    if (rc != FL_OK) return rc;
    FL_CHECK(grad_stride >= D, "%s: rows of grad overlap", name);
    FL_CHECK(grad_weight && (N == 0 || (grad && index)), "%s: NULL pointer argument", name);
    FL_CHECK(aligned(grad, dtype) && aligned(grad_weight, dtype), "%s: pointers are not element-aligned", name);
    const Ws w = ws_layout(N, V, D);
    FL_CHECK((int64_t)workspace_bytes >= w.bytes, "%s: workspace of %llu bytes, %lld needed", name,
             (unsigned long long)workspace_bytes, (long long)w.bytes);
    FL_CHECK(w.bytes == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0),
             "%s: workspace is not 256-byte aligned", name);
    char* ws = static_cast<char*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    int passes, bits;
    digits(V, passes, bits);
    Entry* sorted = reinterpret_cast<Entry*>(ws + w.a);
    const FirstKey first{index, V, padding, (1 << bits) - 1};
    if (N > 0 && N <= key_sort::kChunk) {
        sort_alone<<<1, key_sort::kThreads, 0, s>>>(first, (int)N, bits, passes, sorted);
    } else if (N > 0) {
        int* hist = reinterpret_cast<int*>(ws + w.hist);
        int* total = reinterpret_cast<int*>(ws + w.total);
        const unsigned blocks = (unsigned)key_sort::chunks(N);
        const int bins = 1 << bits;
        Entry* other = reinterpret_cast<Entry*>(ws + w.b);
        // the last pass ends in `sorted`
        Entry* to = passes % 2 ? sorted : other;
        for (int pass = 0; pass < passes; ++pass) {
            Entry* from = to == sorted ? other : sorted;
            const NextKey next{from, pass * bits, bins - 1};
            if (pass == 0) key_sort::count_kernel<<<blocks, key_sort::kThreads, 0, s>>>(first, N, bins, hist);
            else key_sort::count_kernel<<<blocks, key_sort::kThreads, 0, s>>>(next, N, bins, hist);
            key_sort::sum_kernel<<<(unsigned)((bins + 3) / 4), 256, 0, s>>>(hist, blocks, bins, total);
            if (pass == 0) place_kernel<<<blocks, key_sort::kThreads, 0, s>>>(first, N, bits, hist, total, to);
            else place_kernel<<<blocks, key_sort::kThreads, 0, s>>>(next, N, bits, hist, total, to);
            to = from;
        }
    }
    GradArgs a{};
    a.g = grad;
    a.ldg = grad_stride;
    a.e = sorted;
    a.n = N;
    a.V = V;
    a.D = D;
    a.scale = scale;
    a.dw = grad_weight;
    a.part = reinterpret_cast<float*>(ws + w.part);
    a.runs = (N + kRun - 1) / kRun;
    a.steps = row_steps(vectors(D, dtype));
    a.sum_blocks = (a.runs * a.steps + kThreads / 64 - 1) / (kThreads / 64);
    const int64_t fill = (V + kFillRows - 1) / kFillRows;
    const int64_t joins = a.runs > 1 ? (a.runs - 1) * a.steps : 0;
    if (a.sum_blocks + fill > max_grid_blocks(kThreads) || joins > max_grid_blocks(kJoin))
        return set_error(FL_ERANGE, "%s: too many tokens for rows of %lld columns", name, (long long)D);
    by_type(dtype, [&](auto t) {
        grad_kernel<decltype(t)><<<(unsigned)(a.sum_blocks + fill), kThreads, 0, s>>>(a);
        if (joins) join_kernel<decltype(t)><<<(unsigned)joins, kJoin, 0, s>>>(a);
    });
    return launch_status(name);
}

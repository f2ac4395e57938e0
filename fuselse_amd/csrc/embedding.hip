// Embedding lookup with scaling, and the gradient of its matrix, on gfx950.
//
//   out[i] = scale W[id_i];   dW[v] = scale sum_{i: id_i = v} g_i
//
// The lookup copies rows and is bound by memory.  The gradient sorts the token
// ids (stably, so a run's sum is in the tokens' order and takes no atomics), sums
// runs of equal ids in fp32 and rounds a row once.  A sorted run is cut where it
// crosses a border of 16 or 64 entries, so a token that comes often is summed by many
// waves; its pieces are joined in an order that their number alone decides (every
// fourth by a wave, then the waves).  All of dW is zeroed by further
// blocks of the sort's launches, which leave most of the chip idle: rows that no
// token takes, most of them where the vocabulary is large, need nothing more, and
// the time the sort takes is hidden.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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
    float scale;
    void* out;
    int lanes, steps;
    int64_t items;
    bool through;  // a wave an item, rows of out that are written through
};

// Lanes share a token's row, or a wave takes U times 64 vectors of it: a row's loads
// wait for its index, and two of them in flight a lane take (65536, 4096) in bf16 from
// 174 to 141 us (5.8 TB/s), four to 137 to 164 by the tokens' order.
template <typename T, int U>
__global__ __launch_bounds__(kThreads) void lookup_kernel(LookupArgs p) {
    constexpr int VE = Elem<T>::kVec;
    const int nvec = row_vectors<T>(p.D);
    const int sub = (int)threadIdx.x % p.lanes, per = kThreads / p.lanes;
    for (int64_t it = (int64_t)blockIdx.x * per + (int)threadIdx.x / p.lanes; it < p.items;
         it += (int64_t)gridDim.x * per) {
        const int64_t i = p.steps == 1 ? it : it / p.steps;
        const int v = (int)(it - i * p.steps) * 64 * U + sub;
        const int64_t id = p.index[i];
        const bool inside = id >= 0 && id < p.V;
        const T* row = static_cast<const T*>(p.w) + (inside ? id : 0) * p.ldw;
        T* out = static_cast<T*>(p.out) + i * p.D;
        u32x4 r[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v + 64 * u < nvec) r[u] = row_load(row, p.D, v + 64 * u);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (v + 64 * u >= nvec) continue;
            if (!inside || p.scale != 1.0f) {
                float f[VE];
                Elem<T>::cvt(r[u], f);
#pragma unroll
                for (int k = 0; k < VE; ++k) f[k] = inside ? f[k] * p.scale : __builtin_nanf("");
                r[u] = pack_vec<T>(f);
            }
            if (p.through) row_store_through(out, p.D, v + 64 * u, r[u]);
            else row_store(out, p.D, v + 64 * u, r[u]);
        }
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

// Zeros over a launch's share of dW, and in the list's length: two blocks a CU, which
// walk the share together, 128 KB at a time each, written through to memory: 525 MB
// in 83 us, 95 with the nontemporal hint alone, 106 in steps of 16 KB.
struct Zeros {
    char* at;
    int64_t bytes;
    int* joins;  // cleared too, by the first block
    static constexpr int kBlocks = 511, kSteps = 8, kBytes = 16 * kSteps * key_sort::kThreads;
    __device__ __forceinline__ void operator()(int64_t block) const {
        if (block == 0 && threadIdx.x == 0) *joins = 0;
        int64_t first = block * kBytes;
        if ((reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
            for (; first + kBytes <= bytes; first += (int64_t)kBlocks * kBytes) {
                const __amdgpu_buffer_rsrc_t rsrc =
                    __builtin_amdgcn_make_buffer_rsrc(at + first, 0, kBytes, 0x00020000);
#pragma unroll
                for (int j = 0; j < kSteps; ++j)
                    __builtin_amdgcn_raw_buffer_store_b128(u32x4{0, 0, 0, 0}, rsrc,
                                                           16 * (j * key_sort::kThreads + (int)threadIdx.x), 0,
                                                           kStoreStreamAux);
            }
        } else {
            for (; first + kBytes <= bytes; first += (int64_t)kBlocks * kBytes)
#pragma unroll
                for (int j = 0; j < kSteps; ++j)
                    *(reinterpret_cast<u32x4_any*>(at + first) + j * key_sort::kThreads + (int)threadIdx.x) =
                        u32x4{0, 0, 0, 0};
        }
        if (first >= bytes) return;
        // the share's end, to whole elements, of two bytes at least
        int64_t k = first + 16 * (int)threadIdx.x;
        for (; k + 16 <= bytes; k += 16 * key_sort::kThreads) *reinterpret_cast<u32x4_any*>(at + k) = u32x4{0, 0, 0, 0};
        for (; k < bytes; k += 2) *reinterpret_cast<uint16_t*>(at + k) = 0;
    }
    unsigned blocks() const {
        const int64_t want = (bytes + kBytes - 1) / kBytes;
        return (unsigned)(want < 1 ? 1 : want < kBlocks ? want : kBlocks);
    }
};

template <typename Key>
__global__ __launch_bounds__(key_sort::kThreads) void place_kernel(Key key, int64_t n, int bits, int blocks,
                                                                   const int* hist, const int* total, Entry* to,
                                                                   Zeros zeros) {
    __shared__ key_sort::Shared<1024> sh;
    if ((int)blockIdx.x >= blocks) return zeros((int)blockIdx.x - blocks);
    const int64_t first = (int64_t)blockIdx.x * key_sort::kChunk;
    const int m = (int)(n - first < key_sort::kChunk ? n - first : key_sort::kChunk);
    const int bins = 1 << bits;
    int k[key_sort::kRounds], place[key_sort::kRounds], all[2], before[2], own[2], start[2];
#pragma unroll
    for (int j = 0; j < key_sort::kRounds; ++j)
        k[j] = key_sort::entry(j) < m ? key(first + key_sort::entry(j)) : 0;
    key_sort::load_counts(hist, total, blocks, bins, all, before);
    key_sort::rank(sh, k, m, bins, bits, place, own);
    key_sort::block_starts(sh, all, before, bins, start);
#pragma unroll
    for (int j = 0; j < key_sort::kRounds; ++j)
        if (key_sort::entry(j) < m)
            to[key_sort::placed(sh, k[j], place[j], bins)] = key.entry(first + key_sort::entry(j));
}

// Up to 8192 entries: one block sorts them by all digits, in shared memory, of which
// short digits leave enough for two blocks a CU, as the zeros' blocks need.
constexpr int kAloneBits = 6, kAloneRounds = 8, kAlone = kAloneRounds * key_sort::kThreads;
__global__ __launch_bounds__(key_sort::kThreads) void sort_alone(FirstKey src, int n, int bits, int passes, Entry* to,
                                                                 Zeros zeros) {
    constexpr int R = kAloneRounds;
    __shared__ key_sort::Shared<1 << kAloneBits> sh;
    __shared__ Entry e[kAlone];
    if (blockIdx.x > 0) return zeros((int64_t)blockIdx.x - 1);
    Entry mine[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int i = key_sort::entry<R>(j);
        mine[j] = i < n ? src.entry(i) : Entry{0, 0};
    }
    const int bins = 1 << bits;
    for (int pass = 0; pass < passes; ++pass) {
        int k[R], place[R], total[2], start[2];
#pragma unroll
        for (int j = 0; j < R; ++j) k[j] = (int)(mine[j].id >> (pass * bits)) & (bins - 1);
        key_sort::rank(sh, k, n, bins, bits, place, total);
        key_sort::starts(sh, total, bins, start);
        if ((int)threadIdx.x < bins) sh.start[threadIdx.x] = start[0];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (key_sort::entry<R>(j) < n) e[key_sort::placed(sh, k[j], place[j], bins)] = mine[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (key_sort::entry<R>(j) < n) mine[j] = e[key_sort::entry<R>(j)];
    }
#pragma unroll
    for (int j = 0; j < R; ++j)
        if (key_sort::entry<R>(j) < n) to[key_sort::entry<R>(j)] = mine[j];
}

constexpr int kAhead = 16;  // sorted entries whose rows' loads are in flight
constexpr int kPieces = 8;  // pieces of a row whose loads are in flight

struct GradArgs {
    const void* g;
    int64_t ldg;
    const Entry* e;
    int64_t n, V, D;
    float scale;
    void* dw;
    float* part;  // [runs][2][D]: a run's first and last pieces where they go on beyond it
    int run;  // entries of a run
    int64_t runs;
    int steps;
    int* joins;  // number of rows of several pieces
    int* list;   // [runs]: the runs they begin in
};

// Sums of the sorted entries [run RUN, (run + 1) RUN) of equal ids, 64 vectors of
// columns a wave.  SHORT: rows may be shorter than a vector; where they are known not to
// be, loads need no branches: (65536, 2048) in bf16, all of one token, 112 us, 125 with
// them, (60000, 2016) into 32000 rows 107 and 110.
template <typename T, int RUN, bool SHORT>
__device__ __forceinline__ void sum_run(const GradArgs& p, int64_t run, int step) {
    constexpr int VE = Elem<T>::kVec, AHEAD = RUN > kAhead ? kAhead / 2 : kAhead;
    if constexpr (!SHORT) __builtin_assume(p.D >= VE);
    const int lane = (int)threadIdx.x & 63, v = step * 64 + lane;
    const bool live = v < row_vectors<T>(p.D);
    const int64_t first = run * RUN;
    const int m = (int)(p.n - first < RUN ? p.n - first : RUN);
    Entry mine{0xFFFFFFFFu, 0};  // entry `lane` of the run
    if (lane < m) mine = p.e[first + lane];
    const uint32_t behind = first + m < p.n ? p.e[first + m].id : 0xFFFFFFFFu;
    const uint32_t ahead = run > 0 ? p.e[first - 1].id : 0xFFFFFFFFu;
    const auto id_of = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane((int)mine.id, i); };
    float acc[VE] = {};
    bool head = id_of(0) == ahead;  // the piece began before
    // Loads without conditions, AHEAD in flight (entries that are not there have row
    // 0); the next ones before this batch's stores, whose end they would wait for:
    // (65536, 4096) of 32000 rows in bf16 140 us for 125.
    u32x4 coming[AHEAD];
    const auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)mine.at, i0 + u);
            coming[u] = row_load<true>(static_cast<const T*>(p.g) + at * p.ldg, p.D, live ? v : 0);
        }
    };
    if (id_of(0) >= p.V) return;
    load(0);
    for (int i0 = 0; i0 < m; i0 += AHEAD) {
        u32x4 raw[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) raw[u] = coming[u];
        if constexpr (RUN > AHEAD)
            if (i0 + AHEAD < m) load(i0 + AHEAD);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u;
            const uint32_t id = id_of(i);
            if (id >= p.V) return;  // nothing but such entries, or none, from here on
            const uint32_t next = i + 1 < m ? id_of(i + 1) : behind;
            float f[VE];
            Elem<T>::cvt(raw[u], f);
#pragma unroll
            for (int k = 0; k < VE; ++k) acc[k] += f[k];
            if (next == id && i + 1 < m) continue;
            const bool tail = next == id;  // the piece goes on behind the run
            if (live && (head || tail)) {
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
            } else if (live) {
#pragma unroll
                for (int k = 0; k < VE; ++k) acc[k] *= p.scale;
                row_store(static_cast<T*>(p.dw) + id * p.D, p.D, v, pack_vec<T>(acc));
            }
            // the list of runs in which a row of several pieces begins, in any order
            if (tail && !head && step == 0 && lane == 0) p.list[atomicAdd(p.joins, 1)] = (int)run;
#pragma unroll
            for (int k = 0; k < VE; ++k) acc[k] = 0.0f;
            head = false;
        }
    }
}

template <typename T, int RUN, bool SHORT>
__global__ __launch_bounds__(kThreads) void sum_kernel(GradArgs p) {
    const int64_t it = (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (it < p.runs * p.steps) sum_run<T, RUN, SHORT>(p, it / p.steps, (int)(it % p.steps));
}

// Rows of several pieces: a block adds them for 64 vectors of columns, a wave each
// fourth of them, eight at a time.
constexpr int kJoinBlocks = 2048;
template <typename T, bool SHORT>
__global__ __launch_bounds__(kThreads) void join_kernel(GradArgs p) {
    constexpr int VE = Elem<T>::kVec, WAVES = kThreads / 64;
    if constexpr (!SHORT) __builtin_assume(p.D >= VE);
    __shared__ float sh[WAVES][64 * VE];
    const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    const int64_t items = (int64_t)*p.joins * p.steps;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int64_t run = p.list[it / p.steps];
        const int v = (int)(it % p.steps) * 64 + lane;
        const uint32_t id = p.e[run * p.run + p.run - 1].id;
        // the row has a piece in each following run that begins with it
        int64_t pieces = 1;
        for (bool on = true; on;) {
            const int64_t r = run + pieces + lane;
            const uint64_t not_its = __ballot(r >= p.runs || p.e[r * p.run].id != id);
            pieces += not_its ? __builtin_ctzll(not_its) : 64;
            on = not_its == 0;
        }
        const bool live = v < row_vectors<T>(p.D);
        const int64_t at = live && p.D >= VE ? row_vec_at<T>(p.D, v) : 0;
        float acc[VE] = {};
        for (int64_t k0 = wave; k0 < pieces; k0 += WAVES * kPieces) {
            // loads at places that are there in any case, all in flight; what is too much
            // is not added
            float f[kPieces][VE];
#pragma unroll
            for (int u = 0; u < kPieces; ++u) {
                const int64_t k = k0 + u * WAVES < pieces ? k0 + u * WAVES : pieces - 1;
                const float* from = p.part + ((run + k) * 2 + (k == 0 ? 1 : 0)) * p.D + at;
                if (p.D >= VE) {
                    __builtin_memcpy(f[u], from, 4 * VE);
                } else {
#pragma unroll
                    for (int j = 0; j < VE; ++j) f[u][j] = j < p.D ? from[j] : 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < kPieces; ++u)
#pragma unroll
                for (int j = 0; j < VE; ++j) acc[j] += k0 + u * WAVES < pieces ? f[u][j] : 0.0f;
        }
        __syncthreads();  // the item before is done with sh
#pragma unroll
        for (int j = 0; j < VE; ++j) sh[wave][lane * VE + j] = acc[j];
        __syncthreads();
        if (wave == 0 && live) {
#pragma unroll
            for (int w = 1; w < WAVES; ++w)
#pragma unroll
                for (int j = 0; j < VE; ++j) acc[j] += sh[w][lane * VE + j];
#pragma unroll
            for (int j = 0; j < VE; ++j) acc[j] *= p.scale;
            row_store(static_cast<T*>(p.dw) + id * p.D, p.D, v, pack_vec<T>(acc));
        }
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

// Digits that the ids 0 .. V (V: no gradient) are sorted by, of ten bits at most, of six where one block sorts.
void digits(int64_t n, int64_t V, int& passes, int& bits) {
    const int most = n <= kAlone ? kAloneBits : 10;
    int all = 1;
    while (((int64_t)1 << all) <= V) ++all;
    passes = (all + most - 1) / most;
    bits = (all + passes - 1) / passes;
}

int64_t align256(int64_t v) { return (v + 255) & ~(int64_t)255; }

// Entries of a run: as many as a wave has loads in flight, or 64, which leave fewer
// pieces to join, where that many waves keep the memory busy (steps of 512 columns):
// (65536, 2048), all of one token, 136 us for 266, (65536, 4096) 188 for 226, (2^20, 4)
// of 100000 rows in fp32 180 for 370, but (32768, 1024) 90 for 69.
int run_of(int64_t n, int64_t D) { return n * ((D + 511) / 512) >= (1 << 17) ? 64 : kAhead; }
int64_t runs_of(int64_t n, int64_t D) { return (n + run_of(n, D) - 1) / run_of(n, D); }

struct Ws {
    int64_t joins, list, a, b, hist, total, part, bytes;
};
Ws ws_layout(int64_t n, int64_t V, int64_t D) {
    int passes, bits;
    digits(n, V, passes, bits);
    Ws w{};
    const bool alone = n <= kAlone;
    w.joins = 0;
    w.list = 256;
    w.a = w.list + align256(4 * runs_of(n, D));
    w.b = w.a + align256(8 * n);
    w.hist = w.b + (alone || passes == 1 ? 0 : align256(8 * n));
    w.total = w.hist + (alone ? 0 : align256(4 * (key_sort::chunks(n) << bits)));
    w.part = w.total + (alone ? 0 : align256((int64_t)4 << bits));
    w.bytes = w.part + (n <= kAhead ? 0 : 8 * D * runs_of(n, D));
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
    LookupArgs a{weight, row_stride, V, D, index, scale, out, 0, 0, 0, false};
    const int nvec = vectors(D, dtype);
    a.lanes = row_lanes(nvec);
    a.steps = row_steps(nvec);
    const bool more = a.steps > 1 && N * a.steps >= 1024;  // fewer waves would not fill the chip
    if (more) a.steps = (a.steps + 1) / 2;
    a.items = N * a.steps;
    a.through = a.lanes == 64 && row_through(out, D * (dtype == 0 ? 4 : 2));
    const int per = kThreads / a.lanes;
    const int64_t want = (a.items + per - 1) / per;
    const unsigned blocks = (unsigned)(want < (1 << 22) ? want : (1 << 22));
    by_type(dtype, [&](auto t) {
        if (more) lookup_kernel<decltype(t), 2><<<blocks, kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
        else lookup_kernel<decltype(t), 1><<<blocks, kThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
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
    FL_CHECK((workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0),
             "%s: workspace is not 256-byte aligned", name);
    const int steps = row_steps(vectors(D, dtype));
    const int64_t sums = (runs_of(N, D) * steps + kThreads / 64 - 1) / (kThreads / 64);
    if (sums > max_grid_blocks(kThreads))
        return set_error(FL_ERANGE, "%s: N=%lld, V=%lld, D=%lld are too many for a launch", name, (long long)N,
                         (long long)V, (long long)D);
    char* ws = static_cast<char*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    int passes, bits;
    digits(N, V, passes, bits);
    Entry* sorted = reinterpret_cast<Entry*>(ws + w.a);
    const FirstKey first{index, V, padding, (1 << bits) - 1};
    int* joins = reinterpret_cast<int*>(ws + w.joins);
    // dW's zeros in `shares` parts, of which each launch takes the next ones
    char* dw = static_cast<char*>(grad_weight);
    const int64_t dw_bytes = V * D * (dtype == 0 ? 4 : 2);
    const bool alone = N <= kAlone;
    const int shares = alone ? 1 : 3 * passes;
    const int64_t per = align256(dw_bytes / shares + 1);
    int64_t done = 0;
    const auto zeros = [&](int parts) {
        int64_t bytes = per * parts < dw_bytes - done ? per * parts : dw_bytes - done;
        const Zeros z{dw + done, bytes, joins};
        done += bytes;
        return z;
    };
    if (alone) {
        const Zeros z = zeros(1);
        sort_alone<<<1 + z.blocks(), key_sort::kThreads, 0, s>>>(first, (int)N, bits, passes, sorted, z);
    } else {
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
            const auto go = [&](auto key) {
                const Zeros z1 = zeros(1), z2 = zeros(2);
                key_sort::count_kernel<<<blocks + z1.blocks(), key_sort::kThreads, 0, s>>>(key, N, bins, hist, z1);
                if (blocks > (unsigned)key_sort::kFewBlocks)
                    key_sort::sum_kernel<<<(unsigned)((bins + 63) / 64), key_sort::kThreads, 0, s>>>(hist, (int)blocks,
                                                                                                    bins, total);
                place_kernel<<<blocks + z2.blocks(), key_sort::kThreads, 0, s>>>(key, N, bits, (int)blocks, hist, total,
                                                                                 to, z2);
            };
            if (pass == 0) go(first);
            else go(next);
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
    a.run = run_of(N, D);
    a.runs = runs_of(N, D);
    a.steps = steps;
    a.joins = joins;
    a.list = reinterpret_cast<int*>(ws + w.list);
    if (N == 0) return launch_status(name);
    const int64_t most = (a.runs - 1) * a.steps;
    const unsigned blocks = (unsigned)(most < kJoinBlocks ? most : kJoinBlocks);
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        const auto go = [&](auto is_short) {
            constexpr bool SHORT = decltype(is_short)::value;
            if (a.run == 64) sum_kernel<T, 64, SHORT><<<(unsigned)sums, kThreads, 0, s>>>(a);
            else sum_kernel<T, kAhead, SHORT><<<(unsigned)sums, kThreads, 0, s>>>(a);
            if (blocks) join_kernel<T, SHORT><<<blocks, kThreads, 0, s>>>(a);
        };
        if (D < Elem<T>::kVec) go(std::true_type{});
        else go(std::false_type{});
    });
    return launch_status(name);
}

// Tokens in their experts' order and back, on gfx950.
//
//   order:    entries (t, k) sorted by expert, tokens in order within one; entries
//             of masked tokens and of no expert behind all others.
//   dispatch: rows[pos(t, k)] = x[t], 0 for entries that are dropped
//   combine:  y[t] = sum_k w_tk rows[pos(t, k)]           (w = 1: dispatch's gradient)
//   gradient: drows[pos(t, k)] = w_tk dy[t], dw_tk = dy[t] . rows[pos(t, k)]
//
// All run from the token's side, which knows its rows: x and dy are then read
// once and no row is found by a search.  Nothing is added by atomics, so results
// do not depend on the order of blocks.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/fuselse_amd.h"
#include "fl_status.hpp"
#include "key_sort.hpp"
#include "row_vec.hpp"

namespace fl {
namespace experts {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// The order
// ---------------------------------------------------------------------------
struct Key {
    const int64_t* index;
    const uint8_t* mask;  // NULL: every token takes part
    uint32_t top;
    int experts;
    // an entry's expert, or `experts` where it has none
    __device__ __forceinline__ int operator()(int64_t i) const {
        if (mask && !mask[(uint32_t)i / top]) return experts;
        const int64_t e = index[i];
        return e >= 0 && e < experts ? (int)e : experts;
    }
};

struct OrderArgs {
    Key key;
    int64_t n;
    int bits;
    int32_t* position;
    int64_t* counts;
    int32_t* offsets;
    // more than one block
    int* hist;
    int* total;
    int64_t blocks;
};

__device__ __forceinline__ void write_counts(const OrderArgs& p, const int (&total)[2], const int (&start)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int b = (int)threadIdx.x + j * key_sort::kThreads;
        if (b < p.key.experts) p.counts[b] = total[j];
        if (b <= p.key.experts) p.offsets[b] = start[j];
    }
}

template <bool ALONE>
__global__ __launch_bounds__(key_sort::kThreads) void place_kernel(OrderArgs p) {
    __shared__ key_sort::Shared<> sh;
    const int64_t first = (int64_t)blockIdx.x * key_sort::kChunk;
    const int m = (int)(p.n - first < key_sort::kChunk ? p.n - first : key_sort::kChunk);
    const int bins = p.key.experts + 1;
    int key[key_sort::kRounds], place[key_sort::kRounds], total[2], start[2], before[2] = {}, own[2];
#pragma unroll
    for (int j = 0; j < key_sort::kRounds; ++j)
        key[j] = key_sort::entry(j) < m ? p.key(first + key_sort::entry(j)) : 0;
    if constexpr (!ALONE) key_sort::load_counts(p.hist, p.total, (int)p.blocks, bins, total, before);
    key_sort::rank(sh, key, m, bins, p.bits, place, own);
    if constexpr (ALONE) {
        total[0] = own[0];
        total[1] = own[1];
    }
    key_sort::block_starts(sh, total, before, bins, start);
    if (blockIdx.x == 0) write_counts(p, total, start);
#pragma unroll
    for (int j = 0; j < key_sort::kRounds; ++j)
        if (key_sort::entry(j) < m) {
            const int at = key_sort::placed(sh, key[j], place[j], bins);
            p.position[first + key_sort::entry(j)] = key[j] == p.key.experts ? ~at : at;
        }
}

// ---------------------------------------------------------------------------
// Rows
// ---------------------------------------------------------------------------
struct RowArgs {
    const void* in;  // x, rows, or dy
    int64_t ldi;
    int64_t D, n;  // n rows, of all tokens' choices
    const int32_t* position;
    int top;
    const void* weights;  // [tokens, top], NULL: 1
    bool weights_f32;
    void* out;  // rows, y, or drows
    const void* rows;  // gradient: the experts' rows
    int64_t ldr;
    void* dweights;
    int lanes, steps, groups;  // groups of a token's rows
    int64_t items;
    bool ragged;   // rows are no whole vectors
    bool through;  // rows of out are written through
};

template <typename T>
__device__ __forceinline__ float weight_of(const RowArgs& p, int64_t i) {
    if (!p.weights) return 1.0f;
    return p.weights_f32 ? static_cast<const float*>(p.weights)[i] : Elem<T>::scalar(static_cast<const T*>(p.weights) + i);
}

// Item of this thread's lanes and its lane among them.  With WAVE a wave has one item.
template <bool WAVE>
__device__ __forceinline__ int64_t first_item(const RowArgs& p, int& sub) {
    if constexpr (WAVE) {
        sub = (int)threadIdx.x & 63;
        return (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    } else {
        sub = (int)threadIdx.x % p.lanes;
        return (int64_t)blockIdx.x * (kThreads / p.lanes) + (int)threadIdx.x / p.lanes;
    }
}
template <bool WAVE>
__device__ __forceinline__ int64_t item_stride(const RowArgs& p) {
    return (int64_t)gridDim.x * (kThreads / (WAVE ? 64 : p.lanes));
}

constexpr int kAhead = 8;  // rows whose loads are in flight

// Token of item `it` of a group of A of its rows, and the first of them.  Groups are
// items of their own, so that few tokens of many rows fill the chip too: 4 tokens of
// 1024 rows of 512 in fp32 7 us to dispatch and 13 for the gradient, 166 and 1313 by
// a loop over a token's; (8192, 2048) in bf16 of 16 rows each 100 for 104, 211 for 219.
template <int A>
__device__ __forceinline__ int64_t token_of(const RowArgs& p, int64_t it, int& k0) {
    const int64_t t = p.groups == 1 ? it : it / p.groups;
    k0 = (int)(it - t * p.groups) * A;
    return t;
}

// Places of the token's entries k0, k0 + 1, ..; INT_MAX, outside all rows, past
// the last.  A load each, which a wave waits for one by one.  All at once, as below, are
// there sooner: 100 tokens of 2048 in bf16 from 32 experts each 9.4 us for 11.0, the
// gradient of (40000, 2048) from two 141 for 147.  But the rows' loads then come in
// bursts, and those of (131072, 512) from 8 take 211 us for 200.
template <int A>
__device__ __forceinline__ void load_places(const RowArgs& p, int64_t t, int k0, int (&at)[A]) {
#pragma unroll
    for (int u = 0; u < A; ++u) at[u] = k0 + u < p.top ? p.position[t * p.top + k0 + u] : 0x7FFFFFFF;
}

// The same with their weights, by one load a wave, a lane an entry, for which all of it
// has to be there.
template <typename T, bool WAVE, int A>
__device__ __forceinline__ void load_entries(const RowArgs& p, int64_t t, int k0, int (&at)[A], float (&w)[A]) {
    const auto load = [&](int k, int& place, float& weight) {
        const int64_t i = t * p.top + (k < p.top ? k : p.top - 1);
        place = p.position[i];
        weight = weight_of<T>(p, i);
    };
    if constexpr (WAVE) {
        int place;
        float weight;
        load(k0 + (int)threadIdx.x % A, place, weight);
#pragma unroll
        for (int u = 0; u < A; ++u) {
            at[u] = __builtin_amdgcn_readlane(place, u);
            w[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), u));
        }
    } else {
#pragma unroll
        for (int u = 0; u < A; ++u) load(k0 + u, at[u], w[u]);
    }
#pragma unroll
    for (int u = 0; u < A; ++u) at[u] = k0 + u < p.top ? at[u] : 0x7FFFFFFF;
}

// x is read with plain loads, since what made it has often left it in the caches
// (with the nontemporal hint (16383, 2048) in bf16 to 6 experts each takes 98 us
// for 80), and a wave's rows are written through to memory (77).  MANY: tokens may have
// more rows than a group; whoever has one group is spared the division, for which the
// load of x would wait ((60000, 4096) in bf16 to one expert each 158 us for 163).  A is 1
// where tokens are few: 8 of 2048 in bf16 to 8 experts each 3.1 us, 5.6 with all of a
// token's rows by a wave.
template <typename T, bool WAVE, int A, bool MANY>
__global__ __launch_bounds__(kThreads) void dispatch_kernel(RowArgs p) {
    if constexpr (WAVE) __builtin_assume(p.D >= Elem<T>::kVec);  // more than 32 vectors
    const int nvec = row_vectors<T>(p.D);
    int sub;
    for (int64_t it = first_item<WAVE>(p, sub); it < p.items; it += item_stride<WAVE>(p)) {
        const int64_t group = p.steps == 1 ? it : it / p.steps;
        const int v = (int)(it - group * p.steps) * 64 + sub;
        if (v >= nvec) continue;
        int k0 = 0, at[A];
        int64_t t = group;
        if constexpr (MANY) t = token_of<A>(p, group, k0);
        const u32x4 x = row_load(static_cast<const T*>(p.in) + t * p.ldi, p.D, v);
        load_places(p, t, k0, at);
#pragma unroll
        for (int u = 0; u < A; ++u) {
            const int row = at[u] < 0 ? ~at[u] : at[u];
            if (row >= p.n) continue;
            T* to = static_cast<T*>(p.out) + row * p.D;
            u32x4 r = x;
            if (at[u] < 0) r = u32x4{0, 0, 0, 0};
            if (WAVE && p.through) row_store_through(to, p.D, v, r);
            else row_store(to, p.D, v, r);
        }
    }
}

// The experts' rows are read once, with the nontemporal hint: (131072, 512) in
// bf16 from 8 experts each 200 us (6.0 TB/s), without it 217.  A wave takes A rows'
// loads and U times 64 vectors of them together: eight rows of one, or, where rows
// are longer than that, up to four of two ((60000, 4096) from one expert each 225 us
// with one vector a lane, 156 with two; (60000, 999) from 5 141 and 130).
template <typename T, bool WAVE, int A, int U, bool FEW = false>
__global__ __launch_bounds__(kThreads) void combine_kernel(RowArgs p) {
    constexpr int VE = Elem<T>::kVec;
    if constexpr (WAVE) __builtin_assume(p.D >= Elem<T>::kVec);  // more than 32 vectors
    const int nvec = row_vectors<T>(p.D);
    int sub;
    for (int64_t it = first_item<WAVE>(p, sub); it < p.items; it += item_stride<WAVE>(p)) {
        const int64_t t = p.steps == 1 ? it : it / p.steps;
        const int first = (int)(it - t * p.steps) * 64 * U + sub;
        const int v = first < nvec ? first : nvec - 1;  // lanes behind the row load places too
        float acc[U][VE] = {};
        for (int k0 = 0; k0 < p.top; k0 += A) {
            int at[A];
            u32x4 raw[A][U];
            float w[A];
            if constexpr (FEW) {
                load_entries<T, WAVE>(p, t, k0, at, w);
            } else {
                load_places(p, t, k0, at);
#pragma unroll
                for (int u = 0; u < A; ++u) w[u] = k0 + u < p.top ? weight_of<T>(p, t * p.top + k0 + u) : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < A; ++u)
                if (at[u] >= 0 && at[u] < p.n)
#pragma unroll
                    for (int j = 0; j < U; ++j)
                        raw[u][j] = row_load<true>(static_cast<const T*>(p.in) + at[u] * p.ldi, p.D,
                                                   v + 64 * j < nvec ? v + 64 * j : v);
#pragma unroll
            for (int u = 0; u < A; ++u)
                if (at[u] >= 0 && at[u] < p.n)
#pragma unroll
                    for (int j = 0; j < U; ++j) {
                        float r[VE];
                        Elem<T>::cvt(raw[u][j], r);
#pragma unroll
                        for (int k = 0; k < VE; ++k) acc[j][k] = __builtin_fmaf(w[u], r[k], acc[j][k]);
                    }
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (first + 64 * j < nvec) row_store(static_cast<T*>(p.out) + t * p.D, p.D, v + 64 * j, pack_vec<T>(acc[j]));
    }
}

// Sums of eight values over lanes that share a token (8, 16, 32 or 64): three
// exchanges halve the values a lane holds, the rest add one value, so that lane
// l ends with value 4 (l & 1) + (l & 2) + (l >> 2 & 1) of its lanes' eight.
__device__ __forceinline__ float sum_eight(const float (&v)[8], int lanes) {
    const int lane = (int)threadIdx.x & 63;
    float a[4], b[2], c;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const float give = lane & 1 ? v[u] : v[u + 4], keep = lane & 1 ? v[u + 4] : v[u];
        a[u] = keep + reduce_partner<1>(give);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const float give = lane & 2 ? a[u] : a[u + 2], keep = lane & 2 ? a[u + 2] : a[u];
        b[u] = keep + reduce_partner<2>(give);
    }
    {
        const float give = lane & 4 ? b[0] : b[1], keep = lane & 4 ? b[1] : b[0];
        c = keep + exact_xor<4>(give);
    }
    if (lanes >= 16) c += exact_xor<8>(c);
    if (lanes >= 32) c += exact_xor<16>(c);
    if (lanes >= 64) c += exact_xor<32>(c);
    return c;
}
__device__ __forceinline__ int eighth(int sub) { return 4 * (sub & 1) + (sub & 2) + ((sub >> 2) & 1); }

// The gradient of a combination, a token by its lanes or by the block: dy is read
// once for A rows, and the loads of U vectors a lane of all of them are in flight
// together, ahead of the stores, whose end a later load would wait for.  A wave's
// rows are written through: (131072, 512) in bf16 from 8 experts each 434 us for 441.
template <typename T, int TEAM, int A, int U>  // TEAM 0: p.lanes, 1: a wave, 2: the block
__global__ __launch_bounds__(kThreads) void combine_bwd_kernel(RowArgs p) {
    constexpr int VE = Elem<T>::kVec;
    constexpr bool BLOCK = TEAM == 2;
    __shared__ float sh[2][kThreads / 64][kAhead];
    if constexpr (TEAM > 0) __builtin_assume(p.D >= VE);  // more than 32 vectors
    const int nvec = row_vectors<T>(p.D);
    int sub = (int)threadIdx.x, turn = 0;
    const int team = BLOCK ? kThreads : TEAM == 1 ? 64 : p.lanes;
    int64_t it = blockIdx.x, stride = gridDim.x;
    if constexpr (!BLOCK) {
        it = first_item<TEAM == 1>(p, sub);
        stride = item_stride<TEAM == 1>(p);
    }
    for (; it < p.items; it += stride, turn ^= 1) {
        int k0;
        const int64_t t = token_of<A>(p, it, k0);
        const T* dy = static_cast<const T*>(p.in) + t * p.ldi;
        float dot[kAhead] = {};
        int at[A];
        float w[A];
        load_entries<T, (TEAM > 0)>(p, t, k0, at, w);
        for (int v0 = sub; v0 < nvec; v0 += team * U) {
            u32x4 raw[A][U], gr[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int v = v0 + j * team;
                gr[j] = row_load(dy, p.D, v < nvec ? v : v0);
            }
            if (p.dweights)
#pragma unroll
                for (int u = 0; u < A; ++u)
                    if (at[u] >= 0 && at[u] < p.n)
#pragma unroll
                        for (int j = 0; j < U; ++j) {
                            const int v = v0 + j * team;
                            raw[u][j] = row_load<true>(static_cast<const T*>(p.rows) + at[u] * p.ldr, p.D,
                                                       v < nvec ? v : v0);
                        }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int v = v0 + j * team;
                if (v >= nvec) continue;
                float g[VE];
                Elem<T>::cvt(gr[j], g);
                if (p.out)
#pragma unroll
                    for (int u = 0; u < A; ++u) {
                        const int row = at[u] < 0 ? ~at[u] : at[u];
                        if (row >= p.n) continue;
                        u32x4 r{0, 0, 0, 0};
                        if (at[u] >= 0) {
                            float d[VE];
#pragma unroll
                            for (int k = 0; k < VE; ++k) d[k] = w[u] * g[k];
                            r = pack_vec<T>(d);
                        }
                        T* to = static_cast<T*>(p.out) + row * p.D;
                        if (TEAM == 1 && p.through) row_store_through(to, p.D, v, r);
                        else row_store(to, p.D, v, r);
                    }
                if (!p.dweights) continue;
                // elements that the vector before has too
                const int skip = p.ragged && p.D >= VE ? (int)((int64_t)v * VE - row_vec_at<T>(p.D, v)) : 0;
#pragma unroll
                for (int u = 0; u < A; ++u)
                    if (at[u] >= 0 && at[u] < p.n) {
                        float r[VE];
                        Elem<T>::cvt(raw[u][j], r);
#pragma unroll
                        for (int k = 0; k < VE; ++k)
                            if (k >= skip) dot[u] = __builtin_fmaf(g[k], r[k], dot[u]);
                    }
            }
        }
        if (!p.dweights) continue;
        float s = sum_eight(dot, BLOCK ? 64 : team);
        int u = eighth(sub);
        bool mine = sub < kAhead;
        if constexpr (BLOCK) {
            // two turns' values, so that one barrier a turn is enough
            if (((int)threadIdx.x & 63) < kAhead) sh[turn][threadIdx.x >> 6][u] = s;
            __syncthreads();
            u = sub;
            if (mine) {
                s = sh[turn][0][u];
#pragma unroll
                for (int w = 1; w < kThreads / 64; ++w) s += sh[turn][w][u];
            }
        }
        if (mine && u < A && k0 + u < p.top) {
            const int64_t i = t * p.top + k0 + u;
            if (p.weights_f32) static_cast<float*>(p.dweights)[i] = s;
            else Elem<T>::put(static_cast<T*>(p.dweights) + i, s);
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check_sizes(const char* name, int64_t tokens, int64_t top) {
    FL_CHECK(tokens >= 0 && top >= 1, "%s: bad shape (tokens=%lld, top=%lld)", name, (long long)tokens,
             (long long)top);
    if (top > 1024 || tokens > (1 << 30) || tokens * top >= ((int64_t)1 << 31))
        return set_error(FL_ERANGE, "%s: at most 2^30 tokens, 1024 choices each and 2^31 - 1 choices", name);
    return ok();
}

int check_rows(const char* name, int64_t tokens, int64_t D, int dtype, int64_t top) {
    const int rc = check_sizes(name, tokens, top);
    if (rc != FL_OK) return rc;
    FL_CHECK(D >= 1, "%s: bad shape (D=%lld)", name, (long long)D);
    FL_CHECK(dtype >= 0 && dtype <= 2, "%s: dtype %d", name, dtype);
    if (D > (1 << 24)) return set_error(FL_ERANGE, "%s: at most 2^24 columns", name);
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

void split_rows(RowArgs& a, int dtype) {
    const int nvec = vectors(a.D, dtype);
    a.lanes = row_lanes(nvec);
    a.steps = row_steps(nvec);
    a.groups = (a.top + kAhead - 1) / kAhead;
    a.ragged = a.D % (dtype == 0 ? 4 : 8) != 0;
    a.through = row_through(a.out, a.D * (dtype == 0 ? 4 : 2));
}

unsigned grid_of(int64_t items, int per_block) {
    const int64_t want = (items + per_block - 1) / per_block;
    return (unsigned)(want < (1 << 22) ? want : (1 << 22));
}

}  // namespace
}  // namespace experts
}  // namespace fl

using namespace fl;
using namespace fl::experts;

extern "C" size_t fl_expert_order_workspace_bytes(int64_t tokens, int64_t top, int64_t experts) {
    if (tokens < 0 || top < 1 || experts < 1 || experts > kMaxExperts || tokens > (1 << 30) || top > 1024) return 0;
    const int64_t blocks = key_sort::chunks(tokens * top);
    return blocks <= 1 ? 0 : (size_t)(4 * (blocks + 1) * (experts + 1));
}

extern "C" int fl_expert_order(const int64_t* index, int64_t tokens, int64_t top, int64_t experts, const uint8_t* mask,
                               int32_t* position, int64_t* counts, int32_t* offsets, void* workspace,
                               size_t workspace_bytes, void* stream) {
    const char* name = "fl_expert_order";
    FL_CHECK(experts >= 1, "%s: bad shape (experts=%lld)", name, (long long)experts);
    const int rc = check_sizes(name, tokens, top);
    if (rc != FL_OK) return rc;
    if (experts > kMaxExperts) return set_error(FL_ERANGE, "%s: at most %d experts", name, kMaxExperts);
    FL_CHECK(counts && offsets && (tokens == 0 || (index && position)), "%s: NULL pointer argument", name);
    const size_t need = fl_expert_order_workspace_bytes(tokens, top, experts);
    FL_CHECK(workspace_bytes >= need, "%s: workspace of %llu bytes, %llu needed", name,
             (unsigned long long)workspace_bytes, (unsigned long long)need);
    FL_CHECK(need == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 3u) == 0),
             "%s: workspace is not 4-byte aligned", name);
    OrderArgs a{};
    a.key = Key{index, mask, (uint32_t)top, (int)experts};
    a.n = tokens * top;
    a.bits = key_sort::bits_of((int)experts + 1);
    a.position = position;
    a.counts = counts;
    a.offsets = offsets;
    a.blocks = key_sort::chunks(a.n);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.blocks <= 1) {
        place_kernel<true><<<1, key_sort::kThreads, 0, s>>>(a);
        return launch_status(name);
    }
    const int bins = (int)experts + 1;
    a.total = static_cast<int*>(workspace);
    a.hist = a.total + bins;
    const unsigned blocks = (unsigned)a.blocks;
    key_sort::count_kernel<<<blocks, key_sort::kThreads, 0, s>>>(a.key, a.n, bins, a.hist, key_sort::NoWork{});
    if (a.blocks > key_sort::kFewBlocks)
        key_sort::sum_kernel<<<(unsigned)((bins + 63) / 64), key_sort::kThreads, 0, s>>>(a.hist, (int)a.blocks, bins,
                                                                                        a.total);
    place_kernel<false><<<blocks, key_sort::kThreads, 0, s>>>(a);
    return launch_status(name);
}

extern "C" int fl_expert_dispatch(const void* x, int64_t row_stride, int64_t tokens, int64_t D, int dtype,
                                  const int32_t* position, int64_t top, void* rows, void* stream) {
    const char* name = "fl_expert_dispatch";
    const int rc = check_rows(name, tokens, D, dtype, top);
    if (rc != FL_OK || tokens == 0) return rc;
    FL_CHECK(row_stride >= D, "%s: rows of x overlap", name);
    FL_CHECK(x && position && rows, "%s: NULL pointer argument", name);
    FL_CHECK(aligned(x, dtype) && aligned(rows, dtype), "%s: pointers are not element-aligned", name);
    RowArgs a{};
    a.in = x;
    a.ldi = row_stride;
    a.D = D;
    a.n = tokens * top;
    a.position = position;
    a.top = (int)top;
    a.out = rows;
    split_rows(a, dtype);
    const bool few = a.lanes == 64 && tokens * a.groups * a.steps < 1024;  // so few waves do not fill the chip
    if (few) a.groups = a.top;
    a.items = tokens * a.groups * a.steps;
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type(dtype, [&](auto t) {
        const unsigned grid = grid_of(a.items, kThreads / a.lanes);
        if (a.lanes < 64) dispatch_kernel<decltype(t), false, kAhead, true><<<grid, kThreads, 0, s>>>(a);
        else if (few) dispatch_kernel<decltype(t), true, 1, true><<<grid, kThreads, 0, s>>>(a);
        else if (a.groups > 1) dispatch_kernel<decltype(t), true, kAhead, true><<<grid, kThreads, 0, s>>>(a);
        else dispatch_kernel<decltype(t), true, kAhead, false><<<grid, kThreads, 0, s>>>(a);
    });
    return launch_status(name);
}

extern "C" int fl_expert_combine(const void* rows, int64_t row_stride, int64_t tokens, int64_t D, int dtype,
                                 const int32_t* position, int64_t top, const void* weights, int weights_dtype,
                                 void* out, void* stream) {
    const char* name = "fl_expert_combine";
    const int rc = check_rows(name, tokens, D, dtype, top);
    if (rc != FL_OK || tokens == 0) return rc;
    FL_CHECK(row_stride >= D, "%s: the experts' rows overlap", name);
    FL_CHECK(!weights || weights_dtype == 0 || weights_dtype == dtype, "%s: weights' dtype %d", name, weights_dtype);
    FL_CHECK(rows && position && out, "%s: NULL pointer argument", name);
    FL_CHECK(aligned(rows, dtype) && aligned(out, dtype) && aligned(weights, weights_dtype),
             "%s: pointers are not element-aligned", name);
    RowArgs a{};
    a.in = rows;
    a.ldi = row_stride;
    a.D = D;
    a.n = tokens * top;
    a.position = position;
    a.top = (int)top;
    a.weights = weights;
    a.weights_f32 = weights_dtype == 0;
    a.out = out;
    split_rows(a, dtype);
    const bool few = tokens * a.steps < 1024, two = a.steps > 1 && !few;  // so few waves do not fill the chip
    if (two) a.steps = (a.steps + 1) / 2;
    a.items = tokens * a.steps;
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        const unsigned grid = grid_of(a.items, kThreads / a.lanes);
        if (a.lanes < 64) combine_kernel<T, false, 8, 1><<<grid, kThreads, 0, s>>>(a);
        else if (few) combine_kernel<T, true, 8, 1, true><<<grid, kThreads, 0, s>>>(a);
        else if (!two) combine_kernel<T, true, 8, 1><<<grid, kThreads, 0, s>>>(a);
        else if (top == 1) combine_kernel<T, true, 1, 2><<<grid, kThreads, 0, s>>>(a);
        else if (top == 2) combine_kernel<T, true, 2, 2><<<grid, kThreads, 0, s>>>(a);
        else combine_kernel<T, true, 4, 2><<<grid, kThreads, 0, s>>>(a);
    });
    return launch_status(name);
}

extern "C" int fl_expert_combine_bwd(const void* grad, int64_t grad_stride, const void* rows, int64_t row_stride,
                                     int64_t tokens, int64_t D, int dtype, const int32_t* position, int64_t top,
                                     const void* weights, int weights_dtype, void* grad_rows, void* grad_weights,
                                     void* stream) {
    const char* name = "fl_expert_combine_bwd";
    const int rc = check_rows(name, tokens, D, dtype, top);
    if (rc != FL_OK || tokens == 0) return rc;
    FL_CHECK(grad_stride >= D && (!grad_weights || row_stride >= D), "%s: rows overlap", name);
    FL_CHECK(weights_dtype == 0 || weights_dtype == dtype, "%s: weights' dtype %d", name, weights_dtype);
    FL_CHECK(grad && position && weights && (rows || !grad_weights), "%s: NULL pointer argument", name);
    FL_CHECK(aligned(grad, dtype) && aligned(rows, dtype) && aligned(grad_rows, dtype) &&
                 aligned(weights, weights_dtype) && aligned(grad_weights, weights_dtype),
             "%s: pointers are not element-aligned", name);
    if (!grad_rows && !grad_weights) return ok();
    RowArgs a{};
    a.in = grad;
    a.ldi = grad_stride;
    a.D = D;
    a.n = tokens * top;
    a.position = position;
    a.top = (int)top;
    a.weights = weights;
    a.weights_f32 = weights_dtype == 0;
    a.out = grad_rows;
    a.rows = rows;
    a.ldr = row_stride;
    a.dweights = grad_weights;
    split_rows(a, dtype);
    a.items = tokens * a.groups;
    hipStream_t s = static_cast<hipStream_t>(stream);
    by_type(dtype, [&](auto t) {
        using T = decltype(t);
        const unsigned by_wave = grid_of(a.items, kThreads / 64);
        // Steps of a wave over a row.  With one or two rows a token a wave takes up to
        // eight loads a lane of them in one step ((60000, 4096) from one expert each, bf16:
        // 260 us, 284 by a block; (40000, 2048) from two 147 and 167).  With more, a block
        // shares a token from 193 vectors on: (16383, 2048) from six 162 us for 186 by a
        // wave, but (60000, 999) 338 for 312.
        const int u = a.steps;
        if (a.lanes < 64) combine_bwd_kernel<T, 0, 8, 1><<<grid_of(a.items, kThreads / a.lanes), kThreads, 0, s>>>(a);
        else if (u == 1) combine_bwd_kernel<T, 1, 8, 1><<<by_wave, kThreads, 0, s>>>(a);
        else if (top == 1 && u <= 2) combine_bwd_kernel<T, 1, 1, 2><<<by_wave, kThreads, 0, s>>>(a);
        else if (top == 1 && u <= 4) combine_bwd_kernel<T, 1, 1, 4><<<by_wave, kThreads, 0, s>>>(a);
        else if (top == 1 && u <= 8) combine_bwd_kernel<T, 1, 1, 8><<<by_wave, kThreads, 0, s>>>(a);
        else if (top == 2 && u <= 2) combine_bwd_kernel<T, 1, 2, 2><<<by_wave, kThreads, 0, s>>>(a);
        else if (top == 2 && u <= 4) combine_bwd_kernel<T, 1, 2, 4><<<by_wave, kThreads, 0, s>>>(a);
        else if (u > 3) combine_bwd_kernel<T, 2, 8, 1><<<grid_of(a.items, 1), kThreads, 0, s>>>(a);
        else combine_bwd_kernel<T, 1, 8, 1><<<by_wave, kThreads, 0, s>>>(a);
    });
    return launch_status(name);
}

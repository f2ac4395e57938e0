// Linear cross entropy on gfx950: the softmax cross entropy of hidden states
// against a vocabulary projection, forward and backward, in pieces of the
// vocabulary and without the logits in memory (formulas: linear_ce.hpp).
//
// Forward: a plan kernel lists the live rows, a packing kernel lays their
// hidden states out, the logits product reduces each of its tiles to a (max,
// sum) pair per row and keeps the target's logit, and a finishing kernel joins
// the pairs.  Backward, per piece of the vocabulary: the logits again, turned
// into G in 16 bits; dx += G w in fp32; dw = G^T x.
//
// Bound by the matrix cores but for few rows, which are bound by reading w.
// (4096, 2048, 128256) in bf16 with 2867 live rows: forward 1.2 ms, backward 4.1 ms,
// of which G 1.3, dx 1.4 and dw 1.35, 5.3 ms in all for 4.65 of four large library
// products; (8, 2048, 128256) forward 95 us, w's 525 MB at the copy rate 77.
// (2048, 1024, 32000) in fp32, both directions: 2.2 ms, for 3.0 of three products
// on the fp32 matrix pipe.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/fuselse_amd.h"
#include "fl_status.hpp"
#include "linear_ce.hpp"
#include "linear_ce_tile.hpp"
#include "row_stream.hpp"

namespace fl {
namespace lce {
namespace {

// ---------------------------------------------------------------------------
// Element types
// ---------------------------------------------------------------------------
template <int DT> struct Io;
template <> struct Io<kF32> { typedef float T; };
template <> struct Io<kF16> { typedef _Float16 T; };
template <> struct Io<kBF16> { typedef bf16_t T; };

// How a product takes its operands: the number of parts and their type.
template <int DT> struct Logits {  // x and w in the logits
    static constexpr int kParts = DT == kF32 ? 2 : 1;
    static constexpr bool kHalf = DT != kBF16;
};
template <int DT> struct Grads {   // G, w and x in dx and dw
    static constexpr int kParts = DT == kF32 ? 3 : 1;
    static constexpr bool kHalf = DT == kF16;
};

template <int DT>
__device__ __forceinline__ uint16_t half_bits(float v) {
    if constexpr (DT == kF16) return __builtin_bit_cast(uint16_t, (_Float16)v);
    else return __builtin_bit_cast(uint16_t, (__bf16)v);
}

template <int DT>
__device__ __forceinline__ float widen(uint16_t bits) {
    if constexpr (DT == kF16) return (float)__builtin_bit_cast(_Float16, bits);
    else return __builtin_bit_cast(float, (uint32_t)bits << 16);
}

// A value as its matrix operands.  x and w are exact in fp16 and bf16; G,
// computed in fp32, is rounded to nearest even there.  What the rounding of a
// row's largest entry, its target's, takes off is kept and added to dx and dw
// in fp32: their error is then that of their own rounding within 5%, against
// up to 1.5 times as much without (64-bit results, 60 drawn cases).
template <int DT, int PARTS>
__device__ __forceinline__ void to_parts(float v, uint16_t (&o)[PARTS]) {
    if constexpr (PARTS == 3) split3(v, o);
    else if constexpr (PARTS == 2) split2(v, o);
    else o[0] = half_bits<DT>(v);
}

// ---------------------------------------------------------------------------
// What the host lays out in the workspace for one call
// ---------------------------------------------------------------------------
struct Head {          // at the workspace's start, written by the plan kernel
    int live;          // rows whose target is not ignore_index
    float inv_scale;   // undoes the power of two that a and b carry
    int splits;        // of K in dx
};

// ---------------------------------------------------------------------------
// Plan: one block lists the live rows in order, and for the backward their
// coefficients a and b, scaled by a power of two that brings the largest to
// [2^13, 2^14) for fp16: G then loses 2^-39 of the largest at most to the type's
// smallest values.  The others have room below, and need it above, where w or x
// near the type's largest enter the sums: [2^9, 2^10).
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

// Sum of v over the threads before this one, and over all.
__device__ __forceinline__ int block_scan_excl(int v, int* sh, int* total) {
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    int inc = v;
    for (int d = 1; d < 64; d *= 2) {
        const int up = __shfl_up(inc, d, 64);
        inc += lane >= d ? up : 0;
    }
    if (lane == 63) sh[wave] = inc;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        const int t = sh[w];
        before += w < wave ? t : 0;
        all += t;
    }
    *total = all;
    return before + inc - v;
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
    float* lse_out;    // NULL: no backward follows
    // backward
    const float* grad;
    int grad_stride;
    const float* lse_in;
    float z;
    int mean;
    int scale_to;              // the exponent above
    float* a;
    float* b;
    float* lse;
    int tile, tiles_m, steps;  // dx: its tiles, and products of a step's depth of the first piece
    int most_splits;
    int64_t room;              // rows of sums there is room for
    float sum_cost;            // what a split's sums of a row cost at the end, in steps
    int* list;                 // fp16, bf16: live rows by their target's group of 64, in order
    int* list_at;              // [groups + 1]: where a group's rows begin
    int* rest_row;             // [groups * 64]: a target's place among the targets' rows, else -1
    int groups;                // 0: no lists
};

// What a split's start and its sums of a tile cost: a tile is written and read
// at the card's memory rate in about 16 steps.
constexpr int kSplitSteps = 16;

// Splits of K in dx over tiles that fill the chip's places unevenly: the
// number with the least rounds of blocks times steps a block takes, and sums at
// the end.  All lanes of a wave call it.
__device__ __forceinline__ int dx_splits(const PlanArgs& p, int live) {
    const int s = lane_id() + 1;
    const int tiles = p.tiles_m * ((live + p.tile - 1) / p.tile), slots = 256 * (256 / p.tile);
    const bool fits = s <= p.most_splits && (int64_t)s * live <= p.room;
    const float cost = (float)((tiles * s + slots - 1) / slots) * (float)((p.steps + s - 1) / s + kSplitSteps) +
                       p.sum_cost * (float)s * (float)live;
    // the least cost, and the least s of those: positive floats order as their bits
    uint64_t best = fits || s == 1 ? (uint64_t)__builtin_bit_cast(uint32_t, cost) << 32 | (uint32_t)s : ~0ull;
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t other = __shfl_xor(best, d, 64);
        best = other < best ? other : best;
    }
    return (int)(best & 127);
}

__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, reduce_partner<1>(v));
    v = fmaxf(v, reduce_partner<2>(v));
    v = fmaxf(v, reduce_partner<4>(v));
    v = fmaxf(v, reduce_partner<8>(v));
    v = fmaxf(v, reduce_partner<16>(v));
    return fmaxf(v, reduce_partner<32>(v));
}
// Maximum over the block's waves of each wave's v; all threads get it.
template <int THREADS>
__device__ __forceinline__ float block_max(float v, float* sh) {
    v = wave_max(v);
    if (lane_id() == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
    for (int w = 1; w < THREADS / 64; ++w) v = fmaxf(v, sh[w]);
    return v;
}

// Live rows by their targets' groups of 64 vocabulary entries, a wave a group: an
// entry is the live row and, from bit 24, the target's place in its group.
constexpr int kGroup = 64, kSlotShift = 24;
__device__ __forceinline__ void target_lists(const PlanArgs& p, int block) {
    const int group = block * (kPlanThreads / 64) + (int)(threadIdx.x >> 6), lane = lane_id();
    if (group >= p.groups) return;
    const int64_t lo = (int64_t)group * kGroup, hi = lo + kGroup < p.v ? lo + kGroup : p.v;
    constexpr int U = 8;
    auto targets = [&](int64_t r0, int64_t (&t)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) t[u] = r0 + u * 64 + lane < p.n ? p.target[r0 + u * 64 + lane] : p.ignore;
    };
    int before = 0, mine = 0;
    for (int64_t r0 = 0; r0 < p.n; r0 += 64 * U) {
        int64_t t[U];
        targets(r0, t);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = t[u] != p.ignore && t[u] >= 0;
            before += __popcll(__ballot(in && t[u] < lo));
            mine += __popcll(__ballot(in && t[u] >= lo && t[u] < hi));
        }
    }
    if (lane == 0) {
        p.list_at[group] = before;
        if (group == p.groups - 1) p.list_at[p.groups] = before + mine;
    }
    const int begin = before;
    int live = 0;
    bool comes = false;  // this lane's entry of the group is a target
    for (int64_t r0 = 0; mine > 0 && r0 < p.n; r0 += 64 * U) {
        int64_t t[U];
        targets(r0, t);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t below = (1ull << lane) - 1;
            const uint64_t any = __ballot(t[u] != p.ignore);
            const bool in = t[u] != p.ignore && t[u] >= lo && t[u] < hi;
            uint64_t b = __ballot(in);
            for (uint64_t left = b; left; left &= left - 1) {
                const int l = __builtin_ctzll(left);
                comes |= lane == __builtin_amdgcn_readlane((int)(t[u] - lo), l);
            }
            if (in)
                p.list[before + __popcll(b & below)] = (live + __popcll(any & below)) | (int)(t[u] - lo) << kSlotShift;
            before += __popcll(b);
            mine -= __popcll(b);
            live += __popcll(any);
        }
    }
    const uint64_t there = __ballot(comes);
    p.rest_row[lo + lane] = comes ? begin + __popcll(there & ((1ull << lane) - 1)) : -1;
}

// Block 0 makes the plan; blocks after it take the lists.
template <bool BWD>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs p) {
    if (blockIdx.x > 0) {
        target_lists(p, (int)blockIdx.x - 1);
        return;
    }
    __shared__ int sh[kPlanThreads / 64];
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
                if (p.lse_out) p.lse_out[r] = 0.0f;
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
        __shared__ float shf[kPlanThreads / 64];
        big = block_max<kPlanThreads>(big, shf);
        const int e = scale_exp(big, p.scale_to);
        const float scale = __builtin_ldexpf(1.0f, e);
        if (threadIdx.x == 0) p.head->inv_scale = __builtin_ldexpf(1.0f, -e);
        if (threadIdx.x < 64) {
            const int splits = dx_splits(p, live);
            if (threadIdx.x == 0) p.head->splits = splits;
        }
        at = at - mine;
        for (int k = 0; k < mine; ++k) {
            p.a[at + k] *= scale;
            p.b[at + k] *= scale;
        }
    }
    if (threadIdx.x == 0) p.head->live = live;
    if constexpr (!BWD) {
        if (p.lse_out && threadIdx.x < 2) p.lse_out[p.n + threadIdx.x] = 0.0f;
    }
}

// fp32 logits: `undo` takes back both operands' rows' scales (as one step: one of
// the two may leave the type's range where both together do not).
template <int DT>
__device__ __forceinline__ float logit(float acc, int undo) {
    return DT == kF32 ? __builtin_ldexpf(acc, undo) : acc;
}

// ---------------------------------------------------------------------------
// Packing: the live rows of x and a piece's rows of w as 16-bit operands of ldp
// elements (a multiple of 64), zero beyond D; 8 elements a thread at a time.
// ---------------------------------------------------------------------------
struct PackSide {
    const void* src;   // NULL: nothing to pack
    int64_t ld, n;     // rows there are, or may be
    const int* rows;   // x: the live rows
    uint16_t* logits;
    int64_t logits_part;
    // fp32: parts for dx and dw (NULL: not wanted), and a row's undoing exponent
    uint16_t* grads;
    int64_t grads_part;
    int8_t* undo;
};
struct PackArgs {
    PackSide x, w;
    const Head* head;
    int64_t d, ldp;
    int lanes;         // fp32: of a row
    int64_t block0;    // fp16, bf16: blocks of the launches before
};

template <typename T>
__device__ __forceinline__ void load8(const T* src, int64_t left, float (&v)[8]) {
    constexpr int VE = Elem<T>::kVec;
#pragma unroll
    for (int h = 0; h < 8; h += VE) {
        float t[VE];
        load_vec_part<T>(src + h, left - h, 0.0f, t);
#pragma unroll
        for (int k = 0; k < VE; ++k) v[h + k] = t[k];
    }
}

template <int DT, int P>
__device__ __forceinline__ void store_parts(const float (&v)[8], float scale, uint16_t* dst, int64_t part) {
    uint16_t o[8][P];
#pragma unroll
    for (int k = 0; k < 8; ++k) to_parts<DT>(P == 2 ? v[k] * scale : v[k], o[k]);
#pragma unroll
    for (int k = 0; k < P; ++k) {
        u32x4 w;
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = o[2 * q][k] | (uint32_t)o[2 * q + 1][k] << 16;
        *reinterpret_cast<u32x4*>(dst + k * part) = w;
    }
}

// fp16 and bf16.
template <int DT>
__global__ __launch_bounds__(256) void pack(PackArgs p) {
    typedef typename Io<DT>::T T;
    const int64_t chunks = p.ldp / 8;
    int64_t i = (p.block0 + blockIdx.x) * 256 + threadIdx.x;
    const bool is_x = i < p.x.n * chunks;
    const PackSide& s = is_x ? p.x : p.w;
    if (!is_x) i -= p.x.n * chunks;
    const int64_t r = i / chunks, c = i % chunks * 8;
    if (r >= (is_x ? (int64_t)p.head->live : s.n)) return;
    float v[8];
    load8(static_cast<const T*>(s.src) + (s.rows ? (int64_t)s.rows[r] : r) * s.ld + c, p.d - c, v);
    store_parts<DT, 1>(v, 1.0f, s.logits + r * p.ldp + c, s.logits_part);
}

// fp32: a group of lanes, of a wave or (BLOCK) the whole block, takes a row's largest
// finite magnitude, and with it the row's scale, then writes the row for the
// logits and, where `grads` is not NULL, for dx and dw.  The first C of a lane's
// chunks stay in registers; what a row has beyond is read twice, the second time
// from the caches.
template <int C, bool BLOCK>
__global__ __launch_bounds__(256) void pack_f32(PackArgs p) {
    const int lanes = BLOCK ? 256 : p.lanes;
    const int sub = (int)threadIdx.x % lanes;
    int64_t r = (int64_t)blockIdx.x * (256 / lanes) + (int)threadIdx.x / lanes;
    const bool is_x = r < p.x.n;
    const PackSide& s = is_x ? p.x : p.w;
    if (!is_x) r -= p.x.n;
    if (r >= (is_x ? (int64_t)p.head->live : s.n)) return;  // whole groups
    const float* src = static_cast<const float*>(s.src) + (s.rows ? (int64_t)s.rows[r] : r) * s.ld;
    const int64_t first = sub * 8, step = lanes * 8;
    float kept[C][8], big = 0.0f;
    auto take = [&](const float (&v)[8]) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float a = __builtin_fabsf(v[k]);
            big = a < kInf ? fmaxf(big, a) : big;
        }
    };
#pragma unroll
    for (int j = 0; j < C; ++j) load8(src + first + j * step, p.d - first - j * step, kept[j]);
#pragma unroll
    for (int j = 0; j < C; ++j) take(kept[j]);
    for (int64_t c = first + C * step; c < p.ldp; c += step) {
        float v[8];
        load8(src + c, p.d - c, v);
        take(v);
    }
    if constexpr (BLOCK) {
        __shared__ float sh[4];
        big = block_max<256>(big, sh);
    } else {
        for (int d = 1; d < lanes; d *= 2) big = fmaxf(big, __shfl_xor(big, d, 64));
    }
    const int e = scale_exp(big, 15);
    const float scale = __builtin_ldexpf(1.0f, e);
    if (sub == 0) s.undo[r] = (int8_t)-e;
    auto put = [&](int64_t c, const float (&v)[8]) {
        store_parts<kF32, 2>(v, scale, s.logits + r * p.ldp + c, s.logits_part);
        if (s.grads) store_parts<kF32, 3>(v, 1.0f, s.grads + r * p.ldp + c, s.grads_part);
    };
#pragma unroll
    for (int j = 0; j < C; ++j)
        if (first + j * step < p.ldp) put(first + j * step, kept[j]);
    for (int64_t c = first + C * step; c < p.ldp; c += step) {
        float v[8];
        load8(src + c, p.d - c, v);
        put(c, v);
    }
}

// ---------------------------------------------------------------------------
// The products.  Large ones take tiles of 256 x 256 in eight waves of 128 x 64:
// two waves a SIMD, so that one's LDS reads run beside the other's matrix
// instructions.  Ones with too few such tiles take 128 x 128 (two blocks a CU)
// or 64 x 64 in four waves.  Measured, bf16, K-major, us: 8192^3 897 / 957 /
// 1452; (4096, 2048, K 1024) 29.2 / 21.7 / 29.1; (4096, 512, 768) 22.5 / 10.0 /
// 8.6; (1024, 128, 256) 10.4 / 6.2 / 4.0.
// ---------------------------------------------------------------------------
typedef Shape<2, 4, 8, 4> Big;
typedef Shape<2, 2, 4, 4> Mid;
typedef Shape<2, 2, 2, 2> Small;

#define FL_LCE_BUFFERS(S)                                     \
    __shared__ __attribute__((aligned(1024))) char buf0[kBufferBytes<S>]; \
    __shared__ __attribute__((aligned(1024))) char buf1[kBufferBytes<S>]

// A lane's place in the results: that of acc[0][0][0].  PERM: A's rows are
// permuted (acc[i][j][q] is then perm_at(i, q) rows further).
template <class S, bool PERM = false>
struct Place {
    int m, n;
    __device__ __forceinline__ Place(int m0, int n0) {
        const int lane = threadIdx.x & 63, wave = scalar(threadIdx.x >> 6);
        m = m0 + wave % S::WM * (S::FM * 16) + (lane >> 4) * (PERM ? 8 : 4);
        n = n0 + wave / S::WM * (S::FN * 16) + (lane & 15);
    }
};

constexpr int perm_at(int i, int q) { return i / 2 * 32 + i % 2 * 4 + q; }

// fp32: what undoes the scales of a lane's permuted rows of w, perm_at(i, q) from
// `from` on, for FM fragments (past the piece: of no meaning, in the buffer).
// A byte each, since as whole registers they spilled, and loaded before the tile's
// products: at their end the loads stand behind the next tile's, and G of
// (2048, 1024, 16128) took 198 us for 180.
template <int DT, int FM>
struct Undo {
    uint2 e[DT == kF32 ? FM / 2 : 1];
    __device__ __forceinline__ void load(const int8_t* from) {
        if constexpr (DT == kF32) {
#pragma unroll
            for (int i = 0; i < FM; i += 2) e[i / 2] = *reinterpret_cast<const uint2*>(from + perm_at(i, 0));
        }
    }
    // of the lane's result k = 4 i + q
    __device__ __forceinline__ int at(int k) const {
        if constexpr (DT != kF32) return 0;
        const uint32_t word = k & 4 ? e[k / 8].y : e[k / 8].x;
        return (int8_t)(word >> 8 * (k & 3));
    }
};

struct StatArgs {
    Operand w, x;      // M: vocabulary rows, N: live rows
    int steps;
    const Head* head;
    const int* tgt;
    int v0, v;         // the piece's first row, and its rows
    int tiles_m;
    float2* part;      // [live row][parts]: (max, sum)
    int64_t parts;
    float* at_target;  // [live row]
    const int8_t *undo_w, *undo_x;  // fp32: of the piece's rows, of the live rows
};

template <int DT, class S>
struct StatJob {
    StatArgs p;
    int live;
    int tiles_n;

    typedef Side<S, S::TM, true> SA;
    typedef Side<S, S::TN, true> SB;
    struct Rows {
        int target[S::FN], undo_x[DT == kF32 ? S::FN : 1];
        Undo<DT, S::FM> undo_w;
    };
    __device__ __forceinline__ void place(int t, SA& A, SB& B) const {
        const TileAt tile = tile_at(t, p.tiles_m, tiles_n);
        A.template init<true>(p.w, tile.m * S::TM);
        B.init(p.x, tile.n * S::TN);
    }
    __device__ __forceinline__ int first(int) const { return 0; }
    __device__ __forceinline__ int steps(int) const { return p.steps; }
    __device__ __forceinline__ Rows rows(int t) const {
        const TileAt tile = tile_at(t, p.tiles_m, tiles_n);
        const Place<S, true> at(tile.m * S::TM, tile.n * S::TN);
        Rows r;
        r.undo_w.load(p.undo_w + at.m);
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int n = at.n + j * 16;
            r.target[j] = n < live ? p.tgt[n] : -1;
            if constexpr (DT == kF32) r.undo_x[j] = n < live ? p.undo_x[n] : 0;
        }
        return r;
    }
    __device__ __forceinline__ void finish(int t, const Rows& r, const f32x4 (&acc)[S::FM][S::FN]) const {
        const TileAt tile = tile_at(t, p.tiles_m, tiles_n);
        const Place<S, true> at(tile.m * S::TM, tile.n * S::TN);
        const int mw = at.m / (S::FM * 16);
        const int left = p.v - at.m;  // the piece's rows from this lane's first
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int64_t n = at.n + j * 16;
            const int undo_x = DT == kF32 ? r.undo_x[j] : 0;
            const int hit = r.target[j] >= 0 && r.target[j] < p.v0 + p.v ? r.target[j] - p.v0 - at.m : -1;
            float v[S::FM * 4];
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float l = logit<DT>(acc[i][j][q], r.undo_w.at(i * 4 + q) + undo_x);
                    v[i * 4 + q] = perm_at(i, q) < left ? l : -kInf;
                    if (perm_at(i, q) == hit) p.at_target[n] = l;
                }
            float m = -kInf, s = 0.0f;
            lse_fold<true>(m, s, v);
            lse_merge(m, s, exact_xor<16>(m), exact_xor<16>(s));
            lse_merge(m, s, exact_xor<32>(m), exact_xor<32>(s));
            if ((threadIdx.x & 63) < 16 && n < live && mw * (S::FM * 16) < p.v)
                p.part[n * p.parts + mw] = make_float2(m, s);
        }
    }
};

template <int DT, class S>
__global__ __launch_bounds__(S::kThreads, 2) void logits_stats(StatArgs p) {
    FL_LCE_BUFFERS(S);
    StatJob<DT, S> job{p, p.head->live};
    job.p.x.rows = job.live;
    job.tiles_n = (job.live + S::TN - 1) / S::TN;
    run_tiles<S, true, true, Logits<DT>::kHalf, Logits<DT>::kParts>(job, p.tiles_m * job.tiles_n, (lds_char*)buf0,
                                                                    (lds_char*)buf1);
}

// ---------------------------------------------------------------------------
// Few rows (16 in fp16 and bf16, 64 in fp32): bound by reading w once.  Each wave
// takes 32 rows of w after another, 512 bytes of each at a time through two LDS
// buffers of its own, so that a row's loads are consecutive and no wave waits
// for another; x's fragments come from the caches, a stage ahead.  A lane keeps
// one running (max, sum) of its tokens over all its wave's rows.  (8, 2048,
// 128256) in bf16: 87 us, 6.0 TB/s, against 123 us through tiles; without the
// nontemporal hint 102; rows of 256 bytes a load 106.  fp32 is split into bf16
// parts in registers here, which saves writing and reading w's parts.
// ---------------------------------------------------------------------------
struct FewArgs {
    const void* w;
    int64_t ldw;
    const void* x;
    int64_t ldx;
    const int* rows;   // the live ones
    int k, v;          // k: a multiple of 64; fp32: of 4
    const Head* head;
    const int* tgt;
    float2* part;      // [live row][parts]
    int64_t parts;     // the waves
    float* at_target;
};

constexpr int kFewWaves = 2;
// One pass / tiles, us: bf16 (16, 2048, 128256) 99 / 131, 32 rows of it 124 / 123, 64
// 182 / 125 (x's fragments, read for every 32 rows of w, outweigh w); fp32 (16,
// 1024, 32000) 39 / 110, 64 rows 79 / 113.
constexpr int few_rows(int dtype) { return dtype == kF32 ? 64 : 16; }

// split3 of 8 fp32 values, two to a conversion.
__device__ __forceinline__ void split_frag(const f32x4& lo, const f32x4& hi, u32x4 (&o)[3]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float a = q < 2 ? lo[2 * q] : hi[2 * q - 4], b = q < 2 ? lo[2 * q + 1] : hi[2 * q - 3];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const uint32_t u = bf16_pack2(a, b);
            o[p][q] = u;
            a -= __builtin_bit_cast(float, u << 16);
            b -= __builtin_bit_cast(float, u & 0xFFFF0000u);
        }
    }
}

template <int DT, int FN>
__global__ __launch_bounds__(kFewWaves * 64) void logits_few(FewArgs p) {
    typedef typename Io<DT>::T T;
    constexpr bool F32 = DT == kF32;
    constexpr int FM = 2, R = FM * 16, ROW = 512, KC = ROW / (int)sizeof(T), STAGE = R * ROW, LOADS = STAGE / 1024;
    constexpr int KS = KC / 32, XV = F32 ? 2 : 1;  // K of a product; 16-byte vectors of a fragment
    __shared__ __attribute__((aligned(1024))) char lds[kFewWaves * 2 * STAGE];
    const int lane = threadIdx.x & 63, wave = scalar(threadIdx.x >> 6);
    lds_char* mine = (lds_char*)lds + wave * 2 * STAGE;
    const int live = p.head->live;
    const int me = (int)blockIdx.x * kFewWaves + wave, waves = (int)gridDim.x * kFewWaves;
    const int groups = (p.v + R - 1) / R, stages = (p.k + KC - 1) / KC;
    if (live == 0) return;
    const T* x[FN];
    int target[FN];
    float m[FN], s[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = j * 16 + (lane & 15), at = n < live ? n : live - 1;
        x[j] = static_cast<const T*>(p.x) + (int64_t)p.rows[at] * p.ldx;
        target[j] = n < live ? p.tgt[n] : -1;
        m[j] = -kInf;
        s[j] = 0.0f;
    }

    // where the loads are: stage ls of rows lg R ..
    int lg = me, ls = 0;
    const char* base = nullptr;
    uint32_t row[LOADS];
    auto place = [&]() {
        base = uniform(reinterpret_cast<const char*>(static_cast<const T*>(p.w) + (int64_t)lg * R * p.ldw));
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int r = j * 2 + (lane >> 5);
            row[j] = (uint32_t)((lg * R + r < p.v ? r : p.v - 1 - lg * R) * p.ldw * (int)sizeof(T));
        }
    };
    u32x4 next[KS][FN][XV], now[KS][FN][XV];
    auto load = [&](lds_char* buf) {
        const int left = p.k - ls * KC;  // of K, from this stage on
#pragma unroll
        for (int t = 0; t < KS; ++t)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                const int k = t * 32 + (lane >> 4) * 8;
#pragma unroll
                for (int h = 0; h < XV; ++h) {
                    // past K: zero, so that what w's side holds there adds nothing
                    next[t][j][h] = u32x4{0, 0, 0, 0};
                    if (k + h * 4 < left) __builtin_memcpy(&next[t][j][h], x[j] + ls * KC + k + h * 4, 16);
                }
            }
        const char* b = uniform(base + (int64_t)ls * ROW);
        const uint32_t to = scalar((int)(uint32_t)(uintptr_t)buf);
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            // the 16 chunks of 256 bytes permuted by the row number, as in a tile;
            // past K: the row's last chunk
            const int r = j * 2 + (lane >> 5), c = lane & 31;
            int col = ((c & 16) | ((c ^ r) & 15)) * 16;
            const int end = left * (int)sizeof(T);
            if (col > end - 16) col = end - 16;
            load_to_lds<true>(b, row[j] + col, to + j * 1024);
        }
    };
    auto advance = [&]() {
        if (ls + 1 < stages) {
            ++ls;
        } else if (lg + waves < groups) {
            lg += waves;
            ls = 0;
            place();
        }
    };
    // chunk c of row r, in a stage's buffer
    auto chunk = [](const lds_char* buf, int r, int c) {
        return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(buf + r * ROW +
                                                                                 ((c & 16) | ((c ^ r) & 15)) * 16);
    };
    lds_char *cur = mine, *nxt = mine + STAGE;
    if (me < groups) {
        place();
        load(cur);
        advance();
    }
    for (int g = me; g < groups; g += waves) {
        f32x4 acc[FM][FN];
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int st = 0; st < stages; ++st) {
            // the wave's own copies and x's fragments are there, and its reads of the
            // buffer that is filled next are done
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int t = 0; t < KS; ++t)
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int h = 0; h < XV; ++h) {
                        asm volatile("" : "+v"(next[t][j][h]));
                        now[t][j][h] = next[t][j][h];
                    }
            load(nxt);
            advance();
            const int left = p.k - st * KC;
#pragma unroll
            for (int t = 0; t < KS; ++t) {
                if (t * 32 >= left) break;
                u32x4 b[FN][Grads<DT>::kParts];
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    if constexpr (F32)
                        split_frag(__builtin_bit_cast(f32x4, now[t][j][0]), __builtin_bit_cast(f32x4, now[t][j][XV - 1]), b[j]);
                    else b[j][0] = now[t][j][0];
                }
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const int r = i * 16 + (lane & 15);
                    u32x4 a[Grads<DT>::kParts];
                    if constexpr (F32) {
                        const int c = t * 8 + (lane >> 4) * 2;
                        split_frag(__builtin_bit_cast(f32x4, chunk(cur, r, c)), __builtin_bit_cast(f32x4, chunk(cur, r, c + 1)), a);
                    } else {
                        a[0] = chunk(cur, r, t * 4 + (lane >> 4));
                    }
                    constexpr int kTerms = terms(Grads<DT>::kParts);
                    unrolled<kTerms>([&](auto tc) {
                        constexpr int k = decltype(tc)::value;
#pragma unroll
                        for (int j = 0; j < FN; ++j)
                            acc[i][j] = mfma<Grads<DT>::kHalf>(a[term_a(k)], b[j][term_b(k)], acc[i][j]);
                    });
                }
            }
            lds_char* const done = cur;
            cur = nxt;
            nxt = done;
        }
        const int first = g * R + (lane >> 4) * 4;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            float v[FM * 4];
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int at = first + i * 16 + q;
                    v[i * 4 + q] = at < p.v ? acc[i][j][q] : -kInf;
                    if (at == target[j]) p.at_target[j * 16 + (lane & 15)] = acc[i][j][q];
                }
            lse_fold<true>(m[j], s[j], v);
        }
    }
    wait_copies();
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = j * 16 + (lane & 15);
        lse_merge(m[j], s[j], exact_xor<16>(m[j]), exact_xor<16>(s[j]));
        lse_merge(m[j], s[j], exact_xor<32>(m[j]), exact_xor<32>(s[j]));
        if (lane < 16 && n < live) p.part[n * p.parts + me] = make_float2(m[j], s[j]);
    }
}

// Joins a live row's pairs begin .. end - 1; one wave a row.  With `more` pieces to
// come the joined pair goes to the row's first place.
__global__ __launch_bounds__(256) void finish_rows(const Head* head, const int* rows, const int* tgt, float2* part,
                                                   int64_t parts, int64_t begin, int64_t end, bool more,
                                                   const float* at_target, float z, float* loss_rows, float* lse_out) {
    const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= head->live) return;
    const int lane = threadIdx.x & 63;
    float m = -kInf, s = 0.0f;
    // the pairs lie in other XCDs' memory: eight loads a lane in flight
    constexpr int U = 8;
    for (int64_t k0 = begin + lane; k0 < end; k0 += 64 * U) {
        float2 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = k0 + u * 64 < end ? part[r * parts + k0 + u * 64] : make_float2(-kInf, 0.0f);
#pragma unroll
        for (int u = 0; u < U; ++u) lse_merge(m, s, q[u].x, q[u].y);
    }
    group_merge<64>(m, s);
    if (lane == 0) {
        if (more) {
            part[r * parts] = make_float2(m, s);
            return;
        }
        const float lse = lse_finish<true>(m, s);
        const int row = rows[r];
        if (lse_out) lse_out[row] = lse;
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
    int steps;
    const Head* head;
    const int* tgt;
    const float *a, *b, *lse;
    int v0, v;           // the piece: vocabulary rows v0 .. v - 1 are w's rows 0 ..
    int tiles_m;
    uint16_t* g;         // [live row][ldg]
    int64_t ldg, g_part;
    const int8_t *undo_w, *undo_x;  // fp32: of the piece's rows, of the live rows
    float* rest;         // fp16, bf16: [live row] what rounding took off the target's entry
};

// G of a piece.  Rows from the live ones up to a multiple of 64 are zero, and so
// are columns up to the tiles' end: the products' K runs over whole steps.
template <int DT, class S>
struct GradJob {
    GradArgs p;
    int live;
    int tiles_n;

    typedef Side<S, S::TM, true> SA;
    typedef Side<S, S::TN, true> SB;
    struct Rows {
        int target[S::FN], undo_x[DT == kF32 ? S::FN : 1];
        Undo<DT, S::FM> undo_w;
        float a[S::FN], b[S::FN], lse[S::FN];
    };
    __device__ __forceinline__ void place(int t, SA& A, SB& B) const {
        const TileAt tile = tile_at(t, p.tiles_m, tiles_n);
        A.template init<true>(p.w, tile.m * S::TM);
        B.init(p.x, tile.n * S::TN);
    }
    __device__ __forceinline__ int first(int) const { return 0; }
    __device__ __forceinline__ int steps(int) const { return p.steps; }
    __device__ __forceinline__ Rows rows(int t) const {
        const TileAt tile = tile_at(t, p.tiles_m, tiles_n);
        const Place<S, true> at(tile.m * S::TM, tile.n * S::TN);
        Rows r;
        r.undo_w.load(p.undo_w + at.m);
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int64_t n = at.n + j * 16;
            const bool in = n < live;
            r.target[j] = in ? p.tgt[n] : -1;
            r.a[j] = in ? p.a[n] : 0.0f;
            r.b[j] = in ? p.b[n] : 0.0f;
            r.lse[j] = in ? p.lse[n] : 0.0f;
            if constexpr (DT == kF32) r.undo_x[j] = in ? p.undo_x[n] : 0;
        }
        return r;
    }
    __device__ __forceinline__ void finish(int t, const Rows& r, const f32x4 (&acc)[S::FM][S::FN]) const {
        constexpr int P = Grads<DT>::kParts;
        const TileAt tile = tile_at(t, p.tiles_m, tiles_n);
        const Place<S, true> at(tile.m * S::TM, tile.n * S::TN);
        const int n_end = (live + kStep - 1) / kStep * kStep;
        const int left = p.v - p.v0 - at.m;  // the piece's rows from this lane's first
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int64_t n = at.n + j * 16;
            const int hit = r.target[j] >= 0 ? r.target[j] - p.v0 - at.m : -1;
            // rows past the live ones have a = 0, but an exponential of anything
            const int cols = n < live ? left : 0;
            const int undo_x = DT == kF32 ? r.undo_x[j] : 0;
            float hit_g = 0.0f;
#pragma unroll
            for (int i = 0; i < S::FM; i += 2) {
                uint16_t o[8][P];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const int m = perm_at(i, q);  // q runs over both fragments
                    float g = r.a[j] * fexp2((logit<DT>(acc[i + q / 4][j][q % 4], r.undo_w.at(i * 4 + q) + undo_x) - r.lse[j]) * kLog2e);
                    if (m == hit) hit_g = g += r.b[j];
                    to_parts<DT>(m < cols ? g : 0.0f, o[q]);
                }
                if (n < n_end) {
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        u32x4 u;
#pragma unroll
                        for (int q = 0; q < 4; ++q) u[q] = o[2 * q][k] | (uint32_t)o[2 * q + 1][k] << 16;
                        *reinterpret_cast<u32x4*>(p.g + k * p.g_part + n * p.ldg + at.m + i * 16) = u;
                    }
                }
            }
            if constexpr (DT != kF32) {
                // of the rows that a lane's results cover: hit is one of them
                if (hit >= 0 && hit < S::FM * 16 && hit % 32 < 8)
                    p.rest[n] = hit_g - widen<DT>(half_bits<DT>(hit_g));
            }
        }
    }
};

template <int DT, class S>
__global__ __launch_bounds__(S::kThreads, 2) void logits_grad(GradArgs p) {
    FL_LCE_BUFFERS(S);
    GradJob<DT, S> job{p, p.head->live};
    job.p.x.rows = job.live;
    job.tiles_n = (job.live + S::TN - 1) / S::TN;
    run_tiles<S, true, true, Logits<DT>::kHalf, Logits<DT>::kParts>(job, p.tiles_m * job.tiles_n, (lds_char*)buf0,
                                                                    (lds_char*)buf1);
}

struct ProductArgs {
    Operand a, b;       // M and N rows
    const Head* head;
    int steps;          // of K; dw: the live rows'
    int m, n;           // results
    int tiles_m;
    float* acc;         // [split][live row, or row of the piece][ldc] fp32 sums
    int64_t ldc;
    int add;            // dx: the sums are added to
    int splits;         // dw's
    void* out;          // dw: [n][ldc] results
    // dw in fp16, bf16: result row n is also wanted in fp32, at this place (-1: not)
    float* rests;
    const int* rest_row;
};

// kDx: C[n][d] = sum_v G[n][v] w[v][d] over a piece, added to the splits' sums.
// kDw: C[v][d] = sum_n G[n][v] x[n][d], the piece's rows of the result; in
// kDwSplit the splits' sums of them.
enum Mode { kDx, kDw, kDwSplit };
template <int DT, class S, int MODE>
struct ProductJob {
    static constexpr bool DX = MODE == kDx, SUMS = MODE != kDw;
    ProductArgs p;
    int n_end, tiles_n, tiles, splits;
    float inv;
    bool whole;  // four results of a lane are one store

    typedef typename Io<DT>::T T;
    typedef Side<S, S::TM, false> SA;
    typedef Side<S, S::TN, DX> SB;
    static constexpr bool kRests = MODE == kDw && DT != kF32;
    struct Rows {
        int rest[kRests ? S::FN : 1];
    };
    __device__ __forceinline__ int split(int t) const { return SUMS ? scalar((unsigned)t / (unsigned)tiles) : 0; }
    __device__ __forceinline__ TileAt at(int t) const { return tile_at(t - split(t) * tiles, p.tiles_m, tiles_n); }
    // K's steps are cut evenly
    __device__ __forceinline__ int first(int t) const {
        return SUMS ? scalar((unsigned)(p.steps * split(t)) / (unsigned)splits) : 0;
    }
    __device__ __forceinline__ int steps(int t) const {
        return SUMS ? scalar((unsigned)(p.steps * (split(t) + 1)) / (unsigned)splits) - first(t) : p.steps;
    }
    __device__ __forceinline__ void place(int t, SA& A, SB& B) const {
        const TileAt tile = at(t);
        A.init(p.a, tile.m * S::TM);
        B.init(p.b, tile.n * S::TN);
    }
    __device__ __forceinline__ Rows rows(int t) const {
        Rows r{};
        if constexpr (kRests) {
            const Place<S> at(0, this->at(t).n * S::TN);
#pragma unroll
            for (int j = 0; j < S::FN; ++j) r.rest[j] = at.n + j * 16 < n_end ? p.rest_row[at.n + j * 16] : -1;
        }
        return r;
    }
    __device__ __forceinline__ void finish(int t, const Rows& r, const f32x4 (&acc)[S::FM][S::FN]) const {
        const TileAt tile = at(t);
        const Place<S> at(tile.m * S::TM, tile.n * S::TN);
        float* sums = SUMS ? p.acc + (int64_t)split(t) * n_end * p.ldc : nullptr;
#pragma unroll
        for (int j = 0; j < S::FN; ++j) {
            const int64_t n = at.n + j * 16;
            if (n >= n_end) continue;
#pragma unroll
            for (int i = 0; i < S::FM; ++i) {
                const int64_t m = at.m + i * 16;
                if (m >= p.m) continue;
                f32x4 v = acc[i][j];
                if constexpr (SUMS) {
                    float* c = sums + n * p.ldc + m;
                    if (whole) {
                        if (DX && p.add) v += *reinterpret_cast<const f32x4*>(c);
                        *reinterpret_cast<f32x4*>(c) = v;
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (m + q < p.m) c[q] = DX && p.add ? c[q] + v[q] : v[q];
                    }
                } else {
                    T* c = static_cast<T*>(p.out) + n * p.ldc + m;
                    if constexpr (kRests) {
                        if (r.rest[j] >= 0) {
                            float* f = p.rests + r.rest[j] * p.ldc + m;
                            if (whole) {
                                *reinterpret_cast<f32x4*>(f) = v;
                            } else {
#pragma unroll
                                for (int q = 0; q < 4; ++q)
                                    if (m + q < p.m) f[q] = v[q];
                            }
                        }
                    }
                    v *= inv;
                    if (whole && sizeof(T) == 4) {
                        *reinterpret_cast<f32x4*>(c) = v;
                    } else if (whole) {
                        uint16_t o[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) o[q] = half_bits<DT>(v[q]);
                        uint2 u;
                        u.x = o[0] | (uint32_t)o[1] << 16;
                        u.y = o[2] | (uint32_t)o[3] << 16;
                        *reinterpret_cast<uint2*>(c) = u;
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (m + q < p.m) Elem<T>::put(c + q, v[q]);
                    }
                }
            }
        }
    }
};

template <int DT, class S, int MODE>
__global__ __launch_bounds__(S::kThreads, 2) void product(ProductArgs p) {
    FL_LCE_BUFFERS(S);
    constexpr bool DX = MODE == kDx;
    const int live = p.head->live;
    ProductJob<DT, S, MODE> job{p};
    if constexpr (DX) {
        job.p.b.rows = live;
        job.n_end = live;
    } else {
        job.p.steps = (live + kStep - 1) / kStep;
        job.p.a.rows = live;
        job.p.b.rows = job.p.steps * kStep;
        job.n_end = p.n;
    }
    // no split without a step: a short last piece of dx adds to the first ones
    const int splits = DX ? p.head->splits : MODE == kDwSplit ? p.splits : 1;
    job.splits = splits < job.p.steps ? splits : job.p.steps;
    job.tiles_n = (job.n_end + S::TN - 1) / S::TN;
    job.tiles = p.tiles_m * job.tiles_n;
    job.inv = p.head->inv_scale;
    job.whole = (p.ldc & 3) == 0;
    if (MODE == kDw && live == 0) {  // no step of K: dw is zero
        f32x4 none[S::FM][S::FN] = {};
        for (Walk w(job.tiles); w.t < w.end; w.t += w.stride) job.finish(w.t, job.rows(w.t), none);
        return;
    }
    run_tiles<S, false, DX, Grads<DT>::kHalf, Grads<DT>::kParts>(job, job.tiles * (MODE == kDw ? 1 : job.splits),
                                                                 (lds_char*)buf0, (lds_char*)buf1);
}

// dw's rows that are targets: the product's fp32 sums and, for each of the
// target's rows in order, rest times x.  A wave a group of 64 entries, 256 columns
// and every `parts`-th of the group's targets.
struct RestArgs {
    const Head* head;
    const float* rest;
    const int *list, *list_at, *rest_row;
    const uint16_t* x;   // packed live rows
    int64_t ldx;
    int d, group0, cols, parts;  // cols: blocks of 256 columns
    const float* rests;  // [place][d]
    void* dw;            // [vocabulary entry][d]
};
template <int DT>
__global__ __launch_bounds__(64) void finish_targets(RestArgs p) {
    typedef typename Io<DT>::T T;
    const int group = p.group0 + (int)blockIdx.x, lane = lane_id();
    const int part = (int)blockIdx.y / p.cols, c = (int)blockIdx.y % p.cols * 256 + lane * 4;
    const int begin = p.list_at[group], end = p.list_at[group + 1];
    if (begin == end) return;
    const int place = p.rest_row[group * kGroup + lane];
    const float inv = p.head->inv_scale;
    // packed rows are whole multiples of 64 elements; past them: not stored
    const uint16_t* x = p.x + (c < p.ldx ? c : 0);
    int at = 0;
    for (uint64_t left = __ballot(place >= 0); left; left &= left - 1, ++at) {
        if (at % p.parts != part) continue;
        const int slot = __builtin_ctzll(left);
        const float* base = p.rests + (int64_t)__builtin_amdgcn_readlane(place, slot) * p.d + c;
        f32x4 s;
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] = c + q < p.d ? base[q] : 0.0f;
        for (int e0 = begin; e0 < end; e0 += 64) {
            const int e = e0 + lane < end ? p.list[e0 + lane] : -1;
            const bool mine = e >= 0 && e >> kSlotShift == slot;
            const int row = e & ((1 << kSlotShift) - 1);
            const float rest = mine ? p.rest[row] : 0.0f;
            uint64_t hits = __ballot(mine);
            // a number of rows' loads at a time (16 where a target comes often: (16384,
            // 768, 32000) in bf16, half of the rows the same target, 4.64 ms in all for
            // 5.22 with 4); past the hits: a rest of 0
            auto add = [&](auto rows) {
                constexpr int R = decltype(rows)::value;
                uint2 u[R];
                float f[R];
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    const int l = hits ? __builtin_ctzll(hits) : 0;
                    f[k] = hits ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, rest), l)) : 0.0f;
                    const int r = hits ? __builtin_amdgcn_readlane(row, l) : 0;
                    hits &= hits - 1;
                    u[k] = *reinterpret_cast<const uint2*>(x + (int64_t)r * p.ldx);
                }
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    if (f[k] == 0.0f) continue;  // and what row 0 holds adds nothing
                    s[0] += f[k] * widen<DT>((uint16_t)u[k].x);
                    s[1] += f[k] * widen<DT>((uint16_t)(u[k].x >> 16));
                    s[2] += f[k] * widen<DT>((uint16_t)u[k].y);
                    s[3] += f[k] * widen<DT>((uint16_t)(u[k].y >> 16));
                }
            };
            while (__popcll(hits) > 4) add(std::integral_constant<int, 16>{});
            if (hits) add(std::integral_constant<int, 4>{});
        }
        T* to = static_cast<T*>(p.dw) + (int64_t)(group * kGroup + slot) * p.d + c;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (c + q < p.d) Elem<T>::put(to + q, s[q] * inv);
    }
}

// dw rows of a piece from the splits' sums; targets' sums go to `rests` as they
// are.
template <int DT>
__global__ __launch_bounds__(256) void finish_dw(const Head* head, const float* acc, int splits, int64_t rows, int64_t d,
                                                 void* dw, const int* rest_row, float* rests) {
    typedef typename Io<DT>::T T;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * d) return;
    // a split of no step wrote nothing
    const int steps = (head->live + kStep - 1) / kStep;
    splits = splits < steps ? splits : steps;
    float s = 0.0f;
    for (int k = 0; k < splits; ++k) s += acc[k * rows * d + i];
    if constexpr (DT != kF32) {
        const int place = rest_row[i / d];
        if (place >= 0) rests[place * d + i % d] = s;
    }
    Elem<T>::put(static_cast<T*>(dw) + i, s * head->inv_scale);
}

// dx rows from the splits' sums, and what rounding took off the targets' entries;
// ignored rows are zero.  Q columns a thread: 4 where rows of sums are whole
// 16-byte vectors.
template <int DT, int Q>
__global__ __launch_bounds__(256) void finish_dx(const Head* head, const int* pos, const float* acc, int64_t d, void* dx,
                                                 const float* rest, const int* tgt, const void* w, int64_t ldw) {
    typedef typename Io<DT>::T T;
    typedef float vec __attribute__((ext_vector_type(Q)));
    const int64_t r = blockIdx.x;
    const int at = pos[r];
    const float inv = head->inv_scale;
    const int splits = head->splits;
    const int64_t stride = head->live * d;
    const int target = at >= 0 && DT != kF32 ? tgt[at] : -1;
    const float more = target >= 0 ? rest[at] : 0.0f;
    const T* wt = static_cast<const T*>(w) + target * ldw;
    for (int64_t c = (int64_t)threadIdx.x * Q; c < d; c += 256 * Q) {
        vec s = (vec)(0.0f);
        if (at >= 0) {
            const float* from = acc + at * d + c;
#pragma unroll 4
            for (int k = 0; k < splits; ++k) s += *reinterpret_cast<const vec*>(from + k * stride);
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                if (target >= 0) s[q] += more * Elem<T>::scalar(wt + c + q);
                s[q] *= inv;
            }
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) Elem<T>::put(static_cast<T*>(dx) + r * d + c + q, s[q]);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
constexpr int64_t div_up(int64_t v, int64_t by) { return (v + by - 1) / by; }

// G of a piece takes at most this many bytes: enough vocabulary rows for the
// products to fill the chip, and a workspace that stays small beside w.  Training
// calls with 128 / 256 / 512 / 1024 MB, us: bf16 (4096, 2048, 128256) 5055 / 5034 /
// 4999 / 4862; fp32 (2048, 1024, 32000) 2399 / 1974 / 1952 / 1953.
constexpr int64_t kPieceBytes = 256 << 20;

struct Layout {
    int64_t piece;       // vocabulary rows of a piece, a multiple of 256
    int64_t ldx;         // a packed row of x and w
    bool pack_w;         // w is packed a piece at a time
    int splits;          // of K in dx, with every row live
    int64_t room;        // rows of its sums
    int few;             // forward of few rows: its blocks, or 0
    int logits, dx, dw;  // the products' tiles: 256, 128 or 64
    bool join;           // forward: a row's pairs are joined after every piece
    int dw_splits;
    int64_t head, rows, pos, tgt, at_target, loss_rows, part, parts, a, b, lse, xp, xg, wp, wg, undo_x, undo_w, rest, list,
        list_at, rest_row, rests, dw_acc, g, acc, bytes;
};

// A product's tiles: the largest that fill most of the chip (both sides beside the
// shapes: 128 tiles of 256 29.2 us, as 512 of 128 21.7; 128 of 128 10.0, as 512 of
// 64 8.6).
int tile_size(int64_t m, int64_t n) {
    if (n > 128 && div_up(m, 256) * div_up(n, 256) >= 192) return 256;
    return div_up(m, 128) * div_up(n, 128) >= 200 ? 128 : 64;
}

// Tiles and splits of K of dx or dw, m x n results of `steps` of K, as dx_splits
// chooses them with every row live.
void split_plan(int64_t m, int64_t n, int64_t steps, int terms, int& tile, int& splits) {
    double best = 0.0;
    for (int t = 256; t >= 64; t /= 2) {
        const int64_t tiles = div_up(m, t) * div_up(n, t), slots = 256 * (256 / t);
        // a step of a tile in 1/256 of the chip, by the times beside the shapes
        const double step = t == 256 ? 1.0 : t == 128 ? 0.55 : 0.4;
        for (int s = 1; s <= 64 && s <= steps; ++s) {
            const double c = div_up(tiles * s, slots) * step * (div_up(steps * terms, s) + kSplitSteps);
            if (best == 0.0 || c < best) {
                best = c;
                tile = t;
                splits = s;
            }
        }
    }
}

// aligned: w's rows can be read as matrix operands where they are.
// alone: a forward that no backward follows.  One that is followed takes the tiles
// also for few rows: the backward makes its logits again, and they have to be
// the ones its lse was taken of, to the bit, where a probability is near 1.
Layout layout(int64_t N, int64_t V, int64_t D, int dtype, bool bwd, bool alone, bool aligned) {
    Layout l{};
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    const int64_t lparts = dtype == kF32 ? 2 : 1, parts = dtype == kF32 ? 3 : 1;
    int64_t most = kPieceBytes / (2 * parts * round_up(N, 64)) / 256 * 256;
    if (most < 2048) most = 2048;
    l.ldx = round_up(D, 64);
    if (alone && N <= few_rows(dtype) && aligned && D % (dtype == kF32 ? 4 : 64) == 0) {
        const int64_t blocks = div_up(div_up(V, 32), kFewWaves);
        l.few = (int)(blocks < 512 ? blocks : 512);
    }
    l.pack_w = !l.few && (dtype == kF32 || !aligned || D % 64 != 0);
    if (l.pack_w) {
        const int64_t fit = kPieceBytes / (2 * parts * l.ldx) / 256 * 256;
        if (most > fit) most = fit < 2048 ? 2048 : fit;
    } else if (!bwd) {
        most = V;
    }
    // A forward's pairs, 8 bytes for each row and half tile, cover the vocabulary
    // where they fit, and else one piece beside the join of those before.  (Tiles of
    // 64 never have that many.)
    if (!bwd && !l.few && 8 * N * div_up(V, tile_size(V, N) / 2) > kPieceBytes) {
        l.join = true;
        const int64_t fit = kPieceBytes / (8 * N) * (N > 128 ? 128 : 64) / 256 * 256;
        if (most > fit) most = fit < 2048 ? 2048 : fit;
    }
    l.piece = round_up(div_up(V, div_up(V, most)), 256);
    l.head = take(sizeof(Head));
    l.rows = take(4 * N);
    l.pos = take(4 * N);
    l.tgt = take(4 * N);
    l.xp = take(l.few ? 0 : 2 * lparts * N * l.ldx);
    l.wp = take(l.pack_w ? 2 * lparts * l.piece * l.ldx : 0);
    l.undo_x = take(dtype == kF32 && !l.few ? N : 0);
    l.undo_w = take(dtype == kF32 && !l.few ? l.piece : 0);
    l.logits = tile_size(l.piece, N);
    if (!bwd) {
        l.parts = l.few ? l.few * kFewWaves : l.join ? 1 + l.piece / (l.logits / 2) : div_up(V, l.logits / 2);
        l.at_target = take(4 * N);
        l.loss_rows = take(4 * N);
        l.part = take(8 * N * l.parts);
    } else {
        split_plan(D, N, l.piece / kStep, terms((int)parts), l.dx, l.splits);
        split_plan(D, l.piece, div_up(N, kStep), terms((int)parts), l.dw, l.dw_splits);
        // without splits a partly filled round of large tiles is the better one:
        // (2047, 768, 50257) in fp16, 591 tiles of 256 in three rounds: dw 221 us;
        // 2358 of 128 in five shorter ones: 258
        if (l.dw_splits == 1) l.dw = tile_size(D, l.piece);
        l.a = take(4 * N);
        l.b = take(4 * N);
        l.lse = take(4 * N);
        l.rest = take(4 * N);
        l.list = take(4 * N);
        l.list_at = take(4 * (div_up(V, kGroup) + 1));
        l.rest_row = take(4 * round_up(V, kGroup));
        l.rests = take(dtype == kF32 ? 0 : 4 * N * D);
        l.dw_acc = take(l.dw_splits > 1 ? 4 * l.dw_splits * l.piece * D : 0);
        // fp32: x and w again in the gradients' parts
        l.xg = dtype == kF32 ? take(2 * parts * N * l.ldx) : l.xp;
        l.wg = dtype == kF32 ? take(2 * parts * l.piece * l.ldx) : l.wp;
        l.g = take(2 * parts * round_up(N, 64) * l.piece);
        // room for more splits where fewer rows are live
        const int64_t rows = kPieceBytes / (4 * D);
        l.room = l.splits * N > rows ? l.splits * N : rows > 64 * N ? 64 * N : rows;
        l.acc = take(4 * l.room * D);
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

// Operands of x and of rows v0 .. of w: for the logits, and for dw and dx.
struct Operands {
    Operand x, xg, w, wg;
};

// Packs what has to be packed for the piece at v0 (x with the first piece) and
// sets up its operands.
template <int DT>
void operands(const Call& c, const Layout& l, int64_t v0, int64_t rows, bool dx, bool dw, Operands& o) {
    typedef typename Io<DT>::T T;
    const T* w = static_cast<const T*>(c.w) + v0 * c.ldw;
    PackArgs p{};
    p.head = at<Head>(c, l.head);
    p.d = c.D;
    p.ldp = l.ldx;
    if (v0 == 0) {
        const int64_t part = c.N * l.ldx;
        uint16_t* to = at<uint16_t>(c, l.xp);
        o.x = o.xg = Operand{to, l.ldx, part, (int)c.N, l.ldx};
        p.x = PackSide{c.x, c.ldx, c.N, at<int>(c, l.rows), to, part, nullptr, part, at<int8_t>(c, l.undo_x)};
        if (DT == kF32 && dw) p.x.grads = at<uint16_t>(c, l.xg);
        if (DT == kF32) o.xg.p = p.x.grads;
    }
    if (l.pack_w) {
        const int64_t part = l.piece * l.ldx;
        uint16_t* to = at<uint16_t>(c, l.wp);
        o.w = o.wg = Operand{to, l.ldx, part, (int)rows, l.ldx};
        p.w = PackSide{w, c.ldw, rows, nullptr, to, part, nullptr, part, at<int8_t>(c, l.undo_w)};
        if (DT == kF32 && dx) p.w.grads = at<uint16_t>(c, l.wg);
        if (DT == kF32) o.wg.p = p.w.grads;
    } else {
        o.w = o.wg = Operand{reinterpret_cast<const uint16_t*>(w), c.ldw, 0, (int)rows, l.ldx};
    }
    const int64_t packed = p.x.n + p.w.n;
    if (packed == 0) return;
    if constexpr (DT == kF32) {
        // By a wave / a block a row, us: (2921, 3776) for the logits alone 21.0 / 17.1,
        // with the gradients' parts 30.7 / 24.4.  One / two chunks a lane, whole
        // forwards: (513, 64, 32000) 40.6 / 41.3, (500, 768, 50257) 192 / 188.
        if (l.ldx > 1024) {
            pack_f32<2, true><<<dim3((unsigned)packed), 256, 0, c.s>>>(p);
            return;
        }
        p.lanes = 8;  // a row is 64 elements at least
        while (p.lanes < 64 && p.lanes * 8 < l.ldx) p.lanes *= 2;
        const dim3 grid((unsigned)div_up(packed * p.lanes, 256));
        if (l.ldx <= 512) pack_f32<1, false><<<grid, 256, 0, c.s>>>(p);
        else pack_f32<2, false><<<grid, 256, 0, c.s>>>(p);
    } else {
        for_grid_chunks(div_up(packed * (l.ldx / 8), 256), 256, [&](int64_t first, int64_t count) {
            p.block0 = first;
            pack<DT><<<dim3((unsigned)count), 256, 0, c.s>>>(p);
        });
    }
}

// Blocks for `tiles` tiles: no more than run at a time, in multiples of 8.
template <class S>
dim3 grid_of(int64_t tiles) {
    constexpr int64_t most = 256 * (S::TM == 256 ? 1 : S::TM == 128 ? 2 : 4);
    return dim3((unsigned)(tiles < most ? round_up(tiles, 8) : most));
}

// Calls f with the shape of `tile`.
template <typename F>
void by_shape(int tile, F f) {
    if (tile == 256) f(Big{});
    else if (tile == 128) f(Mid{});
    else f(Small{});
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
void run_fwd(const Call& c, const Layout& l, float* loss, float* lse) {
    PlanArgs p = plan_args(c, l);
    p.loss_rows = c.reduction == 0 ? loss : at<float>(c, l.loss_rows);
    p.lse_out = lse;
    plan_kernel<false><<<1, kPlanThreads, 0, c.s>>>(p);
    Operands o{};
    auto finish = [&](int64_t begin, int64_t end, bool more) {
        finish_rows<<<dim3((unsigned)div_up(c.N, 4)), 256, 0, c.s>>>(p.head, p.rows, p.tgt, at<float2>(c, l.part), l.parts,
                                                                     begin, end, more, at<float>(c, l.at_target), c.z,
                                                                     p.loss_rows, lse);
    };
    const int64_t half = l.logits / 2;
    for (int64_t v0 = 0; v0 < c.V; v0 += l.piece) {
        const int64_t rows = c.V - v0 < l.piece ? c.V - v0 : l.piece;
        if (l.few) {
            const FewArgs f{c.w,    c.ldw,  c.x,   c.ldx, p.rows,  (int)c.D, (int)c.V,
                            p.head, p.tgt, at<float2>(c, l.part), l.parts, at<float>(c, l.at_target)};
            const dim3 grid((unsigned)l.few), block(kFewWaves * 64);
            if constexpr (DT == kF32) {
                if (c.N > 32) logits_few<DT, 4><<<grid, block, 0, c.s>>>(f);
                else if (c.N > 16) logits_few<DT, 2><<<grid, block, 0, c.s>>>(f);
                else logits_few<DT, 1><<<grid, block, 0, c.s>>>(f);
            } else {
                logits_few<DT, 1><<<grid, block, 0, c.s>>>(f);
            }
            break;  // one piece
        }
        operands<DT>(c, l, v0, rows, false, false, o);
        StatArgs a{};
        a.w = o.w;
        a.x = o.x;
        a.undo_w = at<int8_t>(c, l.undo_w);
        a.undo_x = at<int8_t>(c, l.undo_x);
        a.steps = (int)(l.ldx / kStep);
        a.head = p.head;
        a.tgt = p.tgt;
        a.v0 = (int)v0;
        a.v = (int)rows;
        a.part = at<float2>(c, l.part) + (l.join ? 1 : v0 / half);
        a.parts = l.parts;
        a.at_target = at<float>(c, l.at_target);
        by_shape(l.logits, [&](auto shape) {
            typedef decltype(shape) S;
            a.tiles_m = (int)div_up(rows, S::TM);
            logits_stats<DT, S><<<grid_of<S>(div_up(c.N, S::TN) * a.tiles_m), S::kThreads, 0, c.s>>>(a);
        });
        if (l.join) finish(v0 == 0, 1 + div_up(rows, half), v0 + rows < c.V);
    }
    if (!l.join) finish(0, l.parts, false);
    if (c.reduction != 0) reduce_rows<<<1, 1024, 0, c.s>>>(p.head, p.loss_rows, c.N, p.mean, loss);
}

template <int DT>
void run_bwd(const Call& c, const Layout& l, const float* grad, const float* lse, void* dx, void* dw) {
    typedef typename Io<DT>::T T;
    PlanArgs p = plan_args(c, l);
    p.grad = grad;
    p.grad_stride = c.reduction == 0 ? 1 : 0;
    p.lse_in = lse;
    p.scale_to = DT == kF16 ? 14 : 10;
    p.a = at<float>(c, l.a);
    p.b = at<float>(c, l.b);
    p.lse = at<float>(c, l.lse);
    p.tile = l.dx;
    p.tiles_m = (int)div_up(c.D, l.dx);
    p.most_splits = (int)div_up(c.V < l.piece ? c.V : l.piece, kStep);
    p.steps = p.most_splits * terms(Grads<DT>::kParts);
    // a row's sums, 4 D bytes, at about 5 TB/s, once for all pieces; a step takes
    // about 1.35 us
    p.sum_cost = (float)((double)c.D * 4 / (5e12 * 1.35e-6) / (double)div_up(c.V, l.piece));
    p.room = l.room;
    p.list = at<int>(c, l.list);
    p.list_at = at<int>(c, l.list_at);
    p.rest_row = at<int>(c, l.rest_row);
    p.groups = DT != kF32 && dw ? (int)div_up(c.V, kGroup) : 0;
    const int64_t beside = div_up(p.groups, kPlanThreads / 64);
    plan_kernel<true><<<dim3((unsigned)(1 + beside)), kPlanThreads, 0, c.s>>>(p);
    Operands o{};
    const int64_t g_part = round_up(c.N, 64) * l.piece;
    for (int64_t v0 = 0; v0 < c.V; v0 += l.piece) {
        const int64_t rows = c.V - v0 < l.piece ? c.V - v0 : l.piece;
        operands<DT>(c, l, v0, rows, dx != nullptr, dw != nullptr, o);
        GradArgs g{};
        g.w = o.w;
        g.x = o.x;
        g.undo_w = at<int8_t>(c, l.undo_w);
        g.undo_x = at<int8_t>(c, l.undo_x);
        g.rest = at<float>(c, l.rest);
        g.steps = (int)(l.ldx / kStep);
        g.head = p.head;
        g.tgt = p.tgt;
        g.a = p.a;
        g.b = p.b;
        g.lse = p.lse;
        g.v0 = (int)v0;
        g.v = (int)(v0 + rows);
        g.g = at<uint16_t>(c, l.g);
        g.ldg = l.piece;
        g.g_part = g_part;
        by_shape(l.logits, [&](auto shape) {
            typedef decltype(shape) S;
            g.tiles_m = (int)div_up(rows, S::TM);
            logits_grad<DT, S><<<grid_of<S>(div_up(c.N, S::TN) * g.tiles_m), S::kThreads, 0, c.s>>>(g);
        });
        ProductArgs a{};
        a.head = p.head;
        a.m = (int)c.D;
        a.ldc = c.D;
        a.rests = at<float>(c, l.rests);
        a.rest_row = p.rest_row + v0;
        if (dx) {
            a.a = o.wg;
            a.b = Operand{g.g, l.piece, g_part, (int)c.N, l.piece};
            a.steps = (int)div_up(rows, kStep);
            a.n = (int)c.N;
            a.acc = at<float>(c, l.acc);
            a.add = v0 > 0;
            by_shape(l.dx, [&](auto shape) {
                typedef decltype(shape) S;
                a.tiles_m = (int)div_up(c.D, S::TM);
                product<DT, S, kDx><<<grid_of<S>((int64_t)a.tiles_m * (div_up(c.N, S::TN) * l.splits + 64)), S::kThreads, 0, c.s>>>(a);
            });
        }
        if (dw) {
            a.a = o.xg;
            a.b = Operand{g.g, l.piece, g_part, 0, l.piece};
            a.n = (int)rows;
            a.out = static_cast<T*>(dw) + v0 * c.D;
            a.acc = at<float>(c, l.dw_acc);
            a.splits = l.dw_splits;
            by_shape(l.dw, [&](auto shape) {
                typedef decltype(shape) S;
                a.tiles_m = (int)div_up(c.D, S::TM);
                const int64_t tiles = (int64_t)a.tiles_m * div_up(rows, S::TN);
                if (a.splits > 1) product<DT, S, kDwSplit><<<grid_of<S>(tiles * a.splits), S::kThreads, 0, c.s>>>(a);
                else product<DT, S, kDw><<<grid_of<S>(tiles), S::kThreads, 0, c.s>>>(a);
            });
            if (a.splits > 1)
                finish_dw<DT><<<dim3((unsigned)div_up(rows * c.D, 256)), 256, 0, c.s>>>(
                    p.head, a.acc, a.splits, rows, c.D, a.out, a.rest_row, a.rests);
            if constexpr (DT != kF32) {
                // many rows a group (small vocabularies): its targets in 16 waves.
                // (2469, 64, 125) in bf16: 162 us for 412 in one; with fewer rows than
                // that most waves would find no target.  A grid has 65535 rows.
                const int cols = (int)div_up(c.D, 256);
                const int parts = c.N * kGroup > 128 * c.V && cols <= 65535 / 16 ? 16 : 1;
                finish_targets<DT><<<dim3((unsigned)div_up(rows, kGroup), (unsigned)(cols * parts)), 64, 0, c.s>>>(
                    RestArgs{p.head, g.rest, p.list, p.list_at, p.rest_row, o.x.p, o.x.ld, (int)c.D, (int)(v0 / kGroup),
                             cols, parts, a.rests, dw});
            }
        }
    }
    if (dx) {
        auto finish = [&](auto q) {
            finish_dx<DT, decltype(q)::value><<<dim3((unsigned)c.N), 256, 0, c.s>>>(
                p.head, p.pos, at<float>(c, l.acc), c.D, dx, at<float>(c, l.rest), p.tgt, c.w, c.ldw);
        };
        if (c.D % 4 == 0) finish(std::integral_constant<int, 4>{});
        else finish(std::integral_constant<int, 1>{});
    }
}

// w's rows can be read as operands where they are: 16-byte loads at 16-byte
// addresses, and a tile's rows within 32-bit offsets.
bool is_aligned(const void* w, int64_t ldw, int dtype) {
    return (reinterpret_cast<uintptr_t>(w) & 15u) == 0 && ldw % (dtype == kF32 ? 4 : 8) == 0 && ldw <= (1 << 22);
}

int check(const char* name, const Call& c, int dtype, size_t ws_bytes, bool bwd, bool alone) {
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
    const int64_t need = layout(c.N, c.V, c.D, dtype, bwd, alone, is_aligned(c.w, c.ldw, dtype)).bytes;
    FL_CHECK((int64_t)ws_bytes >= need, "%s: workspace of %llu bytes, %lld needed", name, (unsigned long long)ws_bytes,
             (long long)need);
    FL_CHECK(c.ws && (reinterpret_cast<uintptr_t>(c.ws) & 255u) == 0, "%s: workspace is not 256-byte aligned", name);
    return ok();
}

}  // namespace
}  // namespace lce
}  // namespace fl

using namespace fl::lce;

extern "C" size_t fl_linear_ce_workspace_bytes(int64_t N, int64_t V, int64_t D, int dtype, int pass,
                                               const void* w, int64_t ldw) {
    if (N < 1 || V < 1 || D < 1 || dtype < 0 || dtype > 2 || pass < 0 || pass > 2 || N > (1 << 23) || V > (1 << 28) ||
        D > (1 << 20))
        return 0;
    return (size_t)layout(N, V, D, dtype, pass == 2, pass == 0, is_aligned(w, ldw, dtype)).bytes;
}

extern "C" int fl_linear_ce_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* target,
                                int64_t N, int64_t V, int64_t D, int dtype, int64_t ignore_index, float z_loss,
                                int reduction, float* loss, float* lse, void* workspace, size_t workspace_bytes,
                                void* stream) {
    const Call c{x,      ldx, w, ldw, target, N, V, D, ignore_index, z_loss, reduction, static_cast<char*>(workspace),
                 static_cast<hipStream_t>(stream)};
    const int rc = check("fl_linear_ce_fwd", c, dtype, workspace_bytes, false, !lse);
    if (rc != FL_OK || N == 0) return rc;
    FL_CHECK(loss, "fl_linear_ce_fwd: NULL pointer argument");
    const Layout l = layout(N, V, D, dtype, false, !lse, is_aligned(c.w, c.ldw, dtype));
    if (dtype == kF32) run_fwd<kF32>(c, l, loss, lse);
    else if (dtype == kF16) run_fwd<kF16>(c, l, loss, lse);
    else run_fwd<kBF16>(c, l, loss, lse);
    return fl::launch_status("fl_linear_ce_fwd");
}

extern "C" int fl_linear_ce_bwd(const float* grad, const void* x, int64_t ldx, const void* w, int64_t ldw,
                                const int64_t* target, const float* lse, int64_t N, int64_t V, int64_t D, int dtype,
                                int64_t ignore_index, float z_loss, int reduction, void* dx, void* dw,
                                void* workspace, size_t workspace_bytes, void* stream) {
    const Call c{x,      ldx, w, ldw, target, N, V, D, ignore_index, z_loss, reduction, static_cast<char*>(workspace),
                 static_cast<hipStream_t>(stream)};
    const int rc = check("fl_linear_ce_bwd", c, dtype, workspace_bytes, true, false);
    if (rc != FL_OK || N == 0) return rc;
    FL_CHECK(grad && lse, "fl_linear_ce_bwd: NULL pointer argument");
    if (!dx && !dw) return fl::ok();
    const Layout l = layout(N, V, D, dtype, true, false, is_aligned(c.w, c.ldw, dtype));
    if (dtype == kF32) run_bwd<kF32>(c, l, grad, lse, dx, dw);
    else if (dtype == kF16) run_bwd<kF16>(c, l, grad, lse, dx, dw);
    else run_bwd<kBF16>(c, l, grad, lse, dx, dw);
    return fl::launch_status("fl_linear_ce_bwd");
}

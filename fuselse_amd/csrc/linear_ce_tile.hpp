// The matrix-core tile product of the linear cross entropy (linear_ce.hip):
// C[m][n] += sum_k A[m][k] B[n][k] for one tile of TM x TN results per block.
//
// Operands are 16-bit and may lie either way round in memory, so that no
// matrix is transposed in HBM: K-major (rows of K, as x and w in the logits) or
// row-major across K (K rows of the tile's M or N entries, as w in dx = G w).
// Both are copied to LDS as they lie by 16-byte direct-to-LDS loads, 64 of K a
// step, into two buffers in turn.  K-major fragments are 16-byte LDS reads; the
// others come through ds_read_b64_tr_b16, which hands each lane four
// consecutive K entries of its column.  The 16-byte chunks of an LDS row are
// permuted by an exclusive or with bits of the row number, so that the lanes
// that one cycle of a read serves meet different banks (counted: no conflict
// cycle in either kind of read); the loads' lane addresses apply the
// permutation, since a direct-to-LDS load writes its lanes' data in lane order.
//
// A block takes one tile after another, and its loads run ahead of its products
// across tiles: while a tile's results are written, the next tile's first steps
// arrive.  A step is four phases of a quarter of its products each (one half of K, one
// half of the wave's rows).  A phase's fragments are read during the phase
// before, and the loads for the step after next are spread over two phases,
// one behind every few matrix instructions: issued together they stall a wave
// for as long as half a step's products take.  One barrier a step, before the
// phase that first reads the next buffer.
//
// Measured at 8192^3 in bf16: 830 us, 1324 TFLOP/s (the library's product:
// 849 us); with all of a step's loads issued at its start 870 us, with v_mfma
// 32x32x16 in place of 16x16x32 7% more.  In the logits of (4096, 4096, 32000) the
// matrix pipes are busy 72% of cycles.
#pragma once

#include <type_traits>
#include <utility>

#include "linear_ce.hpp"

namespace fl {
namespace lce {

constexpr int kStep = 64;  // K of a step

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(1))) const char glb_char;

template <bool HALF>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
}

// Starts a copy of 16 bytes a lane from base + off to LDS at lds + 16 lane; base
// and lds are the wave's.  It has no register result; what reads the LDS
// bytes first waits for vmcnt and a barrier.  Written as assembly because the
// compiler, which cannot tell the two step buffers apart at every read, put a
// wait for all copies in flight before reads of the other buffer.
template <bool NT = false>
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t off, uint32_t lds) {
    // The compiler does not see what the assembly is, so the wait states it would
    // put in are written out: one from m0's write, and five from a vector
    // instruction's write of base's registers (readfirstlane) to their use as
    // an address.
    if constexpr (NT)  // nontemporal: data that is read once
        asm volatile(
            "s_nop 4\n\t"
            "global_load_lds_dwordx4 %1, %2 nt"
            :
            : "{m0}"(lds), "v"(off), "s"(base)
            : "memory");
    else
        asm volatile(
            "s_nop 4\n\t"
            "global_load_lds_dwordx4 %1, %2"
            :
            : "{m0}"(lds), "v"(off), "s"(base)
            : "memory");
}
// A value all lanes share, in scalar registers.
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const char* uniform(const char* p) {
    const uint64_t u = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
    return (const char*)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <int N, typename F, int... I>
__device__ __forceinline__ void unrolled_(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
// f(integral_constant 0), .., f(integral_constant N - 1)
template <int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
    unrolled_<N>(f, std::make_integer_sequence<int, N>{});
}

// WM x WN waves of FM x FN results of 16 x 16 each.
template <int WM_, int WN_, int FM_, int FN_>
struct Shape {
    static constexpr int WM = WM_, WN = WN_, FM = FM_, FN = FN_;
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int TM = WM * FM * 16, TN = WN * FN * 16;
};

// One operand's side of a tile: T rows of it, K-major (KMAJOR) or across K.
template <class S, int T, bool KMAJOR>
struct Side {
    static constexpr int kBytes = T * kStep * 2;
    static constexpr int kLoads = kBytes / (S::kThreads * 16);  // a thread and step
    static constexpr int kRowBytes = KMAJOR ? kStep * 2 : T * 2;

    const char* base;   // uniform: the tile's first row at k = 0 (K-major), column at k = 0 (across)
    int64_t part;       // bytes between an fp32 operand's parts
    int64_t step;       // bytes a step of K advances
    int64_t ld;         // bytes a row
    int rows;           // across: K rows there are
    uint32_t off[kLoads];

    // K-major: rows of the operand past its last are read as the last.  With
    // PERM the side's fragments hold its rows in another order, that of
    // perm_row.  Across: columns past the last whole chunk are read as that chunk.
    template <bool PERM = false>
    __device__ __forceinline__ void init(const Operand& o, int64_t first) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        part = o.part * 2;
        ld = o.ld * 2;
        if constexpr (KMAJOR) {
            base = reinterpret_cast<const char*>(o.p) + first * ld;
            step = kStep * 2;
            rows = 0;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                int64_t r = (j * S::kWaves + wave) * 8 + (lane >> 3);
                if (PERM) r = perm_row((int)r);
                if (first + r >= o.rows) r = o.rows - 1 - first;
                off[j] = (uint32_t)(r * ld) + ((lane & 7) ^ (lane >> 3)) * 16;
            }
        } else {
            base = reinterpret_cast<const char*>(o.p) + first * 2;
            step = kStep * ld;
            rows = o.rows;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) off[j] = (uint32_t)(krow(j) * ld) + col(j, first, o.cols);
        }
    }
    // Row r of LDS, of fragment i of a wave's, is row
    // 32 (i / 2) + 8 (r % 16 / 4) + 4 (i % 2) + r % 4 of the wave's: two fragments'
    // results of a lane are 8 consecutive rows of C, and the four lanes that
    // share a column hold 32: whole 64-byte stores of 16-bit results.
    __device__ __forceinline__ static int perm_row(int r) {
        const int w = r % (S::FM * 16), i = w / 16;
        return r - w + i / 2 * 32 + w % 16 / 4 * 8 + i % 2 * 4 + w % 4;
    }
    // across: the permutation of K row k's chunks.  The 32 lanes that a cycle of
    // a transposing read serves hold 2 chunks each of K rows 0 .. 3 and of those
    // 8 or 16 further; their 16 chunks have to differ in the 256 bytes that the
    // banks span, in which a row of 64 has a half of its own.
    __device__ __forceinline__ static int swz(int k) {
        const int far = ((k >> 3) ^ (k >> 4)) & 1;
        if constexpr (T == 64) return (k & 2) | (far << 2);
        else return ((k & 3) << 1) | (far << 3);
    }
    // across: the K row and the column's byte of this lane's chunk in load j
    __device__ __forceinline__ static int krow(int j) {
        return ((j * S::kWaves + (int)(threadIdx.x >> 6)) * 1024 + (int)(threadIdx.x & 63) * 16) / kRowBytes;
    }
    __device__ __forceinline__ static uint32_t col(int j, int64_t first, int64_t cols) {
        const int slot = (int)(threadIdx.x & 63) * 16 % kRowBytes / 16;
        int64_t c = (slot ^ swz(krow(j))) * 8;
        if (first + c > cols - 8) c = cols - 8 - first;
        return (uint32_t)(c * 2);  // never before the row: first < cols
    }

    // Starts load J of step k (of part p) into buf.  Where the K rows end inside
    // the step, those past the last are read as the last.
    template <int J>
    __device__ __forceinline__ void load(lds_char* buf, int k, int p) const {
        const char* b = uniform(base + k * step + p * part);
        const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)buf + (threadIdx.x >> 6) * 1024);
        uint32_t o = off[J];
        if (!KMAJOR && (k + 1) * kStep > rows) {
            const int last = rows - 1 - k * kStep;
            o -= krow(J) > last ? (uint32_t)((krow(J) - last) * ld) : 0u;
        }
        load_to_lds(b, o, lds + J * S::kWaves * 1024);
    }

    // Fragment of 16 rows from row0 (a multiple of 16) and K half kk.
    __device__ __forceinline__ static u32x4 frag(const lds_char* buf, int row0, int kk) {
        const int lane = threadIdx.x & 63;
        if constexpr (KMAJOR) {
            const int chunk = (kk * 4 + (lane >> 4)) ^ (lane & 7);
            return *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(buf + (row0 + (lane & 15)) * 128 +
                                                                                     chunk * 16);
        } else {
            const int i = lane & 15;
            const int k = kk * 32 + (lane >> 4) * 8 + (i >> 2);
            const int m = row0 + (i & 3) * 4;
            const int at = k * kRowBytes + ((m >> 3) ^ swz(k)) * 16 + (m & 7) * 2;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(buf + at));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(buf + at + 4 * kRowBytes));
            struct { s16x4 a, b; } both = {lo, hi};
            return __builtin_bit_cast(u32x4, both);
        }
    }
};

// The tiles a block takes, of `total` in the order of tile_at.  The dispatcher
// deals blocks to the 8 XCDs in turn; each XCD has an eighth of the tiles, in
// one run, and its blocks take consecutive ones at a time.
struct Walk {
    int t, end, stride;
    __device__ __forceinline__ explicit Walk(int total) {
        const int xcd = blockIdx.x & 7;
        end = (int)((xcd + 1) * (int64_t)total / 8);
        stride = (int)(gridDim.x / 8);
        t = (int)(xcd * (int64_t)total / 8) + (int)(blockIdx.x >> 3);
    }
};
// Tile t's place among tiles_m x tiles_n: down columns of 4 in M before a step in
// N, so that the 32 tiles an XCD runs at a time read 4 row strips and 8 column
// strips.  In scalar registers, which the compiler's division does not keep to.
struct TileAt {
    int m, n;
};
__device__ __forceinline__ TileAt tile_at(int t, int tiles_m, int tiles_n) {
    constexpr int kRows = 4;
    const int group = scalar((int)((unsigned)t / (unsigned)(kRows * tiles_n))), first = group * kRows;
    const int gm = tiles_m - first < kRows ? tiles_m - first : kRows;
    const int r = t - group * kRows * tiles_n;
    const int n = scalar((int)((unsigned)r / (unsigned)gm));
    return {first + r - n * gm, n};
}

// Bytes of one step's buffer.
template <class S>
constexpr int kBufferBytes = (S::TM + S::TN) * kStep * 2;

// Runs a block's tiles.  job.place(t, A, B) sets up tile t's sides; job.first(t)
// and job.steps(t), at least one, are its steps of K; job.rows(t) loads what its results need;
// job.finish(t, rows, acc) takes them.  acc[i][j][q] of a lane is
// C[wm + 16 i + 4 (lane / 16) + q][wn + 16 j + lane % 16] of the tile, or, where A
// was set up with PERM, C[wm + 32 (i / 2) + 8 (lane / 16) + 4 (i % 2) + q][..], with
// (wm, wn) the wave's corner.
template <class S, bool AK, bool BK, bool HALF, int PARTS, class Job>
__device__ __forceinline__ void run_tiles(const Job& job, int total, lds_char* buf0, lds_char* buf1) {
    typedef Side<S, S::TM, AK> SA;
    typedef Side<S, S::TN, BK> SB;
    constexpr int TERMS = terms(PARTS);
    constexpr int kLoads = SA::kLoads + SB::kLoads, kHalf = kLoads / 2;
    constexpr int H = S::FM / 2;
    static_assert(S::FM % 2 == 0 && kLoads >= 2, "phases take half of a wave's rows");
    typedef std::integral_constant<int, 0> C0;
    typedef std::integral_constant<int, kHalf> CHalf;
    typedef std::integral_constant<int, kLoads - kHalf> CRest;

    Walk walk(total);
    if (walk.t >= walk.end) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % S::WM * (S::FM * 16), wn = wave / S::WM * (S::FN * 16);

    // where the loads are: step ls of tile lt
    SA A;
    SB B;
    int lt = walk.t, ls = 0;
    int lk0 = job.first(lt), ln = job.steps(lt) * TERMS;
    job.place(lt, A, B);
    // loads J0 .. J0 + N - 1 of that step
    auto load = [&](auto j0, auto n, lds_char* buf) {
        const int k = lk0 + (TERMS > 1 ? scalar((unsigned)ls / TERMS) : ls);
        const int t = TERMS > 1 ? ls - (k - lk0) * TERMS : 0;
        unrolled<decltype(n)::value>([&](auto i) {
            constexpr int J = decltype(j0)::value + decltype(i)::value;
            if constexpr (J < SA::kLoads) A.template load<J>(buf, k, term_a(t));
            else B.template load<J - SA::kLoads>(buf + SA::kBytes, k, term_b(t));
        });
    };
    // to the next step; past the last one it is loaded again, and not used
    auto advance = [&]() {
        if (ls + 1 < ln) {
            ++ls;
        } else if (lt + walk.stride < walk.end) {
            lt += walk.stride;
            ls = 0;
            lk0 = job.first(lt);
            ln = job.steps(lt) * TERMS;
            job.place(lt, A, B);
        }
    };

    f32x4 acc[S::FM][S::FN];
    u32x4 fa[2][H], fb[2][S::FN];
    auto read_a = [&](const lds_char* buf, auto p, int i) {
        constexpr int P = decltype(p)::value;
        fa[P & 1][i] = SA::frag(buf, wm + ((P & 1) * H + i) * 16, P >> 1);
    };
    auto read_b = [&](const lds_char* buf, auto p, int j) {
        constexpr int P = decltype(p)::value;
        fb[P >> 1][j] = SB::frag(buf + SA::kBytes, wn + j * 16, P >> 1);
    };
    // Phase P: its products, with the reads of the phase after it (from rd) and
    // loads J0 .. J0 + N - 1 (to ld) between them, in this order.
    auto phase = [&](auto p, const lds_char* rd, auto j0, auto n, lds_char* ld) {
        constexpr int P = decltype(p)::value, Q = (P + 1) & 3;
        typedef std::integral_constant<int, Q> CQ;
        unrolled<H>([&](auto ic) {
            constexpr int i = decltype(ic)::value, N = decltype(n)::value;
            read_a(rd, CQ{}, i);
            if constexpr ((Q & 1) == 0) {
#pragma unroll
                for (int j = i * S::FN / H; j < (i + 1) * S::FN / H; ++j) read_b(rd, CQ{}, j);
            }
#pragma unroll
            for (int j = 0; j < S::FN; ++j)
                acc[(P & 1) * H + i][j] = mfma<HALF>(fa[P & 1][i], fb[P >> 1][j], acc[(P & 1) * H + i][j]);
            constexpr int first = i * N / H, count = (i + 1) * N / H - first;
            if constexpr (count > 0)
                load(std::integral_constant<int, decltype(j0)::value + first>{}, std::integral_constant<int, count>{}, ld);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // A step in cur.  The loads of the step after next begin in phase 3, when
    // every wave has read cur, and end in phase 0 of the next step.
    auto step = [&](lds_char* cur, lds_char* nxt) {
        phase(C0{}, cur, CHalf{}, CRest{}, nxt);
        advance();
        phase(std::integral_constant<int, 1>{}, cur, C0{}, C0{}, nxt);
        phase(std::integral_constant<int, 2>{}, cur, C0{}, C0{}, nxt);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        phase(std::integral_constant<int, 3>{}, nxt, C0{}, CHalf{}, cur);
    };

    load(C0{}, std::integral_constant<int, kLoads>{}, buf0);
    advance();
    load(C0{}, CHalf{}, buf1);
    wait_copies();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < H; ++i) read_a(buf0, C0{}, i);
#pragma unroll
    for (int j = 0; j < S::FN; ++j) read_b(buf0, C0{}, j);
    // one copy of the step for both buffers: with one for each, the compiler kept
    // two sets of accumulators
    lds_char *cur = buf0, *nxt = buf1;
    for (; walk.t < walk.end; walk.t += walk.stride) {
        const auto rows = job.rows(walk.t);
        const int steps = job.steps(walk.t) * TERMS;
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int j = 0; j < S::FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < steps; ++s) {
            step(cur, nxt);
            lds_char* const done = cur;
            cur = nxt;
            nxt = done;
        }
        job.finish(walk.t, rows, acc);
    }
    wait_copies();
}

}  // namespace lce
}  // namespace fl

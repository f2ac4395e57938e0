// The matrix-core tile product of the linear cross entropy (linear_ce.hip):
// C[m][n] += sum_k A[m][k] B[n][k] for one tile of TM x TN results per block.
//
// Operands are 16-bit and may lie either way round in memory, so that no
// matrix is transposed in HBM: K-major (rows of K, as x and w in the logits) or
// row-major across K (K rows of the tile's M or N entries, as w in dx = G w).
// Both are copied to LDS as they lie by 16-byte direct-to-LDS loads, 64 of K a
// step, two steps' buffers in turn: while a step's products run, the next
// step's loads are in flight, and one barrier a step orders them.  K-major
// fragments are 16-byte LDS reads; the others come through ds_read_b64_tr_b16,
// which hands each lane four consecutive K entries of its column.  The 16-byte
// chunks of an LDS row are permuted by an exclusive or with the row number, so
// that the lanes of one read meet different banks; the loads' lane addresses
// apply it, since a direct-to-LDS load writes its lanes' data in lane order.
#pragma once

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
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t off, uint32_t lds) {
    // The compiler does not see what the assembly is, so the wait states it would
    // put in are written out: one from m0's write, and five from a vector
    // instruction's write of base's registers (readfirstlane) to their use as
    // an address.
    asm volatile(
        "s_nop 4\n\t"
        "global_load_lds_dwordx4 %1, %2"
        :
        : "{m0}"(lds), "v"(off), "s"(base)
        : "memory");
}
// A value all lanes share, in scalar registers.
__device__ __forceinline__ const char* uniform(const char* p) {
    const uint64_t u = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
    return (const char*)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

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

    // K-major: rows of the operand past its last are read as the last.
    // Across: columns past the last whole chunk are read as that chunk.
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
    // across: the K row and the column's byte of this lane's chunk in load j
    __device__ __forceinline__ static int krow(int j) {
        return ((j * S::kWaves + (int)(threadIdx.x >> 6)) * 1024 + (int)(threadIdx.x & 63) * 16) / kRowBytes;
    }
    __device__ __forceinline__ static uint32_t col(int j, int64_t first, int64_t cols) {
        const int slot = (int)(threadIdx.x & 63) * 16 % kRowBytes / 16;
        int64_t c = (slot ^ ((krow(j) & 3) << 1)) * 8;
        if (first + c > cols - 8) c = cols - 8 - first;
        return (uint32_t)(c * 2);  // never before the row: first < cols
    }

    // Starts the loads of step k (and part p) into buf.  `ragged`: the K rows
    // end inside this step; those past the last are read as the last.
    __device__ __forceinline__ void load(lds_char* buf, int64_t k, int p) const {
        const char* b = uniform(base + k * step + p * part);
        const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)buf + (threadIdx.x >> 6) * 1024);
        const bool ragged = !KMAJOR && (k + 1) * kStep > rows;
        const int last = rows - 1 - (int)(k * kStep);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            uint32_t o = off[j];
            if (ragged) o -= krow(j) > last ? (uint32_t)((krow(j) - last) * ld) : 0u;
            load_to_lds(b, o, lds + j * S::kWaves * 1024);
        }
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
            const int at = k * kRowBytes + ((m >> 3) ^ ((i >> 2) << 1)) * 16 + (m & 7) * 2;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(buf + at));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(buf + at + 4 * kRowBytes));
            struct { s16x4 a, b; } both = {lo, hi};
            return __builtin_bit_cast(u32x4, both);
        }
    }
};

// Tile t of tiles_m x tiles_n, counted so that blocks that run together share
// operands: the dispatcher deals blocks to the 8 XCDs in turn, so block b
// takes tile (b mod 8) total / 8 + b / 8, consecutive tiles of one XCD; and tiles
// go down columns of 4 in M before they step in N, so that the 32 tiles an XCD
// runs at a time read 4 row strips and 8 column strips.
__device__ __forceinline__ int64_t xcd_tile(int64_t b, int64_t total) {
    const int64_t per = total / 8;
    return b < per * 8 ? (b & 7) * per + (b >> 3) : b;
}
__device__ __forceinline__ void tile_at(int64_t t, int64_t tiles_m, int64_t tiles_n, int64_t& m, int64_t& n) {
    constexpr int64_t kGroup = 4;
    const int64_t group = t / (kGroup * tiles_n), first = group * kGroup;
    const int64_t gm = tiles_m - first < kGroup ? tiles_m - first : kGroup;
    const int64_t r = t - group * kGroup * tiles_n;
    m = first + r % gm;
    n = r / gm;
}

// Bytes of one step's buffer.
template <class S>
constexpr int kBufferBytes = (S::TM + S::TN) * kStep * 2;

// acc[i][j][q] of a lane is C[wm + 16 i + 4 (lane / 16) + q][wn + 16 j + lane % 16]
// of the tile, with (wm, wn) the wave's corner.
template <class S, bool AK, bool BK, bool HALF, int PARTS>
__device__ __forceinline__ void tile_product(const Side<S, S::TM, AK>& A, const Side<S, S::TN, BK>& B, int64_t k0,
                                             int64_t k1, f32x4 (&acc)[S::FM][S::FN], lds_char* buf0, lds_char* buf1) {
    typedef Side<S, S::TM, AK> SA;
    typedef Side<S, S::TN, BK> SB;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % S::WM * (S::FM * 16), wn = wave / S::WM * (S::FN * 16);
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int TERMS = PARTS == 3 ? kTerms : 1;
    const int64_t steps = (k1 - k0) * TERMS;
    auto load = [&](lds_char* buf, int64_t s) {
        if constexpr (PARTS == 3) {
            const int64_t k = k0 + s / kTerms;
            const int t = (int)(s % kTerms);
            A.load(buf, k, kTermA[t]);
            B.load(buf + SA::kBytes, k, kTermB[t]);
        } else {
            A.load(buf, k0 + s, 0);
            B.load(buf + SA::kBytes, k0 + s, 0);
        }
    };
    auto compute = [&](const lds_char* buf) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 fa[S::FM], fb[S::FN];
#pragma unroll
            for (int j = 0; j < S::FN; ++j) fb[j] = SB::frag(buf + SA::kBytes, wn + j * 16, kk);
#pragma unroll
            for (int i = 0; i < S::FM; ++i) fa[i] = SA::frag(buf, wm + i * 16, kk);
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int j = 0; j < S::FN; ++j) acc[i][j] = mfma<HALF>(fa[i], fb[j], acc[i][j]);
        }
    };
    if (steps <= 0) return;
    load(buf0, 0);
    for (int64_t s = 0; s < steps; s += 2) {
        wait_copies();
        __syncthreads();
        if (s + 1 < steps) load(buf1, s + 1);
        compute(buf0);
        if (s + 1 >= steps) break;
        wait_copies();
        __syncthreads();
        if (s + 2 < steps) load(buf0, s + 2);
        compute(buf1);
    }
    __syncthreads();
}

}  // namespace lce
}  // namespace fl

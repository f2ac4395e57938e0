// Stable counting sort of entries by a small key (at most 1025 bins), for the
// experts' order and, digit by digit, for an embedding's gradient.
//
// A block takes 4096 entries in their order, a wave 256 of them, 64 at a time.
// Lanes of equal keys find each other with a ballot a key bit; a lane's place
// among its wave's entries of that key is the wave's count so far plus the lanes
// below it, so nothing depends on the order of atomics.  Up to 4096 entries one
// block does it all; beyond, one launch counts and one places, with one between them
// that sums the blocks' counts where there are many.
#pragma once

#include "lse_common.hpp"

namespace fl {
namespace key_sort {

constexpr int kWaves = 16, kThreads = 64 * kWaves, kRounds = 4, kChunk = kThreads * kRounds;
constexpr int kMaxBins = 1025;

template <int BINS = kMaxBins>
struct Shared {
    int base[kWaves * BINS];  // entries of a bin in the waves before
    int start[BINS];          // place of a bin's first entry of this block
    int waves[kWaves];
};

// Key bits that `bins` bins take.
inline int bits_of(int bins) {
    int b = 0;
    while ((1 << b) < bins) ++b;
    return b;
}

inline int64_t chunks(int64_t n) { return (n + kChunk - 1) / kChunk; }

// Entry that round j of this thread takes, of the block's.
template <int ROUNDS = kRounds>
__device__ __forceinline__ int entry(int j) {
    return ((int)(threadIdx.x >> 6) * ROUNDS + j) * 64 + (int)(threadIdx.x & 63);
}

// Places of the block's n entries (key[j] of entry(j)) among those of their bin
// in their wave; sh.base then holds the waves' counts before.  total[j] becomes
// the block's count of bin threadIdx.x + j * kThreads.
template <int BINS, int ROUNDS>
__device__ __forceinline__ void rank(Shared<BINS>& sh, const int (&key)[ROUNDS], int n, int bins, int bits,
                                     int (&place)[ROUNDS], int (&total)[2]) {
    const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    for (int b = threadIdx.x; b < kWaves * bins; b += kThreads) sh.base[b] = 0;
    __syncthreads();
    int* mine = sh.base + wave * bins;
    const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
        place[j] = 0;
        if ((wave * ROUNDS + j) * 64 >= n) continue;  // the same for all of the wave
        const bool live = entry<ROUNDS>(j) < n;
        uint64_t same = __ballot(live);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((key[j] >> b) & 1);
            same &= (key[j] >> b) & 1 ? set : ~set;
        }
        if (live) {
            const int before = __popcll(same & below), all = __popcll(same);
            const int old = __hip_atomic_load(mine + key[j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
            place[j] = old + before;
            // lanes run together, so all of a key have read before one writes
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (before == all - 1)
                __hip_atomic_store(mine + key[j], old + all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int b = (int)threadIdx.x + j * kThreads;
        int s = 0;
        if (b < bins) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const int c = sh.base[w * bins + b];
                sh.base[w * bins + b] = s;
                s += c;
            }
        }
        total[j] = s;
    }
}

// Sum over the threads below of v; all is the sum over all of them.
template <int BINS>
__device__ __forceinline__ int scan(Shared<BINS>& sh, int v, int& all) {
    const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    int s = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(s, d, 64);
        if (lane >= d) s += o;
    }
    __syncthreads();
    if (lane == 63) sh.waves[wave] = s;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const int c = sh.waves[w];
        if (w < wave) before += c;
        all += c;
    }
    return before + s - v;
}

// The bins' starts, from the counts over all entries of this thread's bins
// (threadIdx.x and kThreads, of which there is at most the one).
template <int BINS>
__device__ __forceinline__ void starts(Shared<BINS>& sh, const int (&total)[2], int bins, int (&start)[2]) {
    int all;
    start[0] = scan(sh, (int)threadIdx.x < bins ? total[0] : 0, all);
    start[1] = all;
}

// What the blocks beyond the entries' do in the same launch: nothing.
struct NoWork {
    __device__ __forceinline__ void operator()(int64_t) const {}
};

// Blocks' counts of their entries: hist[block * bins + bin].
template <typename Key, typename Work>
__global__ __launch_bounds__(kThreads) void count_kernel(Key key, int64_t n, int bins, int* hist, Work work) {
    __shared__ int count[kMaxBins];
    const int64_t first = (int64_t)blockIdx.x * kChunk;
    if (first >= n) return work((int64_t)blockIdx.x - (n + kChunk - 1) / kChunk);
    const int m = (int)(n - first < kChunk ? n - first : kChunk);
    for (int b = threadIdx.x; b < bins; b += kThreads) count[b] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kRounds; ++j)
        if (entry(j) < m) atomicAdd(&count[key(first + entry(j))], 1);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) hist[(int64_t)blockIdx.x * bins + b] = count[b];
}

// Blocks' counts of which every placing block makes the sums itself: beyond, a
// launch for the sums costs less (3 us, as 16 blocks' counts do).
constexpr int kFewBlocks = 16;

// Over the blocks, 64 bins a block in 16 runs of blocks: counts become the sums of
// those before, total[bin] the sum of all.
static __global__ __launch_bounds__(kThreads) void sum_kernel(int* hist, int blocks, int bins, int* total) {
    __shared__ int sh[kWaves][64];
    const int lane = (int)threadIdx.x & 63, run = (int)threadIdx.x >> 6, bin = (int)blockIdx.x * 64 + lane;
    const int per = (blocks + kWaves - 1) / kWaves;
    const int first = run * per, last = first + per < blocks ? first + per : blocks;
    int s = 0;
    if (bin < bins)
#pragma unroll 8
        for (int b = first; b < last; ++b) s += hist[(int64_t)b * bins + bin];
    sh[run][lane] = s;
    __syncthreads();
    if (bin >= bins) return;
    int before = 0;
    for (int r = 0; r < run; ++r) before += sh[r][lane];
#pragma unroll 8
    for (int b = first; b < last; ++b) {
        const int v = hist[(int64_t)b * bins + bin];
        hist[(int64_t)b * bins + bin] = before;
        before += v;
    }
    if (run == kWaves - 1) total[bin] = before;
}

// The counts of this thread's bins over all blocks and over those before this one.
// With few blocks hist holds their counts, else the sums of those before and total
// the sums of all.
__device__ __forceinline__ void load_counts(const int* hist, const int* total, int blocks, int bins, int (&all)[2],
                                            int (&before)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int b = (int)threadIdx.x + j * kThreads;
        all[j] = before[j] = 0;
        if (b >= bins) continue;
        if (blocks <= kFewBlocks) {
#pragma unroll
            for (int k = 0; k < kFewBlocks; ++k) {
                const int v = k < blocks ? hist[(int64_t)k * bins + b] : 0;
                before[j] += k < (int)blockIdx.x ? v : 0;
                all[j] += v;
            }
        } else {
            all[j] = total[b];
            before[j] = hist[(int64_t)blockIdx.x * bins + b];
        }
    }
}

// Leaves in sh.start the places of this block's first entries of each bin, and in
// start those of all blocks'.
template <int BINS>
__device__ __forceinline__ void block_starts(Shared<BINS>& sh, const int (&all)[2], const int (&before)[2], int bins,
                                             int (&start)[2]) {
    starts(sh, all, bins, start);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int b = (int)threadIdx.x + j * kThreads;
        if (b < bins) sh.start[b] = start[j] + before[j];
    }
    __syncthreads();
}

// The place over all entries of round j's, once sh.start is set.
template <int BINS>
__device__ __forceinline__ int placed(const Shared<BINS>& sh, int key, int place, int bins) {
    return sh.start[key] + sh.base[((int)threadIdx.x >> 6) * bins + key] + place;
}

}  // namespace key_sort
}  // namespace fl

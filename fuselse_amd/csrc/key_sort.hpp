// Stable counting sort of entries by a small key (at most 1025 bins), for the
// experts' order and, digit by digit, for an embedding's gradient.
//
// A block takes 4096 entries in their order, a wave 256 of them, 64 at a time.
// Lanes of equal keys find each other with a ballot a key bit; a lane's place
// among its wave's entries of that key is the wave's count so far plus the lanes
// below it, so nothing depends on the order of atomics.  Up to 4096 entries one
// block does it all; beyond, one launch counts, one sums the blocks' counts a bin
// and one places.
#pragma once

#include "lse_common.hpp"

namespace fl {
namespace key_sort {

constexpr int kWaves = 16, kThreads = 64 * kWaves, kRounds = 4, kChunk = kThreads * kRounds;
constexpr int kMaxBins = 1025;

struct Shared {
    int base[kWaves * kMaxBins];  // entries of a bin in the waves before
    int start[kMaxBins];          // place of a bin's first entry of this block
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
__device__ __forceinline__ int entry(int j) {
    return ((int)(threadIdx.x >> 6) * kRounds + j) * 64 + (int)(threadIdx.x & 63);
}

// Places of the block's n entries (key[j] of entry(j)) among those of their bin
// in their wave; sh.base then holds the waves' counts before.  total[j] becomes
// the block's count of bin threadIdx.x + j * kThreads.
__device__ __forceinline__ void rank(Shared& sh, const int (&key)[kRounds], int n, int bins, int bits,
                                     int (&place)[kRounds], int (&total)[2]) {
    const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    for (int b = threadIdx.x; b < kWaves * bins; b += kThreads) sh.base[b] = 0;
    __syncthreads();
    int* mine = sh.base + wave * bins;
    const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
        place[j] = 0;
        if ((wave * kRounds + j) * 64 >= n) continue;  // the same for all of the wave
        const bool live = entry(j) < n;
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
__device__ __forceinline__ int scan(Shared& sh, int v, int& all) {
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
__device__ __forceinline__ void starts(Shared& sh, const int (&total)[2], int bins, int (&start)[2]) {
    int all;
    start[0] = scan(sh, (int)threadIdx.x < bins ? total[0] : 0, all);
    start[1] = all;
}

// Blocks' counts of their entries: hist[bin * chunks + block].
template <typename Key>
__global__ __launch_bounds__(kThreads) void count_kernel(Key key, int64_t n, int bins, int* hist) {
    __shared__ int count[kMaxBins];
    for (int b = threadIdx.x; b < bins; b += kThreads) count[b] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * kChunk;
    const int m = (int)(n - first < kChunk ? n - first : kChunk);
#pragma unroll
    for (int j = 0; j < kRounds; ++j)
        if (entry(j) < m) atomicAdd(&count[key(first + entry(j))], 1);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) hist[(int64_t)b * gridDim.x + blockIdx.x] = count[b];
}

// Over the blocks of a bin, a wave a bin: counts become the sums of those
// before, total[bin] the sum of all.
static __global__ __launch_bounds__(256) void sum_kernel(int* hist, int64_t blocks, int bins, int* total) {
    const int bin = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
    if (bin >= bins) return;
    int* h = hist + (int64_t)bin * blocks;
    int sum = 0;
    for (int64_t first = 0; first < blocks; first += 64) {
        const int64_t b = first + lane;
        const int v = b < blocks ? h[b] : 0;
        int s = v;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(s, d, 64);
            if (lane >= d) s += o;
        }
        if (b < blocks) h[b] = sum + s - v;
        sum += __shfl(s, 63, 64);
    }
    if (lane == 0) total[bin] = sum;
}

// Loads the bins' totals and starts over all blocks, and leaves in sh.start the
// places of this block's first entries; sh.base and place from rank().
__device__ __forceinline__ void block_starts(Shared& sh, const int* hist, const int* total, int64_t blocks, int bins,
                                             int (&all)[2], int (&start)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int b = (int)threadIdx.x + j * kThreads;
        all[j] = b < bins ? total[b] : 0;
    }
    starts(sh, all, bins, start);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int b = (int)threadIdx.x + j * kThreads;
        if (b < bins) sh.start[b] = start[j] + hist[(int64_t)b * blocks + blockIdx.x];
    }
    __syncthreads();
}

// The place over all entries of round j's, once sh.start is set.
__device__ __forceinline__ int placed(const Shared& sh, int key, int place, int bins) {
    return sh.start[key] + sh.base[((int)threadIdx.x >> 6) * bins + key] + place;
}

}  // namespace key_sort
}  // namespace fl

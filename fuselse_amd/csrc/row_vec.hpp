// Rows of any length and alignment as 16-byte vectors, for the kernels that move
// whole rows (embedding.hip, experts.hip).
#pragma once

#include "row_stream.hpp"

namespace fl {

template <typename T>
constexpr int row_vectors(int64_t D) {
    return (int)((D + Elem<T>::kVec - 1) / Elem<T>::kVec);
}

// Vector v of a row of D elements begins here: the last one is moved back to end
// with the row, so that every vector of a row of at least kVec elements is whole.
// Elements that two vectors share have the same value in both.
template <typename T>
__device__ __forceinline__ int64_t row_vec_at(int64_t D, int v) {
    const int64_t e = (int64_t)v * Elem<T>::kVec, last = D - Elem<T>::kVec;
    return e < last ? e : last;
}

// STREAM: with the nontemporal hint, for rows that are read once.
template <bool STREAM = false, typename T>
__device__ __forceinline__ u32x4 row_load(const T* row, int64_t D, int v) {
    if (D >= Elem<T>::kVec) {
        const T* at = row + row_vec_at<T>(D, v);
        if constexpr (STREAM) return load_raw_stream(at);
        else return *reinterpret_cast<const u32x4_any*>(at);
    }
    T part[Elem<T>::kVec];
#pragma unroll
    for (int k = 0; k < Elem<T>::kVec; ++k) part[k] = k < D ? row[k] : T{};
    u32x4 r;
    __builtin_memcpy(&r, part, 16);
    return r;
}

template <typename T>
__device__ __forceinline__ void row_store(T* row, int64_t D, int v, u32x4 r) {
    if (D >= Elem<T>::kVec) {
        __builtin_nontemporal_store(r, reinterpret_cast<u32x4_any*>(row + row_vec_at<T>(D, v)));
        return;
    }
    T part[Elem<T>::kVec];
    __builtin_memcpy(part, &r, 16);
#pragma unroll
    for (int k = 0; k < Elem<T>::kVec; ++k)
        if (k < D) row[k] = part[k];
}

// The same written through to memory, for a row that all of a wave has and that is
// whole, aligned vectors, of 64 MB at most.
template <typename T>
__device__ __forceinline__ void row_store_through(T* row, int64_t D, int v, u32x4 r) {
    const uint64_t a = reinterpret_cast<uint64_t>(row);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)a);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32));
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<void*>((uint64_t)hi << 32 | lo), 0, (int)(D * sizeof(T)), 0x00020000);
    __builtin_amdgcn_raw_buffer_store_b128(r, rsrc, (int)(row_vec_at<T>(D, v) * sizeof(T)), 0, kStoreStreamAux);
}

// Whether rows are written through: those that begin and end with 64-byte units.
// Others lose time, as units that two rows share are written in parts: the experts'
// rows of (40000, 1000) in fp32 from 6 each take 262 us so and 249 else, of (30000,
// 1992) in bf16 200 and 181, but of (30000, 2016) 138 and 143.
inline bool row_through(const void* out, int64_t bytes) {
    return bytes % 64 == 0 && (reinterpret_cast<uintptr_t>(out) & 63u) == 0;
}

// fp32 values rounded to the type, once.
template <typename T>
__device__ __forceinline__ u32x4 pack_vec(const float (&v)[Elem<T>::kVec]) {
    u32x4 r;
    if constexpr (sizeof(T) == 4) {
        __builtin_memcpy(&r, v, 16);
    } else if constexpr (__is_same(T, _Float16)) {
        f16x8 t;
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = (_Float16)v[k];
        r = __builtin_bit_cast(u32x4, t);
    } else {
        r = Elem<T>::pack(v);
    }
    return r;
}

// Lanes that share a row of nvec vectors (a power of two from 8 up to a wave) and
// the steps of 64 vectors that longer rows take.
inline int row_lanes(int nvec) {
    int lanes = 8;
    while (lanes < nvec && lanes < 64) lanes *= 2;
    return lanes;
}
inline int row_steps(int nvec) { return (nvec + 63) / 64; }

}  // namespace fl

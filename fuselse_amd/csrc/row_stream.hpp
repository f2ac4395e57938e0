// Row vectors at any alignment, and rows of a two-level strided batch, for the
// loss kernels (distill.hip, router.hip).
#pragma once

#include "lse_common.hpp"

namespace fl {

// One 16-byte vector of row elements at any element alignment (gfx950 takes
// unaligned global accesses; one load instruction either way), as it lies and
// streamed with the nontemporal hint, or widened.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
__device__ __forceinline__ u32x4 load_raw_stream(const T* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
}
template <typename T>
__device__ __forceinline__ void load_vec_any(const T* p, float (&o)[Elem<T>::kVec]) {
    u32x4 r;
    __builtin_memcpy(&r, p, 16);
    Elem<T>::cvt(r, o);
}

// The same, elements at and past `n` (of those left in the row) replaced.
template <typename T>
__device__ __forceinline__ void load_vec_part(const T* p, int64_t n, float fill, float (&o)[Elem<T>::kVec]) {
    if (n >= Elem<T>::kVec) {
        load_vec_any<T>(p, o);
        return;
    }
#pragma unroll
    for (int k = 0; k < Elem<T>::kVec; ++k) o[k] = k < n ? Elem<T>::scalar(p + k) : fill;
}

// Row r of a batch of n1 rows each: base + (r / n1) s0 + (r % n1) s1.
struct RowMap {
    int64_t n1, s0, s1;
    __device__ __forceinline__ int64_t offset(int64_t r) const { return r / n1 * s0 + r % n1 * s1; }
};

}  // namespace fl

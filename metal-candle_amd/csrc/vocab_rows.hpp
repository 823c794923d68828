// What the kernels over rows of a vocabulary share: a row of any length and
// start as aligned vectors, and stores past the caches.
#pragma once

#include "common.hpp"

namespace mc {

// A row as aligned 16-byte vectors between up to N - 1 elements on each side,
// for rows of any length and start: vector c holds elements head + N c ..
template <typename T> struct RowSpan {
    int64_t head, nvec, tail;  // elements before the vectors, vectors, first element after them
    __device__ RowSpan(const T* p, int64_t dim) {
        constexpr int N = Vec16<T>::N;
        const int64_t mis = (int64_t)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
        head = mis ? N - mis : 0;
        if (head > dim) head = dim;
        nvec = (dim - head) / N;
        tail = head + nvec * N;
    }
    // The element of an edge that thread t (of at least 2 N) takes, or -1.
    __device__ int64_t edge(int t, int64_t dim) const {
        constexpr int N = Vec16<T>::N;
        if (t < N) return t < head ? t : -1;
        return t < 2 * N && tail + t - N < dim ? tail + t - N : -1;
    }
};

__device__ __forceinline__ void store_nt16(float* p, const float (&v)[4]) {
    __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(p));
}
__device__ __forceinline__ void store_nt16(uint16_t* p, const float (&v)[8]) {
    const u32x4 q = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    __builtin_nontemporal_store(q, reinterpret_cast<u32x4*>(p));
}
// Sixteen bytes at any element.
__device__ __forceinline__ void store_any16(float* p, const float (&v)[4]) {
    typedef f32x4 __attribute__((aligned(4))) any;
    *reinterpret_cast<any*>(p) = f32x4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ void store_any16(uint16_t* p, const float (&v)[8]) {
    typedef u32x4 __attribute__((aligned(2))) any;
    *reinterpret_cast<any*>(p) =
        u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}

}  // namespace mc

// What the kernels of the memory over decisions share (include/flyguy_memory.h): value types, views, wave sums.
#pragma once
#include "../../include/flyguy_memory.h"
#include "common.h"

namespace fg {

using bf16 = __bf16;
using f16 = _Float16;

template <class T>
__device__ __forceinline__ float widen(T v) { return (float)v; }
// to the nearest, ties to even: the one rounding of an output
template <class T>
__device__ __forceinline__ T narrow(float v) { return (T)v; }

// x exp(g) with the factor kept to more than 24 bits near 1: a state is multiplied by it once a moment (or a chunk) for as
// long as it remembers, and a rounded factor's errors would all point the same way (g = -1e-5 over 20,000 moments: 3e-4).
// A factor of 1 keeps infinities, and zero stays zero where the factor overflows.
struct Keep {
    float one, f;                        // exp(g) = one + f
    __device__ __forceinline__ explicit Keep(float g) : one(g > -0.5f ? 1.f : 0.f), f(g > -0.5f ? expm1f(g) : expf(g)) {}
    // (of the common kind: neither of those)
    __device__ __forceinline__ bool plain() const { return f != 0.f && f < INFINITY; }
    __device__ __forceinline__ float times(float x) const { return fmaf(f, x, one * x); }
    __device__ __forceinline__ float operator()(float x) const {
        return f == 0.f || (x == 0.f && f > 0.f) ? one * x : times(x);
    }
};

// values of a 16-byte load
template <class T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
};

__device__ __forceinline__ float wave_sum(float v, int width) {
    for (int m = 1; m < width; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// an entry of an index array of either width
__device__ __forceinline__ long long index_at(const void* p, long long i, bool wide) {
    return wide ? reinterpret_cast<const long long*>(p)[i] : reinterpret_cast<const int*>(p)[i];
}

// a launch of any number of workgroups (a grid's x holds 2^32 threads)
inline dim3 blocks_of(long long n) {
    const long long x = n < 1 << 20 ? n : 1 << 20;
    return dim3((unsigned)x, (unsigned)((n + x - 1) / x));
}
__device__ __forceinline__ long long block_number() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }

inline bool aligned16(const fm_view& v, int size) {
    return !(((uintptr_t)v.data | (uintptr_t)(v.seq * size) | (uintptr_t)(v.moment * size) | (uintptr_t)(v.head * size)) & 15);
}

inline int fail(const char* what) {
    set_error(what);
    return -1;
}

}  // namespace fg

// Tensors of float32 or bfloat16: the same element reads and writes for both, float32 in registers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace slayer {

typedef __bf16 bf16;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <typename T> struct Elements;
template <> struct Elements<float> {
    static constexpr int kVec = 4;                 // elements of one 16-byte access
    typedef f4 Vec;
};
template <> struct Elements<bf16> {
    static constexpr int kVec = 8;
    typedef b8 Vec;
};

// 16 bytes as float32 and back (rounded to nearest)
__device__ __forceinline__ void to_floats(float (&out)[4], f4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = v[i];
}
__device__ __forceinline__ void to_floats(float (&out)[8], b8 v) {
    const f8 f = __builtin_convertvector(v, f8);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = f[i];
}
__device__ __forceinline__ f4 from_floats(const float (&in)[4]) { return f4{in[0], in[1], in[2], in[3]}; }
__device__ __forceinline__ b8 from_floats(const float (&in)[8]) {
    return __builtin_convertvector(f8{in[0], in[1], in[2], in[3], in[4], in[5], in[6], in[7]}, b8);
}

// kVec elements from `p`, of which the first `n` exist (the others read as 0): one access where `whole` (p is a multiple
// of 16 bytes) and all exist, one by one otherwise.
template <typename T>
__device__ __forceinline__ typename Elements<T>::Vec load_vec(const T* p, int n, bool whole) {
    constexpr int V = Elements<T>::kVec;
    typename Elements<T>::Vec v = {};
    if (whole && n >= V) {
        v = *reinterpret_cast<const typename Elements<T>::Vec*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) v[i] = p[i];
    }
    return v;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, typename Elements<T>::Vec v, int n, bool whole) {
    constexpr int V = Elements<T>::kVec;
    if (whole && n >= V) {
        *reinterpret_cast<typename Elements<T>::Vec*>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = v[i];
    }
}

}  // namespace slayer

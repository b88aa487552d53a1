// Tensors of float32 or bfloat16: the same element reads and writes for both, float32 in registers; what kernels on them share.
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

// Neighbouring elements at any address that suits one of them: the hardware takes wide accesses that are not aligned.
// `n`: how many of them exist (the others read as 0 and are not written).
typedef f4 f4_any __attribute__((aligned(4)));
typedef b4 b4_any __attribute__((aligned(2)));
template <typename T> struct Four;
template <typename T> struct Wide;             // as many as 16 bytes hold
typedef b8 b8_any __attribute__((aligned(2)));
template <> struct Wide<float> { typedef f4_any Any; };
template <> struct Wide<bf16> { typedef b8_any Any; };
template <> struct Four<float> { typedef f4 Vec; typedef f4_any Any; };
template <> struct Four<bf16> { typedef b4 Vec; typedef b4_any Any; };
template <typename T> __device__ __forceinline__ typename Four<T>::Vec load_four(const T* p, int n) {
    if (n >= 4) return *reinterpret_cast<const typename Four<T>::Any*>(p);
    typename Four<T>::Vec v = {};
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < n) v[i] = p[i];
    return v;
}
template <typename T> __device__ __forceinline__ void store_four(T* p, f4 x, int n) {
    const typename Four<T>::Vec v = __builtin_convertvector(x, typename Four<T>::Vec);
    if (n >= 4) {
        *reinterpret_cast<typename Four<T>::Any*>(p) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < n) p[i] = v[i];
}

// 1 / (1 + exp(-z)) from the hardware's base-two exponential and reciprocal, a unit in the last place each.  For bfloat16 tensors as they
// are: the argument's rounding makes it (3 + 1.5 |z|) 2^-24 where it matters (for negative z it is the exponential that falls), far below
// the rounding of the result.  For float32 tensors what the argument's rounding leaves goes into the exponential, 2^x (1 + r ln 2), and the
// reciprocal takes a step of Newton's: 6 2^-24.  Rows of [480000,256] in 4 groups, forward, as they are / with the two / with the precise
// functions: bfloat16 114 / 139 / 177 us, float32 193 / 216 / 250 us.
template <typename T> __device__ __forceinline__ float logistic(float z) {
    constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;
    constexpr float hi = (float)-kLog2e, lo = (float)(-kLog2e - (double)hi);
    const float x = z * hi;
    float e = __builtin_amdgcn_exp2f(x);
    if constexpr (sizeof(T) != 4) return __builtin_amdgcn_rcpf(1.f + e);
    e = fmaf(e, fmaf(z, lo, fmaf(z, hi, -x)) * (float)kLn2, e);
    const float r = __builtin_amdgcn_rcpf(1.f + e);
    return x < 126.f ? fmaf(fmaf(-(1.f + e), r, 1.f), r, r) : __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x));
}

// Sum over `lanes` neighbouring lanes (a power of two), in all of them.
__device__ __forceinline__ float sum_lanes(float v, int lanes) {
    for (int d = lanes >> 1; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

}  // namespace slayer

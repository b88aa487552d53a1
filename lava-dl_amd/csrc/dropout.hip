// Dropout whose mask is a function of (seed, offset, index): nothing is stored, and the gradient is the same call.
//   Philox-4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: Parallel Random Numbers: As Easy as 1, 2, 3, SC 2011):
// key = seed, counter = (block, offset), 128 bits a block = eight decisions of sixteen bits, decision i in half word i % 8 of
// block i / 8.  A decision is "keep" at or above limit = round(p * 65536), so the share that is dropped is limit / 65536
// (within 2^-17 of p), and what is kept is scaled by the inverse of what that share really leaves.
//   Sixteen bits rather than 32: the ten rounds of a block, twenty products of 32 bits, then serve eight decisions and not four.  Bound:
// memory, at the rate of a copy.  12.3 million bfloat16 in 9.1 us (5.4 TB/s), 131 million float32 with a decision for each 2000 in
// 188 us (5.6 TB/s).
#include "common.h"
#include "elements.h"

namespace slayer {

struct Philox { unsigned w[4]; };
__device__ __forceinline__ Philox philox(uint64_t block, uint64_t seed, uint64_t offset) {
    unsigned c0 = (unsigned)block, c1 = (unsigned)(block >> 32), c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
    unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
        c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c1 = (unsigned)b;
        c3 = (unsigned)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}
__device__ __forceinline__ unsigned decision(const Philox& r, int i) { return i & 1 ? r.w[i >> 1] >> 16 : r.w[i >> 1] & 0xffffu; }

constexpr int kSpan = 8;                       // elements of a thread: one block of the generator

// A decision for each element: eight elements and one block of the generator a thread.
template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(T* __restrict__ out, const T* __restrict__ in, uint64_t seed, uint64_t offset,
                                                      unsigned limit, float scale, int64_t n, bool whole) {
    constexpr int V = Elements<T>::kVec;
    const int64_t block = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (block * kSpan >= n) return;
    const Philox r = philox((uint64_t)block, seed, offset);
#pragma unroll
    for (int h = 0; h < kSpan / V; ++h) {
        const int64_t at = block * kSpan + h * V;
        const int left = n - at < V ? (n > at ? (int)(n - at) : 0) : V;
        float x[V];
        to_floats(x, load_vec(in + at, left, whole));
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = decision(r, h * V + i) >= limit ? x[i] * scale : 0.f;
        store_vec(out + at, from_floats(x), left, whole);
    }
}

// One decision for the `steps` elements of a row.
template <typename T>
__global__ __launch_bounds__(256) void dropout_rows_kernel(T* __restrict__ out, const T* __restrict__ in, uint64_t seed, uint64_t offset,
                                                           unsigned limit, float scale, int64_t n, int64_t steps, bool whole) {
    constexpr int V = Elements<T>::kVec;
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (at >= n) return;
    const int left = n - at < V ? (int)(n - at) : V;
    int64_t row = at / steps, next = (row + 1) * steps;      // the row the elements begin in, and where it ends
    bool keep = decision(philox((uint64_t)row / 8, seed, offset), (int)(row % 8)) >= limit;
    float x[V];
    to_floats(x, load_vec(in + at, left, whole));
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (at + i == next) {
            ++row;
            next += steps;
            keep = decision(philox((uint64_t)row / 8, seed, offset), (int)(row % 8)) >= limit;
        }
        x[i] = keep ? x[i] * scale : 0.f;
    }
    store_vec(out + at, from_floats(x), left, whole);
}

template <typename T>
int launch_dropout(void* out, const void* in, int64_t n, int64_t steps, unsigned limit, float scale, uint64_t seed, uint64_t offset,
                   hipStream_t stream) {
    const bool whole = ((uintptr_t)out | (uintptr_t)in) % 16 == 0;
    const int64_t span = 256 * (steps > 0 ? Elements<T>::kVec : kSpan);
    const int64_t blocks = (n + span - 1) / span;
    if (blocks > (1 << 24) - 1) return SLAYER_ERANGE;         // fewer than 2^32 threads in a launch
    if (steps > 0)
        hipLaunchKernelGGL(dropout_rows_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, (T*)out, (const T*)in, seed, offset,
                           limit, scale, n, steps, whole);
    else
        hipLaunchKernelGGL(dropout_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, stream, (T*)out, (const T*)in, seed, offset, limit,
                           scale, n, whole);
    return (int)hipGetLastError();
}

}  // namespace slayer

using namespace slayer;

extern "C" int slayer_dropout(void* out, const void* in, int dtype, int64_t n, int64_t steps, int limit, float scale, uint64_t seed,
                              uint64_t offset, void* stream) {
    if (n < 0 || steps < 0 || limit < 0 || limit > 65536 || (steps > 0 && n % steps != 0)) return SLAYER_EINVAL;
    if (dtype != SLAYER_FLOAT32 && dtype != SLAYER_BFLOAT16) return SLAYER_EINVAL;
    if (n == 0) return 0;
    if (!out || !in) return SLAYER_ENULL;
    if (n > ((int64_t)1 << 40)) return SLAYER_ERANGE;
    return dtype == SLAYER_FLOAT32 ? launch_dropout<float>(out, in, n, steps, (unsigned)limit, scale, seed, offset, (hipStream_t)stream)
                                   : launch_dropout<bf16>(out, in, n, steps, (unsigned)limit, scale, seed, offset, (hipStream_t)stream);
}

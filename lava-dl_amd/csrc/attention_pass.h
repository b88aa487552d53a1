// The kernel of leaky attention (attention.hip says what it computes), for attention_f32.hip and attention_bf16.hip.
#pragma once
#include "common.h"
#include "elements.h"
#include <type_traits>

namespace slayer {

constexpr int kChunk = 64;

// One pass of the recurrence, as its kernels see it.  `query`, `key`, `value` are the tensors in the three places.
struct LeakyPass {
    void* out;
    const void *query, *key, *value;
    const float* decay;
    const void* lengths;
    const float* first;            // states in front of the first token, [samples * heads], or nullptr: zeros
    float* starts;                 // states in front of the segments, [samples * heads][segments] of them (not `joined`: what the
                                   // segment before each adds)
    float* last;                   // state behind the last token, or nullptr
    float* slope_starts;           // LEAKY_SLOPE: derivatives of the states in `starts`
    const float* grad_last;        // LEAKY_SLOPE: gradient of the last state, or nullptr
    const void* query2;            // LEAKY_BOTH
    void* out2;
    const void* other;             // LEAKY_SLOPE: what the derivative of the results is multiplied with, laid out as they are
    double* slopes;                // LEAKY_SLOPE: [samples][heads][segments][slices]
    int64_t out_n, out_t, out_h, query_n, query_t, query_h, key_n, key_t, key_h, value_n, value_t, value_h, other_n, other_t, other_h;
    int64_t query2_n, query2_t, query2_h, out2_n, out2_t, out2_h;
    int tokens, heads, keys, values, state_k, state_v;      // the strides of a state's axes
    int units;                     // samples * heads
    // slices of the values, `tiles` sixteens each (1 to 4; 2 or 4 where rows are not made of whole pieces)
    int one_decay, lengths64, segments, segment, slices, tiles, backwards, joined;
    int whole_other;               // `other` comes in fours that can be read at once
    int whole_out2;
    int whole_out;                 // values come in fours that can be written at once, within the reach of a 32-bit offset
    float score_scale, state_scale, key_scale;      // of scores, of the state in results, of keys in the state
};

// ---- fragments of the matrix instructions.  A fragment holds kDepth terms of a product for 16 rows (or columns): lane l has
// row l % 16 and, with g = l / 16,
//   float32 : terms 4g ... 4g+3 of 16, one v_mfma_f32_16x16x4_f32 for each of the four;
//   bfloat16: eight of 32, for one v_mfma_f32_16x16x32_bf16: 8g ... 8g+7 where both operands lie along the terms in LDS, or
//             4g ... 4g+3 and 16+4g ... 16+4g+3 ("halves") where one of them is a pair of results (whose lane l has rows
//             4g ... 4g+3 of column l % 16 of a 16 x 16 tile) or is read across its rows.
template <typename T> struct Frag;
template <> struct Frag<float> {
    static constexpr int kDepth = 16;
    typedef f4 Type;
};
template <> struct Frag<bf16> {
    static constexpr int kDepth = 32;
    typedef b8 Type;
};
__device__ __forceinline__ f4 mma(f4 a, f4 b, f4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f4 mma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// terms along the row of `tile`
template <typename T>
__device__ __forceinline__ typename Frag<T>::Type along(const T* tile, int pitch, int row, int term, int lane) {
    return *reinterpret_cast<const typename Frag<T>::Type*>(tile + (row + (lane & 15)) * pitch + term + (lane >> 4) * Elements<T>::kVec);
}
// ... in halves (float32: the same)
__device__ __forceinline__ f4 along_halves(const float* tile, int pitch, int row, int term, int lane) { return along(tile, pitch, row, term, lane); }
__device__ __forceinline__ b8 along_halves(const bf16* tile, int pitch, int row, int term, int lane) {
    const bf16* p = tile + (row + (lane & 15)) * pitch + term + (lane >> 4) * 4;
    return __builtin_shufflevector(*reinterpret_cast<const b4*>(p), *reinterpret_cast<const b4*>(p + 16), 0, 1, 2, 3, 4, 5, 6, 7);
}
// terms across the rows of `tile`, the sixteen columns from `column` on
__device__ __forceinline__ f4 across(const float* tile, int pitch, int column, int term, int lane) {
    const float* p = tile + (term + (lane >> 4) * 4) * pitch + column + (lane & 15);
    return f4{p[0], p[pitch], p[2 * pitch], p[3 * pitch]};
}
typedef __attribute__((address_space(3))) short LdsShort;
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
// ds_read_b64_tr_b16: the sixteen lanes of a group read four rows of sixteen columns, lane i gets column i of the four
__device__ __forceinline__ b8 across(const bf16* tile, int pitch, int column, int term, int lane) {
    const int i = lane & 15;
    const bf16* p = tile + (term + (lane >> 4) * 4 + (i >> 2)) * pitch + column + (i & 3) * 4;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(LdsShort*)p);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(LdsShort*)(p + 16 * pitch));
    const b4 a = __builtin_bit_cast(b4, lo), b = __builtin_bit_cast(b4, hi);
    return b8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// A float32 operand: in float32, or as three bfloat16 numbers that sum to it, so that what the kernel makes itself (scores, states, leaked
// keys) keeps float32's digits on the way.  Two would leave 2^-16 of every term, which is more than the rounding of a bfloat16
// result as soon as the terms cancel to a 256th of their magnitudes; [64,1000,8,64], forward, calls in a row: 65 us with two, 82 with
// three.  A value that is not finite, or beyond the largest bfloat16, leaves a NaN.
constexpr int kParts = 3;
struct Split { b8 part[kParts]; };
__device__ __forceinline__ Split split(f8 v) {
    Split o;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
        o.part[i] = __builtin_convertvector(v, b8);
        if (i + 1 < kParts) v -= __builtin_convertvector(o.part[i], f8);
    }
    return o;
}

__device__ __forceinline__ double power(double a, int n) {
    double p = 1;
    for (; n > 0; n >>= 1) {
        if (n & 1) p *= a;
        a *= a;
    }
    return p;
}

__device__ __forceinline__ int sample_length(const LeakyPass& a, int n) {
    if (!a.lengths) return a.tokens;
    const int64_t l = a.lengths64 ? static_cast<const int64_t*>(a.lengths)[n] : static_cast<const int*>(a.lengths)[n];
    return l < 0 ? 0 : (l > a.tokens ? a.tokens : (int)l);
}


enum { LEAKY_STATE, LEAKY_MAIN, LEAKY_BOTH, LEAKY_STATE_SLOPE, LEAKY_SLOPE };

// Values that are not finite.  A score that the mask leaves out is 0, and 0 times such a value is not: a strip with masked scores takes
// the products without these values and says which results they belong to.
__device__ __forceinline__ bool any_not_finite(f4 v) {
    const u4 x = __builtin_bit_cast(u4, v) & 0x7fffffffu;
    return max(max(x[0], x[1]), max(x[2], x[3])) >= 0x7f800000u;
}
__device__ __forceinline__ bool any_not_finite(b8 v) {
    const u4 x = (__builtin_bit_cast(u4, v) & 0x7f807f80u) + 0x00800080u;     // an exponent of all ones carries into the sign
    return ((x[0] | x[1]) | (x[2] | x[3])) & 0x80008000u;
}
template <typename F> __device__ __forceinline__ F where_not_finite(F v, F yes, F no) {
    constexpr int count = sizeof(F) == 16 && sizeof(v[0]) == 4 ? 4 : 8;
    F r;
#pragma unroll
    for (int i = 0; i < count; ++i) {
        const float x = (float)v[i];
        r[i] = x - x == 0.f ? no[i] : yes[i];
    }
    return r;
}

// a^n and its derivative n a^(n-1); both 0 for n < 0
__device__ __forceinline__ float power_at(const float* powers, int n) { return n >= 0 ? powers[n] : 0.f; }
__device__ __forceinline__ float slope_at(const float* powers, int n) { return n >= 1 ? (float)n * powers[n - 1] : 0.f; }

// A workgroup of four waves takes one segment of one head of one sample, chunk after chunk, and one slice of 16 VT values.
// Wave w makes the outputs of places 16w ... 16w+15 (transposed: lane = place) and the rows of the state w, w+4, ... (16 each).
// The first chunk is the one that is not full, with its tokens at the end, so that weights behind a token are the same in all.
//   LEAKY_STATE: only the state, from zero, into `starts` behind the segment's place (for the segments but the last).
//   LEAKY_MAIN:  results, and the last state.
//   LEAKY_BOTH:  the gradients of value and key together: beside out[i], from query and key, also out2[i], from query2 and value,
//       out2[i] = a^i query2[i] S^T + sum over j <= i of a^(i-j) (query2[i] . value[j]) key[j],
//     for which the state and the chunk's keys and values (queries and gradients) are there already.  One slice.
//   LEAKY_SLOPE: results, and the derivative of each with respect to a, in which the state's derivative W takes the place of S:
//       dout[i] = a^(i+1) query[i] W + (i+1) a^i query[i] S + sum over j of (i-j) a^(i-j-1) (query[i] . key[j]) value[j]
//       W'      = a^64 W + 64 a^63 S + sum over j of (63-j) a^(62-j) key[j] (outer) value[j]
//     of which the workgroup returns the sum of its products with `other`.  LEAKY_STATE_SLOPE: S and W from zero.
//   WHOLE: the rows of all tensors are made of whole, aligned 16-byte pieces.
//
//   What bounds it (64 keys and values, two workgroups a compute unit).  float32: the matrix cores, whose 3.25 products of 64 x 64 x 64
// a chunk take 6 656 cycles of each SIMD; [32,1500,4,64] in four segments 64 us, of which 37 are those and 39 would be a copy of the
// same bytes.  bfloat16: vector instructions, 55 % of a compute unit's busy cycles (about half of them, counted in the
// code, split scores, states and keys into parts), LDS 38 %, the matrix cores 23 %; [64,1000,8,64], calls in a row, 82 us from the last-level cache and 91 from memory,
// 262 MB, where a kernel that only moves the tensors takes 52 and 63: pieces of 128 bytes cost it a fifth.  A third workgroup a compute
// unit, slices of 32 values, priorities for one of the two and two sets of tiles (one barrier a chunk) were no faster.
//   Registers decide: versions of the forward and joint kernels with more than 256 of them, or with many in scratch memory (whose
// accesses wait for the chunk on its way), took 1.4 to 2 times as long.  So a strip is compiled for its wave, addresses are made anew in
// every chunk, the values are read twice, and `phase_end` keeps the compiler from starting the reads of a later phase.  What does
// not fit all the same: float32 LEAKY_SLOPE spills at KT, VT = 4, 4 (9 registers), 6, 3 (64) and 8, 2 (10), float32 LEAKY_BOTH at 6, 4 (26; 219 us,
// 236 as two passes, [32,1500,4] with 96 keys and 64 values), bfloat16 LEAKY_SLOPE at 6, 3 (2); LEAKY_SLOPE with VT = 4 and KT = 6 or 8, or
// 8, 3, and float32 LEAKY_MAIN at 8, 4 leave room for one workgroup a compute unit.
__device__ __forceinline__ void phase_end() { __builtin_amdgcn_sched_barrier(0); }

template <typename T, int KT, int VT, int MODE, bool WHOLE>
__global__ __launch_bounds__(256, 2) void leaky_kernel(LeakyPass a) {
    typedef typename Frag<T>::Type F;
    typedef typename Elements<T>::Vec Vec;
    constexpr bool BOTH = MODE == LEAKY_BOTH, SLOPE = MODE >= LEAKY_STATE_SLOPE, F32 = sizeof(T) == 4;
    constexpr bool MAIN = MODE != LEAKY_STATE && MODE != LEAKY_STATE_SLOPE;
    constexpr int V = Elements<T>::kVec, D = Frag<T>::kDepth, P = F32 ? 1 : kParts;      // parts of a state in LDS
    constexpr int KP = KT * 16, VP = VT * 16;
    // rows of LDS: sixteen rows of keys, read along, start in different banks; so do the eight (float32: four) rows of values that
    // an access across them touches
    constexpr int kPitch = KP + V, vPitch = F32 ? VP + 4 : VP + (VT % 2 ? 0 : 16);
    constexpr int KV = KP / V, VV = VP / V;                                  // 16-byte pieces of a row
    constexpr int kLoads = (kChunk * KV + 255) / 256, vLoads = (kChunk * VV + 255) / 256;
    constexpr int ST = (KT + 3) / 4;                                         // strips of the state of a wave
    constexpr int kStates = MAIN ? (SLOPE ? 2 : 1) : 0;                      // states in LDS
    constexpr int kTile = kChunk * kPitch, vTile = kChunk * vPitch, sTile = kStates * P * VP * kPitch;
    __shared__ __align__(16) T keys[kTile];
    __shared__ __align__(16) T values[vTile];
    __shared__ __align__(16) T state[sTile > 0 ? sTile : 8];                 // [state][part][value][key]
    __shared__ __align__(16) float powers[kChunk + 4];                       // a^i
    __shared__ float weights[MAIN ? 48 : 1];                                 // of scores: a^(i - 16), 0 for i < 16
    __shared__ __align__(16) float behind[SLOPE ? 2 : 1][kChunk];            // what key j counts behind the chunk; its derivative
    __shared__ double sums[4];

    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    // Strips of the later places cost more (float32, 64 keys and values: 10, 12, 14 and 16 times sixteen instructions), and waves with the
    // same place in their workgroups share a SIMD: the second workgroup of a compute unit has them the other way round.
    const int wave = __builtin_amdgcn_readfirstlane(blockIdx.x & 256 ? 3 - (threadIdx.x >> 6) : threadIdx.x >> 6);
    const int segments = MAIN ? a.segments : a.segments - 1;
    // The slices of a segment, which read the same queries and keys, eight workgroups apart: on the same XCD, with one L2.  (Heads and
    // samples are left spread over the XCDs: samples of different lengths then load them alike.)
    int slice, at_segment = blockIdx.x;
    if (at_segment < (a.units * segments & ~7) * a.slices) {
        slice = at_segment / 8 % a.slices;
        at_segment = at_segment / (8 * a.slices) * 8 + at_segment % 8;
    } else {
        slice = at_segment % a.slices;
        at_segment /= a.slices;
    }
    const int seg = at_segment % segments, unit = at_segment / segments;
    const int n = unit / a.heads, h = unit % a.heads;
    const int v0 = slice * VP, vleft = a.values - v0, length = sample_length(a, n);
    const double leak = 1.0 - (double)a.decay[a.one_decay ? 0 : h] / 4096.0;
    const int begin = seg * a.segment, end = min(begin + a.segment, a.tokens), stop = min(end, length);
    if (!MAIN && end > length) return;                                       // no segment behind it needs this one's state
    const int64_t state_size = (int64_t)a.keys * a.values;
    T* out = (T*)a.out + n * a.out_n + h * a.out_h + v0;
    T* out2 = BOTH ? (T*)a.out2 + n * a.out2_n + h * a.out2_h : nullptr;
    const int shift = a.backwards ? 0 : 1;
    f4 S[ST][VT], W[SLOPE ? ST : 1][SLOPE ? VT : 1];
    auto share = [&](f4 x, int which, int strip, int v, int g, int col) {
        T* p = state + which * P * VP * kPitch + (v * 16 + col) * kPitch + strip * 16 + 4 * g;
        if constexpr (F32) {
            *reinterpret_cast<f4*>(p) = x;
        } else {
#pragma unroll
            for (int part = 0; part < P; ++part) {
                const b4 y = __builtin_convertvector(x, b4);
                *reinterpret_cast<b4*>(p + part * VP * kPitch) = y;
                x -= __builtin_convertvector(y, f4);
            }
        }
    };

    // What the next chunk needs, on its way.  WHOLE: a thread's pieces are an offset from the chunk's first address (kNowhere
    // lies outside of every buffer and reads 0); otherwise they are read element by element.
    const int count0 = stop > begin ? (stop - begin - 1) % kChunk + 1 : 0;   // tokens of the first chunk
    int p0 = stop > begin ? begin - (kChunk - count0) : stop;                // place of the chunk's first row
    auto place = [&](int p) { return (int64_t)(a.backwards ? length - 1 - p : p); };
    const int64_t low0 = place(a.backwards ? p0 + kChunk - 1 : p0), turn = a.backwards ? -kChunk : kChunk;
    const T* key = (const T*)a.key + n * a.key_n + h * a.key_h + low0 * a.key_t;             // the chunk's first address
    const T* value = (const T*)a.value + n * a.value_n + h * a.value_h + v0 + low0 * a.value_t;
    const T* query = MAIN ? (const T*)a.query + n * a.query_n + h * a.query_h + low0 * a.query_t : nullptr;
    Vec nk[kLoads], nv[vLoads];
    F qf[MAIN ? KP / D : 1];
    constexpr int kNowhere = (int)0x80000000;
    // `missing`: rows of the chunk that are not there (the first chunk's)
    auto fetch = [&](auto& to, const T* base, int64_t stride, int left, int missing, auto pieces, int thread) {
        constexpr int per = decltype(pieces)::value;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int i = 0; i < (kChunk * per + 255) / 256; ++i) {
            const int at = i * 256 + thread, row = at / per, c = at % per * V, from = a.backwards ? kChunk - 1 - row : row;
            const bool on = row >= missing && (kChunk * per % 256 == 0 || at < kChunk * per);
            if constexpr (WHOLE) {
                const int off = (from * (int)stride + c) * (int)sizeof(T);
                to[i] = __builtin_bit_cast(Vec, __builtin_amdgcn_raw_buffer_load_b128(r, on && c < left ? off : kNowhere, 0, 0));
            } else {
                to[i] = load_vec(base + (on ? from * stride : 0) + c, on ? left - c : 0, false);
            }
        }
    };
    auto fetch_rows = [&](int missing, int thread) {
        fetch(nk, key, a.key_t, a.keys, missing, std::integral_constant<int, KV>{}, thread);
        fetch(nv, value, a.value_t, vleft, missing, std::integral_constant<int, VV>{}, thread);
        key += turn * a.key_t;
        value += turn * a.value_t;
    };
    auto fetch_query = [&](int missing, int g, int col) {                    // this lane's place: row 16 wave + col
        if constexpr (MAIN) {
            const int row = wave * 16 + col, from = a.backwards ? kChunk - 1 - row : row;
            const bool on = row >= missing;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(query), 0, 0x7fffffff, 0x00020000);
            const int off = (from * (int)a.query_t + g * V) * (int)sizeof(T);
#pragma unroll
            for (int d = 0; d < KP / D; ++d) {
                const int c = d * D + g * V;
                if constexpr (WHOLE) qf[d] = __builtin_bit_cast(F, __builtin_amdgcn_raw_buffer_load_b128(r, on && c < a.keys ? off + d * D * (int)sizeof(T) : kNowhere, 0, 0));
                else qf[d] = load_vec(query + (on ? from * a.query_t : 0) + c, on ? a.keys - c : 0, false);
            }
            query += turn * a.query_t;
        }
    };
    // LEAKY_BOTH: the terms of query2 in halves, as the state is read across its rows
    F qf2[BOTH ? VP / D : 1];
    const T* query2 = BOTH ? (const T*)a.query2 + n * a.query2_n + h * a.query2_h + low0 * a.query2_t : nullptr;
    auto fetch_query2 = [&](int missing, int g, int col) {
        if constexpr (BOTH) {
            const int row = wave * 16 + col, from = a.backwards ? kChunk - 1 - row : row;
            const bool on = row >= missing;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(query2), 0, 0x7fffffff, 0x00020000);
            const int off = (from * (int)a.query2_t + 4 * g) * (int)sizeof(T);
#pragma unroll
            for (int d = 0; d < VP / D; ++d) {
                const int c = d * D + 4 * g;
                if constexpr (F32) {
                    qf2[d] = __builtin_bit_cast(F, __builtin_amdgcn_raw_buffer_load_b128(r, on && c < a.values ? off + d * D * (int)sizeof(T) : kNowhere, 0, 0));
                } else {
                    const b4 lo = __builtin_bit_cast(b4, __builtin_amdgcn_raw_buffer_load_b64(r, on && c < a.values ? off + d * D * (int)sizeof(T) : kNowhere, 0, 0));
                    const b4 hi = __builtin_bit_cast(b4, __builtin_amdgcn_raw_buffer_load_b64(r, on && c + 16 < a.values ? off + (d * D + 16) * (int)sizeof(T) : kNowhere, 0, 0));
                    qf2[d] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                }
            }
            query2 += turn * a.query2_t;
        }
    };
    // LEAKY_SLOPE: what this lane's results are multiplied with
    typedef std::conditional_t<F32, f4, b4> Quad;
    Quad other[MODE == LEAKY_SLOPE ? VT : 1];
    const T* others = MODE == LEAKY_SLOPE ? (const T*)a.other + n * a.other_n + h * a.other_h + v0 + low0 * a.other_t : nullptr;
    auto fetch_other = [&](int missing, int g, int col) {
        if constexpr (MODE == LEAKY_SLOPE) {
            const int row = wave * 16 + col, from = a.backwards ? kChunk - 1 - row : row;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(others), 0, 0x7fffffff, 0x00020000);
#pragma unroll
            for (int v = 0; v < VT; ++v) {
                const int c = v * 16 + 4 * g;
                if (a.whole_other) {
                    const int off = row >= missing && c < vleft ? (from * (int)a.other_t + c) * (int)sizeof(T) : kNowhere;
                    if constexpr (F32) other[v] = __builtin_bit_cast(Quad, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
                    else other[v] = __builtin_bit_cast(Quad, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) other[v][e] = row >= missing && c + e < vleft ? others[from * a.other_t + c + e] : (T)0.f;
                }
            }
            others += turn * a.other_t;
        }
    };
    if (stop > begin) {
        fetch_query(begin - p0, g, col);
        fetch_query2(begin - p0, g, col);
        fetch_other(begin - p0, g, col);
        fetch_rows(begin - p0, threadIdx.x);
    }

    __shared__ int not_finite;                                               // the last chunk with such values
    if (threadIdx.x == 0) not_finite = p0 - 1;
    if (threadIdx.x <= kChunk) powers[threadIdx.x] = (float)power(leak, threadIdx.x);
    __syncthreads();
    if (threadIdx.x < kChunk) {
        const int left = kChunk - 1 - (int)threadIdx.x;
        behind[0][threadIdx.x] = powers[left + (a.backwards ? 1 : 0)] * a.key_scale;
        if (SLOPE) behind[SLOPE ? 1 : 0][threadIdx.x] = slope_at(powers, left);
    }
    if (MAIN && threadIdx.x < 48) weights[MAIN ? threadIdx.x : 0] = power_at(powers, (int)threadIdx.x - 16) * a.score_scale;
    const double whole_leak = power(leak, kChunk);

    // the state, in strips of 16 keys: lane has keys 4g ... 4g+3 of column `col`
    {
        // in front of the segment: from `starts` where the states are joined, or what the segments before it have left there, added up
        const int from = !MAIN || begin > length ? seg + 1 : a.joined && seg > 0 ? seg : 0;
        const double past = from < seg ? power(leak, a.segment) : 1;
        const float past_hi = (float)past, past_lo = (float)(past - (double)past_hi);
        const float past_slope = SLOPE && from < seg ? (float)(a.segment * power(leak, a.segment - 1)) : 0.f;
#pragma unroll
        for (int s = 0; s < ST; ++s)
#pragma unroll
            for (int v = 0; v < VT; ++v) {
                S[s][v] = f4{0, 0, 0, 0};
                if constexpr (SLOPE) W[s][v] = f4{0, 0, 0, 0};
            }
        for (int j = from; j <= seg; ++j) {
            const int64_t at = ((int64_t)unit * a.segments + j) * state_size;
            const float* first = j > 0 ? a.starts + at : (a.first ? a.first + unit * state_size : nullptr);
            const float* slope_first = SLOPE && j > 0 ? a.slope_starts + at : nullptr;
#pragma unroll
            for (int s = 0; s < ST; ++s)
#pragma unroll
                for (int v = 0; v < VT; ++v)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int k = (s * 4 + wave) * 16 + 4 * g + r, c = v * 16 + col;
                        const bool on = k < a.keys && c < vleft;
                        const int64_t element = (int64_t)k * a.state_k + (int64_t)(v0 + c) * a.state_v;
                        const float x = S[s][v][r];
                        if constexpr (SLOPE) W[s][v][r] = fmaf(W[s][v][r], past_hi, fmaf(x, past_slope, slope_first && on ? slope_first[element] : 0.f));
                        S[s][v][r] = fmaf(x, past_hi, fmaf(x, past_lo, first && on ? first[element] : 0.f));
                    }
        }
    }
    const float apart[3] = {1.f, powers[16], powers[32]};
    float total = 0;                                                         // LEAKY_SLOPE

    auto fill = [&](int thread, int g, int col) {                            // LDS for the next chunk
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = i * 256 + thread;
            if (kChunk * KV % 256 == 0 || at < kChunk * KV) *reinterpret_cast<Vec*>(keys + at / KV * kPitch + at % KV * V) = nk[i];
            if (BOTH) bad = bad || any_not_finite(nk[i]);
        }
#pragma unroll
        for (int i = 0; i < vLoads; ++i) {
            const int at = i * 256 + thread;
            if (kChunk * VV % 256 == 0 || at < kChunk * VV) *reinterpret_cast<Vec*>(values + at / VV * vPitch + at % VV * V) = nv[i];
            if (MAIN) bad = bad || any_not_finite(nv[i]);
        }
        if (MAIN && bad) not_finite = p0;
        if constexpr (MAIN) {
#pragma unroll
            for (int s = 0; s < ST; ++s) {
                if (KT % 4 != 0 && s * 4 + wave >= KT) continue;
#pragma unroll
                for (int v = 0; v < VT; ++v) {
                    share(S[s][v], 0, s * 4 + wave, v, g, col);
                    if constexpr (SLOPE) share(W[s][v], 1, s * 4 + wave, v, g, col);
                }
            }
        }
    };
    for (; p0 < stop; p0 += kChunk) {
        // the thread's place, worked out anew: kept, the addresses made of it for the four strips would take 60 registers
        int thread = threadIdx.x;
        asm volatile("" : "+v"(thread));
        const int lane = thread & 63, g = lane >> 4, col = lane & 15;
        __syncthreads();                                                     // the chunk before is done with LDS
        fill(thread, g, col);
        __syncthreads();
        const bool odd_values = MAIN && __builtin_amdgcn_readfirstlane(not_finite) == p0;
        const bool more = p0 + kChunk < stop;
        if (more) fetch_rows(0, thread);

        const int missing = p0 < begin ? begin - p0 : 0;
        const double step = missing ? power(leak, kChunk - missing) : whole_leak;
        const float step_hi = (float)step, step_lo = (float)(step - (double)step_hi);
        const float step_slope = SLOPE ? (float)(kChunk - missing) * powers[kChunk - 1 - missing] : 0.f;

        auto chunk = [&](auto which) {
            constexpr int w = decltype(which)::value;
            f4 scores[4];
            // adds the products of weighted scores and values
            auto weigh = [&](F v, const f4 (&from)[4], int d, f4 to) {
                if constexpr (F32) {
                    return mma(v, from[d], to);
                } else {
                    const Split x = split(__builtin_shufflevector(from[2 * d], from[2 * d + 1], 0, 1, 2, 3, 4, 5, 6, 7));
                    for (int part = 0; part < kParts; ++part) to = mma(v, x.part[part], to);
                    return to;
                }
            };
            auto add_values = [&](auto& to, const f4 (&from)[4], int d, const auto& vf) {
                constexpr int N = sizeof(vf) / sizeof(F);
                if (odd_values && (d + 1) * D > w * 16) {                    // some of these scores are masked
                    F there, none, one;                                      // `there`: 1 for places up to this lane's
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        there[e] = (T)(d * D + (e >> 2) * 16 + 4 * g + (e & 3) <= w * 16 + col ? 1.f : 0.f);
                        none[e] = (T)0.f;
                        one[e] = (T)1.f;
                    }
#pragma unroll
                    for (int v = 0; v < N; ++v) {
                        const f4 reached = mma(where_not_finite(vf[v], one, none), there, f4{0, 0, 0, 0});
                        to[v] = weigh(where_not_finite(vf[v], none, vf[v]), from, d, to[v]);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (reached[r] > 0.f) to[v][r] = __builtin_nanf("");
                    }
                    return;
                }
                if constexpr (F32) {
#pragma unroll
                    for (int v = 0; v < N; ++v) to[v] = mma(vf[v], from[d], to[v]);
                } else {
                    const Split x = split(__builtin_shufflevector(from[2 * d], from[2 * d + 1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int part = 0; part < kParts; ++part)
#pragma unroll
                        for (int v = 0; v < N; ++v) to[v] = mma(vf[v], x.part[part], to[v]);
                }
            };
            // the state's part of the results
            auto of_state = [&](f4 (&to)[VT], int which) {
#pragma unroll
                for (int v = 0; v < VT; ++v) to[v] = f4{0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < KP / D; ++d)
#pragma unroll
                    for (int part = 0; part < P; ++part)
#pragma unroll
                        for (int v = 0; v < VT; ++v)
                            to[v] = mma(along(state + (which * P + part) * VP * kPitch, kPitch, v * 16, d * D, lane), qf[d], to[v]);
            };
            if constexpr (MAIN) {
                // scores, transposed: lane has keys 4g ... 4g+3 of each strip for its place
#pragma unroll
                for (int s = 0; s < 4; ++s) scores[s] = f4{0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < KP / D; ++d)
#pragma unroll
                    for (int s = 0; s <= w; ++s) scores[s] = mma(along(keys, kPitch, s * 16, d * D, lane), qf[d], scores[s]);
            }
            phase_end();
            const int i = w * 16 + col - missing + shift;                    // places of the chunk up to this lane's
            const float reach = MAIN ? power_at(powers, i) * a.state_scale : 0.f;
            const int p = p0 + w * 16 + col;
            auto store = [&](const auto& acc, T* out, int64_t out_t, int left, bool whole) {
                constexpr int N = sizeof(acc) / sizeof(f4);
                if (whole) {                                                 // four results that are all there or not at all
                    const int row = w * 16 + col, from = a.backwards ? kChunk - 1 - row : row;
                    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                        out + (int64_t)(a.backwards ? length - kChunk - p0 : p0) * out_t, 0, 0x7fffffff, 0x00020000);
                    const int off = (from * (int)out_t + 4 * g) * (int)sizeof(T);
#pragma unroll
                    for (int v = 0; v < N; ++v) {
                        const int to = p >= begin && v * 16 + 4 * g < left ? off + v * 16 * (int)sizeof(T) : kNowhere;
                        if constexpr (F32) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, acc[v]), r, to, 0, 0);
                        else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, __builtin_convertvector(acc[v], b4)), r, to, 0, 0);
                    }
                } else if (p >= begin) {
                    T* o = out + place(p) * out_t;
#pragma unroll
                    for (int v = 0; v < N; ++v)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (v * 16 + 4 * g + r < left) o[v * 16 + 4 * g + r] = (T)acc[v][r];
                }
            };
            if constexpr (MODE == LEAKY_SLOPE) {
                f4 dacc[VT], dscores[4];
                of_state(dacc, 1);
                {
                    f4 acc[VT];
                    of_state(acc, 0);
                    const float reach_slope = slope_at(powers, i) * a.state_scale;
#pragma unroll
                    for (int v = 0; v < VT; ++v) dacc[v] = dacc[v] * reach + acc[v] * reach_slope;
                }
#pragma unroll
                for (int d = 0; d < kChunk / D; ++d) {
                    if (d * D > w * 16) continue;
                    phase_end();
#pragma unroll
                    for (int s = d * D / 16; s < (d + 1) * D / 16; ++s)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int back = (w - s) * 16 + col - 4 * g - r;
                            dscores[s][r] = s > w || back < 1 ? 0.f : scores[s][r] * (slope_at(powers, s > w ? 0 : back) * a.score_scale);
                        }
                    F vf[VT];
#pragma unroll
                    for (int v = 0; v < VT; ++v) vf[v] = across(values, vPitch, v * 16, d * D, lane);
                    add_values(dacc, dscores, d, vf);
                }
#pragma unroll
                for (int v = 0; v < VT; ++v)                                 // (0 for places and values that are not there)
#pragma unroll
                    for (int r = 0; r < 4; ++r) total = fmaf((float)other[v][r], dacc[v][r], total);
                if (more) fetch_other(0, g, col);
                phase_end();
            }
            auto weigh_scores = [&]() {
                // key 4g + r of the strip of this lane's place, and of strips in front of it, in which a factor a^(16 strips) is left out
                float near[4], far[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    near[r] = weights[16 + col - 4 * g - r];
                    far[r] = weights[32 + col - 4 * g - r];
                }
#pragma unroll
                for (int s = 0; s <= w; ++s)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        scores[s][r] = s == w ? (col >= 4 * g + r ? scores[s][r] * near[r] : 0.f)
                                              : scores[s][r] * (s + 1 == w ? far[r] : far[r] * apart[w - s - 1]);
            };
            f4 acc[VT];
            if constexpr (MAIN) {
                of_state(acc, 0);
                phase_end();
                if (more) fetch_query(0, g, col);
#pragma unroll
                for (int v = 0; v < VT; ++v) acc[v] *= reach;
                weigh_scores();
            }
            if constexpr (MAIN) {                                            // (values are read twice: fewer sums are kept at once)
#pragma unroll
                for (int d = 0; d < kChunk / D; ++d) {
                    if (d * D > w * 16) continue;
                    phase_end();
                    F vf[VT];
#pragma unroll
                    for (int v = 0; v < VT; ++v) vf[v] = across(values, vPitch, v * 16, d * D, lane);
                    add_values(acc, scores, d, vf);
                }
                store(acc, out, a.out_t, vleft, a.whole_out);
            }
            if constexpr (BOTH) {
                phase_end();
#pragma unroll
                for (int s = 0; s < 4; ++s) scores[s] = f4{0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < VP / D; ++d)
#pragma unroll
                    for (int s = 0; s <= w; ++s) scores[s] = mma(along_halves(values, vPitch, s * 16, d * D, lane), qf2[d], scores[s]);
                f4 acc2[KT];
#pragma unroll
                for (int k = 0; k < KT; ++k) acc2[k] = f4{0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < VP / D; ++d)
#pragma unroll
                    for (int part = 0; part < P; ++part)
#pragma unroll
                        for (int k = 0; k < KT; ++k) acc2[k] = mma(across(state + part * VP * kPitch, kPitch, k * 16, d * D, lane), qf2[d], acc2[k]);
                phase_end();
                if (more) fetch_query2(0, g, col);
#pragma unroll
                for (int k = 0; k < KT; ++k) acc2[k] *= reach;
                weigh_scores();
#pragma unroll
                for (int d = 0; d < kChunk / D; ++d) {
                    if (d * D > w * 16) continue;
                    phase_end();
                    F kf[KT];
#pragma unroll
                    for (int k = 0; k < KT; ++k) kf[k] = across(keys, kPitch, k * 16, d * D, lane);
                    add_values(acc2, scores, d, kf);
                }
                store(acc2, out2, a.out2_t, a.keys, a.whole_out2);
            }
#pragma unroll
            for (int s = 0; s < ST; ++s)
#pragma unroll
                for (int v = 0; v < VT; ++v) {
                    if constexpr (SLOPE) W[s][v] = W[s][v] * step_hi + S[s][v] * step_slope;
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[s][v][r] = fmaf(S[s][v][r], step_hi, S[s][v][r] * step_lo);
                }
#pragma unroll
            for (int d = 0; d < kChunk / D; ++d) {
                phase_end();
                F vf[VT];                                                    // values, terms across the places
#pragma unroll
                for (int v = 0; v < VT; ++v) vf[v] = across(values, vPitch, v * 16, d * D, lane);
#pragma unroll
                for (int s = 0; s < ST; ++s) {
                    if (s * 4 + w >= KT) continue;
                    const F kf = across(keys, kPitch, (s * 4 + w) * 16, d * D, lane);
                    auto add_keys = [&](f4 (&to)[VT], const float* weights) {
                        const f4 w0 = *reinterpret_cast<const f4*>(weights + d * D + 4 * g);
                        if constexpr (F32) {
                            const f4 x = kf * w0;
#pragma unroll
                            for (int v = 0; v < VT; ++v) to[v] = mma(x, vf[v], to[v]);
                        } else {
                            const f4 w1 = *reinterpret_cast<const f4*>(weights + d * D + 16 + 4 * g);
                            const Split x = split(__builtin_convertvector(kf, f8) * __builtin_shufflevector(w0, w1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                            for (int part = 0; part < kParts; ++part)
#pragma unroll
                                for (int v = 0; v < VT; ++v) to[v] = mma(x.part[part], vf[v], to[v]);
                        }
                    };
                    add_keys(S[s], behind[0]);
                    if constexpr (SLOPE) add_keys(W[s], behind[1]);
                }
            }
        };
        if (wave == 0) chunk(std::integral_constant<int, 0>{});
        else if (wave == 1) chunk(std::integral_constant<int, 1>{});
        else if (wave == 2) chunk(std::integral_constant<int, 2>{});
        else chunk(std::integral_constant<int, 3>{});
    }

    const bool last = MAIN && ((begin < length && length <= begin + a.segment) || (length == 0 && seg == 0));
    float *to = nullptr, *slope_to = nullptr;
    if (!MAIN) {
        const int64_t at = ((int64_t)unit * a.segments + seg + 1) * state_size;
        to = a.starts + at;
        if (SLOPE) slope_to = a.slope_starts + at;
    } else if (last && a.last) {
        to = a.last + unit * state_size;
    }
    const float* grad_last = MODE == LEAKY_SLOPE && last && a.grad_last ? a.grad_last + unit * state_size : nullptr;
    double slope = total;
    if (to || grad_last) {
#pragma unroll
        for (int s = 0; s < ST; ++s)
#pragma unroll
            for (int v = 0; v < VT; ++v)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int k = (s * 4 + wave) * 16 + 4 * g + r, c = v * 16 + col;
                    const int64_t at = (int64_t)k * a.state_k + (int64_t)(v0 + c) * a.state_v;
                    if (k < a.keys && c < vleft) {
                        if (to) to[at] = S[s][v][r];
                        if constexpr (SLOPE) {
                            if (slope_to) slope_to[at] = W[s][v][r];
                            if (grad_last) slope += (double)W[s][v][r] * grad_last[at];
                        }
                    }
                }
    }
    if (MODE == LEAKY_SLOPE) {
        for (int d = 32; d > 0; d >>= 1) slope += __shfl_xor(slope, d);
        if (lane == 0) sums[wave] = slope;
        __syncthreads();
        if (threadIdx.x == 0) a.slopes[((int64_t)unit * a.segments + seg) * a.slices + slice] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
    // tokens behind the sample's end
    if (MAIN) {
        for (int64_t at = threadIdx.x; at < (int64_t)(end - max(begin, length)) * VP; at += 256) {
            const int p = max(begin, length) + (int)(at / VP), c = (int)(at % VP);
            if (c < vleft) out[p * a.out_t + c] = (T)0.f;
        }
        if constexpr (BOTH)
            for (int64_t at = threadIdx.x; at < (int64_t)(end - max(begin, length)) * KP; at += 256) {
                const int p = max(begin, length) + (int)(at / KP), c = (int)(at % KP);
                if (c < a.keys) out2[p * a.out2_t + c] = (T)0.f;
            }
    }
}

template <typename T, int MODE>
int launch_leaky_mode(const LeakyPass& p, dim3 grid, bool whole, hipStream_t s) {
    const int vt = p.tiles;
#define LAUNCH(K, V, WHOLE) hipLaunchKernelGGL((leaky_kernel<T, K, V, MODE, WHOLE>), grid, dim3(256), 0, s, p)
#define BY_KEYS(V, WHOLE)                           \
    if (p.keys <= 32) LAUNCH(2, V, WHOLE);          \
    else if (p.keys <= 64) LAUNCH(4, V, WHOLE);     \
    else if (p.keys <= 96) LAUNCH(6, V, WHOLE);     \
    else LAUNCH(8, V, WHOLE)
    if (!whole) {
        if (vt == 2) { if (p.keys <= 64) LAUNCH(4, 2, false); else LAUNCH(8, 2, false); }
        else { if (p.keys <= 64) LAUNCH(4, 4, false); else LAUNCH(8, 4, false); }
    }
    else if (vt == 1) { BY_KEYS(1, true); }
    else if (vt == 2) { BY_KEYS(2, true); }
    else if (vt == 3) { BY_KEYS(3, true); }
    else { BY_KEYS(4, true); }
#undef BY_KEYS
#undef LAUNCH
    return (int)hipGetLastError();
}

// LEAKY_BOTH: up to 96 keys and 64 values, in whole pieces
template <typename T>
int launch_leaky_both(const LeakyPass& p, dim3 grid, hipStream_t s) {
#define LAUNCH(K, V) hipLaunchKernelGGL((leaky_kernel<T, K, V, LEAKY_BOTH, true>), grid, dim3(256), 0, s, p)
#define BY_VALUES(K) if (p.tiles == 2) LAUNCH(K, 2); else LAUNCH(K, 4)
    if (p.keys <= 32) { BY_VALUES(2); }
    else if (p.keys <= 64) { BY_VALUES(4); }
    else { BY_VALUES(6); }
#undef BY_VALUES
#undef LAUNCH
    return (int)hipGetLastError();
}

template <typename T> int launch_leaky(const LeakyPass& p, int mode, bool whole, hipStream_t stream);    // attention_f32.hip, attention_bf16.hip

}  // namespace slayer

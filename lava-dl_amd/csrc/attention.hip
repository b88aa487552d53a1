// Leaky attention: linear attention whose state, a [keys][values] matrix for each sample and head, leaks like the current of a
// neuron (a = 1 - decay / 4096):
//     S[t] = a S[t-1] + key[t] (outer) value[t],     out[t] = scale * query[t] S[t].
// A prompt is taken in chunks of 64 tokens.  With S the state in front of a chunk and i, j the places inside it,
//     out[i] = a^(i+1) query[i] S + sum over j <= i of a^(i-j) (query[i] . key[j]) value[j]
//     S'     = a^64 S + sum over j of a^(63-j) key[j] (outer) value[j],
// four products on the matrix cores.  The gradients are the same recurrence with other tensors in its three places:
//     grad query: forwards,  query = grad out, key = value,    value = key    (state transposed)
//     grad value: backwards, query = key,      key = query,    value = grad out
//     grad key:   backwards, query = value,    key = grad out, value = query  (state transposed)
// where "backwards" counts places from a sample's end and the state G, the gradient of the state behind the chunk, meets
// place i with a^i (not a^(i+1)): G' = a^64 G + sum over i of a^(64-i) query[i] (outer) grad[i].
#include "common.h"
#include "elements.h"

namespace slayer {

constexpr int kChunk = 64;

// One pass of the recurrence, as its kernels see it.  `query`, `key`, `value` are the tensors in the three places.
struct LeakyPass {
    void* out;
    const void *query, *key, *value;
    const float* decay;
    const void* lengths;
    const float* first;            // [samples][heads] states with strides first_k, first_v, or nullptr: zeros
    float* starts;                 // states in front of the segments, [samples * heads][segments] of them
    float* last;                   // state behind the last token, or nullptr
    int64_t out_n, out_t, out_h, query_n, query_t, query_h, key_n, key_t, key_h, value_n, value_t, value_h;
    int tokens, heads, keys, values, state_k, state_v;      // the strides of a state's axes
    int one_decay, lengths64, segments, segment, slices, backwards;
    int whole_query, whole_key, whole_value, whole_out;
    float out_scale, key_scale;    // of the results; of what `key` stands for, in scores and in the state
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
__device__ __forceinline__ typename Frag<T>::Type along(const T* tile, int pitch, int row, int term) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const typename Frag<T>::Type*>(tile + (row + (lane & 15)) * pitch + term + (lane >> 4) * Elements<T>::kVec);
}
// terms across the rows of `tile`, the sixteen columns from `column` on
__device__ __forceinline__ f4 across(const float* tile, int pitch, int column, int term) {
    const int lane = threadIdx.x & 63;
    const float* p = tile + (term + (lane >> 4) * 4) * pitch + column + (lane & 15);
    return f4{p[0], p[pitch], p[2 * pitch], p[3 * pitch]};
}
typedef __attribute__((address_space(3))) short LdsShort;
typedef short s4 __attribute__((ext_vector_type(4)));
// ds_read_b64_tr_b16: the sixteen lanes of a group read four rows of sixteen columns, lane i gets column i of the four
__device__ __forceinline__ b8 across(const bf16* tile, int pitch, int column, int term) {
    const int lane = threadIdx.x & 63, i = lane & 15;
    const bf16* p = tile + (term + (lane >> 4) * 4 + (i >> 2)) * pitch + column + (i & 3) * 4;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(LdsShort*)p);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(LdsShort*)(p + 16 * pitch));
    const b4 a = __builtin_bit_cast(b4, lo), b = __builtin_bit_cast(b4, hi);
    return b8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// A float32 operand: in float32, or as two bfloat16 numbers whose sum is within 2^-17 of it, so that what the kernel makes
// itself (scores, the state, leaked keys) is not rounded to the type of the tensors on the way.
template <typename T> struct Operand;
template <> struct Operand<float> {
    static constexpr int kParts = 1;
    f4 part[1];
};
template <> struct Operand<bf16> {
    static constexpr int kParts = 2;
    b8 part[2];
};
__device__ __forceinline__ Operand<bf16> split(f8 v) {
    Operand<bf16> o;
    o.part[0] = __builtin_convertvector(v, b8);
    o.part[1] = __builtin_convertvector(v - __builtin_convertvector(o.part[0], f8), b8);
    return o;
}
template <typename T>
__device__ __forceinline__ f4 mma(const Operand<T>& a, typename Frag<T>::Type b, f4 c) {
#pragma unroll
    for (int i = 0; i < Operand<T>::kParts; ++i) c = mma(a.part[i], b, c);
    return c;
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

// A workgroup of four waves takes one segment of one head of one sample, chunk after chunk, and one slice of 16 VT values.
// Wave w makes the outputs of places 16w ... 16w+15 (transposed: lane = place) and the rows of the state w, w+4, ... (16 each).
//   MAIN false: only the state, from zero, into `starts` behind the segment's place (for the segments but the last).
template <typename T, int KT, int VT, bool MAIN>
__global__ __launch_bounds__(256) void leaky_kernel(LeakyPass a) {
    typedef typename Frag<T>::Type F;
    constexpr int V = Elements<T>::kVec, D = Frag<T>::kDepth, P = Operand<T>::kParts;
    constexpr int KP = KT * 16, VP = VT * 16, kPitch = KP + V, vPitch = VP + V;
    constexpr int KV = KP / V, VV = VP / V;                                  // 16-byte pieces of a row
    constexpr int kLoads = (kChunk * KV + 255) / 256, vLoads = (kChunk * VV + 255) / 256;
    constexpr int ST = (KT + 3) / 4;                                         // strips of the state of a wave
    __shared__ __align__(16) T keys[kChunk * kPitch];
    __shared__ __align__(16) T values[kChunk * vPitch];
    __shared__ __align__(16) T state[MAIN ? P * VP * kPitch : 8];            // transposed: [part][value][key]
    __shared__ float powers[kChunk + 1], weights[kChunk + 1];                // a^i; what a key counts i places on

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
    int b = blockIdx.x;
    const int slice = b % a.slices; b /= a.slices;
    const int segments = MAIN ? a.segments : a.segments - 1;
    const int seg = b % segments, unit = b / segments;
    const int n = unit / a.heads, h = unit % a.heads;
    const int v0 = slice * VP, length = sample_length(a, n);
    const double leak = 1.0 - (double)a.decay[a.one_decay ? 0 : h] / 4096.0;
    const int begin = seg * a.segment, end = min(begin + a.segment, a.tokens);
    if (!MAIN && end > length) return;                                       // no segment behind it needs this one's state
    if (threadIdx.x <= kChunk) {
        const double p = power(leak, threadIdx.x);
        powers[threadIdx.x] = (float)p;
        weights[threadIdx.x] = (float)(p * a.key_scale);
    }
    const double whole_leak = power(leak, kChunk);

    const T* query = (const T*)a.query + n * a.query_n + h * a.query_h;
    const T* key = (const T*)a.key + n * a.key_n + h * a.key_h;
    const T* value = (const T*)a.value + n * a.value_n + h * a.value_h + v0;
    T* out = (T*)a.out + n * a.out_n + h * a.out_h + v0;
    const int64_t state_size = (int64_t)a.keys * a.values;
    const int vleft = a.values - v0;
    auto place = [&](int p) { return (int64_t)(a.backwards ? length - 1 - p : p); };     // the token of a place in front of the end

    // the state, in strips of 16 keys: lane has keys 4g ... 4g+3 of column `col`
    f4 S[ST][VT];
    const float* first = nullptr;
    if (MAIN) first = seg > 0 ? a.starts + ((int64_t)unit * a.segments + seg) * state_size : (a.first ? a.first + unit * state_size : nullptr);
#pragma unroll
    for (int s = 0; s < ST; ++s)
#pragma unroll
        for (int v = 0; v < VT; ++v)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int k = (s * 4 + wave) * 16 + 4 * g + r, c = v * 16 + col;
                S[s][v][r] = first && begin <= length && k < a.keys && c < vleft ? first[(int64_t)k * a.state_k + (int64_t)(v0 + c) * a.state_v] : 0.f;
            }
    auto share_state = [&]() {
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            if ((s * 4 + wave) * 16 >= KP) continue;
#pragma unroll
            for (int v = 0; v < VT; ++v) {
                T* p = state + (v * 16 + col) * kPitch + (s * 4 + wave) * 16 + 4 * g;
                if constexpr (P == 1) {
                    *reinterpret_cast<f4*>(p) = S[s][v];
                } else {
                    const b4 hi = __builtin_convertvector(S[s][v], b4);
                    *reinterpret_cast<b4*>(p) = hi;
                    *reinterpret_cast<b4*>(p + VP * kPitch) = __builtin_convertvector(S[s][v] - __builtin_convertvector(hi, f4), b4);
                }
            }
        }
    };
    if (MAIN) share_state();

    // what the next chunk needs, on its way
    typename Elements<T>::Vec nk[kLoads], nv[vLoads];
    auto fetch = [&](int p0) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = i * 256 + threadIdx.x, p = p0 + at / KV, k = at % KV * V;
            nk[i] = load_vec(key + (p < length && p < end ? place(p) : 0) * a.key_t + k,
                             at < kChunk * KV && p < length && p < end ? a.keys - k : 0, a.whole_key);
        }
#pragma unroll
        for (int i = 0; i < vLoads; ++i) {
            const int at = i * 256 + threadIdx.x, p = p0 + at / VV, c = at % VV * V;
            nv[i] = load_vec(value + (p < length && p < end ? place(p) : 0) * a.value_t + c,
                             at < kChunk * VV && p < length && p < end ? vleft - c : 0, a.whole_value);
        }
    };
    if (begin < length) fetch(begin);

    for (int p0 = begin; p0 < end && p0 < length; p0 += kChunk) {
        const int count = min(min(end, length) - p0, kChunk);
        __syncthreads();                                                     // the chunk before is done with LDS
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = i * 256 + threadIdx.x;
            if (at < kChunk * KV) *reinterpret_cast<typename Elements<T>::Vec*>(keys + at / KV * kPitch + at % KV * V) = nk[i];
        }
#pragma unroll
        for (int i = 0; i < vLoads; ++i) {
            const int at = i * 256 + threadIdx.x;
            if (at < kChunk * VV) *reinterpret_cast<typename Elements<T>::Vec*>(values + at / VV * vPitch + at % VV * V) = nv[i];
        }
        __syncthreads();
        if (p0 + kChunk < end && p0 + kChunk < length) fetch(p0 + kChunk);

        F vf[kChunk / D][VT];                                                // value, terms across the places
#pragma unroll
        for (int d = 0; d < kChunk / D; ++d)
#pragma unroll
            for (int v = 0; v < VT; ++v) vf[d][v] = across(values, vPitch, v * 16, d * D);

        if (MAIN) {
            const int i = wave * 16 + col, p = p0 + i;                       // this lane's place
            const bool there = i < count;
            F qf[KP / D];
#pragma unroll
            for (int d = 0; d < KP / D; ++d) {
                const int k = d * D + g * V;
                qf[d] = load_vec(query + (there ? place(p) : 0) * a.query_t + k, there ? a.keys - k : 0, a.whole_query);
            }
            // scores, transposed: lane has keys 4g ... 4g+3 of each strip for its place
            f4 scores[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                scores[s] = f4{0, 0, 0, 0};
                if (s > wave) continue;
#pragma unroll
                for (int d = 0; d < KP / D; ++d) scores[s] = mma(along(keys, kPitch, s * 16, d * D), qf[d], scores[s]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int back = i - (s * 16 + 4 * g + r);
                    scores[s][r] = back >= 0 ? scores[s][r] * weights[back >= 0 ? back : 0] : 0.f;
                }
            }
            f4 acc[VT];
            const float reach = a.backwards ? powers[i] : powers[i + 1];
#pragma unroll
            for (int v = 0; v < VT; ++v) {
                acc[v] = f4{0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < KP / D; ++d)
#pragma unroll
                    for (int part = 0; part < P; ++part)
                        acc[v] = mma(along(state + part * VP * kPitch, kPitch, v * 16, d * D), qf[d], acc[v]);
                acc[v] *= reach;
            }
#pragma unroll
            for (int d = 0; d < kChunk / D; ++d) {
                if (d * D > wave * 16 + 15) continue;
                Operand<T> w;
                if constexpr (P == 1) w.part[0] = scores[d];
                else w = split(f8{scores[2 * d][0], scores[2 * d][1], scores[2 * d][2], scores[2 * d][3], scores[2 * d + 1][0],
                                  scores[2 * d + 1][1], scores[2 * d + 1][2], scores[2 * d + 1][3]});
#pragma unroll
                for (int v = 0; v < VT; ++v)
#pragma unroll
                    for (int part = 0; part < P; ++part) acc[v] = mma(vf[d][v], w.part[part], acc[v]);
            }
            if (there) {
                T* o = out + place(p) * a.out_t;
#pragma unroll
                for (int v = 0; v < VT; ++v) {
                    const int c = v * 16 + 4 * g;
                    const f4 y = acc[v] * a.out_scale;
                    if (a.whole_out && c + 4 <= vleft) {
                        if constexpr (P == 1) *reinterpret_cast<f4*>(o + c) = y;
                        else *reinterpret_cast<b4*>(o + c) = __builtin_convertvector(y, b4);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (c + r < vleft) o[c + r] = (T)y[r];
                    }
                }
            }
        }

        // the state
        const double step = count == kChunk ? whole_leak : power(leak, count);
        const float step_hi = (float)step, step_lo = (float)(step - (double)step_hi);
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            const int strip = s * 4 + wave;
            if (strip >= KT) continue;
#pragma unroll
            for (int v = 0; v < VT; ++v)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[s][v][r] = fmaf(S[s][v][r], step_hi, S[s][v][r] * step_lo);
#pragma unroll
            for (int d = 0; d < kChunk / D; ++d) {
                const F kf = across(keys, kPitch, strip * 16, d * D);
                float w[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int j = d * D + (e >> 2) * 16 + 4 * g + (e & 3);
                    const int left = count - 1 - j + (a.backwards ? 1 : 0);
                    w[e] = j < count ? (float)kf[e] * weights[j < count ? left : 0] : 0.f;
                }
                Operand<T> leaked;
                if constexpr (P == 1) leaked.part[0] = f4{w[0], w[1], w[2], w[3]};
                else leaked = split(f8{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]});
#pragma unroll
                for (int v = 0; v < VT; ++v) S[s][v] = mma<T>(leaked, vf[d][v], S[s][v]);
            }
        }
        if (MAIN && p0 + kChunk < end && p0 + kChunk < length) {
            __syncthreads();
            share_state();
        }
    }

    float* to = nullptr;
    if (!MAIN) to = a.starts + ((int64_t)unit * a.segments + seg + 1) * state_size;
    else if (a.last && ((begin < length && length <= begin + a.segment) || (length == 0 && seg == 0))) to = a.last + unit * state_size;
    if (to) {
#pragma unroll
        for (int s = 0; s < ST; ++s)
#pragma unroll
            for (int v = 0; v < VT; ++v)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int k = (s * 4 + wave) * 16 + 4 * g + r, c = v * 16 + col;
                    if (k < a.keys && c < vleft) to[(int64_t)k * a.state_k + (int64_t)(v0 + c) * a.state_v] = S[s][v][r];
                }
    }
    // tokens behind the sample's end
    if (MAIN) {
        for (int64_t at = threadIdx.x; at < (int64_t)(end - max(begin, length)) * VP; at += 256) {
            const int p = max(begin, length) + (int)(at / VP), c = (int)(at % VP);
            if (c < vleft) out[p * a.out_t + c] = (T)0.f;
        }
    }
}

// starts[unit][seg], which holds what the segment in front of it adds, becomes the state in front of segment seg.
__global__ __launch_bounds__(256) void leaky_join_kernel(LeakyPass a) {
    const int64_t size = (int64_t)a.keys * a.values;
    const int64_t per = (size + 255) / 256;
    const int64_t unit = blockIdx.x / per, at = blockIdx.x % per * 256 + threadIdx.x;
    if (at >= size) return;
    const int n = (int)(unit / a.heads), h = (int)(unit % a.heads), length = sample_length(a, n);
    const double step = power(1.0 - (double)a.decay[a.one_decay ? 0 : h] / 4096.0, a.segment);
    const float hi = (float)step, lo = (float)(step - (double)hi);
    float s = a.first ? a.first[unit * size + at] : 0.f;
    float* starts = a.starts + unit * a.segments * size + at;
    for (int seg = 1; seg < a.segments && (int64_t)seg * a.segment <= length; ++seg) {
        s = fmaf(s, hi, fmaf(s, lo, starts[seg * size]));
        starts[seg * size] = s;
    }
}

// Gradient of the leak, with W[t] = dS[t] / da = S[t-1] + a W[t-1]: the sum over t of query[t] W[t] grad[t], and of the last W with
// the gradient of the last state.  A workgroup walks one head of one sample, a thread has E elements of S and W.
constexpr int kWalk = 16;                      // tokens in LDS at once
template <typename T, int E>
__global__ __launch_bounds__(256) void leaky_slope_kernel(double* __restrict__ slopes, const T* __restrict__ grad, const float* __restrict__ grad_last,
                                                          int64_t grad_n, int64_t grad_t, int64_t grad_h, LeakyPass a) {
    __shared__ float q[kWalk][128], k[kWalk][128], v[kWalk][128], g[kWalk][128];
    __shared__ double sums[4];
    const int unit = blockIdx.x, n = unit / a.heads, h = unit % a.heads, length = sample_length(a, n), size = a.keys * a.values;
    const float leak = (float)(1.0 - (double)a.decay[a.one_decay ? 0 : h] / 4096.0);
    const T* query = (const T*)a.query + n * a.query_n + h * a.query_h;
    const T* key = (const T*)a.key + n * a.key_n + h * a.key_h;
    const T* value = (const T*)a.value + n * a.value_n + h * a.value_h;
    grad += n * grad_n + h * grad_h;
    float S[E], W[E], sum = 0;
    int row[E], column[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int at = e * 256 + threadIdx.x;
        row[e] = at < size ? at / a.values : 0;
        column[e] = at < size ? at % a.values : 0;
        S[e] = a.first && at < size ? a.first[(int64_t)unit * size + at] : 0.f;
        W[e] = 0;
    }
    for (int t0 = 0; t0 < length; t0 += kWalk) {
        __syncthreads();
        for (int at = threadIdx.x; at < kWalk * 128; at += 256) {
            const int t = t0 + at / 128, c = at % 128;
            const bool on = t < length;
            q[at / 128][c] = on && c < a.keys ? (float)query[t * a.query_t + c] : 0.f;
            k[at / 128][c] = on && c < a.keys ? (float)key[t * a.key_t + c] : 0.f;
            v[at / 128][c] = on && c < a.values ? (float)value[t * a.value_t + c] : 0.f;
            g[at / 128][c] = on && c < a.values ? (float)grad[t * grad_t + c] : 0.f;
        }
        __syncthreads();
        for (int i = 0; i < kWalk && t0 + i < length; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (e * 256 + (int)threadIdx.x >= size) continue;
                W[e] = fmaf(leak, W[e], S[e]);
                S[e] = fmaf(leak, S[e], k[i][row[e]] * v[i][column[e]]);
                sum = fmaf(q[i][row[e]] * g[i][column[e]], W[e], sum);
            }
    }
    double total = (double)sum * a.out_scale;
    if (grad_last) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int at = e * 256 + threadIdx.x;
            if (at < size) total += (double)W[e] * grad_last[(int64_t)unit * size + at];
        }
    }
    for (int d = 32; d > 0; d >>= 1) total += __shfl_xor(total, d);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = total;
    __syncthreads();
    if (threadIdx.x == 0) slopes[unit] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// grad decay = - slope / 4096, summed over the samples (and the heads that share one decay)
__global__ __launch_bounds__(256) void leaky_decay_kernel(float* __restrict__ grad_decay, const double* __restrict__ slopes, int samples,
                                                          int heads, int one_decay, int parts) {
    __shared__ double sums[4];
    const int64_t count = (int64_t)samples * parts * (one_decay ? heads : 1);
    double total = 0;
    for (int64_t i = threadIdx.x; i < count; i += 256)       // slopes[sample][head][part]
        total += one_decay ? slopes[i] : slopes[(i / parts * heads + blockIdx.x) * parts + i % parts];
    for (int d = 32; d > 0; d >>= 1) total += __shfl_xor(total, d);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = total;
    __syncthreads();
    if (threadIdx.x == 0) grad_decay[blockIdx.x] = (float)(((sums[0] + sums[1]) + (sums[2] + sums[3])) / -4096.0);
}

// One token a sample: the state is read, leaked, added to, multiplied with the query and written back.  A workgroup takes QP
// quads of values and all keys of one head; 256 / QP rows of keys at a time.
template <typename T, int QP>
__global__ __launch_bounds__(256) void leaky_step_kernel(T* __restrict__ out, float* __restrict__ state, const T* __restrict__ query,
                                                         const T* __restrict__ key, const T* __restrict__ value,
                                                         const float* __restrict__ decay, int one_decay, int heads, int keys, int values,
                                                         int64_t query_n, int64_t query_h, int64_t key_n, int64_t key_h, int64_t value_n,
                                                         int64_t value_h, int tiles, int whole, float scale) {
    constexpr int ROWS = 256 / QP;
    __shared__ f4 sums[256];
    const int tile = blockIdx.x % tiles, unit = blockIdx.x / tiles, n = unit / heads, h = unit % heads;
    const int quad = threadIdx.x % QP, row = threadIdx.x / QP, c = (tile * QP + quad) * 4;
    const float leak = (float)(1.0 - (double)decay[one_decay ? 0 : h] / 4096.0);
    query += n * query_n + h * query_h;
    key += n * key_n + h * key_h;
    value += n * value_n + h * value_h;
    float* S = state + (int64_t)unit * keys * values + c;
    const int left = values - c;
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? (float)value[c + i] : 0.f;
    f4 sum = {0, 0, 0, 0};
    if (left > 0) {
        for (int k = row; k < keys; k += ROWS) {
            const float kk = (float)key[k], q = (float)query[k];
            f4 s = load_vec(S + (int64_t)k * values, left, whole);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = fmaf(kk, v[i], s[i] * leak);
                sum[i] = fmaf(q, s[i], sum[i]);
            }
            store_vec(S + (int64_t)k * values, s, left, whole);
        }
    }
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (row == 0 && left > 0) {
        for (int r = 1; r < ROWS; ++r) sum += sums[r * QP + quad];
        T* o = out + (int64_t)unit * values + c;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) o[i] = (T)(sum[i] * scale);
    }
}

}  // namespace slayer

using namespace slayer;

namespace {

int check_leaky(const slayer_attention* a) {
    if (!a) return SLAYER_ENULL;
    if (a->samples < 0 || a->tokens < 0 || a->heads < 1 || a->keys < 1 || a->values < 1) return SLAYER_EINVAL;
    if (a->dtype != SLAYER_FLOAT32 && a->dtype != SLAYER_BFLOAT16) return SLAYER_EINVAL;
    if (a->num_decays != 1 && a->num_decays != a->heads) return SLAYER_EINVAL;
    if (a->lengths && a->lengths_bytes != 4 && a->lengths_bytes != 8) return SLAYER_EINVAL;
    if (!a->decay) return SLAYER_ENULL;
    if (a->tokens > (1 << 30) || a->keys > 128 || a->values > 128 || a->heads > (1 << 20) || a->samples > (1 << 24) ||
        a->samples * a->heads > (1 << 24))
        return SLAYER_ERANGE;
    return 0;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Segments of a pass: enough workgroups for the chip (512: two a compute unit), and chunks enough in each that reading keys and
// values a second time for the states in front of them pays.
int segment_tokens(const slayer_attention* a, int slices) {
    const int64_t chunks = a->tokens > 0 ? ceil_div(a->tokens, kChunk) : 1, units = a->samples * a->heads * slices;
    int64_t segments = units > 0 ? 512 / units : 1;
    if (segments > chunks / 4) segments = chunks / 4;
    if (segments < 1) segments = 1;
    return ceil_div(chunks, segments) * kChunk;
}
int slice_tiles(int64_t values) { return values <= 16 ? 1 : values <= 32 ? 2 : 4; }

template <typename T, bool MAIN>
int launch_pass(const LeakyPass& p, int64_t units, hipStream_t stream) {
    const int kt = p.keys <= 32 ? 2 : p.keys <= 64 ? 4 : 8, vt = slice_tiles(p.values);
    const int64_t blocks = units * (MAIN ? p.segments : p.segments - 1) * p.slices;
    if (blocks == 0) return 0;
    if (blocks > (1 << 24) - 1) return SLAYER_ERANGE;
#define LAUNCH(K, V) hipLaunchKernelGGL((leaky_kernel<T, K, V, MAIN>), dim3((unsigned)blocks), dim3(256), 0, stream, p)
    if (kt == 2) { if (vt == 1) LAUNCH(2, 1); else if (vt == 2) LAUNCH(2, 2); else LAUNCH(2, 4); }
    else if (kt == 4) { if (vt == 1) LAUNCH(4, 1); else if (vt == 2) LAUNCH(4, 2); else LAUNCH(4, 4); }
    else { if (vt == 1) LAUNCH(8, 1); else if (vt == 2) LAUNCH(8, 2); else LAUNCH(8, 4); }
#undef LAUNCH
    return (int)hipGetLastError();
}

// aligned: every row that starts at `p` with these strides is a multiple of `bytes`
bool aligned(const void* p, const int64_t (&stride)[3], int size, int bytes) {
    return ((uintptr_t)p | (uintptr_t)(stride[0] * size) | (uintptr_t)(stride[1] * size) | (uintptr_t)(stride[2] * size)) % bytes == 0;
}

struct Place { const void* p; const int64_t (&stride)[3]; };

// One pass with its segments: states in front of them, joined, and the main kernel.
int run_pass(const slayer_attention* a, void* out, const int64_t (&out_stride)[3], Place query, Place key, Place value, int keys,
             int values, bool transposed, bool backwards, const float* first, float* last, float* workspace, hipStream_t stream) {
    const int size = a->dtype == SLAYER_FLOAT32 ? 4 : 2;
    LeakyPass p = {};
    p.out = out;
    p.query = query.p; p.key = key.p; p.value = value.p;
    p.decay = a->decay;
    p.lengths = a->lengths;
    p.first = first;
    p.starts = workspace;
    p.last = last;
    p.out_n = out_stride[0]; p.out_t = out_stride[1]; p.out_h = out_stride[2];
    p.query_n = query.stride[0]; p.query_t = query.stride[1]; p.query_h = query.stride[2];
    p.key_n = key.stride[0]; p.key_t = key.stride[1]; p.key_h = key.stride[2];
    p.value_n = value.stride[0]; p.value_t = value.stride[1]; p.value_h = value.stride[2];
    p.tokens = (int)a->tokens; p.heads = (int)a->heads; p.keys = keys; p.values = values;
    p.state_k = transposed ? 1 : values;
    p.state_v = transposed ? keys : 1;
    p.one_decay = a->num_decays == 1;
    p.lengths64 = a->lengths_bytes == 8;
    p.slices = ceil_div(values, slice_tiles(values) * 16);
    p.segment = segment_tokens(a, p.slices);
    p.segments = a->tokens > 0 ? ceil_div(a->tokens, p.segment) : 1;
    p.backwards = backwards;
    p.whole_query = aligned(query.p, query.stride, size, 16);
    p.whole_key = aligned(key.p, key.stride, size, 16);
    p.whole_value = aligned(value.p, value.stride, size, 16);
    p.whole_out = aligned(out, out_stride, size, 4 * size);
    p.out_scale = backwards ? 1.f : (float)a->scale;
    p.key_scale = backwards ? (float)a->scale : 1.f;      // the state it starts from is not scaled
    const int64_t units = a->samples * a->heads;
    if (p.segments > 1) {
        if (int e = size == 4 ? launch_pass<float, false>(p, units, stream) : launch_pass<bf16, false>(p, units, stream)) return e;
        const int64_t blocks = units * ceil_div((int64_t)keys * values, 256);
        if (blocks > (1 << 24) - 1) return SLAYER_ERANGE;
        hipLaunchKernelGGL(leaky_join_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p);
        if (int e = (int)hipGetLastError()) return e;
    }
    return size == 4 ? launch_pass<float, true>(p, units, stream) : launch_pass<bf16, true>(p, units, stream);
}

int64_t workspace_floats(const slayer_attention* a, int64_t values) {
    const int slices = ceil_div(values, slice_tiles(values) * 16);
    const int64_t segments = ceil_div(a->tokens, segment_tokens(a, slices));
    return segments > 1 ? a->samples * a->heads * segments * a->keys * a->values : 0;
}

template <typename T>
int launch_step(void* out, float* state, const void* query, const void* key, const void* value, const slayer_attention* a,
                hipStream_t stream) {
    const int quads = ceil_div(a->values, 4);
    const int qp = quads <= 4 ? 4 : quads <= 8 ? 8 : quads <= 16 ? 16 : 32, tiles = ceil_div(quads, qp);
    const int64_t blocks = a->samples * a->heads * tiles;
    if (blocks > (1 << 24) - 1) return SLAYER_ERANGE;
    const int whole = a->values % 4 == 0 && (uintptr_t)state % 16 == 0;
#define LAUNCH(Q)                                                                                                                \
    hipLaunchKernelGGL((leaky_step_kernel<T, Q>), dim3((unsigned)blocks), dim3(256), 0, stream, (T*)out, state, (const T*)query,   \
                       (const T*)key, (const T*)value, a->decay, a->num_decays == 1, (int)a->heads, (int)a->keys, (int)a->values, \
                       a->query_stride[0], a->query_stride[2], a->key_stride[0], a->key_stride[2], a->value_stride[0],            \
                       a->value_stride[2], tiles, whole, (float)a->scale)
    if (qp == 4) LAUNCH(4);
    else if (qp == 8) LAUNCH(8);
    else if (qp == 16) LAUNCH(16);
    else LAUNCH(32);
#undef LAUNCH
    return (int)hipGetLastError();
}

template <typename T>
int launch_slope(double* slopes, const void* grad, const float* grad_last, const slayer_attention* a, const LeakyPass& p, hipStream_t stream) {
    const int64_t units = a->samples * a->heads, size = a->keys * a->values;
#define LAUNCH(E)                                                                                                              \
    hipLaunchKernelGGL((leaky_slope_kernel<T, E>), dim3((unsigned)units), dim3(256), 0, stream, slopes, (const T*)grad, grad_last, \
                       a->grad_stride[0], a->grad_stride[1], a->grad_stride[2], p)
    if (size <= 4 * 256) LAUNCH(4);
    else if (size <= 16 * 256) LAUNCH(16);
    else LAUNCH(64);
#undef LAUNCH
    return (int)hipGetLastError();
}

// [samples][tokens][heads][width] as it lies in a new tensor
struct Contiguous {
    int64_t stride[3];
    Contiguous(const slayer_attention* a, int64_t width) : stride{a->tokens * a->heads * width, a->heads * width, width} {}
};

}  // namespace

extern "C" int64_t slayer_leaky_attention_workspace(const slayer_attention* a, int backward) {
    if (int e = check_leaky(a)) return e;
    const int64_t k = workspace_floats(a, a->keys), v = workspace_floats(a, a->values);
    if (!backward) return v;
    return (k > v ? k : v) + 2 * a->samples * a->heads;
}

extern "C" int slayer_leaky_attention_fwd(void* out, float* last, const void* query, const void* key, const void* value, const float* state,
                                          const slayer_attention* a, float* workspace, int64_t floats, void* stream) {
    if (int e = check_leaky(a)) return e;
    if (a->samples == 0) return 0;
    if (a->tokens > 0 && (!out || !query || !key || !value)) return SLAYER_ENULL;
    const int64_t need = slayer_leaky_attention_workspace(a, 0);
    if (need > 0 && !workspace) return SLAYER_ENULL;
    if (floats < need) return SLAYER_EINVAL;
    const Contiguous o(a, a->values);
    return run_pass(a, out, o.stride, {query, a->query_stride}, {key, a->key_stride}, {value, a->value_stride}, (int)a->keys, (int)a->values,
                    false, false, state, last, workspace, (hipStream_t)stream);
}

extern "C" int slayer_leaky_attention_bwd(void* grad_query, void* grad_key, void* grad_value, float* grad_decay, float* grad_state,
                                          const void* grad_out, const float* grad_last, const void* query, const void* key, const void* value,
                                          const float* state, const slayer_attention* a, float* workspace, int64_t floats, void* stream) {
    if (int e = check_leaky(a)) return e;
    hipStream_t s = (hipStream_t)stream;
    if (a->samples == 0) return grad_decay ? launch_zero_fill(grad_decay, a->num_decays, s) : 0;
    if (a->tokens > 0 && (!grad_out || !query || !key || !value)) return SLAYER_ENULL;
    const int64_t need = slayer_leaky_attention_workspace(a, 1);
    if (!workspace || (grad_state && !grad_value)) return SLAYER_ENULL;
    if (floats < need) return SLAYER_EINVAL;
    const int K = (int)a->keys, V = (int)a->values;
    const Contiguous k(a, K), v(a, V);
    double* slopes = (double*)workspace;
    float* rest = workspace + 2 * a->samples * a->heads;
    const Place q{query, a->query_stride}, kk{key, a->key_stride}, vv{value, a->value_stride}, g{grad_out, a->grad_stride};
    if (grad_query)
        if (int e = run_pass(a, grad_query, k.stride, g, vv, kk, V, K, true, false, state, nullptr, rest, s)) return e;
    if (grad_value || grad_state)
        if (int e = run_pass(a, grad_value, v.stride, kk, q, g, K, V, false, true, grad_last, grad_state, rest, s)) return e;
    if (grad_key)
        if (int e = run_pass(a, grad_key, k.stride, vv, g, q, V, K, true, true, grad_last, nullptr, rest, s)) return e;
    if (!grad_decay) return 0;
    LeakyPass p = {};
    p.query = query; p.key = key; p.value = value;
    p.decay = a->decay;
    p.lengths = a->lengths;
    p.first = state;
    p.query_n = a->query_stride[0]; p.query_t = a->query_stride[1]; p.query_h = a->query_stride[2];
    p.key_n = a->key_stride[0]; p.key_t = a->key_stride[1]; p.key_h = a->key_stride[2];
    p.value_n = a->value_stride[0]; p.value_t = a->value_stride[1]; p.value_h = a->value_stride[2];
    p.tokens = (int)a->tokens; p.heads = (int)a->heads; p.keys = K; p.values = V;
    p.one_decay = a->num_decays == 1;
    p.lengths64 = a->lengths_bytes == 8;
    p.out_scale = (float)a->scale;
    if (int e = a->dtype == SLAYER_FLOAT32 ? launch_slope<float>(slopes, grad_out, grad_last, a, p, s)
                                           : launch_slope<bf16>(slopes, grad_out, grad_last, a, p, s)) return e;
    hipLaunchKernelGGL(leaky_decay_kernel, dim3((unsigned)a->num_decays), dim3(256), 0, s, grad_decay, slopes, (int)a->samples, (int)a->heads,
                       (int)(a->num_decays == 1), 1);
    return (int)hipGetLastError();
}

extern "C" int slayer_leaky_attention_step(void* out, float* state, const void* query, const void* key, const void* value,
                                           const slayer_attention* a, void* stream) {
    if (int e = check_leaky(a)) return e;
    if (a->samples == 0) return 0;
    if (!out || !state || !query || !key || !value) return SLAYER_ENULL;
    return a->dtype == SLAYER_FLOAT32 ? launch_step<float>(out, state, query, key, value, a, (hipStream_t)stream)
                                      : launch_step<bf16>(out, state, query, key, value, a, (hipStream_t)stream);
}

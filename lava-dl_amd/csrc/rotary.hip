// Rotary positions: pairs of a head's features turned by an angle that grows with the token's position, of queries and keys in one
// launch.  With c = magnitude cos(position * frequency[i]) and s = magnitude sin(position * frequency[i]) a pair (x, y) becomes
// (c x - s y, c y + s x); the pairs are (i, i + turned / 2) or (2i, 2i + 1), features behind the first `turned` are copied.  The gradient is
// the same call with the angle's sign changed.
//   Angles: the whole turns are taken off in float64, with what the roundings of the products leave, so that a far position costs no
// digits; sine and cosine of the rest are made in float64 as well and rounded once.  All heads of a token share them: a workgroup makes those of
// its tokens once, in LDS.
//   Bound: memory, each tensor read and written once.  [64,1000,8,64] bfloat16, queries and keys from a projection: 53 us (4.9 TB/s); [16,1450,8,80]
// float32 with 48 features turned: 42 (5.7 TB/s).  One token of 256 samples, 16 heads of 128: 4.4 us, a launch and two steps that wait for memory.
#include "common.h"
#include "elements.h"

namespace slayer {
namespace {

constexpr int kAngles = 2048;                  // pairs of all tokens of a workgroup: 16 KB of LDS
constexpr int kSpan = 64;                      // most tokens of a workgroup
constexpr int kMostFeatures = 4096;            // of a head

struct RotaryArgs {
    void* out[2];
    const void* in[2];
    const double* frequency;
    const void* position;
    int64_t all;                               // samples * tokens
    int64_t tokens;
    int64_t in_stride[2][3];
    int heads[2];
    int features, pairs, position_bytes, each, span;          // span: tokens of a workgroup
    int units, rest;                           // accesses of a head: of W pairs each, then of W of the features that are copied
    int step_unit, step_head, step_token;      // 256 accesses on
    float magnitude, sign;
};

__device__ __forceinline__ int64_t position_of(const RotaryArgs& a, int64_t n, int64_t t) {
    if (!a.position) return t;
    const int64_t at = a.each ? n * a.tokens + t : n;
    const int64_t p = a.position_bytes == 4 ? ((const int*)a.position)[at] : ((const int64_t*)a.position)[at];
    return a.each ? p : p + t;
}

// Where an access lies: the head's features, the first pair (-1: features that are copied), the first feature of either half.
template <typename T> struct Place {
    const T* in;
    T* out;
    int pair, at[2];
    bool wide;                                 // W of them; otherwise all there are, one by one
};
template <typename T, bool HALVES>
__device__ __forceinline__ Place<T> place_of(const RotaryArgs& a, const int64_t (*in_at)[kSpan], const int64_t (*out_at)[kSpan], int token,
                                             int head, int unit) {
    constexpr int W = Elements<T>::kVec;
    const bool key = head >= a.heads[0];
    const int h = key ? head - a.heads[0] : head;
    Place<T> p;
    p.in = (const T*)(key ? a.in[1] : a.in[0]) + in_at[key][token] + h * (key ? a.in_stride[1][2] : a.in_stride[0][2]);
    p.out = (T*)(key ? a.out[1] : a.out[0]) + out_at[key][token] + (int64_t)h * a.features;
    if (unit < a.units) {
        p.wide = a.pairs >= W;
        p.pair = !p.wide ? 0 : unit * W < a.pairs - W ? unit * W : a.pairs - W;
        p.at[0] = HALVES ? p.pair : 2 * p.pair;
        p.at[1] = HALVES ? a.pairs + p.pair : 2 * p.pair + W;
    } else {
        const int at = 2 * a.pairs + (unit - a.units) * W;
        p.wide = a.features - 2 * a.pairs >= W;
        p.pair = -1;
        p.at[0] = at < a.features - W ? at : a.features - W;
        p.at[1] = 0;
    }
    return p;
}

// Cosine and sine of a part of a turn between -1/2 and 1/2: quarters are taken off, and Taylor's series of the angle that is left, at most pi / 4, stop
// where the next term is below 2^-28 of the sum.  float64 fused multiply-adds run at float32's rate here, so this costs what float32's functions do.
struct Turn { double cosine, sine; };
__device__ __forceinline__ Turn turn_of(double rest) {
    const double quarters = rint(4 * rest), x = (rest - 0.25 * quarters) * 6.283185307179586, z = x * x;
    const double s = fma(fma(fma(fma(1.0 / 362880, z, -1.0 / 5040), z, 1.0 / 120), z, -1.0 / 6) * z, x, x);
    const double c = fma(fma(fma(fma(fma(-1.0 / 3628800, z, 1.0 / 40320), z, -1.0 / 720), z, 1.0 / 24), z, -0.5), z, 1.0);
    const int q = (int)quarters;
    const double first = q & 1 ? s : c, second = q & 1 ? c : s;
    return {(q + 1) & 2 ? -first : first, q & 2 ? -second : second};
}

// Angles of a workgroup's tokens, then its accesses: for each token and head the pairs, W at a time, and what is copied.  The last access of
// either, where there are W, ends with the last feature and so may do some of the one before it again, with the same values: no access is
// cut.  The angles are being made while the first features are on their way.
template <typename T, bool HALVES>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    constexpr int W = Elements<T>::kVec;
    typedef typename Wide<T>::Any Any;
    typedef typename Elements<T>::Vec Vec;
    __shared__ __align__(16) float cosines[kAngles + W], sines[kAngles + W];
    __shared__ double positions[kSpan];
    __shared__ int64_t in_at[2][kSpan], out_at[2][kSpan];
    const int64_t first = (int64_t)blockIdx.x * a.span;
    const int count = a.all - first < a.span ? (int)(a.all - first) : a.span;
    if (threadIdx.x < count) {
        const int64_t at = first + threadIdx.x, n = at / a.tokens, t = at - n * a.tokens;
        positions[threadIdx.x] = (double)position_of(a, n, t);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            in_at[w][threadIdx.x] = n * a.in_stride[w][0] + t * a.in_stride[w][1];
            out_at[w][threadIdx.x] = at * a.heads[w] * a.features;
        }
    }
    __syncthreads();
    const int heads = a.heads[0] + a.heads[1], per = a.units + a.rest;
    int unit = threadIdx.x % per, head = threadIdx.x / per % heads, token = threadIdx.x / (per * heads);
    Place<T> place = {};
    Vec x = {}, y = {};
    if (token < count) {
        place = place_of<T, HALVES>(a, in_at, out_at, token, head, unit);
        if (place.wide) {
            x = *reinterpret_cast<const Any*>(place.in + place.at[0]);
            if (place.pair >= 0) y = *reinterpret_cast<const Any*>(place.in + place.at[1]);
        }
    }
    for (int i = threadIdx.x; i < count * a.pairs; i += 256) {
        const int t = i / a.pairs;
        constexpr double kHigh = 0x1.45f306dc9c883p-3, kLow = -0x1.6b01ec5417056p-57;           // 1 / (2 pi)
        const double radians = a.frequency[i - t * a.pairs], f = radians * kHigh, turns = positions[t] * f;
        const double rest = (turns - rint(turns)) + (fma(positions[t], f, -turns) + positions[t] * fma(radians, kLow, fma(radians, kHigh, -f)));
        const Turn turn = turn_of(rest);
        cosines[i] = (float)(a.magnitude * turn.cosine);
        sines[i] = (float)(a.sign * a.magnitude * turn.sine);
    }
    __syncthreads();
    while (token < count) {
        if (place.wide) {
            if (place.pair >= 0) {
                const float *c = cosines + token * a.pairs + place.pair, *s = sines + token * a.pairs + place.pair;
                float u[W], v[W], p[W], q[W];
                to_floats(u, x);
                to_floats(v, y);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const float left = HALVES ? u[e] : e < W / 2 ? u[2 * e % W] : v[2 * e % W];
                    const float right = HALVES ? v[e] : e < W / 2 ? u[2 * e % W + 1] : v[2 * e % W + 1];
                    const float l = fmaf(c[e], left, -(s[e] * right)), r = fmaf(c[e], right, s[e] * left);
                    if (HALVES) {
                        p[e] = l;
                        q[e] = r;
                    } else {
                        (e < W / 2 ? p : q)[2 * e % W] = l;
                        (e < W / 2 ? p : q)[2 * e % W + 1] = r;
                    }
                }
                x = from_floats(p);
                y = from_floats(q);
                *reinterpret_cast<Any*>(place.out + place.at[1]) = y;
            }
            *reinterpret_cast<Any*>(place.out + place.at[0]) = x;
        } else if (place.pair >= 0) {                              // fewer pairs than W
            const float *c = cosines + token * a.pairs, *s = sines + token * a.pairs;
            for (int e = 0; e < a.pairs; ++e) {
                const int i = HALVES ? e : 2 * e, j = HALVES ? a.pairs + e : 2 * e + 1;
                const float left = (float)place.in[i], right = (float)place.in[j];
                place.out[i] = (T)fmaf(c[e], left, -(s[e] * right));
                place.out[j] = (T)fmaf(c[e], right, s[e] * left);
            }
        } else {
            for (int i = 2 * a.pairs; i < a.features; ++i) place.out[i] = place.in[i];
        }
        unit += a.step_unit;
        head += a.step_head;
        token += a.step_token;
        if (unit >= per) {
            unit -= per;
            ++head;
        }
        if (head >= heads) {
            head -= heads;
            ++token;
        }
        if (token >= count) break;
        place = place_of<T, HALVES>(a, in_at, out_at, token, head, unit);
        if (place.wide) {
            x = *reinterpret_cast<const Any*>(place.in + place.at[0]);
            if (place.pair >= 0) y = *reinterpret_cast<const Any*>(place.in + place.at[1]);
        }
    }
}

}  // namespace
}  // namespace slayer

using namespace slayer;

extern "C" int slayer_rotary(void* out_query, void* out_key, const void* query, const void* key, const slayer_rotary_call* r, int inverse,
                             void* stream) {
    if (!r) return SLAYER_ENULL;
    if (r->samples < 0 || r->tokens < 0 || r->query_heads < 0 || r->key_heads < 0 || r->features < 1) return SLAYER_EINVAL;
    if (r->turned < 0 || r->turned % 2 != 0 || r->turned > r->features) return SLAYER_EINVAL;
    if (r->dtype != SLAYER_FLOAT32 && r->dtype != SLAYER_BFLOAT16) return SLAYER_EINVAL;
    if (r->layout != SLAYER_ROTARY_HALVES && r->layout != SLAYER_ROTARY_PAIRS) return SLAYER_EINVAL;
    if (r->position && r->position_bytes != 4 && r->position_bytes != 8) return SLAYER_EINVAL;
    if (r->features > kMostFeatures || r->query_heads > 65536 || r->key_heads > 65536) return SLAYER_ERANGE;
    if (r->tokens > kMaxT || r->samples > ((int64_t)1 << 32) || (r->tokens > 0 && r->samples > ((int64_t)1 << 32) / r->tokens)) return SLAYER_ERANGE;
    const int64_t all = r->samples * r->tokens, heads = r->query_heads + r->key_heads;
    if (all == 0 || heads == 0) return 0;
    if ((r->turned > 0 && !r->frequency) || (r->query_heads > 0 && (!out_query || !query)) || (r->key_heads > 0 && (!out_key || !key)))
        return SLAYER_ENULL;
    RotaryArgs a = {};
    a.out[0] = out_query; a.out[1] = out_key;
    a.in[0] = query; a.in[1] = key;
    a.frequency = r->frequency; a.position = r->position; a.position_bytes = r->position_bytes; a.each = r->position_each;
    a.all = all; a.tokens = r->tokens;
    for (int i = 0; i < 3; ++i) {
        a.in_stride[0][i] = r->query_stride[i];
        a.in_stride[1][i] = r->key_stride[i];
    }
    a.heads[0] = (int)r->query_heads; a.heads[1] = (int)r->key_heads;
    a.features = (int)r->features; a.pairs = (int)r->turned / 2;
    const int w = r->dtype == SLAYER_FLOAT32 ? 4 : 8;
    a.units = (a.pairs + w - 1) / w;
    a.rest = (a.features - 2 * a.pairs + w - 1) / w;
    const int per = a.units + a.rest;
    a.step_unit = 256 % per;
    a.step_head = 256 / per % (int)heads;
    a.step_token = 256 / per / (int)heads;
    a.magnitude = r->magnitude; a.sign = inverse ? -1.f : 1.f;
    // Tokens of a workgroup: an access for each of its threads, as long as the angles fit; fewer where that leaves compute units idle.  Of
    // [64,1000,8,64] bfloat16, 64 accesses a token: 52 us with four tokens, 55 with eight, 60 with sixteen.
    int span = (256 + per * (int)heads - 1) / (per * (int)heads);
    if (span > kSpan) span = kSpan;
    if (a.pairs > 0 && span > kAngles / a.pairs) span = kAngles / a.pairs;
    while (span > 1 && (all + span - 1) / span < 512) span /= 2;
    a.span = span;
    const int64_t blocks = (all + span - 1) / span;
    if (blocks > (1 << 24) - 1) return SLAYER_ERANGE;
    const bool halves = r->layout == SLAYER_ROTARY_HALVES;
#define LAUNCH(T, HALVES) hipLaunchKernelGGL((rotary_kernel<T, HALVES>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a)
    if (r->dtype == SLAYER_FLOAT32) {
        if (halves) LAUNCH(float, true);
        else LAUNCH(float, false);
    } else {
        if (halves) LAUNCH(bf16, true);
        else LAUNCH(bf16, false);
    }
#undef LAUNCH
    return (int)hipGetLastError();
}

// Rotary positions: pairs of a head's features turned by an angle that grows with the token's position, of queries and keys in one
// launch.  With c = magnitude cos(position * frequency[i]) and s = magnitude sin(position * frequency[i]) a pair (x, y) becomes
// (c x - s y, c y + s x); the pairs are (i, i + turned / 2) or (2i, 2i + 1), features behind the first `turned` are copied.  The gradient is
// the same call with the angle's sign changed.
//   Angles: the whole turns are taken off in float64, with what the product's rounding leaves, so that a position of 2^31 costs no
// digits; sine and cosine of the rest are float32.  All heads of a token share them: a workgroup makes those of its tokens once, in LDS.
//   Bound: memory, each tensor read and written once.
#include "common.h"
#include "elements.h"

namespace slayer {
namespace {

constexpr int kAngles = 2048;                  // pairs of all tokens of a workgroup: 16 KB of LDS
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
    int units, rest;                           // accesses of a head: four pairs each, then four of the features that are copied
    float magnitude, sign;
};

__device__ __forceinline__ int64_t position_of(const RotaryArgs& a, int64_t n, int64_t t) {
    if (!a.position) return t;
    const int64_t at = a.each ? n * a.tokens + t : n;
    const int64_t p = a.position_bytes == 4 ? ((const int*)a.position)[at] : ((const int64_t*)a.position)[at];
    return a.each ? p : p + t;
}

template <typename T, bool HALVES>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    __shared__ float cosines[kAngles], sines[kAngles];
    const int64_t first = (int64_t)blockIdx.x * a.span;
    const int count = a.all - first < a.span ? (int)(a.all - first) : a.span;
    for (int i = threadIdx.x; i < count * a.pairs; i += 256) {
        const int64_t token = first + i / a.pairs, n = token / a.tokens;
        const double p = (double)position_of(a, n, token - n * a.tokens), f = a.frequency[i % a.pairs] * 0.15915494309189533577;
        const double turns = p * f, rest = (turns - rint(turns)) + fma(p, f, -turns);
        float s, c;
        sincospif(2.f * (float)rest, &s, &c);
        cosines[i] = a.magnitude * c;
        sines[i] = a.sign * a.magnitude * s;
    }
    __syncthreads();
    const int heads = a.heads[0] + a.heads[1], per = a.units + a.rest, items = count * heads * per;
    for (int item = threadIdx.x; item < items; item += 256) {
        const int unit = item % per, row = item / per, token = row / heads;
        int head = row % heads;
        const int which = head >= a.heads[0];
        head -= which ? a.heads[0] : 0;
        const int64_t at = first + token, n = at / a.tokens;
        const T* in = (const T*)a.in[which] + n * a.in_stride[which][0] + (at - n * a.tokens) * a.in_stride[which][1] +
                      head * a.in_stride[which][2];
        T* out = (T*)a.out[which] + (at * a.heads[which] + head) * a.features;
        if (unit >= a.units) {
            const int i = 2 * a.pairs + (unit - a.units) * 4, left = a.features - i;
            store_four(out + i, __builtin_convertvector(load_four(in + i, left), f4), left);
            continue;
        }
        const int i = unit * 4, left = a.pairs - i;
        const float *c = cosines + token * a.pairs + i, *s = sines + token * a.pairs + i;
        f4 x, y, u = {}, w = {};
        if (HALVES) {
            x = __builtin_convertvector(load_four(in + i, left), f4);
            y = __builtin_convertvector(load_four(in + a.pairs + i, left), f4);
        } else {
            const f4 p = __builtin_convertvector(load_four(in + 2 * i, 2 * left), f4);
            const f4 q = __builtin_convertvector(load_four(in + 2 * i + 4, 2 * left - 4), f4);
            x = f4{p[0], p[2], q[0], q[2]};
            y = f4{p[1], p[3], q[1], q[3]};
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) {
                u[e] = fmaf(c[e], x[e], -(s[e] * y[e]));
                w[e] = fmaf(c[e], y[e], s[e] * x[e]);
            }
        if (HALVES) {
            store_four(out + i, u, left);
            store_four(out + a.pairs + i, w, left);
        } else {
            store_four(out + 2 * i, f4{u[0], w[0], u[1], w[1]}, 2 * left);
            store_four(out + 2 * i + 4, f4{u[2], w[2], u[3], w[3]}, 2 * left - 4);
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
    a.units = (a.pairs + 3) / 4;
    a.rest = (a.features - 2 * a.pairs + 3) / 4;
    a.magnitude = r->magnitude; a.sign = inverse ? -1.f : 1.f;
    // tokens of a workgroup: up to sixteen, as the angles fit, fewer where that leaves compute units idle
    int span = a.pairs > 0 ? kAngles / a.pairs : 16;
    if (span > 16) span = 16;
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

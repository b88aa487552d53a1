// Gated leak: the leaky integrator whose leak a token's gate opens, with the channels last.  For every sample and channel
//     open = sigmoid(gate[t]),  leak = decay / 4096 * open,  h[t] = (1 - leak) h[t-1] + drive(leak) x[t],
// drive 1, leak, or sqrt(leak (2 - leak)).  Backwards, with D the derivative with respect to the state behind a token and G with
// respect to the state in front of it,
//     D[t] = dy[t] + G[t+1],  G[t] = (1 - leak) D[t],  dx = drive D,  dleak = D (drive' x - h[t-1]),
//     dgate = dleak leak (1 - open),  ddecay = sum of dleak open / 4096.
// Both are linear recurrences s <- A s + H in one number a channel, and spans of tokens join as pairs (A, H): a thread takes a few
// tokens of four channels in its registers, sixteen lanes the channels next to each other, the other lanes and waves the tokens that
// follow; pairs are joined across lanes, then across waves in LDS, and with the state in front of the tile each thread walks its tokens
// again.  The backward pass makes the states of a tile again from the one in front of it, which the forward pass has kept, so that
// it reads neither the results nor anything rounded.
//   Bound: memory, three tensors forward and five backward.
#include "common.h"
#include "elements.h"

namespace slayer {
namespace {

enum { DRIVE_NONE, DRIVE_GAIN, DRIVE_VARIANCE };

constexpr int kStrip = 64;                     // channels of a workgroup: sixteen lanes, four each
constexpr int kTile = 128;                     // tokens that it holds at a time

struct LeakArgs {
    void *out, *grad_in, *grad_gate;
    const void *in, *gate, *grad, *lengths;
    const float *decay, *state, *grad_last;
    float *last, *starts, *grad_state, *parts;
    int64_t samples, tokens, tiles;
    int64_t in_stride[2], gate_stride[2], grad_stride[2];
    int channels, strips, lengths_bytes, decays;
};

// A gate of +infinity is open, as one of 100 is (the precise form of logistic would make it NaN).
template <typename T> __device__ __forceinline__ float open_gate(float z) {
    return logistic<T>(sizeof(T) == 4 && z > 100.f ? 100.f : z);
}

// drive and its derivative from the leak and what it keeps, 1 - leak.  sqrt(leak (2 - leak)) counts as 0 with derivative 0 where its square
// is below the smallest numbers that the hardware's reciprocal root takes (leaks below 5e-37).
struct Drive { float value, slope; };
template <int DRIVE> __device__ __forceinline__ Drive drive_of(float leak, float keep) {
    if (DRIVE == DRIVE_NONE) return {1.f, 0.f};
    if (DRIVE == DRIVE_GAIN) return {leak, 1.f};
    const float square = leak * (2.f - leak);
    float r = __builtin_amdgcn_rsqf(square);
    r = square < 1e-36f ? 0.f : r;
    return {square * r, keep * r};
}

__device__ __forceinline__ int64_t length_of(const LeakArgs& a, int64_t n) {
    if (!a.lengths) return a.tokens;
    const int64_t length = a.lengths_bytes == 4 ? ((const int*)a.lengths)[n] : ((const int64_t*)a.lengths)[n];
    return length < 0 ? 0 : length < a.tokens ? length : a.tokens;
}

__device__ __forceinline__ f4 decays_of(const LeakArgs& a, int c, int left) {
    f4 d = {};
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (v < left) d[v] = a.decay[a.decays == 1 ? 0 : c + v] * (1.f / 4096.f);
    return d;
}

// ---- forward --------------------------------------------------------------------------------------------------------------------
// A workgroup takes one strip of one sample and walks its tiles.
template <typename T, int DRIVE, int S, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void leak_fwd_kernel(LeakArgs a) {
    static_assert(4 * WAVES * S == kTile, "a tile is four lanes a wave");
    __shared__ f4 total[2][WAVES][2][16];                           // A, H of each wave and channel
    __shared__ f4 carry[2][16];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, lc = lane % 16, lt = lane / 16;
    const int strip = blockIdx.x % a.strips;
    const int64_t n = blockIdx.x / a.strips;
    const int c = strip * kStrip + lc * 4, left = a.channels - c;
    const int64_t length = length_of(a, n);
    const f4 d = decays_of(a, c, left);
    const T* in = (const T*)a.in + n * a.in_stride[0] + c;
    const T* gate = (const T*)a.gate + n * a.gate_stride[0] + c;
    T* out = (T*)a.out + n * a.tokens * a.channels + c;
    if (threadIdx.x < 16) {
        f4 h = {};
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (a.state && v < left) h[v] = a.state[n * a.channels + c + v];
        carry[0][lc] = h;
    }
    for (int64_t tile = 0; tile < a.tiles; ++tile) {
        const int turn = tile % 2;
        const int64_t t0 = tile * kTile + (wave * 4 + lt) * S;
        float keep[S][4], add[S][4];
        typename Four<T>::Vec x[S], z[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const bool on = t0 + s < length;
            x[s] = z[s] = {};
            if (on && left > 0) {
                x[s] = load_four(in + (t0 + s) * a.in_stride[1], left);
                z[s] = load_four(gate + (t0 + s) * a.gate_stride[1], left);
            }
        }
        f4 A = {1.f, 1.f, 1.f, 1.f}, H = {};
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const bool on = t0 + s < length;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float leak = d[v] * open_gate<T>((float)z[s][v]);
                keep[s][v] = on ? 1.f - leak : 1.f;
                add[s][v] = on ? drive_of<DRIVE>(leak, keep[s][v]).value * (float)x[s][v] : 0.f;
                A[v] *= keep[s][v];
                H[v] = fmaf(keep[s][v], H[v], add[s][v]);
            }
        }
        // the pairs of the lanes in front of this one, and of the wave
        f4 before_a = {1.f, 1.f, 1.f, 1.f}, before_h = {};
#pragma unroll
        for (int v = 0; v < 4; ++v) {
#pragma unroll
            for (int by = 16; by < 64; by *= 2) {
                const float oa = __shfl_up(A[v], by), oh = __shfl_up(H[v], by);
                if (lane >= by) {
                    H[v] = fmaf(A[v], oh, H[v]);
                    A[v] *= oa;
                }
            }
            const float oa = __shfl_up(A[v], 16), oh = __shfl_up(H[v], 16);
            if (lane >= 16) {
                before_a[v] = oa;
                before_h[v] = oh;
            }
        }
        if (lt == 3) {
            total[turn][wave][0][lc] = A;
            total[turn][wave][1][lc] = H;
        }
        __syncthreads();
        // the state in front of the wave, and behind the tile
        f4 h = carry[turn][lc];
        if (a.starts && wave == 0 && lt == 0 && left > 0) store_four(a.starts + (n * a.tiles + tile) * a.channels + c, h, left);
        f4 mine = h;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const f4 wa = total[turn][w][0][lc], wh = total[turn][w][1][lc];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                if (w == wave) mine[v] = h[v];
                h[v] = fmaf(wa[v], h[v], wh[v]);
            }
        }
        if (wave == 0 && lt == 0) {
            carry[turn ^ 1][lc] = h;
            if (a.last && tile == a.tiles - 1 && left > 0) store_four(a.last + n * a.channels + c, h, left);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) h[v] = fmaf(before_a[v], mine[v], before_h[v]);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            f4 y;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                h[v] = fmaf(keep[s][v], h[v], add[s][v]);
                y[v] = t0 + s < length ? h[v] : 0.f;
            }
            if (t0 + s < a.tokens && left > 0) store_four(out + (t0 + s) * a.channels, y, left);
        }
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------------
// The same strip, its tiles from the last to the first.  Inside a tile the states go forwards, from the kept one, and G backwards.
template <typename T, int DRIVE, int S, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void leak_bwd_kernel(LeakArgs a) {
    static_assert(4 * WAVES * S == kTile, "a tile is four lanes a wave");
    __shared__ f4 total[2][WAVES][3][16];                           // A, H, G of each wave and channel
    __shared__ f4 carry[2][16];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, lc = lane % 16, lt = lane / 16;
    const int strip = blockIdx.x % a.strips;
    const int64_t n = blockIdx.x / a.strips;
    const int c = strip * kStrip + lc * 4, left = a.channels - c;
    const int64_t length = length_of(a, n);
    const f4 d = decays_of(a, c, left);
    const T* in = (const T*)a.in + n * a.in_stride[0] + c;
    const T* gate = (const T*)a.gate + n * a.gate_stride[0] + c;
    const T* grad = (const T*)a.grad + n * a.grad_stride[0] + c;
    T* grad_in = (T*)a.grad_in + n * a.tokens * a.channels + c;
    T* grad_gate = (T*)a.grad_gate + n * a.tokens * a.channels + c;
    f4 slopes = {};                                                 // sum of dleak * open
    if (threadIdx.x < 16) {
        f4 g = {};
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (a.grad_last && v < left) g[v] = a.grad_last[n * a.channels + c + v];
        carry[0][lc] = g;
    }
    for (int64_t tile = a.tiles - 1; tile >= 0; --tile) {
        const int turn = (a.tiles - 1 - tile) % 2;
        const int64_t t0 = tile * kTile + (wave * 4 + lt) * S;
        typename Four<T>::Vec x[S], z[S], dy[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            x[s] = z[s] = dy[s] = {};
            if (t0 + s < length && left > 0) {
                x[s] = load_four(in + (t0 + s) * a.in_stride[1], left);
                z[s] = load_four(gate + (t0 + s) * a.gate_stride[1], left);
                dy[s] = load_four(grad + (t0 + s) * a.grad_stride[1], left);
            }
        }
        f4 start = {};
        if (left > 0) start = load_four(a.starts + (n * a.tiles + tile) * a.channels + c, left);
        float open[S][4], before[S][4];
        f4 A = {1.f, 1.f, 1.f, 1.f}, H = {}, G = {};
#pragma unroll
        for (int v = 0; v < 4; ++v) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const bool on = t0 + s < length;
                open[s][v] = on ? open_gate<T>((float)z[s][v]) : 0.f;      // what is not there leaks nothing, and x and dy are 0
                const float leak = d[v] * open[s][v], keep = 1.f - leak;
                A[v] *= keep;
                H[v] = fmaf(keep, H[v], drive_of<DRIVE>(leak, keep).value * (float)x[s][v]);
            }
#pragma unroll
            for (int s = S - 1; s >= 0; --s) G[v] = (1.f - d[v] * open[s][v]) * ((float)dy[s][v] + G[v]);
        }
        // the pairs of the lanes in front of this one and behind it, and of the wave
        f4 before_a = {1.f, 1.f, 1.f, 1.f}, before_h = {}, behind_a = {1.f, 1.f, 1.f, 1.f}, behind_g = {}, B = A;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
#pragma unroll
            for (int by = 16; by < 64; by *= 2) {
                const float oa = __shfl_up(A[v], by), oh = __shfl_up(H[v], by);
                const float ob = __shfl_down(B[v], by), og = __shfl_down(G[v], by);
                if (lane >= by) {
                    H[v] = fmaf(A[v], oh, H[v]);
                    A[v] *= oa;
                }
                if (lane < 64 - by) {
                    G[v] = fmaf(B[v], og, G[v]);
                    B[v] *= ob;
                }
            }
            const float oa = __shfl_up(A[v], 16), oh = __shfl_up(H[v], 16);
            const float ob = __shfl_down(B[v], 16), og = __shfl_down(G[v], 16);
            if (lane >= 16) {
                before_a[v] = oa;
                before_h[v] = oh;
            }
            if (lane < 48) {
                behind_a[v] = ob;
                behind_g[v] = og;
            }
        }
        if (lt == 3) {
            total[turn][wave][0][lc] = A;
            total[turn][wave][1][lc] = H;
        }
        if (lt == 0) total[turn][wave][2][lc] = G;
        __syncthreads();
        f4 h = start, g = carry[turn][lc], mine = g;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const f4 wa = total[turn][w][0][lc], wh = total[turn][w][1][lc];
#pragma unroll
            for (int v = 0; v < 4; ++v) h[v] = w < wave ? fmaf(wa[v], h[v], wh[v]) : h[v];
        }
#pragma unroll
        for (int w = WAVES - 1; w >= 0; --w) {
            const f4 wa = total[turn][w][0][lc], wg = total[turn][w][2][lc];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                if (w == wave) mine[v] = g[v];
                g[v] = fmaf(wa[v], g[v], wg[v]);
            }
        }
        if (wave == 0 && lt == 0) {
            carry[turn ^ 1][lc] = g;
            if (a.grad_state && tile == 0 && left > 0) store_four(a.grad_state + n * a.channels + c, g, left);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            h[v] = fmaf(before_a[v], h[v], before_h[v]);
            g[v] = fmaf(behind_a[v], mine[v], behind_g[v]);
        }
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                before[s][v] = h[v];
                const float leak = d[v] * open[s][v], keep = 1.f - leak;
                h[v] = fmaf(keep, h[v], drive_of<DRIVE>(leak, keep).value * (float)x[s][v]);
            }
#pragma unroll
        for (int s = S - 1; s >= 0; --s) {
            const bool on = t0 + s < length;
            f4 dx, dz;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float leak = d[v] * open[s][v], keep = 1.f - leak;
                const Drive drive = drive_of<DRIVE>(leak, keep);
                const float D = (float)dy[s][v] + g[v];
                float dleak = D * fmaf(drive.slope, (float)x[s][v], -before[s][v]);
                dleak = on ? dleak : 0.f;
                dx[v] = on ? drive.value * D : 0.f;
                dz[v] = dleak * leak * (1.f - open[s][v]);
                slopes[v] = fmaf(dleak, open[s][v], slopes[v]);
                g[v] = keep * D;
            }
            if (t0 + s < a.tokens && left > 0) {
                store_four(grad_in + (t0 + s) * a.channels, dx, left);
                store_four(grad_gate + (t0 + s) * a.channels, dz, left);
            }
        }
    }
    if (!a.parts) return;
    __shared__ f4 sums[WAVES * 4][16];
    sums[wave * 4 + lt][lc] = slopes;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const int i = threadIdx.x;
    float sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES * 4; ++w) sum += sums[w][i / 4][i % 4];
    if (a.decays > 1) {
        if (strip * kStrip + i < a.channels) a.parts[n * a.channels + strip * kStrip + i] = sum;
    } else {
        sum = sum_lanes(sum, 64);                                   // (channels that are not there have 0)
        if (i == 0) a.parts[blockIdx.x] = sum;
    }
}

// ---- one token a sample ---------------------------------------------------------------------------------------------------------
template <typename T, int DRIVE>
__global__ __launch_bounds__(256) void leak_step_kernel(LeakArgs a, int quads) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t n = at / quads;
    if (n >= a.samples) return;
    const int c = (int)(at % quads) * 4, left = a.channels - c;
    const f4 d = decays_of(a, c, left);
    const typename Four<T>::Vec x = load_four((const T*)a.in + n * a.in_stride[0] + c, left);
    const typename Four<T>::Vec z = load_four((const T*)a.gate + n * a.gate_stride[0] + c, left);
    f4 h = load_four(a.last + n * a.channels + c, left);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const float leak = d[v] * open_gate<T>((float)z[v]), keep = 1.f - leak;
        h[v] = fmaf(keep, h[v], drive_of<DRIVE>(leak, keep).value * (float)x[v]);
    }
    store_four(a.last + n * a.channels + c, h, left);
    store_four((T*)a.out + n * a.channels + c, h, left);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
int64_t tiles_of(int64_t tokens) { return tokens > 0 ? (tokens + kTile - 1) / kTile : 1; }
int64_t strips_of(int64_t channels) { return (channels + kStrip - 1) / kStrip; }

int check_leak(const slayer_gated_leak* a) {
    if (!a) return SLAYER_ENULL;
    if (a->samples < 0 || a->tokens < 0 || a->channels < 1) return SLAYER_EINVAL;
    if (a->dtype != SLAYER_FLOAT32 && a->dtype != SLAYER_BFLOAT16) return SLAYER_EINVAL;
    if (a->drive < DRIVE_NONE || a->drive > DRIVE_VARIANCE) return SLAYER_EINVAL;
    if (a->num_decays != 1 && a->num_decays != a->channels) return SLAYER_EINVAL;
    if (a->lengths && a->lengths_bytes != 4 && a->lengths_bytes != 8) return SLAYER_EINVAL;
    if (!a->decay) return SLAYER_ENULL;
    if (a->tokens > kMaxT || a->channels > (1 << 24) || a->samples > ((int64_t)1 << 32)) return SLAYER_ERANGE;
    if (a->samples * a->channels > kMaxNumel / (a->tokens > 0 ? a->tokens : 1)) return SLAYER_ERANGE;
    if (a->samples * strips_of(a->channels) > (1 << 23)) return SLAYER_ERANGE;          // a workgroup each
    return 0;
}

LeakArgs args_of(const slayer_gated_leak* s) {
    LeakArgs a = {};
    a.lengths = s->lengths; a.lengths_bytes = s->lengths_bytes;
    a.decay = s->decay; a.decays = (int)s->num_decays;
    a.samples = s->samples; a.tokens = s->tokens; a.tiles = tiles_of(s->tokens);
    a.channels = (int)s->channels; a.strips = (int)strips_of(s->channels);
    for (int i = 0; i < 2; ++i) {
        a.in_stride[i] = s->input_stride[i];
        a.gate_stride[i] = s->gate_stride[i];
        a.grad_stride[i] = s->grad_stride[i];
    }
    return a;
}

#define BY_DRIVE(T, LAUNCH)                                 \
    switch (s->drive) {                                     \
        case DRIVE_NONE: LAUNCH(T, DRIVE_NONE); break;      \
        case DRIVE_GAIN: LAUNCH(T, DRIVE_GAIN); break;      \
        default: LAUNCH(T, DRIVE_VARIANCE); break;          \
    }
#define BY_TYPE(LAUNCH)                                     \
    if (s->dtype == SLAYER_FLOAT32) BY_DRIVE(float, LAUNCH) \
    else BY_DRIVE(bf16, LAUNCH)

}  // namespace
}  // namespace slayer

using namespace slayer;

extern "C" int64_t slayer_gated_leak_starts(const slayer_gated_leak* s) {
    if (int e = check_leak(s)) return e;
    return s->samples * tiles_of(s->tokens) * s->channels;
}

extern "C" int64_t slayer_gated_leak_workspace(const slayer_gated_leak* s, int backward) {
    if (int e = check_leak(s)) return e;
    return backward ? s->samples * (s->num_decays == 1 ? strips_of(s->channels) : s->channels) : 0;
}

extern "C" int slayer_gated_leak_fwd(void* out, float* last, float* starts, const void* input, const void* gate, const float* state,
                                     const slayer_gated_leak* s, float* workspace, int64_t floats, void* stream) {
    if (int e = check_leak(s)) return e;
    if (s->samples == 0) return 0;
    if (s->tokens > 0 && (!out || !input || !gate)) return SLAYER_ENULL;
    LeakArgs a = args_of(s);
    a.out = out; a.last = last; a.starts = starts; a.in = input; a.gate = gate; a.state = state;
#define LAUNCH(T, DRIVE) \
    hipLaunchKernelGGL((leak_fwd_kernel<T, DRIVE, 8, 4>), dim3((unsigned)(a.samples * a.strips)), dim3(256), 0, (hipStream_t)stream, a)
    BY_TYPE(LAUNCH)
#undef LAUNCH
    return (int)hipGetLastError();
}

extern "C" int slayer_gated_leak_bwd(void* grad_input, void* grad_gate, float* grad_decay, float* grad_state, const void* grad_out,
                                     const float* grad_last, const void* input, const void* gate, const float* starts,
                                     const slayer_gated_leak* s, float* workspace, int64_t floats, void* stream) {
    if (int e = check_leak(s)) return e;
    if (s->samples == 0) return grad_decay ? launch_zero_fill(grad_decay, s->num_decays, (hipStream_t)stream) : 0;
    if (!starts || (s->tokens > 0 && (!grad_input || !grad_gate || !grad_out || !input || !gate))) return SLAYER_ENULL;
    const int64_t need = grad_decay ? slayer_gated_leak_workspace(s, 1) : 0;
    if (need > 0 && !workspace) return SLAYER_ENULL;
    if (floats < need) return SLAYER_EINVAL;
    LeakArgs a = args_of(s);
    a.grad_in = grad_input; a.grad_gate = grad_gate; a.grad_state = grad_state; a.grad = grad_out; a.grad_last = grad_last;
    a.in = input; a.gate = gate; a.starts = (float*)starts;
    a.parts = grad_decay ? workspace : nullptr;
#define LAUNCH(T, DRIVE) \
    hipLaunchKernelGGL((leak_bwd_kernel<T, DRIVE, 4, 8>), dim3((unsigned)(a.samples * a.strips)), dim3(512), 0, (hipStream_t)stream, a)
    BY_TYPE(LAUNCH)
#undef LAUNCH
    if (int e = (int)hipGetLastError()) return e;
    if (!grad_decay) return 0;
    ColumnSums sums = {};
    sums.out[0] = grad_decay; sums.parts[0] = workspace; sums.factor = 1.f / 4096.f;
    sums.columns = sums.pitch = s->num_decays;
    sums.rows = need / s->num_decays;
    return launch_column_sums(sums, 1, (hipStream_t)stream);
}

extern "C" int slayer_gated_leak_step(void* out, float* state, const void* input, const void* gate, const slayer_gated_leak* s,
                                      void* stream) {
    if (int e = check_leak(s)) return e;
    if (s->samples == 0) return 0;
    if (!out || !state || !input || !gate) return SLAYER_ENULL;
    LeakArgs a = args_of(s);
    a.out = out; a.last = state; a.in = input; a.gate = gate;
    const int quads = (a.channels + 3) / 4;
    const int64_t blocks = (a.samples * quads + 255) / 256;
    if (blocks > (1 << 23)) return SLAYER_ERANGE;
#define LAUNCH(T, DRIVE) \
    hipLaunchKernelGGL((leak_step_kernel<T, DRIVE>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a, quads)
    BY_TYPE(LAUNCH)
#undef LAUNCH
    return (int)hipGetLastError();
}

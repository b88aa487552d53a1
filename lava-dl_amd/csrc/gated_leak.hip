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

// ---- tiles of a chain -----------------------------------------------------------------------------------------------------------
// A chain is one strip of one sample, from tile to tile in the order of the pass.  Either a workgroup walks all tiles of a chain and
// carries the state in LDS, or there is a workgroup for each tile, and states go through memory:
//   Workgroups take their tiles by a ticket, the first tiles of all chains before the second ones, so a workgroup only ever waits for
// workgroups with lower tickets, which are running or done and wait for lower ones themselves; the lowest waits for nobody, so every wait
// ends.  Tiles form windows.  A tile leaves its pair, then reads those of the tiles before it in its window, and the state in front of
// the window; the last tile of a window leaves the state behind it.  Which values are joined, and in which order, depends on the sizes alone
// and not on who comes first, so that a call computed again has the same bits.
//   What is left is a word of 64 bits that says itself that it is there (the workspace is zeroed before), read and written with relaxed
// atomics of the whole device: no other memory hangs on it, so no fences are needed.
typedef unsigned long long Word;
constexpr int kWindow = 32;                    // largest window

struct Chains {
    unsigned* ticket;
    Word *pairs, *states;                      // [tile][chain][strip], [window][chain][strip]
    int chains, window;
};

__device__ __forceinline__ Word pair_word(float A, float H) {      // A is no NaN of the bits that would make the upper half 0
    const unsigned a = A != A ? 0x7fc00000u : __float_as_uint(A);
    return (Word)~a << 32 | __float_as_uint(H);
}
__device__ __forceinline__ Word state_word(float h) { return (Word)1 << 32 | __float_as_uint(h); }
__device__ __forceinline__ void leave(Word* p, Word w) { __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ Word look(const Word* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct Pair { float a, h; };
__device__ __forceinline__ Pair then(Pair first, Pair second) { return {first.a * second.a, fmaf(second.a, first.h, second.h)}; }

// The state in front of tile `index` of `chain` (counted in the order of the pass), for the strip's 64 channels, into LDS: called by all
// threads of the workgroup, which has left the tile's own pair before.  `initial` is the state in front of the first tile.
template <int THREADS>
__device__ __forceinline__ void state_before(float* to, Pair (*parts)[kStrip], const Chains& k, int64_t index, int chain, float initial) {
    constexpr int kShares = THREADS / kStrip, kMost = kWindow / kShares;
    const int channel = threadIdx.x % kStrip, share = threadIdx.x / kStrip;
    const int64_t window = index / k.window, first = window * k.window;
    const int count = (int)(index - first);                        // tiles before this one in its window, less than kWindow
    const int per = (count + kShares - 1) / kShares, from = share * per, to_read = from + per < count ? per : count - from;
    const Word* pairs = k.pairs + ((first + from) * k.chains + chain) * kStrip + channel;
    Word words[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) words[i] = i < to_read ? 0 : pair_word(1.f, 0.f);
    for (bool all = false; !all;) {
        all = true;
#pragma unroll
        for (int i = 0; i < kMost; ++i)
            if (!(words[i] >> 32)) words[i] = look(pairs + (int64_t)i * k.chains * kStrip);
#pragma unroll
        for (int i = 0; i < kMost; ++i) all = all && words[i] >> 32;
        if (!all) __builtin_amdgcn_s_sleep(1);
    }
    Pair p = {1.f, 0.f};
#pragma unroll
    for (int i = 0; i < kMost; ++i)
        if (i < to_read) p = then(p, {__uint_as_float(~(unsigned)(words[i] >> 32)), __uint_as_float((unsigned)words[i])});
    parts[share][channel] = p;
    float h = initial;
    if (share == 0 && window > 0) {
        const Word* state = k.states + (window * k.chains + chain) * kStrip + channel;
        Word w = look(state);
        while (!(w >> 32)) {
            __builtin_amdgcn_s_sleep(1);
            w = look(state);
        }
        h = __uint_as_float((unsigned)w);
    }
    __syncthreads();
    if (share == 0) {
        for (int i = 1; i < kShares; ++i) p = then(p, parts[i][channel]);
        to[channel] = count > 0 ? fmaf(p.a, h, p.h) : h;
    }
    __syncthreads();
}

// ---- forward --------------------------------------------------------------------------------------------------------------------
template <typename T, int DRIVE, int S, int WAVES, bool LOOK>
__global__ __launch_bounds__(64 * WAVES) void leak_fwd_kernel(LeakArgs a, Chains k) {
    static_assert(4 * WAVES * S == kTile, "a tile is four lanes a wave");
    __shared__ f4 total[2][WAVES][2][16];                           // A, H of each wave and channel
    __shared__ f4 carry[2][16];
    __shared__ Pair parts[WAVES][kStrip];
    __shared__ unsigned ticket;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, lc = lane % 16, lt = lane / 16;
    unsigned chain = blockIdx.x;
    int64_t first = 0, end = a.tiles;
    if (LOOK) {
        if (threadIdx.x == 0) ticket = atomicAdd(k.ticket, 1u);
        __syncthreads();
        first = ticket / (unsigned)k.chains;
        chain = ticket - (unsigned)first * k.chains;
        end = first + 1;
    }
    const int strip = chain % (unsigned)a.strips;
    const int64_t n = chain / (unsigned)a.strips;
    const int c = strip * kStrip + lc * 4, left = a.channels - c;
    const int64_t length = length_of(a, n);
    const f4 d = decays_of(a, c, left);
    const T* in = (const T*)a.in + n * a.in_stride[0] + c;
    const T* gate = (const T*)a.gate + n * a.gate_stride[0] + c;
    T* out = (T*)a.out + n * a.tokens * a.channels + c;
    float initial = 0;                                              // of channel threadIdx.x of the strip
    if (threadIdx.x < kStrip) {
        const int channel = strip * kStrip + threadIdx.x;
        if (a.state && channel < a.channels) initial = a.state[n * a.channels + channel];
        if (!LOOK) ((float*)carry[0])[threadIdx.x] = initial;
    }
    for (int64_t tile = first; tile < end; ++tile) {
        const int turn = LOOK ? 0 : tile % 2;
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
        if (LOOK) {
            if (k.window > 1 && threadIdx.x < kStrip && (tile + 1) % k.window != 0 && tile + 1 < a.tiles) {
                Pair p = {1.f, 0.f};
#pragma unroll
                for (int w = 0; w < WAVES; ++w) p = then(p, {((float*)total[0][w][0])[threadIdx.x], ((float*)total[0][w][1])[threadIdx.x]});
                leave(k.pairs + (tile * k.chains + chain) * kStrip + threadIdx.x, pair_word(p.a, p.h));
            }
            state_before<64 * WAVES>((float*)carry[0], parts, k, tile, chain, initial);
        }
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
            if (!LOOK) carry[turn ^ 1][lc] = h;
            if (a.last && tile == a.tiles - 1 && left > 0) store_four(a.last + n * a.channels + c, h, left);
            if (LOOK && (tile + 1) % k.window == 0 && tile + 1 < a.tiles) {
                Word* to = k.states + ((tile + 1) / k.window * k.chains + chain) * kStrip + lc * 4;
#pragma unroll
                for (int v = 0; v < 4; ++v) leave(to + v, state_word(h[v]));
            }
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
// The same chains, their tiles from the last to the first.  Inside a tile the states go forwards, from the kept one, and G backwards.
template <typename T, int DRIVE, int S, int WAVES, bool LOOK>
__global__ __launch_bounds__(64 * WAVES) void leak_bwd_kernel(LeakArgs a, Chains k) {
    static_assert(4 * WAVES * S == kTile, "a tile is four lanes a wave");
    __shared__ f4 total[2][WAVES][3][16];                           // A, H, G of each wave and channel
    __shared__ f4 carry[2][16];
    __shared__ union {
        Pair parts[WAVES][kStrip];
        f4 sums[WAVES * 4][16];
    } u;
    __shared__ unsigned ticket;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, lc = lane % 16, lt = lane / 16;
    unsigned chain = blockIdx.x;
    int64_t first = 0, end = a.tiles;                               // counted from the last tile
    if (LOOK) {
        if (threadIdx.x == 0) ticket = atomicAdd(k.ticket, 1u);
        __syncthreads();
        first = ticket / (unsigned)k.chains;
        chain = ticket - (unsigned)first * k.chains;
        end = first + 1;
    }
    const int strip = chain % (unsigned)a.strips;
    const int64_t n = chain / (unsigned)a.strips;
    const int c = strip * kStrip + lc * 4, left = a.channels - c;
    const int64_t length = length_of(a, n);
    const f4 d = decays_of(a, c, left);
    const T* in = (const T*)a.in + n * a.in_stride[0] + c;
    const T* gate = (const T*)a.gate + n * a.gate_stride[0] + c;
    const T* grad = (const T*)a.grad + n * a.grad_stride[0] + c;
    T* grad_in = (T*)a.grad_in + n * a.tokens * a.channels + c;
    T* grad_gate = (T*)a.grad_gate + n * a.tokens * a.channels + c;
    f4 slopes = {};                                                 // sum of dleak * open
    float initial = 0;                                              // of channel threadIdx.x of the strip
    if (threadIdx.x < kStrip) {
        const int channel = strip * kStrip + threadIdx.x;
        if (a.grad_last && channel < a.channels) initial = a.grad_last[n * a.channels + channel];
        if (!LOOK) ((float*)carry[0])[threadIdx.x] = initial;
    }
    for (int64_t index = first; index < end; ++index) {
        const int64_t tile = a.tiles - 1 - index;
        const int turn = LOOK ? 0 : index % 2;
        const int64_t t0 = tile * kTile + (wave * 4 + lt) * S;
        typename Four<T>::Vec x[S], dy[S];
        float open[S][4];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            typename Four<T>::Vec z = {};
            x[s] = dy[s] = {};
            const bool on = t0 + s < length;
            if (on && left > 0) {
                x[s] = load_four(in + (t0 + s) * a.in_stride[1], left);
                z = load_four(gate + (t0 + s) * a.gate_stride[1], left);
                dy[s] = load_four(grad + (t0 + s) * a.grad_stride[1], left);
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) open[s][v] = on ? open_gate<T>((float)z[v]) : 0.f;   // what is not there leaks nothing, x and dy are 0
        }
        f4 start = {};
        if (left > 0) start = load_four(a.starts + (n * a.tiles + tile) * a.channels + c, left);
        f4 A = {1.f, 1.f, 1.f, 1.f}, H = {}, G = {};
#pragma unroll
        for (int v = 0; v < 4; ++v) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
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
        if (LOOK) {
            if (k.window > 1 && threadIdx.x < kStrip && (index + 1) % k.window != 0 && index + 1 < a.tiles) {
                Pair p = {1.f, 0.f};
#pragma unroll
                for (int w = WAVES - 1; w >= 0; --w)
                    p = then(p, {((float*)total[0][w][0])[threadIdx.x], ((float*)total[0][w][2])[threadIdx.x]});
                leave(k.pairs + (index * k.chains + chain) * kStrip + threadIdx.x, pair_word(p.a, p.h));
            }
            state_before<64 * WAVES>((float*)carry[0], u.parts, k, index, chain, initial);
        }
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
            if (!LOOK) carry[turn ^ 1][lc] = g;
            if (a.grad_state && tile == 0 && left > 0) store_four(a.grad_state + n * a.channels + c, g, left);
            if (LOOK && (index + 1) % k.window == 0 && index + 1 < a.tiles) {
                Word* to = k.states + ((index + 1) / k.window * k.chains + chain) * kStrip + lc * 4;
#pragma unroll
                for (int v = 0; v < 4; ++v) leave(to + v, state_word(g[v]));
            }
        }
        float before[S][4];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            h[v] = fmaf(before_a[v], h[v], before_h[v]);
            g[v] = fmaf(behind_a[v], mine[v], behind_g[v]);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                before[s][v] = h[v];
                const float leak = d[v] * open[s][v], keep = 1.f - leak;
                h[v] = fmaf(keep, h[v], drive_of<DRIVE>(leak, keep).value * (float)x[s][v]);
            }
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
    // the decays' gradient of this workgroup's tiles: a row of `parts` for each workgroup of a strip, or one number a workgroup
    __syncthreads();                                                // (the pairs' part of the union has been read)
    u.sums[wave * 4 + lt][lc] = slopes;
    __syncthreads();
    if (threadIdx.x >= kStrip) return;
    float sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES * 4; ++w) sum += ((float*)u.sums[w])[threadIdx.x];
    const int channel = strip * kStrip + threadIdx.x;
    if (a.decays > 1) {
        if (channel < a.channels) a.parts[(first * a.samples + n) * a.channels + channel] = sum;
    } else {
        sum = sum_lanes(sum, 64);                                   // (channels that are not there have 0)
        if (threadIdx.x == 0) a.parts[first * k.chains + chain] = sum;
    }
}

__global__ __launch_bounds__(256) void zero_words_kernel(Word* words, int64_t count) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) words[i] = 0;
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

// How the tiles are cut up among workgroups, and the workspace of that: the words, the ticket, the rows of the decays' gradient.
struct Plan {
    bool look;
    int64_t chains, blocks, window, words, rows;        // rows: of partial sums of the decays' gradient
};
Plan plan_of(const slayer_gated_leak* s) {
    Plan p = {};
    const int64_t tiles = tiles_of(s->tokens);
    p.chains = s->samples * strips_of(s->channels);
    p.look = tiles > 2 && p.chains < 2048 && tiles * p.chains < (1 << 23);
    p.blocks = p.look ? tiles * p.chains : p.chains;
    p.window = p.look ? 2048 / p.chains : 1;
    if (p.window > kWindow) p.window = kWindow;
    if (p.window > tiles) p.window = tiles;
    if (p.look) p.words = ((p.window > 1 ? tiles : 0) + (tiles + p.window - 1) / p.window) * p.chains * kStrip + 1;
    p.rows = (p.look ? tiles : 1) * (s->num_decays == 1 ? p.chains : s->samples);
    return p;
}
// The zeroed words at the front of the workspace.
int chains_of(Chains* k, const Plan& p, const slayer_gated_leak* s, float* workspace, hipStream_t stream) {
    if (!p.look) return 0;
    k->chains = (int)p.chains;
    k->window = (int)p.window;
    k->ticket = (unsigned*)workspace;
    k->pairs = (Word*)workspace + 1;
    k->states = k->pairs + (p.window > 1 ? tiles_of(s->tokens) : 0) * p.chains * kStrip;
    const int64_t blocks = (p.words + 1023) / 1024;
    hipLaunchKernelGGL(zero_words_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, stream, (Word*)workspace, p.words);
    return (int)hipGetLastError();
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
    const Plan p = plan_of(s);
    return 2 * p.words + (backward ? p.rows * s->num_decays : 0);
}

extern "C" int slayer_gated_leak_fwd(void* out, float* last, float* starts, const void* input, const void* gate, const float* state,
                                     const slayer_gated_leak* s, float* workspace, int64_t floats, void* stream) {
    if (int e = check_leak(s)) return e;
    if (s->samples == 0) return 0;
    if (s->tokens > 0 && (!out || !input || !gate)) return SLAYER_ENULL;
    const Plan p = plan_of(s);
    if (p.words > 0 && !workspace) return SLAYER_ENULL;
    if (floats < 2 * p.words || (uintptr_t)workspace % 8 != 0) return SLAYER_EINVAL;
    LeakArgs a = args_of(s);
    a.out = out; a.last = last; a.starts = starts; a.in = input; a.gate = gate; a.state = state;
    Chains k = {};
    if (int e = chains_of(&k, p, s, workspace, (hipStream_t)stream)) return e;
#define ONE(T, DRIVE, LOOK) \
    hipLaunchKernelGGL((leak_fwd_kernel<T, DRIVE, 8, 4, LOOK>), dim3((unsigned)p.blocks), dim3(256), 0, (hipStream_t)stream, a, k)
#define LAUNCH(T, DRIVE)                    \
    if (p.look) ONE(T, DRIVE, true);        \
    else ONE(T, DRIVE, false)
    BY_TYPE(LAUNCH)
#undef LAUNCH
#undef ONE
    return (int)hipGetLastError();
}

extern "C" int slayer_gated_leak_bwd(void* grad_input, void* grad_gate, float* grad_decay, float* grad_state, const void* grad_out,
                                     const float* grad_last, const void* input, const void* gate, const float* starts,
                                     const slayer_gated_leak* s, float* workspace, int64_t floats, void* stream) {
    if (int e = check_leak(s)) return e;
    if (s->samples == 0) return grad_decay ? launch_zero_fill(grad_decay, s->num_decays, (hipStream_t)stream) : 0;
    if (!starts || (s->tokens > 0 && (!grad_input || !grad_gate || !grad_out || !input || !gate))) return SLAYER_ENULL;
    const Plan p = plan_of(s);
    const int64_t need = 2 * p.words + (grad_decay ? p.rows * s->num_decays : 0);
    if (need > 0 && !workspace) return SLAYER_ENULL;
    if (floats < need || (uintptr_t)workspace % 8 != 0) return SLAYER_EINVAL;
    LeakArgs a = args_of(s);
    a.grad_in = grad_input; a.grad_gate = grad_gate; a.grad_state = grad_state; a.grad = grad_out; a.grad_last = grad_last;
    a.in = input; a.gate = gate; a.starts = (float*)starts;
    a.parts = grad_decay ? workspace + 2 * p.words : nullptr;
    Chains k = {};
    if (int e = chains_of(&k, p, s, workspace, (hipStream_t)stream)) return e;
#define ONE(T, DRIVE, LOOK) \
    hipLaunchKernelGGL((leak_bwd_kernel<T, DRIVE, 4, 8, LOOK>), dim3((unsigned)p.blocks), dim3(512), 0, (hipStream_t)stream, a, k)
#define LAUNCH(T, DRIVE)                    \
    if (p.look) ONE(T, DRIVE, true);        \
    else ONE(T, DRIVE, false)
    BY_TYPE(LAUNCH)
#undef LAUNCH
#undef ONE
    if (int e = (int)hipGetLastError()) return e;
    if (!grad_decay) return 0;
    ColumnSums sums = {};
    sums.out[0] = grad_decay; sums.parts[0] = a.parts; sums.factor = 1.f / 4096.f;
    sums.columns = sums.pitch = s->num_decays;
    sums.rows = p.rows;
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

// Gated leak: the leaky integrator whose leak a token's gate opens, with the channels last.  For every sample and channel
//     open = sigmoid(gate[t]),  leak = decay / 4096 * open,  h[t] = (1 - leak) h[t-1] + drive(leak) x[t],
// drive 1, leak, or sqrt(leak (2 - leak)).  Backwards, with D the derivative with respect to the state behind a token and G with
// respect to the state in front of it,
//     D[t] = dy[t] + G[t+1],  G[t] = (1 - leak) D[t],  dx = drive D,  dleak = D (drive' x - h[t-1]),
//     dgate = dleak leak (1 - open),  ddecay = sum of dleak open / 4096.
// Both are linear recurrences s <- A s + H in one number a channel, and spans of tokens join as pairs (A, H).  A wave takes eight or sixteen
// tokens of 64 or 128 neighbouring channels, a lane one float32 or two bfloat16 of each token: rows are read and written 256 bytes at a time
// at addresses that are the same for the wave, channels need no joining, and which tokens there are is a scalar question.  Eight waves, one
// behind the other, make a tile; their pairs meet in LDS, where one thread a channel runs through them, and with the state in front of it each
// wave walks its tokens again in its registers.  The backward pass makes the states of a tile again from the one in front of it, which the
// forward pass has kept (one in 64 tokens), so that it reads neither the results nor anything rounded.
//   Bound: memory, three tensors forward and five backward (a copy reaches 5.1 TB/s).  [32,1500,256] float32: forward 30 us (5.0 TB/s), backward 48 (5.1);
// one sample of 32768 tokens of 1024 channels, bfloat16: 47 (4.3).  Not so samples of different lengths, where what lies behind an end is written and not
// read: [16,1450,1021] bfloat16, half of it behind ends, 34 and 53 us, 2.8 and 3.1 TB/s (likely tiles that wait for each other; vector instructions
// 46 and 69 % of the cycles); nor a few tokens, which leave waves of a tile idle: [256,4,4096] bfloat16 77 and 74 us.  The forms before: lanes of four channels with
// tokens across the lanes, 43 and 74, 53 and 122, prompt 69 (joining across lanes takes as many instructions as the recurrence).
#include "common.h"
#include "elements.h"

namespace slayer {
namespace {

enum { DRIVE_NONE, DRIVE_GAIN, DRIVE_VARIANCE };

constexpr int kKept = 64;                      // tokens from one state that is kept for the backward pass to the next

struct LeakArgs {
    void *out, *grad_in, *grad_gate;
    const void *in, *gate, *grad, *lengths;
    const float *decay, *state, *grad_last;
    float *last, *starts, *grad_state, *parts;
    int64_t samples, tokens, tiles, kept;
    int64_t in_stride[2], gate_stride[2], grad_stride[2];
    int channels, strips, lengths_bytes, decays;
};

// sigmoid from the hardware's exponential and reciprocal, a unit in the last place each.  For bfloat16 gates as they are, (3 + 1.5 |z|) 2^-24, most
// of it the rounding of z / ln 2; for float32 ones what that rounding leaves goes into the exponential, 2^x (1 + r ln 2): 6 2^-24 (6 instructions,
// [32,1500,256] forward and backward 0.5 to 1 us).  Infinite gates are open and closed.
template <typename T> __device__ __forceinline__ float open_gate(float z) {
    constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;
    constexpr float hi = (float)-kLog2e, lo = (float)(-kLog2e - (double)hi);
    const float x = z * hi;
    float e = __builtin_amdgcn_exp2f(x);
    if (sizeof(T) == 4) e = __builtin_fabsf(x) < 126.f ? fmaf(e, fmaf(z, lo, fmaf(z, hi, -x)) * (float)kLn2, e) : e;
    return __builtin_amdgcn_rcpf(1.f + e);
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

// What a lane reads and writes of a row: one float32 or bfloat16, or two bfloat16 at any address that suits one of them.  closed(): gates of -inf.
template <typename T, int V> struct Piece;
template <> struct Piece<float, 1> { typedef float Raw; static __device__ Raw closed() { return -__builtin_inff(); } };
template <> struct Piece<bf16, 1> { typedef unsigned short Raw; static __device__ Raw closed() { return 0xff80; } };
template <> struct Piece<bf16, 2> { typedef unsigned Raw; static __device__ Raw closed() { return 0xff80ff80; } };
typedef unsigned unsigned_any __attribute__((aligned(2)));
template <int V> __device__ __forceinline__ typename Piece<bf16, V>::Raw load_piece(const bf16* p) {
    if constexpr (V == 1) return *reinterpret_cast<const unsigned short*>(p);
    else return *reinterpret_cast<const unsigned_any*>(p);
}
template <int V> __device__ __forceinline__ float load_piece(const float* p) { return *p; }
__device__ __forceinline__ float value_of(float raw, int) { return raw; }
__device__ __forceinline__ float value_of(unsigned short raw, int) { return __uint_as_float((unsigned)raw << 16); }
__device__ __forceinline__ float value_of(unsigned raw, int v) { return __uint_as_float(v ? raw & 0xffff0000u : raw << 16); }
__device__ __forceinline__ void store_piece(float* p, const float (&x)[1]) { *p = x[0]; }
__device__ __forceinline__ void store_piece(bf16* p, const float (&x)[1]) { *p = (bf16)x[0]; }
typedef bf16 b2 __attribute__((ext_vector_type(2)));
typedef b2 b2_any __attribute__((aligned(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void store_piece(bf16* p, const float (&x)[2]) {
    *reinterpret_cast<b2_any*>(p) = __builtin_convertvector(f2{x[0], x[1]}, b2);
}
// The channels of a lane.  A last channel without a neighbour (V is 2 and the channels are odd) is read with the one in front of it: `odd`
// lanes have their own channel in value 1, and value 0 goes where a channel behind the last one would be.  Lanes without channels read the
// last ones.
template <int V> struct Lane {
    int c, from, odd, slot;                    // first channel, first channel read, slot of value 0 in the strip
    bool on;
    __device__ __forceinline__ Lane(int strip, int lane, int channels) {
        c = (strip * 64 + lane) * V;
        on = c < channels;
        odd = V == 2 && c + 1 == channels;
        from = on ? c - odd : channels - V;
        slot = lane * V;
    }
    __device__ __forceinline__ int at(int v) const { return slot + (v ^ odd); }
    template <typename T> __device__ __forceinline__ void store(T* row, const float (&x)[V]) const {
        if (!odd) store_piece(row + c, x);
        else row[c] = (T)x[V - 1];
    }
};
// Keeps the compiler from holding on to what it has made of x: that is made again instead of taking up registers.
__device__ __forceinline__ void forget(float& x) { asm volatile("" : "+v"(x)); }

// What a few tokens keep of the state in front of them, the product of 1 - leak, and what they lose of it, by itself: each 1 - leak is a multiple
// of 2^-24, off by the same amount at every token of a steady gate, which would add up along a sample (a leak of 2e-5 at each of 32768 tokens:
// states 1e-3 off).  (As one float64 product: the backward walk spills.)
__device__ __forceinline__ void hold(float& kept, float& lost, float leak, float keep) {
    lost += fmaf(-leak, lost, leak);
    kept *= keep;
}
__device__ __forceinline__ double held(float kept, float lost) { return kept < 0.5f ? (double)kept : 1.0 - (double)lost; }

__device__ __forceinline__ int64_t length_of(const LeakArgs& a, int64_t n) {
    if (!a.lengths) return a.tokens;
    const int64_t length = a.lengths_bytes == 4 ? ((const int*)a.lengths)[n] : ((const int64_t*)a.lengths)[n];
    return length < 0 ? 0 : length < a.tokens ? length : a.tokens;
}

// ---- tiles of a chain -----------------------------------------------------------------------------------------------------------
// A chain is one strip of one sample, from tile to tile in the order of the pass.  Either a workgroup walks all tiles of a chain and
// carries the state in registers, or there is a workgroup for each tile, and states go through memory:
//   A workgroup takes the next tile of its chain by a ticket, so it only ever waits for workgroups of the same chain with lower tickets,
// which are running or done and wait for lower ones themselves; the lowest waits for nobody, so every wait ends.  (One ticket for all
// chains would be taken at 12 ns each, whoever asks: 25 us for the 2048 tiles of a prompt.)  Tiles form windows.  A tile leaves its pair, then
// reads those of the tiles before it in its window, and the state in front of the window; the last tile of a window leaves the state
// behind it.  Which values are joined, and in which order, depends on the sizes alone and not on who comes first, so that a call computed
// again has the same bits.
//   Spans are joined in float64 and states go from wave to wave and tile to tile in it; they are rounded where a wave walks its tokens, so that
// a result carries the roundings of at most 16 tokens, however many there are.
//   What is left is a word of 64 bits that says itself that it is there (the workspace is zeroed before), read and written with relaxed
// atomics of the whole device: no other memory hangs on it, so no fences are needed.
//   Windows of sixteen: of 32 tiles the words a thread waits for take the registers of a workgroup (backward, [16,1450,1021]: 57 us, and 51; one sample of
// 65536 tokens of 256 float32 channels gains, forward 44 us, and 49), of eight the states have too far to go (that sample: 69 us).
typedef unsigned long long Word;
constexpr int kWindow = 16;                    // tiles of a window
constexpr int kApart = 16;                     // words from one chain's ticket to the next: a cache line each

struct Chains {
    Word *tickets, *pairs, *states;            // [chain], [tile][chain][strip], [window][chain][strip]
    int chains;
};

// A's 32 bits: from a half on those of 1 - A, the leak, with the last bit set; below a half its own, with the last bit cleared.  Either is
// within 2^-23 of itself.  A NaN has bits that do not make the upper half 0.
__device__ __forceinline__ Word pair_word(double A, float H) {
    const bool slow = A >= 0.5;
    const float f = (float)(slow ? 1.0 - A : A);
    const unsigned a = f != f ? 0x7fc00000u : __float_as_uint(f);
    return (Word)~((a & ~1u) | slow) << 32 | __float_as_uint(H);
}
__device__ __forceinline__ double kept_of(Word w) {
    const unsigned a = ~(unsigned)(w >> 32);
    const double f = (double)__uint_as_float(a & ~1u);
    return a & 1 ? 1.0 - f : f;
}
__device__ __forceinline__ Word state_word(double h) { return h != h ? ~0x7ff8000000000000ull : ~(Word)__double_as_longlong(h); }
__device__ __forceinline__ double state_of(Word w) { return __longlong_as_double((long long)~w); }
__device__ __forceinline__ void leave(Word* p, Word w) { __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ Word look(const Word* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct Pair { double a, h; };
__device__ __forceinline__ Pair then(Pair first, Pair second) { return {first.a * second.a, fma(second.a, first.h, second.h)}; }

// The pair of all tiles before tile `index` (counted in the order of the pass) in its window, and the state in front of the window
// (`initial` in front of the first one), for channel threadIdx.x % CH: for the first CH threads.  All threads of the workgroup call it.
struct Before { Pair pair; double state; };
template <int THREADS, int CH>
__device__ __forceinline__ Before look_back(Pair (*parts)[CH], const Chains& k, int64_t index, unsigned chain, double initial) {
    constexpr int kShares = THREADS / CH, kMost = kWindow / kShares;
    const int channel = threadIdx.x % CH, share = threadIdx.x / CH;
    const int64_t window = index / kWindow, first = window * kWindow;
    const int count = (int)(index - first);                        // less than kWindow
    const int per = (count + kShares - 1) / kShares, from = share * per, mine = count - from < per ? count - from : per;
    Before b = {{1.0, 0.0}, initial};
    if (count > 0) {
        const Word* pairs = k.pairs + ((first + from) * k.chains + chain) * CH + channel;
        Word words[kMost];
#pragma unroll
        for (int i = 0; i < kMost; ++i) words[i] = i < mine ? 0 : pair_word(1.0, 0.f);
        for (bool all = false; !all;) {
            all = true;
#pragma unroll
            for (int i = 0; i < kMost; ++i)
                if (!(words[i] >> 32)) words[i] = look(pairs + (int64_t)i * k.chains * CH);
#pragma unroll
            for (int i = 0; i < kMost; ++i) all = all && words[i] >> 32;
            if (!all) __builtin_amdgcn_s_sleep(1);
        }
#pragma unroll
        for (int i = 0; i < kMost; ++i)
            if (i < mine) b.pair = then(b.pair, {kept_of(words[i]), (double)__uint_as_float((unsigned)words[i])});
        parts[share][channel] = b.pair;
        __syncthreads();
    }
    if (share > 0) return b;
    for (int i = 1; i < kShares && count > 0; ++i) b.pair = then(b.pair, parts[i][channel]);
    if (window > 0) {
        const Word* state = k.states + (window * k.chains + chain) * CH + channel;
        Word w = look(state);
        while (w == 0) {
            __builtin_amdgcn_s_sleep(1);
            w = look(state);
        }
        b.state = state_of(w);
    }
    return b;
}

// Which chain a workgroup is in, and which of its tiles it takes.
struct Span { unsigned chain; int64_t first, end; };
template <bool LOOK> __device__ __forceinline__ Span span_of(const LeakArgs& a, const Chains& k) {
    if (!LOOK) return {blockIdx.x, 0, a.tiles};
    __shared__ unsigned ticket;
    const unsigned chain = blockIdx.x % (unsigned)k.chains;
    if (threadIdx.x == 0) ticket = (unsigned)atomicAdd(k.tickets + chain * kApart, 1ull);
    __syncthreads();
    const unsigned tile = __builtin_amdgcn_readfirstlane(ticket);
    return {chain, tile, (int64_t)tile + 1};
}

// ---- forward --------------------------------------------------------------------------------------------------------------------
// S tokens a wave, V channels a lane.
template <typename T, int V, int DRIVE, int S, int WAVES, bool LOOK>
__global__ __launch_bounds__(64 * WAVES, 4) void leak_fwd_kernel(LeakArgs a, Chains k) {
    constexpr int CH = 64 * V, kTile = S * WAVES;
    static_assert(kKept % S == 0 && kTile % kKept == 0, "a wave begins where a state is kept");
    __shared__ double total_a[WAVES][CH];
    __shared__ float total_h[WAVES][CH], front[WAVES][CH];          // front: the state in front of each wave
    __shared__ Pair parts[LOOK ? 64 * WAVES / CH : 1][CH];
    const Span span = span_of<LOOK>(a, k);
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int strip = span.chain % (unsigned)a.strips;
    const int64_t n = span.chain / (unsigned)a.strips, length = length_of(a, n);
    const Lane<V> own(strip, lane, a.channels);
    float d[V];
#pragma unroll
    for (int v = 0; v < V; ++v) d[v] = a.decay[a.decays == 1 ? 0 : own.from + v] * (1.f / 4096.f);
    const T* in = (const T*)a.in + n * a.in_stride[0];
    const T* gate = (const T*)a.gate + n * a.gate_stride[0];
    T* out = (T*)a.out + n * a.tokens * a.channels;
    const int channel = strip * CH + threadIdx.x;                  // of the first CH threads
    const bool keeps = threadIdx.x < CH && channel < a.channels;
    double carry = keeps && a.state ? a.state[n * a.channels + channel] : 0.f;
    for (int64_t tile = span.first; tile < span.end; ++tile) {
        const int64_t t0 = tile * kTile + wave * S;
        const int count = length - t0 < S ? (length > t0 ? (int)(length - t0) : 0) : S;
        float keep[S][V], add[S][V], kept[V], lost[V], h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            kept[v] = 1;
            lost[v] = h[v] = 0;
        }
        if (count > 0) {
            typename Piece<T, V>::Raw x[S], z[S];
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int64_t t = t0 + (s < count ? s : count - 1);
                x[s] = load_piece<V>(in + t * a.in_stride[1] + own.from);
                z[s] = load_piece<V>(gate + t * a.gate_stride[1] + own.from);
            }
            if (count < S) {                                       // what is not there leaks nothing
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (s >= count) {
                        x[s] = 0;
                        z[s] = Piece<T, V>::closed();
                    }
            }
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float leak = d[v] * open_gate<T>(value_of(z[s], v));
                    keep[s][v] = 1.f - leak;
                    add[s][v] = drive_of<DRIVE>(leak, keep[s][v]).value * value_of(x[s], v);
                    hold(kept[v], lost[v], leak, keep[s][v]);
                    h[v] = fmaf(keep[s][v], h[v], add[s][v]);
                }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            total_a[wave][own.at(v)] = held(kept[v], lost[v]);
            total_h[wave][own.at(v)] = h[v];
        }
        __syncthreads();
        if (LOOK) {
            if (threadIdx.x < CH && (tile + 1) % kWindow != 0 && tile + 1 < a.tiles) {
                Pair p = {1, 0};
#pragma unroll
                for (int w = 0; w < WAVES; ++w) p = then(p, {total_a[w][threadIdx.x], total_h[w][threadIdx.x]});
                leave(k.pairs + (tile * k.chains + span.chain) * CH + threadIdx.x, pair_word(p.a, (float)p.h));
            }
            const Before b = look_back<64 * WAVES, CH>(parts, k, tile, span.chain, carry);
            carry = tile % kWindow == 0 ? b.state : fma(b.pair.a, b.state, b.pair.h);
        }
        if (threadIdx.x < CH) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                front[w][threadIdx.x] = (float)carry;
                const int64_t start = tile * (kTile / kKept) + w * S / kKept;
                if (w * S % kKept == 0 && a.starts && keeps && start < a.kept) a.starts[(n * a.kept + start) * a.channels + channel] = (float)carry;
                carry = fma(total_a[w][threadIdx.x], carry, (double)total_h[w][threadIdx.x]);
            }
            if (a.last && keeps && tile == a.tiles - 1) a.last[n * a.channels + channel] = (float)carry;
            if (LOOK && (tile + 1) % kWindow == 0 && tile + 1 < a.tiles)
                leave(k.states + ((tile + 1) / kWindow * k.chains + span.chain) * CH + threadIdx.x, state_word(carry));
        }
        __syncthreads();
        if (!own.on) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = front[wave][own.at(v)];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (s < count) {
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = fmaf(keep[s][v], h[v], add[s][v]);
                own.store(out + (t0 + s) * a.channels, h);
            } else if (t0 + s < a.tokens) {
                const float none[V] = {};
                own.store(out + (t0 + s) * a.channels, none);
            }
        }
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------------
// The same chains, their tiles from the last to the first.  Inside a tile the states go forwards, from the kept one, and G backwards.
// LOOK: 80 registers, a third workgroup on a compute unit ([32,1500,256] float32, drive none and root: 44 and 47 us; with 84 registers and two
// workgroups 47 and 50).  G and the states in front of the waves run through threads of their own at the same time ([256,4,4096] bfloat16: 73 us, and 79).
template <typename T, int V, int DRIVE, int S, int WAVES, bool LOOK>
__global__ __launch_bounds__(64 * WAVES, LOOK ? 6 : 4) void leak_bwd_kernel(LeakArgs a, Chains k) {
    constexpr int CH = 64 * V, kTile = S * WAVES;
    static_assert(kTile % kKept == 0, "a tile begins where a state is kept");
    __shared__ double total_a[WAVES][CH];
    __shared__ float total_h[WAVES][CH], total_g[WAVES][CH];
    __shared__ float front[WAVES][CH], behind[WAVES][CH];           // the state in front of each wave, G behind it
    __shared__ Pair parts[LOOK ? 64 * WAVES / CH : 1][CH];
    const Span span = span_of<LOOK>(a, k);
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int strip = span.chain % (unsigned)a.strips;
    const int64_t n = span.chain / (unsigned)a.strips, length = length_of(a, n);
    const Lane<V> own(strip, lane, a.channels);
    float d[V];
    double slopes[V];                                               // sum of dleak * open: of a tile in float32, of the tiles of a walk in float64
#pragma unroll
    for (int v = 0; v < V; ++v) {
        d[v] = a.decay[a.decays == 1 ? 0 : own.from + v] * (1.f / 4096.f);
        slopes[v] = 0;
    }
    const T* in = (const T*)a.in + n * a.in_stride[0];
    const T* gate = (const T*)a.gate + n * a.gate_stride[0];
    const T* grad = (const T*)a.grad + n * a.grad_stride[0];
    T* grad_in = (T*)a.grad_in + n * a.tokens * a.channels;
    T* grad_gate = (T*)a.grad_gate + n * a.tokens * a.channels;
    // the first CH threads have a channel of G each, the next ones a channel of the states
    const int at = threadIdx.x % CH, role = threadIdx.x / CH, channel = strip * CH + at;
    const bool keeps = role == 0 && channel < a.channels;
    double carry = keeps && a.grad_last ? a.grad_last[n * a.channels + channel] : 0.f;
    for (int64_t index = span.first; index < span.end; ++index) {   // counted from the last tile
        const int64_t tile = a.tiles - 1 - index, t0 = tile * kTile + wave * S;
        const int count = length - t0 < S ? (length > t0 ? (int)(length - t0) : 0) : S;
        double start = 0;
        if (role == 1 && channel < a.channels) start = a.starts[(n * a.kept + tile * (kTile / kKept)) * a.channels + channel];
        float open[S][V];
        typename Piece<T, V>::Raw x[S], dy[S];
        float kept[V], lost[V], h[V], g[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            kept[v] = 1;
            lost[v] = h[v] = g[v] = 0;
        }
        if (count > 0) {
            typename Piece<T, V>::Raw z[S];
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int64_t t = t0 + (s < count ? s : count - 1);
                z[s] = load_piece<V>(gate + t * a.gate_stride[1] + own.from);
                x[s] = load_piece<V>(in + t * a.in_stride[1] + own.from);
                dy[s] = load_piece<V>(grad + t * a.grad_stride[1] + own.from);
            }
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int v = 0; v < V; ++v) open[s][v] = open_gate<T>(value_of(z[s], v));
            if (count < S) {                                       // what is not there leaks nothing
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (s >= count) {
                        x[s] = dy[s] = 0;
#pragma unroll
                        for (int v = 0; v < V; ++v) open[s][v] = 0;
                    }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    const float leak = d[v] * open[s][v], keep = 1.f - leak;
                    h[v] = fmaf(keep, h[v], drive_of<DRIVE>(leak, keep).value * value_of(x[s], v));
                    hold(kept[v], lost[v], leak, keep);
                    forget(kept[v]);
                }
#pragma unroll
                for (int s = S - 1; s >= 0; --s) g[v] = fmaf(-d[v], open[s][v], 1.f) * (value_of(dy[s], v) + g[v]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            total_a[wave][own.at(v)] = held(kept[v], lost[v]);
            total_h[wave][own.at(v)] = h[v];
            total_g[wave][own.at(v)] = g[v];
        }
        __syncthreads();
        if (LOOK) {
            if (role == 0 && (index + 1) % kWindow != 0 && index + 1 < a.tiles) {
                Pair p = {1, 0};
#pragma unroll
                for (int w = WAVES - 1; w >= 0; --w) p = then(p, {total_a[w][at], total_g[w][at]});
                leave(k.pairs + (index * k.chains + span.chain) * CH + at, pair_word(p.a, (float)p.h));
            }
            const Before b = look_back<64 * WAVES, CH>(parts, k, index, span.chain, carry);
            carry = index % kWindow == 0 ? b.state : fma(b.pair.a, b.state, b.pair.h);
        }
        if (role == 0) {
#pragma unroll
            for (int w = WAVES - 1; w >= 0; --w) {
                behind[w][at] = (float)carry;
                carry = fma(total_a[w][at], carry, (double)total_g[w][at]);
            }
            if (a.grad_state && keeps && tile == 0) a.grad_state[n * a.channels + channel] = (float)carry;
            if (LOOK && (index + 1) % kWindow == 0 && index + 1 < a.tiles)
                leave(k.states + ((index + 1) / kWindow * k.chains + span.chain) * CH + at, state_word(carry));
        } else if (role == 1) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                front[w][at] = (float)start;
                start = fma(total_a[w][at], start, (double)total_h[w][at]);
            }
        }
        __syncthreads();
        if (!own.on) continue;
        if (count > 0) {
            float before[S][V], slope[V] = {};
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = front[wave][own.at(v)];
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    forget(open[s][v]);
                    before[s][v] = h[v];
                    const float leak = d[v] * open[s][v], keep = 1.f - leak;
                    h[v] = fmaf(keep, h[v], drive_of<DRIVE>(leak, keep).value * value_of(x[s], v));
                }
                g[v] = behind[wave][own.at(v)];
            }
#pragma unroll
            for (int s = S - 1; s >= 0; --s) {
                if (s >= count) continue;
                float dx[V], dz[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    forget(open[s][v]);
                    const float leak = d[v] * open[s][v], keep = 1.f - leak;
                    const Drive drive = drive_of<DRIVE>(leak, keep);
                    const float D = value_of(dy[s], v) + g[v];
                    const float dleak = D * fmaf(drive.slope, value_of(x[s], v), -before[s][v]);
                    dx[v] = drive.value * D;
                    dz[v] = dleak * leak * (1.f - open[s][v]);
                    slope[v] = fmaf(dleak, open[s][v], slope[v]);
                    g[v] = keep * D;
                }
                own.store(grad_in + (t0 + s) * a.channels, dx);
                own.store(grad_gate + (t0 + s) * a.channels, dz);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) slopes[v] += slope[v];
        }
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (s >= count && t0 + s < a.tokens) {
                const float none[V] = {};
                own.store(grad_in + (t0 + s) * a.channels, none);
                own.store(grad_gate + (t0 + s) * a.channels, none);
            }
    }
    if (!a.parts) return;
    // the decays' gradient of this workgroup's tiles: a row of `parts` for all workgroups of a sample's strips, or one number a workgroup
    __syncthreads();                                                // (front has been read)
#pragma unroll
    for (int v = 0; v < V; ++v) front[wave][own.at(v)] = (float)slopes[v];
    __syncthreads();
    if (threadIdx.x >= CH) return;
    float sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += front[w][threadIdx.x];
    if (a.decays > 1) {
        if (channel < a.channels) a.parts[(span.first * a.samples + n) * a.channels + channel] = sum;
        return;
    }
    sum = sum_lanes(channel < a.channels ? sum : 0.f, 64);
    if (lane == 0) a.parts[(span.first * a.samples * a.strips + span.chain) * V + wave] = sum;
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
    f4 d = {};
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (v < left) d[v] = a.decay[a.decays == 1 ? 0 : c + v] * (1.f / 4096.f);
    const typename Four<T>::Vec x = load_four((const T*)a.in + n * a.in_stride[0] + c, left);
    const typename Four<T>::Vec z = load_four((const T*)a.gate + n * a.gate_stride[0] + c, left);
    f4 h = load_four(a.last + n * a.channels + c, left);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const float leak = d[v] * open_gate<T>((float)z[v]), add = drive_of<DRIVE>(leak, 1.f - leak).value * (float)x[v];
        h[v] = (float)fma(1.0 - (double)leak, (double)h[v], (double)add);
    }
    store_four(a.last + n * a.channels + c, h, left);
    store_four((T*)a.out + n * a.channels + c, h, left);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Channels of a lane: two bfloat16 where there are two, so that a wave reads 256 bytes of a row.  (One: [16,1450,1021], ragged, 42 us forward and 67
// backward where two take 33 and 51; the prompt above 52 and 98 where two take 50 and 102.)
int lane_of(const slayer_gated_leak* s) { return s->dtype == SLAYER_BFLOAT16 && s->channels > 1 ? 2 : 1; }
// Tokens of a wave, of the eight waves of a workgroup: as many as leave registers for a second workgroup on a compute unit (backward, pairs of
// bfloat16, sixteen tokens: [16,1450,1021] 109 us where eight take 51).
constexpr int tokens_of(int lane, bool backward) { return lane == 2 && backward ? 8 : 16; }
constexpr int kWaves = 8;
constexpr int64_t kMostBlocks = (int64_t)1 << 23;                  // of 512 threads: fewer than 2^32 threads in a launch

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
    if (a->samples * ceil_div(a->channels, 64 * lane_of(a)) >= kMostBlocks) return SLAYER_ERANGE;          // a workgroup each
    return 0;
}

// How the tiles are cut up among workgroups, and the workspace of that: the words, the ticket, the rows of the decays' gradient.
struct Plan {
    bool look;
    int64_t tiles, strips, chains, blocks, pairs, words, rows, columns;   // rows, columns: of partial sums of the decays' gradient
};
Plan plan_of(const slayer_gated_leak* s, bool backward) {
    Plan p = {};
    const int lane = lane_of(s), tile = kWaves * tokens_of(lane, backward);
    p.tiles = s->tokens > 0 ? ceil_div(s->tokens, tile) : 1;
    p.strips = ceil_div(s->channels, 64 * lane);
    p.chains = s->samples * p.strips;
    // A workgroup for each tile where chains are fewer than compute units; with more, walking saves the words and the launch that zeroes
    // them.  Forward / backward, us, a workgroup for each tile and a walk: [32,512,512] bfloat16, 128 chains, 15 / 27 and 19 / 36; [48,512,512], 192
    // chains, 22 / 34 and 21 / 38; [64,512,512], 256 chains, 25 / 39 and 22 / 39; 400 chains, 37 / 60 and 31 / 63; float32, 200 chains, 30 / 47 and 28 / 47.
    // One rule for both directions: between 192 and 300 chains bfloat16 backward passes would gain up to a fifth from the other form (272 chains:
    // 40 and 50).  Two tiles, [4,200,128] float32: 7.7 / 11.1 and 8.3 / 13.6, but such calls wait for the host, where a launch and an allocation
    // more cost 4.5 us (11.3 us a call with the walk, 15.8 without).
    p.look = p.tiles > 2 && p.chains < 192 && p.tiles * p.chains < kMostBlocks;
    p.blocks = p.look ? p.tiles * p.chains : p.chains;
    if (p.look) {
        p.pairs = p.tiles * p.chains * 64 * lane;
        p.words = p.chains * kApart + p.pairs + ceil_div(p.tiles, kWindow) * p.chains * 64 * lane;
    }
    p.columns = s->num_decays;
    p.rows = (p.look ? p.tiles : 1) * (s->num_decays == 1 ? p.chains * lane : s->samples);
    return p;
}
int64_t floats_of(const Plan& p, bool sums) { return 2 * p.words + (sums ? p.rows * p.columns : 0); }

// The zeroed words at the front of the workspace.
int chains_of(Chains* k, const Plan& p, float* workspace, hipStream_t stream) {
    if (!p.look) return 0;
    k->chains = (int)p.chains;
    k->tickets = (Word*)workspace;
    k->pairs = k->tickets + p.chains * kApart;
    k->states = k->pairs + p.pairs;
    const int64_t blocks = ceil_div(p.words, 1024);
    hipLaunchKernelGGL(zero_words_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, stream, (Word*)workspace, p.words);
    return (int)hipGetLastError();
}

LeakArgs args_of(const slayer_gated_leak* s, const Plan& p) {
    LeakArgs a = {};
    a.lengths = s->lengths; a.lengths_bytes = s->lengths_bytes;
    a.decay = s->decay; a.decays = (int)s->num_decays;
    a.samples = s->samples; a.tokens = s->tokens; a.tiles = p.tiles;
    a.kept = s->tokens > 0 ? ceil_div(s->tokens, kKept) : 1;
    a.channels = (int)s->channels; a.strips = (int)p.strips;
    for (int i = 0; i < 2; ++i) {
        a.in_stride[i] = s->input_stride[i];
        a.gate_stride[i] = s->gate_stride[i];
        a.grad_stride[i] = s->grad_stride[i];
    }
    return a;
}

#define BY_DRIVE(LAUNCH, ...)                                           \
    switch (s->drive) {                                                 \
        case DRIVE_NONE: LAUNCH(DRIVE_NONE, __VA_ARGS__); break;        \
        case DRIVE_GAIN: LAUNCH(DRIVE_GAIN, __VA_ARGS__); break;        \
        default: LAUNCH(DRIVE_VARIANCE, __VA_ARGS__); break;            \
    }
#define BY_TYPE(LAUNCH)                                                 \
    if (s->dtype == SLAYER_FLOAT32) BY_DRIVE(LAUNCH, float, 1)          \
    else if (lane_of(s) == 2) BY_DRIVE(LAUNCH, bf16, 2)                 \
    else BY_DRIVE(LAUNCH, bf16, 1)

}  // namespace
}  // namespace slayer

using namespace slayer;

extern "C" int64_t slayer_gated_leak_starts(const slayer_gated_leak* s) {
    if (int e = check_leak(s)) return e;
    return s->samples * (s->tokens > 0 ? ceil_div(s->tokens, kKept) : 1) * s->channels;
}

extern "C" int64_t slayer_gated_leak_workspace(const slayer_gated_leak* s, int backward) {
    if (int e = check_leak(s)) return e;
    return floats_of(plan_of(s, backward), backward);
}

extern "C" int slayer_gated_leak_fwd(void* out, float* last, float* starts, const void* input, const void* gate, const float* state,
                                     const slayer_gated_leak* s, float* workspace, int64_t floats, void* stream) {
    if (int e = check_leak(s)) return e;
    if (s->samples == 0) return 0;
    if (s->tokens > 0 && (!out || !input || !gate)) return SLAYER_ENULL;
    const Plan p = plan_of(s, false);
    const int64_t need = floats_of(p, false);
    if (need > 0 && !workspace) return SLAYER_ENULL;
    if (floats < need || (uintptr_t)workspace % 8 != 0) return SLAYER_EINVAL;
    LeakArgs a = args_of(s, p);
    a.out = out; a.last = last; a.starts = starts; a.in = input; a.gate = gate; a.state = state;
    Chains k = {};
    if (int e = chains_of(&k, p, workspace, (hipStream_t)stream)) return e;
#define ONE(DRIVE, T, V, LOOK) \
    hipLaunchKernelGGL((leak_fwd_kernel<T, V, DRIVE, tokens_of(V, false), kWaves, LOOK>), dim3((unsigned)p.blocks), dim3(64 * kWaves), 0, (hipStream_t)stream, a, k)
#define LAUNCH(DRIVE, T, V)                    \
    if (p.look) ONE(DRIVE, T, V, true);        \
    else ONE(DRIVE, T, V, false)
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
    const Plan p = plan_of(s, true);
    const int64_t need = floats_of(p, grad_decay);
    if (need > 0 && !workspace) return SLAYER_ENULL;
    if (floats < need || (uintptr_t)workspace % 8 != 0) return SLAYER_EINVAL;
    LeakArgs a = args_of(s, p);
    a.grad_in = grad_input; a.grad_gate = grad_gate; a.grad_state = grad_state; a.grad = grad_out; a.grad_last = grad_last;
    a.in = input; a.gate = gate; a.starts = (float*)starts;
    a.parts = grad_decay ? workspace + 2 * p.words : nullptr;
    Chains k = {};
    if (int e = chains_of(&k, p, workspace, (hipStream_t)stream)) return e;
#define ONE(DRIVE, T, V, LOOK) \
    hipLaunchKernelGGL((leak_bwd_kernel<T, V, DRIVE, tokens_of(V, true), kWaves, LOOK>), dim3((unsigned)p.blocks), dim3(64 * kWaves), 0, (hipStream_t)stream, a, k)
#define LAUNCH(DRIVE, T, V)                    \
    if (p.look) ONE(DRIVE, T, V, true);        \
    else ONE(DRIVE, T, V, false)
    BY_TYPE(LAUNCH)
#undef LAUNCH
#undef ONE
    if (int e = (int)hipGetLastError()) return e;
    if (!grad_decay) return 0;
    ColumnSums sums = {};
    sums.out[0] = grad_decay; sums.parts[0] = a.parts; sums.factor = 1.f / 4096.f;
    sums.columns = sums.pitch = p.columns;
    sums.rows = p.rows;
    return launch_column_sums(sums, 1, (hipStream_t)stream);
}

extern "C" int slayer_gated_leak_step(void* out, float* state, const void* input, const void* gate, const slayer_gated_leak* s,
                                      void* stream) {
    if (int e = check_leak(s)) return e;
    if (s->samples == 0) return 0;
    if (!out || !state || !input || !gate) return SLAYER_ENULL;
    LeakArgs a = args_of(s, plan_of(s, false));
    a.out = out; a.last = state; a.in = input; a.gate = gate;
    const int quads = (a.channels + 3) / 4;
    const int64_t blocks = (a.samples * quads + 255) / 256;
    if (blocks > (1 << 23)) return SLAYER_ERANGE;
#define LAUNCH(DRIVE, T, V) \
    hipLaunchKernelGGL((leak_step_kernel<T, DRIVE>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a, quads)
    BY_TYPE(LAUNCH)
#undef LAUNCH
    return (int)hipGetLastError();
}

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
#include "attention_pass.h"

namespace slayer {

// starts[unit][seg], which holds what the segment in front of it adds, becomes the state in front of segment seg; the same for its
// derivative: W' = a^L W + L a^(L-1) S + what the segment of L tokens adds.
__global__ __launch_bounds__(256) void leaky_join_kernel(LeakyPass a) {
    const int64_t size = (int64_t)a.keys * a.values;
    const int64_t per = (size + 255) / 256;
    const int64_t unit = blockIdx.x / per, at = blockIdx.x % per * 256 + threadIdx.x;
    if (at >= size) return;
    const int n = (int)(unit / a.heads), h = (int)(unit % a.heads), length = sample_length(a, n);
    const double step = power(1.0 - (double)a.decay[a.one_decay ? 0 : h] / 4096.0, a.segment);
    const float hi = (float)step, lo = (float)(step - (double)hi);
    const float step_slope = a.slope_starts ? (float)(a.segment * power(1.0 - (double)a.decay[a.one_decay ? 0 : h] / 4096.0, a.segment - 1)) : 0.f;
    float s = a.first ? a.first[unit * size + at] : 0.f, w = 0;
    float* starts = a.starts + unit * a.segments * size + at;
    float* slope_starts = a.slope_starts ? a.slope_starts + unit * a.segments * size + at : nullptr;
    constexpr int kAhead = 8;                                // segments whose states are on their way at once
    for (int seg0 = 1; seg0 < a.segments && (int64_t)seg0 * a.segment <= length; seg0 += kAhead) {
        float add[kAhead], slope_add[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int seg = seg0 + i;
            const bool on = seg < a.segments && (int64_t)seg * a.segment <= length;
            add[i] = on ? starts[seg * size] : 0.f;
            slope_add[i] = on && slope_starts ? slope_starts[seg * size] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int seg = seg0 + i;
            w = fmaf(w, hi, fmaf(s, step_slope, slope_add[i]));
            s = fmaf(s, hi, fmaf(s, lo, add[i]));
            if (seg < a.segments && (int64_t)seg * a.segment <= length) {
                starts[seg * size] = s;
                if (slope_starts) slope_starts[seg * size] = w;
            }
        }
    }
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
// quads of values and all keys of one head; 256 / QP rows of keys at a time, so that neighbouring lanes have neighbouring quads of a row
// and a result is a sum over a few rows in LDS.  Bound: memory.  256 samples, 16 heads of 128 x 128, bfloat16: 541 MB in 99 us, 5.5 TB/s, more than
// a copy reaches; one sample of 8 heads of 64 x 64: 4.0 us, a launch.
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

// A segment's workgroup adds up the states of up to so many segments itself ([32,1500,4,64] float32, forward: 86 us, 95 with the
// launch that joins them).
constexpr int kJoin = 8;

// Sixteens of values in a slice of up to 64: wide slices, whose scores are worked out once for all of them.
int slice_tiles(int64_t values) {
    const int64_t slices = ceil_div(values, 64);
    return ceil_div(ceil_div(values, slices), 16);
}

// Segments of a pass: up to 512 workgroups, two a compute unit, from two chunks each on.  Keys and values are then read a second time
// for the states in front of them: [8,1000,4,64] float32, forward, 42 us with segments of four chunks, 32 with two; seven chunks
// and fewer are faster in one piece ([4,256,16,64] float32: 20 us, 23 in two).  The same for every pass of a call.
int segment_tokens(const slayer_attention* a) {
    const int64_t chunks = a->tokens > 0 ? ceil_div(a->tokens, kChunk) : 1;
    const int64_t units = a->samples * a->heads * ceil_div(a->keys > a->values ? a->keys : a->values, 64);
    int64_t segments = units > 0 && chunks >= 8 ? 512 / units : 1;
    if (segments > chunks / 2) segments = chunks / 2;
    if (segments < 1) segments = 1;
    return ceil_div(chunks, segments) * kChunk;
}
int segments_of(const slayer_attention* a) { return a->tokens > 0 ? ceil_div(a->tokens, segment_tokens(a)) : 1; }

// ... and narrower slices where the workgroups leave most of the chip idle.
int tiles_of(const slayer_attention* a, int64_t values, bool whole) {
    int tiles = slice_tiles(values);
    if (!whole) return tiles <= 2 ? 2 : 4;
    while (tiles > 1 && a->samples * a->heads * segments_of(a) * ceil_div(values, 16 * tiles) <= 64) tiles /= 2;
    return tiles;
}

// aligned: every row that starts at `p` with these strides is a multiple of `bytes`
bool aligned(const void* p, const int64_t (&stride)[3], int size, int bytes) {
    return ((uintptr_t)p | (uintptr_t)(stride[0] * size) | (uintptr_t)(stride[1] * size) | (uintptr_t)(stride[2] * size)) % bytes == 0;
}

struct Place { const void* p; const int64_t (&stride)[3]; };
// 16-byte accesses to all rows of the three tensors, and a chunk of each within the reach of a 32-bit offset
bool whole_rows(const slayer_attention* a, const Place& query, const Place& key, const Place& value, int keys, int values) {
    const int size = a->dtype == SLAYER_FLOAT32 ? 4 : 2, vec = 16 / size;
    return keys % vec == 0 && values % vec == 0 && aligned(query.p, query.stride, size, 16) && aligned(key.p, key.stride, size, 16) &&
           aligned(value.p, value.stride, size, 16) &&
           query.stride[1] + key.stride[1] + value.stride[1] < ((int64_t)1 << 31) / (kChunk * size) - 256;
}
int slices_of(const slayer_attention* a, const Place& query, const Place& key, const Place& value, int keys, int values) {
    return ceil_div(values, tiles_of(a, values, whole_rows(a, query, key, value, keys, values)) * 16);
}
struct Both { void* out; const int64_t (&out_stride)[3]; Place query; };
struct Slope { double* slopes; const float* grad_last; Place other; float* starts; };

// One pass with its segments: states in front of them, joined, unless they are there already (`ready`), and the main kernel.
int run_pass(const slayer_attention* a, void* out, const int64_t (&out_stride)[3], Place query, Place key, Place value, int keys,
             int values, bool transposed, bool backwards, const float* first, float* last, const Slope* slope, const Both* both, float* starts,
             bool ready, hipStream_t stream) {
    const bool f32 = a->dtype == SLAYER_FLOAT32;
    const int size = f32 ? 4 : 2;
    const bool whole = whole_rows(a, query, key, value, keys, values);
    LeakyPass p = {};
    p.out = out;
    p.query = query.p; p.key = key.p; p.value = value.p;
    p.decay = a->decay;
    p.lengths = a->lengths;
    p.first = first;
    p.starts = starts;
    p.last = last;
    p.out_n = out_stride[0]; p.out_t = out_stride[1]; p.out_h = out_stride[2];
    p.query_n = query.stride[0]; p.query_t = query.stride[1]; p.query_h = query.stride[2];
    p.key_n = key.stride[0]; p.key_t = key.stride[1]; p.key_h = key.stride[2];
    p.value_n = value.stride[0]; p.value_t = value.stride[1]; p.value_h = value.stride[2];
    p.tokens = (int)a->tokens; p.heads = (int)a->heads; p.keys = keys; p.values = values;
    p.units = (int)(a->samples * a->heads);
    p.state_k = transposed ? 1 : values;
    p.state_v = transposed ? keys : 1;
    p.one_decay = a->num_decays == 1;
    p.lengths64 = a->lengths_bytes == 8;
    p.tiles = both ? (values <= 32 ? 2 : 4) : tiles_of(a, values, whole);
    p.slices = ceil_div(values, p.tiles * 16);
    p.segment = segment_tokens(a);
    p.segments = segments_of(a);
    p.joined = p.segments > kJoin;
    p.backwards = backwards;
    p.whole_out = values % 4 == 0 && aligned(out, out_stride, size, 4 * size) && out_stride[1] < ((int64_t)1 << 31) / (kChunk * size) - 256;
    p.score_scale = (float)a->scale;
    p.state_scale = backwards ? 1.f : (float)a->scale;    // backwards the state it starts from is not scaled, but what is added to it
    p.key_scale = backwards ? (float)a->scale : 1.f;
    if (both) {
        p.out2 = both->out;
        p.query2 = both->query.p;
        p.query2_n = both->query.stride[0]; p.query2_t = both->query.stride[1]; p.query2_h = both->query.stride[2];
        p.out2_n = both->out_stride[0]; p.out2_t = both->out_stride[1]; p.out2_h = both->out_stride[2];
        p.whole_out2 = keys % 4 == 0 && aligned(both->out, both->out_stride, size, 4 * size) &&
                       both->out_stride[1] < ((int64_t)1 << 31) / (kChunk * size) - 256;
    }
    if (slope) {
        p.slope_starts = slope->starts;
        p.grad_last = slope->grad_last;
        p.other = slope->other.p;
        p.other_n = slope->other.stride[0]; p.other_t = slope->other.stride[1]; p.other_h = slope->other.stride[2];
        p.slopes = slope->slopes;
        p.whole_other = values % 4 == 0 && aligned(p.other, slope->other.stride, size, 4 * size) &&
                        p.other_t < ((int64_t)1 << 31) / (kChunk * size) - 256;
    }
    auto launch = [&](int mode) { return f32 ? launch_leaky<float>(p, mode, whole, stream) : launch_leaky<bf16>(p, mode, whole, stream); };
    if (p.segments > 1 && !ready) {
        if (int e = launch(slope ? LEAKY_STATE_SLOPE : LEAKY_STATE)) return e;
    }
    if (p.joined && !ready) {
        const int64_t blocks = (int64_t)p.units * ceil_div((int64_t)keys * values, 256);
        if (blocks > (1 << 24) - 1) return SLAYER_ERANGE;
        hipLaunchKernelGGL(leaky_join_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p);
        if (int e = (int)hipGetLastError()) return e;
    }
    return launch(slope ? LEAKY_SLOPE : both ? LEAKY_BOTH : LEAKY_MAIN);
}

// Floats of the states in front of the segments.
int64_t starts_floats(const slayer_attention* a) {
    const int64_t segments = segments_of(a);
    return segments > 1 ? a->samples * a->heads * segments * a->keys * a->values : 0;
}
// Doubles of the slopes of all workgroups: at most eight slices of values each.
int64_t slope_count(const slayer_attention* a) { return a->samples * a->heads * segments_of(a) * 8; }

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

// [samples][tokens][heads][width] as it lies in a new tensor
struct Contiguous {
    int64_t stride[3];
    Contiguous(const slayer_attention* a, int64_t width) : stride{a->tokens * a->heads * width, a->heads * width, width} {}
};

}  // namespace

extern "C" int64_t slayer_leaky_attention_workspace(const slayer_attention* a, int backward) {
    if (int e = check_leaky(a)) return e;
    return backward ? 2 * slope_count(a) + 2 * starts_floats(a) : starts_floats(a);
}

extern "C" int slayer_leaky_attention_fwd(void* out, float* last, const void* query, const void* key, const void* value, const float* state,
                                          const slayer_attention* a, float* workspace, int64_t floats, void* stream) {
    if (int e = check_leaky(a)) return e;
    if (a->samples == 0) return 0;
    if (a->tokens > 0 && (!out || !query || !key || !value)) return SLAYER_ENULL;
    const int64_t need = starts_floats(a);
    if (need > 0 && !workspace) return SLAYER_ENULL;
    if (floats < need) return SLAYER_EINVAL;
    const Contiguous o(a, a->values);
    return run_pass(a, out, o.stride, {query, a->query_stride}, {key, a->key_stride}, {value, a->value_stride}, (int)a->keys, (int)a->values,
                    false, false, state, last, nullptr, nullptr, workspace, false, (hipStream_t)stream);
}

extern "C" int slayer_leaky_attention_bwd(void* grad_query, void* grad_key, void* grad_value, float* grad_decay, float* grad_state,
                                          const void* grad_out, const float* grad_last, const void* query, const void* key, const void* value,
                                          const float* state, const float* starts, const slayer_attention* a, float* workspace, int64_t floats,
                                          void* stream) {
    if (int e = check_leaky(a)) return e;
    hipStream_t s = (hipStream_t)stream;
    if (a->samples == 0) return grad_decay ? launch_zero_fill(grad_decay, a->num_decays, s) : 0;
    if (a->tokens > 0 && (!grad_out || !query || !key || !value)) return SLAYER_ENULL;
    if (!workspace || (a->tokens > 0 && ((grad_state && !grad_value) || (grad_decay && !grad_query)))) return SLAYER_ENULL;
    if (floats < slayer_leaky_attention_workspace(a, 1)) return SLAYER_EINVAL;
    const int K = (int)a->keys, V = (int)a->values;
    const Contiguous k(a, K), v(a, V);
    float *space = workspace + 2 * slope_count(a), *slope_starts = space + starts_floats(a);
    const Place q{query, a->query_stride}, kk{key, a->key_stride}, vv{value, a->value_stride}, g{grad_out, a->grad_stride};
    const Slope slope{(double*)workspace, grad_last, q, slope_starts};
    if (grad_query || grad_decay) {                          // (with no tokens there may be no tensors either)
        const bool ready = starts && !grad_decay;            // the states of the forward call are those of this pass
        if (int e = run_pass(a, grad_query, k.stride, g, vv, kk, V, K, true, false, state, nullptr, grad_decay ? &slope : nullptr, nullptr,
                             ready ? const_cast<float*>(starts) : space, ready, s)) return e;
        if (grad_decay) {
            const int parts = segments_of(a) * slices_of(a, g, vv, kk, V, K);
            hipLaunchKernelGGL(leaky_decay_kernel, dim3((unsigned)a->num_decays), dim3(256), 0, s, grad_decay, slope.slopes, (int)a->samples,
                               (int)a->heads, (int)(a->num_decays == 1), parts);
            if (int e = (int)hipGetLastError()) return e;
        }
    }
    // value's and key's gradients in one pass where a workgroup holds a whole head, up to 96 by 64; in narrow slices, whose chunks take
    // less time, where there are few of them.  The narrower side is the pass's value.  Two passes / one, us, float32 and bfloat16:
    // [32,1500,4,64] 165 / 132, 89 / 66; 96 keys and 64 values 236 / 219, 128 / 108; 80 workgroups, [80,448,1,64], 89 / 71, 46 / 35;
    // 64 of them 65 / 70, 37 / 35; 32 of them 53 / 69, 32 / 34 (with 32 keys and values, 64 of them: 35 / 33, 27 / 20).
    if (grad_value && grad_key && (K < V ? K : V) <= 64 && (K < V ? V : K) <= 96 && whole_rows(a, kk, q, g, K, V) &&
        whole_rows(a, vv, g, q, V, K) && a->samples * a->heads * segments_of(a) > 64) {
        if (V <= 64) {
            const Both both{grad_key, k.stride, vv};
            return run_pass(a, grad_value, v.stride, kk, q, g, K, V, false, true, grad_last, grad_state, nullptr, &both, space, false, s);
        }
        const Both both{grad_value, v.stride, kk};
        return run_pass(a, grad_key, k.stride, vv, g, q, V, K, true, true, grad_last, grad_state, nullptr, &both, space, false, s);
    }
    if (grad_value || grad_state)
        if (int e = run_pass(a, grad_value, v.stride, kk, q, g, K, V, false, true, grad_last, grad_state, nullptr, nullptr, space, false, s)) return e;
    if (grad_key) return run_pass(a, grad_key, k.stride, vv, g, q, V, K, true, true, grad_last, nullptr, nullptr, nullptr, space, grad_value != nullptr, s);
    return 0;
}

extern "C" int slayer_leaky_attention_step(void* out, float* state, const void* query, const void* key, const void* value,
                                           const slayer_attention* a, void* stream) {
    if (int e = check_leaky(a)) return e;
    if (a->samples == 0) return 0;
    if (!out || !state || !query || !key || !value) return SLAYER_ENULL;
    return a->dtype == SLAYER_FLOAT32 ? launch_step<float>(out, state, query, key, value, a, (hipStream_t)stream)
                                      : launch_step<bf16>(out, state, query, key, value, a, (hipStream_t)stream);
}

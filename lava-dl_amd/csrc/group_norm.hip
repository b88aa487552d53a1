// Group norm with the channels last and an activation behind it: x is [samples][pixels][channels], a group is channels / groups
// neighbouring channels over all pixels of a sample,
//     hat = (x - mean) / sqrt(var + eps),   z = hat * weight + bias,   y = act(z).
// Backwards, with dz = dy act'(z), d = dz * weight and means over the group:
//     dx = (d - mean(d) - hat * mean(d * hat)) / sqrt(var + eps),   dweight = sum of dz * hat,   dbias = sum of dz.
// Two forms.  Rows (one pixel a sample, groups of up to 64 * 8 accesses of 16 bytes): a group lies in one piece and in the
// registers of up to 64 lanes, so every tensor is read or written once.  Pixels: a group reaches over many rows, so statistics
// come first, for each channel and piece of the image, are joined, and a second kernel applies them.
//   Rows, 48000 tokens of 256 channels in 4 groups, bfloat16: forward 14 to 15 us (3.2 to 3.5 TB/s), backward 20 (3.8 TB/s), 5 for the sums of the
// weights' gradients.  The first form, whose threads looked up their channels anew for each row and whose activations divided in full
// precision, took 51, 29 and 21.  Pixels, [32,1024,512] float32: statistics 15 us, joining 5, applying 23 (5.7 TB/s); backward 26, 5 and 33 (6.1 TB/s): the
// second reading comes partly from the last-level cache.  Rows of more than 2048 bfloat16 channels a group take up to 512 registers backwards,
// with ReLU some scratch memory.
#include "common.h"
#include "elements.h"

namespace slayer {

enum { ACT_NONE, ACT_RELU, ACT_SILU, ACT_GELU };

template <typename T, int ACT> __device__ __forceinline__ float activate(float z) {
    if (ACT == ACT_RELU) return z > 0.f || z != z ? z : 0.f;
    if (ACT == ACT_SILU) return z * logistic<T>(z);
    if (ACT == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    return z;
}
template <typename T, int ACT> __device__ __forceinline__ float slope(float z) {
    if (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == ACT_SILU) {
        const float s = logistic<T>(z);
        return s * fmaf(z, 1.f - s, 1.f);
    }
    if (ACT == ACT_GELU) return fmaf(z, 0.39894228040143268f * expf(-0.5f * z * z), 0.5f * (1.f + erff(z * 0.70710678118654752f)));
    return 1.f;
}

struct NormArgs {
    void* out;                       // y, or dx
    const void *in, *grad;           // x, dy
    const float *weight, *bias;      // or nullptr: 1, 0
    float *mean, *scale;             // [samples * groups]: mean and 1 / sqrt(var + eps)
    float* work;
    int64_t samples, pixels;
    int channels, groups, width;     // width = channels / groups
    int whole, whole_rows;           // 16-byte accesses to a channel row, to a group's row
    int whole_params;                // ... to weight and bias
    int lanes, splits, tiles;        // lanes of a row; pieces of an image, tiles of channels
    float eps;
};

// weight and bias of the first `n` of V channels
template <int V>
__device__ __forceinline__ void load_params(float (&w)[V], float (&b)[V], const NormArgs& a, int c, int n) {
    const bool whole = n >= V && a.whole_params && c % 4 == 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        w[e] = 1.f;
        b[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < V; e += 4) {
        if (whole) {
            if (a.weight) {
                const f4 v = *reinterpret_cast<const f4*>(a.weight + c + e);
                w[e] = v[0]; w[e + 1] = v[1]; w[e + 2] = v[2]; w[e + 3] = v[3];
            }
            if (a.bias) {
                const f4 v = *reinterpret_cast<const f4*>(a.bias + c + e);
                b[e] = v[0]; b[e + 1] = v[1]; b[e + 2] = v[2]; b[e + 3] = v[3];
            }
        } else {
#pragma unroll
            for (int i = e; i < e + 4; ++i) {
                if (a.weight && i < n) w[i] = a.weight[c + i];
                if (a.bias && i < n) b[i] = a.bias[c + i];
            }
        }
    }
}

// ---- rows ---------------------------------------------------------------------------------------------------------------------
// The rows a workgroup takes at a time (`per`), or those of all workgroups together, are a multiple of the groups, so a thread stays
// with its channels.
template <typename T, int ACT, int IT>
__global__ __launch_bounds__(256) void norm_rows_kernel(NormArgs a, int per) {
    constexpr int V = Elements<T>::kVec;
    const int lane = threadIdx.x % a.lanes, sub = threadIdx.x / a.lanes;
    const int64_t rows = a.samples * a.groups;
    const float inv = 1.f / (float)a.width;
    const int c = (int)((blockIdx.x * (unsigned)per + sub) % (unsigned)a.groups) * a.width;
    float w[IT][V], b[IT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int at = (i * a.lanes + lane) * V, left = a.width - at;
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][e] = b[i][e] = 0;
        if (left > 0) load_params(w[i], b[i], a, c + at, left < V ? left : V);
    }
    if (sub >= per) return;
    for (int64_t row = (int64_t)blockIdx.x * per + sub; row < rows; row += (int64_t)gridDim.x * per) {
        const T* in = (const T*)a.in + row * a.width;
        float x[IT][V], sum = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * a.lanes + lane) * V;
            to_floats(x[i], load_vec(in + at, a.width - at, a.whole_rows));
#pragma unroll
            for (int e = 0; e < V; ++e) sum += x[i][e];
        }
        const float mean = sum_lanes(sum, a.lanes) * inv;
        float square = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = x[i][e] - mean;
                square = (i * a.lanes + lane) * V + e < a.width ? fmaf(d, d, square) : square;
            }
        const float scale = 1.f / sqrtf(sum_lanes(square, a.lanes) * inv + a.eps);
        if (a.mean && lane == 0) {
            a.mean[row] = mean;
            a.scale[row] = scale;
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int at = (i * a.lanes + lane) * V, left = a.width - at;
            if (left <= 0) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) x[i][e] = activate<T, ACT>(fmaf((x[i][e] - mean) * scale, w[i][e], b[i][e]));
            store_vec((T*)a.out + row * a.width + at, from_floats(x[i]), left, a.whole_rows);
        }
    }
}

// dx, and this workgroup's part of the sums over the rows: work[slot][2][width], slot % groups = the group.
//   shared: the rows of a workgroup that have the same channels are summed in LDS first.
template <typename T, int ACT, int IT>
__global__ __launch_bounds__(256) void norm_rows_bwd_kernel(NormArgs a, int per, bool shared) {
    constexpr int V = Elements<T>::kVec;
    extern __shared__ float parts[];                              // [per][2][width] where `shared`
    const int lane = threadIdx.x % a.lanes, sub = threadIdx.x / a.lanes;
    const int64_t rows = a.samples * a.groups;
    const float inv = 1.f / (float)a.width;
    const int c = (int)((blockIdx.x * (unsigned)per + sub) % (unsigned)a.groups) * a.width;
    float w[IT][V], b[IT][V], dw[IT][V], db[IT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int at = (i * a.lanes + lane) * V, left = a.width - at;
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][e] = b[i][e] = dw[i][e] = db[i][e] = 0;
        if (left > 0) load_params(w[i], b[i], a, c + at, left < V ? left : V);
    }
    if (sub < per) {
        for (int64_t row = (int64_t)blockIdx.x * per + sub; row < rows; row += (int64_t)gridDim.x * per) {
            const float mean = a.mean[row], scale = a.scale[row];
            float x[IT][V], d[IT][V], s1 = 0, s2 = 0;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int at = (i * a.lanes + lane) * V;
                to_floats(x[i], load_vec((const T*)a.in + row * a.width + at, a.width - at, a.whole_rows));
                to_floats(d[i], load_vec((const T*)a.grad + row * a.width + at, a.width - at, a.whole_rows));
            }
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const bool on = (i * a.lanes + lane) * V + e < a.width;
                    x[i][e] = on ? (x[i][e] - mean) * scale : 0.f;
                    d[i][e] = on ? d[i][e] * slope<T, ACT>(fmaf(x[i][e], w[i][e], b[i][e])) : 0.f;
                    dw[i][e] = fmaf(d[i][e], x[i][e], dw[i][e]);
                    db[i][e] += d[i][e];
                    d[i][e] *= w[i][e];
                    s1 += d[i][e];
                    s2 = fmaf(d[i][e], x[i][e], s2);
                }
            s1 = sum_lanes(s1, a.lanes) * inv;
            s2 = sum_lanes(s2, a.lanes) * inv;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int at = (i * a.lanes + lane) * V;
#pragma unroll
                for (int e = 0; e < V; ++e) x[i][e] = scale * (d[i][e] - s1 - x[i][e] * s2);
                store_vec((T*)a.out + row * a.width + at, from_floats(x[i]), a.width - at, a.whole_rows);
            }
        }
    }
    if (!a.work) return;
    float* to = shared ? parts + sub * 2 * a.width : a.work + ((int64_t)blockIdx.x * per + sub) * 2 * a.width;
    if (sub < per) {
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int at = (i * a.lanes + lane) * V + e;
                if (at < a.width) {
                    to[at] = dw[i][e];
                    to[a.width + at] = db[i][e];
                }
            }
    }
    if (!shared) return;
    __syncthreads();
    for (int at = threadIdx.x; at < a.groups * 2 * a.width; at += 256) {       // [group][2][width]
        float sum = 0;
        for (int r = 0; r < per; r += a.groups) sum += parts[(int64_t)r * 2 * a.width + at];
        a.work[(int64_t)blockIdx.x * a.groups * 2 * a.width + at] = sum;
    }
}

// dweight and dbias: the sum over the slots of a group.  Sixteen channels and 64 shares of the slots a workgroup.
__global__ __launch_bounds__(1024) void norm_rows_sum_kernel(float* __restrict__ dweight, float* __restrict__ dbias,
                                                             const float* __restrict__ work, int64_t slots, int groups, int width) {
    __shared__ float sums[64][33];
    const int i = threadIdx.x % 16, share = threadIdx.x / 16, c = blockIdx.x * 16 + i, channels = groups * width;
    float w = 0, b = 0;
    if (c < channels) {
#pragma unroll 8
        for (int64_t slot = c / width + (int64_t)share * groups; slot < slots; slot += 64 * groups) {
            w += work[slot * 2 * width + c % width];
            b += work[slot * 2 * width + width + c % width];
        }
    }
    sums[share][i] = w;
    sums[share][16 + i] = b;
    __syncthreads();
    if (threadIdx.x < 512) {                                     // 32 sums, sixteen lanes each
        const int which = threadIdx.x / 16;
        float sum = (sums[i][which] + sums[i + 16][which]) + (sums[i + 32][which] + sums[i + 48][which]);
        sum = sum_lanes(sum, 16);
        const int channel = blockIdx.x * 16 + which % 16;
        float* to = which < 16 ? dweight : dbias;
        if (i == 0 && channel < channels && to) to[channel] = sum;
    }
}

// ---- pixels -------------------------------------------------------------------------------------------------------------------
// A workgroup takes one piece of one image and one tile of channels: `lanes` accesses of 16 bytes, 256 / lanes pixels at a time.
struct Piece {
    int64_t n, p0, p1;
    int split, c, left, row, rows;     // first channel of the thread, its channels, its pixel among `rows`
};
template <int V>
__device__ __forceinline__ Piece piece_of(const NormArgs& a) {
    Piece p;
    int64_t b = blockIdx.x;
    const int tile = (int)(b % a.tiles); b /= a.tiles;
    p.split = (int)(b % a.splits);
    p.n = b / a.splits;
    const int64_t per = (a.pixels + a.splits - 1) / a.splits;
    p.p0 = p.split * per;
    p.p1 = p.p0 + per < a.pixels ? p.p0 + per : a.pixels;
    p.c = (tile * a.lanes + threadIdx.x % a.lanes) * V;
    p.left = a.channels - p.c;
    p.row = threadIdx.x / a.lanes;
    p.rows = 256 / a.lanes;
    return p;
}
// Sums over the pixels of a workgroup, for each of its channels, into work[sample][split][channels][2].
template <int V>
__device__ __forceinline__ void store_sums(float* work, const float (&s1)[V], const float (&s2)[V], const NormArgs& a, const Piece& p) {
    __shared__ float sums[256][2 * V + 1];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        sums[threadIdx.x][2 * e] = s1[e];
        sums[threadIdx.x][2 * e + 1] = s2[e];
    }
    __syncthreads();
    const int base = p.c - (int)(threadIdx.x % a.lanes) * V;
    for (int at = threadIdx.x; at < a.lanes * V * 2; at += 256) {
        const int c = at / 2;
        if (base + c >= a.channels) break;
        float sum = 0;
        for (int r = 0; r < p.rows; ++r) sum += sums[r * a.lanes + c / V][c % V * 2 + at % 2];
        work[((p.n * a.splits + p.split) * a.channels + base) * 2 + at] = sum;
    }
}

// Mean and sum of squares about it, for each channel and piece.  Every mean is that of the values so far, in a thread (Welford, Note on
// a Method for Calculating Corrected Sums of Squares and Products, 1962), and what is joined are squares about means and squares of
// their distances: terms that are not negative, so nothing cancels, wherever the mean lies and whatever a single pixel holds.  What the
// distances leave when they are added up corrects a joined mean, which is rounded where it is large.
template <typename T>
__global__ __launch_bounds__(256) void norm_stats_kernel(NormArgs a) {
    constexpr int V = Elements<T>::kVec;
    __shared__ float parts[256][2 * V + 1];
    const Piece p = piece_of<V>(a);
    const T* in = (const T*)a.in + p.n * a.pixels * a.channels + p.c;
    float mean[V], square[V], count = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) mean[e] = square[e] = 0;
    if (p.left > 0)
        for (int64_t q = p.p0 + p.row; q < p.p1; q += p.rows) {
            float x[V];
            to_floats(x, load_vec(in + q * a.channels, p.left, a.whole));
            count += 1.f;
            const float inv = __builtin_amdgcn_rcpf(count);     // within a unit in the last place, of what the mean moves by
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = x[e] - mean[e];
                mean[e] = fmaf(d, inv, mean[e]);
                square[e] = fmaf(d, x[e] - mean[e], square[e]);
            }
        }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        parts[threadIdx.x][2 * e] = mean[e];
        parts[threadIdx.x][2 * e + 1] = square[e];
    }
    __syncthreads();
    const int base = p.c - (int)(threadIdx.x % a.lanes) * V;
    const int64_t all = p.p1 > p.p0 ? p.p1 - p.p0 : 0;
    const float inv = all > 0 ? 1.f / (float)all : 0.f;
    const float few = (float)(all / p.rows);                    // pixels of a row of threads; the first `more` have one more
    const int more = (int)(all % p.rows);
    for (int c = threadIdx.x; c < a.lanes * V && base + c < a.channels; c += 256) {
        auto pixels_of = [&](int row) { return row < more ? few + 1.f : few; };
        auto part = [&](int row, int which) { return parts[row * a.lanes + c / V][c % V * 2 + which]; };
        float m = 0, off = 0, sq = 0;
        for (int r = 0; r < p.rows; ++r) m = fmaf(pixels_of(r), part(r, 0), m);
        m *= inv;
        for (int r = 0; r < p.rows; ++r) {
            const float d = part(r, 0) - m;
            off = fmaf(pixels_of(r), d, off);
            sq += fmaf(pixels_of(r) * d, d, part(r, 1));
        }
        float* to = a.work + ((p.n * a.splits + p.split) * a.channels + base + c) * 2;
        to[0] = fmaf(off, inv, m);
        to[1] = sq;
    }
}

__device__ __forceinline__ float sum_block(float v, float* shared) {            // of 256 threads
    v = sum_lanes(v, 64);
    __syncthreads();
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
    __syncthreads();
    return (shared[0] + shared[1]) + (shared[2] + shared[3]);
}

// mean and scale of a group from those of its channels and pieces
__global__ __launch_bounds__(256) void norm_join_kernel(NormArgs a) {
    __shared__ float shared[4];
    const int64_t n = blockIdx.x / a.groups, per = (a.pixels + a.splits - 1) / a.splits;
    const int c0 = (int)(blockIdx.x % a.groups) * a.width, count = a.width * a.splits;
    const float* work = a.work + (n * a.splits * a.channels + c0) * 2;
    const float inv = 1.f / ((float)a.pixels * (float)a.width);
    auto pixels_of = [&](int split) {
        const int64_t left = a.pixels - split * per;
        return (float)(left < per ? (left > 0 ? left : 0) : per);
    };
    float sum = 0;
    for (int i = threadIdx.x; i < count; i += 256)
        sum = fmaf(pixels_of(i / a.width), work[((int64_t)(i / a.width) * a.channels + i % a.width) * 2], sum);
    const float mean = sum_block(sum, shared) * inv;
    float off = 0, square = 0;
    for (int i = threadIdx.x; i < count; i += 256) {
        const float* part = work + ((int64_t)(i / a.width) * a.channels + i % a.width) * 2;
        const float d = part[0] - mean;
        off = fmaf(pixels_of(i / a.width), d, off);
        square += fmaf(pixels_of(i / a.width) * d, d, part[1]);
    }
    off = sum_block(off, shared) * inv;
    const float var = sum_block(square, shared) * inv;
    if (threadIdx.x == 0) {
        a.mean[blockIdx.x] = mean + off;
        a.scale[blockIdx.x] = 1.f / sqrtf(var + a.eps);
    }
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void norm_apply_kernel(NormArgs a) {
    constexpr int V = Elements<T>::kVec;
    const Piece p = piece_of<V>(a);
    if (p.left <= 0) return;
    const T* in = (const T*)a.in + p.n * a.pixels * a.channels + p.c;
    T* out = (T*)a.out + p.n * a.pixels * a.channels + p.c;
    float w[V], b[V], mean[V], scale[V];
    load_params(w, b, a, p.c, p.left < V ? p.left : V);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int64_t g = p.n * a.groups + (e < p.left ? (p.c + e) / a.width : 0);
        mean[e] = a.mean[g];
        scale[e] = a.scale[g];
    }
    for (int64_t q = p.p0 + p.row; q < p.p1; q += p.rows) {
        float x[V];
        to_floats(x, load_vec(in + q * a.channels, p.left, a.whole));
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = activate<T, ACT>(fmaf((x[e] - mean[e]) * scale[e], w[e], b[e]));
        store_vec(out + q * a.channels, from_floats(x), p.left, a.whole);
    }
}

// Sums of dz and dz * hat
template <typename T, int ACT>
__global__ __launch_bounds__(256) void norm_bwd_stats_kernel(NormArgs a) {
    constexpr int V = Elements<T>::kVec;
    const Piece p = piece_of<V>(a);
    const int64_t at = p.n * a.pixels * a.channels + p.c;
    float w[V], b[V], mean[V], scale[V], s1[V], s2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int64_t g = p.n * a.groups + (e < p.left ? (p.c + e) / a.width : 0);
        mean[e] = a.mean[g];
        scale[e] = a.scale[g];
        w[e] = b[e] = s1[e] = s2[e] = 0;
    }
    if (p.left > 0) {
        load_params(w, b, a, p.c, p.left < V ? p.left : V);
        for (int64_t q = p.p0 + p.row; q < p.p1; q += p.rows) {
            float x[V], d[V];
            to_floats(x, load_vec((const T*)a.in + at + q * a.channels, p.left, a.whole));
            to_floats(d, load_vec((const T*)a.grad + at + q * a.channels, p.left, a.whole));
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float hat = (x[e] - mean[e]) * scale[e];
                d[e] *= slope<T, ACT>(fmaf(hat, w[e], b[e]));
                s1[e] += d[e];
                s2[e] = fmaf(d[e], hat, s2[e]);
            }
        }
    }
    store_sums<V>(a.work, s1, s2, a, p);
}

// Workgroups up to samples * groups: the two means of a group, into `means`.  The others: dweight and dbias of sixteen channels, in
// sixteen shares of the pieces.
__global__ __launch_bounds__(256) void norm_bwd_join_kernel(NormArgs a, float* __restrict__ means, float* __restrict__ dweight,
                                                            float* __restrict__ dbias) {
    __shared__ float shared[4];
    const int64_t units = a.samples * a.groups;
    if (blockIdx.x < units) {
        const int64_t n = blockIdx.x / a.groups;
        const int c0 = (int)(blockIdx.x % a.groups) * a.width;
        const float* work = a.work + (n * a.splits * a.channels + c0) * 2;
        float s1 = 0, s2 = 0;
        for (int i = threadIdx.x; i < a.width * a.splits; i += 256) {
            const int c = i % a.width;
            const float w = a.weight ? a.weight[c0 + c] : 1.f;
            const float* s = work + ((int64_t)(i / a.width) * a.channels + c) * 2;
            s1 = fmaf(w, s[0], s1);
            s2 = fmaf(w, s[1], s2);
        }
        const float size = (float)a.pixels * (float)a.width;
        s1 = sum_block(s1, shared) / size;
        s2 = sum_block(s2, shared) / size;
        if (threadIdx.x == 0) {
            means[2 * blockIdx.x] = s1;
            means[2 * blockIdx.x + 1] = s2;
        }
    } else {
        __shared__ float sums[16][33];
        const int c = (int)(blockIdx.x - units) * 16 + threadIdx.x % 16, share = threadIdx.x / 16;
        float b = 0, w = 0;
        if (c < a.channels) {
#pragma unroll 8
            for (int64_t s = share; s < a.samples * a.splits; s += 16) {
                b += a.work[(s * a.channels + c) * 2];
                w += a.work[(s * a.channels + c) * 2 + 1];
            }
        }
        sums[share][threadIdx.x % 16] = w;
        sums[share][16 + threadIdx.x % 16] = b;
        __syncthreads();
        if (threadIdx.x < 32 && c < a.channels) {
            float sum = 0;
            for (int s = 0; s < 16; ++s) sum += sums[s][threadIdx.x];
            float* to = threadIdx.x < 16 ? dweight : dbias;
            if (to) to[c] = sum;
        }
    }
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void norm_bwd_apply_kernel(NormArgs a, const float* __restrict__ means) {
    constexpr int V = Elements<T>::kVec;
    const Piece p = piece_of<V>(a);
    if (p.left <= 0) return;
    const int64_t at = p.n * a.pixels * a.channels + p.c;
    float w[V], b[V], mean[V], scale[V], m1[V], m2[V];
    load_params(w, b, a, p.c, p.left < V ? p.left : V);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int64_t g = p.n * a.groups + (e < p.left ? (p.c + e) / a.width : 0);
        mean[e] = a.mean[g];
        scale[e] = a.scale[g];
        m1[e] = means[2 * g];
        m2[e] = means[2 * g + 1];
    }
    for (int64_t q = p.p0 + p.row; q < p.p1; q += p.rows) {
        float x[V], d[V];
        to_floats(x, load_vec((const T*)a.in + at + q * a.channels, p.left, a.whole));
        to_floats(d, load_vec((const T*)a.grad + at + q * a.channels, p.left, a.whole));
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float hat = (x[e] - mean[e]) * scale[e];
            d[e] *= slope<T, ACT>(fmaf(hat, w[e], b[e])) * w[e];
            x[e] = scale[e] * (d[e] - m1[e] - hat * m2[e]);
        }
        store_vec((T*)a.out + at + q * a.channels, from_floats(x), p.left, a.whole);
    }
}

}  // namespace slayer

using namespace slayer;

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int pow2_up(int64_t v) {
    int p = 1;
    while (p < v && p < 64) p *= 2;
    return p;
}

// How a tensor is cut, the same for a call and for its workspace.
struct Cut {
    bool rows;
    int lanes, its;            // rows: lanes of a group and accesses of a lane
    int per;                   // rows, backwards: groups a workgroup takes at a time
    int64_t fwd_blocks, blocks, slots;     // rows; backwards
    bool shared;
    int splits, tiles;         // pixels
};
int64_t gcd(int64_t a, int64_t b) { return b ? gcd(b, a % b) : a; }

Cut cut_of(int dtype, int64_t samples, int64_t pixels, int64_t channels, int64_t groups) {
    Cut c = {};
    const int vec = dtype == SLAYER_FLOAT32 ? 4 : 8;
    const int64_t width = channels / groups, vecs = ceil_div(width, vec);
    c.rows = pixels == 1 && vecs <= 64 * 8;
    if (c.rows) {
        c.lanes = pow2_up(vecs);
        const int64_t its = ceil_div(vecs, c.lanes);
        c.its = its <= 1 ? 1 : its <= 2 ? 2 : its <= 4 ? 4 : 8;
        const int64_t most = 256 / c.lanes, rows = samples * groups;
        int64_t multiple = 1;
        if (groups <= most) c.per = (int)(most / groups * groups);
        else {
            c.per = (int)most;
            multiple = groups / gcd(groups, most);
        }
        const int64_t all = ceil_div(rows, c.per);
        c.fwd_blocks = ceil_div(all < 2048 ? all : 2048, multiple) * multiple;
        c.blocks = ceil_div(all < 1024 ? all : 1024, multiple) * multiple;
        c.shared = groups <= most && c.per * 2 * width * 4 <= 65536;
        c.slots = c.blocks * (c.shared ? groups : c.per);
    } else {
        const int64_t all = ceil_div(channels, vec);
        c.lanes = pow2_up(all);
        c.tiles = (int)ceil_div(all, c.lanes);
        int64_t splits = samples * c.tiles > 0 ? 2048 / (samples * c.tiles) : 1;
        const int64_t most = ceil_div(pixels, 4 * (256 / c.lanes));       // four pixels a thread at least
        if (splits > most) splits = most;
        c.splits = splits < 1 ? 1 : (int)splits;
    }
    return c;
}

int check_norm(int dtype, int64_t samples, int64_t pixels, int64_t channels, int64_t groups, int activation) {
    if (samples < 0 || pixels < 0 || channels < 1 || groups < 1 || channels % groups != 0) return SLAYER_EINVAL;
    if (dtype != SLAYER_FLOAT32 && dtype != SLAYER_BFLOAT16) return SLAYER_EINVAL;
    if (activation < ACT_NONE || activation > ACT_GELU) return SLAYER_EINVAL;
    if (channels > (1 << 24) || samples > ((int64_t)1 << 32) || pixels > ((int64_t)1 << 32)) return SLAYER_ERANGE;
    if (pixels > 0 && samples > ((int64_t)1 << 40) / channels / pixels) return SLAYER_ERANGE;
    const bool rows = pixels == 1 && channels / groups <= 64 * 8 * (dtype == SLAYER_FLOAT32 ? 4 : 8);
    if (!rows && samples * groups > (1 << 23)) return SLAYER_ERANGE;       // a workgroup each
    return 0;
}

#define BY_ACT(LAUNCH)                              \
    switch (activation) {                           \
        case ACT_NONE: LAUNCH(ACT_NONE); break;     \
        case ACT_RELU: LAUNCH(ACT_RELU); break;     \
        case ACT_SILU: LAUNCH(ACT_SILU); break;     \
        default: LAUNCH(ACT_GELU); break;           \
    }

NormArgs args_of(void* out, const void* in, const void* grad, const float* weight, const float* bias, float* mean, float* scale, float* work,
                 int dtype, int64_t samples, int64_t pixels, int64_t channels, int64_t groups, float eps, const Cut& c) {
    NormArgs a = {};
    a.out = out; a.in = in; a.grad = grad; a.weight = weight; a.bias = bias; a.mean = mean; a.scale = scale; a.work = work;
    a.samples = samples; a.pixels = pixels;
    a.channels = (int)channels; a.groups = (int)groups; a.width = (int)(channels / groups);
    const int size = dtype == SLAYER_FLOAT32 ? 4 : 2;
    const bool base = ((uintptr_t)out | (uintptr_t)in | (uintptr_t)grad) % 16 == 0;
    a.whole = base && channels * size % 16 == 0;
    a.whole_rows = base && a.width * size % 16 == 0;
    a.whole_params = ((uintptr_t)weight | (uintptr_t)bias) % 16 == 0;
    a.lanes = c.lanes; a.splits = c.splits; a.tiles = c.tiles;
    a.eps = eps;
    return a;
}

template <typename T>
int launch_fwd(const NormArgs& a, const Cut& c, int activation, hipStream_t s) {
    if (c.rows) {
        if (c.fwd_blocks > (1 << 23)) return SLAYER_ERANGE;
#define ONE(ACT, IT) hipLaunchKernelGGL((norm_rows_kernel<T, ACT, IT>), dim3((unsigned)c.fwd_blocks), dim3(256), 0, s, a, c.per)
#define LAUNCH(ACT)                     \
    if (c.its == 1) ONE(ACT, 1);        \
    else if (c.its == 2) ONE(ACT, 2);   \
    else if (c.its == 4) ONE(ACT, 4);   \
    else ONE(ACT, 8)
        BY_ACT(LAUNCH)
#undef LAUNCH
#undef ONE
        return (int)hipGetLastError();
    }
    const int64_t blocks = a.samples * a.splits * a.tiles;
    if (blocks > (1 << 23)) return SLAYER_ERANGE;
    hipLaunchKernelGGL(norm_stats_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, a);
    hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)(a.samples * a.groups)), dim3(256), 0, s, a);
#define LAUNCH(ACT) hipLaunchKernelGGL((norm_apply_kernel<T, ACT>), dim3((unsigned)blocks), dim3(256), 0, s, a)
    BY_ACT(LAUNCH)
#undef LAUNCH
    return (int)hipGetLastError();
}

template <typename T>
int launch_bwd(const NormArgs& a, const Cut& c, int activation, float* dweight, float* dbias, float* means, hipStream_t s) {
    if (c.rows) {
        if (c.blocks > (1 << 23)) return SLAYER_ERANGE;
        const size_t lds = a.work && c.shared ? (size_t)c.per * 2 * a.width * sizeof(float) : 0;
#define ONE(ACT, IT) hipLaunchKernelGGL((norm_rows_bwd_kernel<T, ACT, IT>), dim3((unsigned)c.blocks), dim3(256), lds, s, a, c.per, c.shared)
#define LAUNCH(ACT)                     \
    if (c.its == 1) ONE(ACT, 1);        \
    else if (c.its == 2) ONE(ACT, 2);   \
    else if (c.its == 4) ONE(ACT, 4);   \
    else ONE(ACT, 8)
        BY_ACT(LAUNCH)
#undef LAUNCH
#undef ONE
        if (int e = (int)hipGetLastError()) return e;
        if (!a.work) return 0;
        hipLaunchKernelGGL(norm_rows_sum_kernel, dim3((unsigned)ceil_div(a.channels, 16)), dim3(1024), 0, s, dweight, dbias, a.work, c.slots,
                           a.groups, a.width);
        return (int)hipGetLastError();
    }
    const int64_t blocks = a.samples * a.splits * a.tiles, units = a.samples * a.groups;
    if (blocks > (1 << 23)) return SLAYER_ERANGE;
#define LAUNCH(ACT) hipLaunchKernelGGL((norm_bwd_stats_kernel<T, ACT>), dim3((unsigned)blocks), dim3(256), 0, s, a)
    BY_ACT(LAUNCH)
#undef LAUNCH
    hipLaunchKernelGGL(norm_bwd_join_kernel, dim3((unsigned)(units + ceil_div(a.channels, 16))), dim3(256), 0, s, a, means, dweight, dbias);
#define LAUNCH(ACT) hipLaunchKernelGGL((norm_bwd_apply_kernel<T, ACT>), dim3((unsigned)blocks), dim3(256), 0, s, a, means)
    BY_ACT(LAUNCH)
#undef LAUNCH
    return (int)hipGetLastError();
}

}  // namespace

extern "C" int64_t slayer_group_norm_workspace(int dtype, int64_t samples, int64_t pixels, int64_t channels, int64_t groups, int backward) {
    if (int e = check_norm(dtype, samples, pixels, channels, groups, ACT_NONE)) return e;
    if (samples == 0 || pixels == 0) return 0;
    const Cut c = cut_of(dtype, samples, pixels, channels, groups);
    if (c.rows) return backward ? c.slots * 2 * (channels / groups) : 0;
    return samples * c.splits * channels * 2 + (backward ? 2 * samples * groups : 0);
}

extern "C" int slayer_group_norm_fwd(void* out, float* mean, float* scale, const void* in, const float* weight, const float* bias, int dtype,
                                     int64_t samples, int64_t pixels, int64_t channels, int64_t groups, float eps, int activation,
                                     float* workspace, int64_t floats, void* stream) {
    if (int e = check_norm(dtype, samples, pixels, channels, groups, activation)) return e;
    if (samples == 0 || pixels == 0) return 0;
    if (!out || !in) return SLAYER_ENULL;
    const Cut c = cut_of(dtype, samples, pixels, channels, groups);
    if ((mean == nullptr) != (scale == nullptr) || (!c.rows && !mean)) return SLAYER_ENULL;
    const int64_t need = slayer_group_norm_workspace(dtype, samples, pixels, channels, groups, 0);
    if (need > 0 && !workspace) return SLAYER_ENULL;
    if (floats < need) return SLAYER_EINVAL;
    const NormArgs a = args_of(out, in, nullptr, weight, bias, mean, scale, workspace, dtype, samples, pixels, channels, groups, eps, c);
    return dtype == SLAYER_FLOAT32 ? launch_fwd<float>(a, c, activation, (hipStream_t)stream) : launch_fwd<bf16>(a, c, activation, (hipStream_t)stream);
}

extern "C" int slayer_group_norm_bwd(void* grad_in, float* grad_weight, float* grad_bias, const void* grad_out, const void* in,
                                     const float* mean, const float* scale, const float* weight, const float* bias, int dtype,
                                     int64_t samples, int64_t pixels, int64_t channels, int64_t groups, int activation, float* workspace,
                                     int64_t floats, void* stream) {
    if (int e = check_norm(dtype, samples, pixels, channels, groups, activation)) return e;
    if (samples == 0 || pixels == 0) {
        if (grad_weight)
            if (int e = launch_zero_fill(grad_weight, channels, (hipStream_t)stream)) return e;
        return grad_bias ? launch_zero_fill(grad_bias, channels, (hipStream_t)stream) : 0;
    }
    if (!grad_in || !grad_out || !in || !mean || !scale) return SLAYER_ENULL;
    const Cut c = cut_of(dtype, samples, pixels, channels, groups);
    const bool sums = grad_weight || grad_bias || !c.rows;
    const int64_t need = sums ? slayer_group_norm_workspace(dtype, samples, pixels, channels, groups, 1) : 0;
    if (need > 0 && !workspace) return SLAYER_ENULL;
    if (floats < need) return SLAYER_EINVAL;
    const NormArgs a = args_of(grad_in, in, grad_out, weight, bias, (float*)mean, (float*)scale, sums ? workspace : nullptr, dtype, samples,
                               pixels, channels, groups, 0.f, c);
    float* means = c.rows ? nullptr : workspace + samples * c.splits * channels * 2;
    return dtype == SLAYER_FLOAT32 ? launch_bwd<float>(a, c, activation, grad_weight, grad_bias, means, (hipStream_t)stream)
                                   : launch_bwd<bf16>(a, c, activation, grad_weight, grad_bias, means, (hipStream_t)stream);
}

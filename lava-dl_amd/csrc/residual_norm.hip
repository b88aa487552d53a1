// A norm behind a block and one in front of the next, with the block's gate and residual scale, in one operator.  Rows x (the block's
// result), r (the residual stream) and z (the gate) of `channels`:
//     u = x / rms(x),  b = act(z) * inner * u,  total = r + factor * scale * b,  hat = total / rms(total),  y = outer * hat,
// rms(v) = sqrt(mean(v^2) + eps).  Without an inner norm u = x, without an outer one there is no y; gate, scale, r may be missing.
// Backwards, with dt the derivative with respect to total, means over the row:
//     dt = dtotal + (dy outer - hat mean(dy outer hat)) / rms(total),  dr = dt,  db = dt factor scale,  dz = db inner u act'(z),
//     d = db act(z) inner,  dx = (d - u mean(d u)) / rms(x);  sums over the rows: dscale of dt factor b, dinner of db act(z) u, douter of dy hat.
//   The norms see the sum as it is, not the one that is rounded to the stream's type.  A row lies in the registers of a part of a wave, a wave, or
// a workgroup where it is longer, four or eight channels a thread, so that each tensor is read or written once; the backward pass makes the row
// again and takes the reciprocals of the two rms from the forward pass.  Parameters stay in registers from row to row, as do the sums of
// their gradients; rows are summed up without LDS inside a wave.
//   Bound: memory.  [48000,256] bfloat16, all there is: forward 23 us (5.3 TB/s), backward 39 (5.0), its sums 4.  [8192,4096] bfloat16 on a float32 stream,
// an outer norm and a scale: 72 (5.6) and 125 (4.8), sums 5.  With four channels a thread, parameters read for every row and sums
// through LDS the same took 44 and 93, 112 and 241.
#include "common.h"
#include "elements.h"

namespace slayer {
namespace {

enum { GATE_NONE, GATE_LINEAR, GATE_SIGMOID, GATE_SILU };

struct ResidualArgs {
    void *out, *total, *grad_in, *grad_residual, *grad_gate;
    const void *in, *residual, *gate, *grad_out, *grad_total;
    const float *inner, *outer, *scale;
    float *stats;                              // [rows][2]: 1 / rms(x), 1 / rms(total)
    float *part_inner, *part_outer, *part_scale;
    int64_t rows, in_stride, residual_stride, gate_stride, grad_out_stride, grad_total_stride;
    int channels, activation;
    float eps, factor;
};

// act(z) and its derivative
struct Gate { float value, slope; };
template <typename T> __device__ __forceinline__ Gate gate_of(int activation, float z) {
    if (activation == GATE_LINEAR) return {z, 1.f};
    const float p = logistic<T>(sizeof(T) == 4 && z > 100.f ? 100.f : z);
    if (activation == GATE_SIGMOID) return {p, p * (1.f - p)};
    return {z * p, p * fmaf(z, 1.f - p, 1.f)};
}

// Sum over LANES neighbouring lanes, in all of them, without LDS: each step adds the other half of 2, 4, 8, 16, 32, 64 lanes.
template <int CTRL> __device__ __forceinline__ float add_moved(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int LANES> __device__ __forceinline__ float sum_wave(float v) {
    v = add_moved<0xb1>(v);                                        // quads: the neighbour
    v = add_moved<0x4e>(v);                                        // quads: the other pair
    if (LANES >= 8) v = add_moved<0x141>(v);                       // eight lanes mirrored
    if (LANES >= 16) v = add_moved<0x140>(v);                      // sixteen lanes mirrored
    if (LANES >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
    if (LANES >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
    return v;
}
// Sum over the LANES threads of a row: a part of a wave, or a whole workgroup.
template <int LANES> __device__ __forceinline__ float sum_row(float v, float* shared) {
    v = sum_wave<LANES < 64 ? LANES : 64>(v);
    if (LANES <= 64) return v;
    __syncthreads();                                               // who reads the sum before
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
    __syncthreads();
    v = shared[threadIdx.x % (LANES / 64)];
    return sum_wave<LANES / 64 < 4 ? 4 : LANES / 64>(LANES == 128 && threadIdx.x % 4 >= 2 ? 0.f : v);
}

// The channels of a thread's access of W: from + lo ... from + hi - 1.  An access at the end of a row that is no multiple of W begins
// earlier than its own channels, so that it is one access all the same; what is not its own reads as 0 and is not written.
struct Own { int from, lo, hi; };
template <int W> __device__ __forceinline__ Own own_of(int c, int channels) {
    if (c >= channels) return {0, 0, 0};
    const int from = c + W <= channels ? c : channels > W ? channels - W : 0;
    return {from, c - from, channels - from < W ? channels - from : W};
}
typedef f8 f8_any __attribute__((aligned(4)));
__device__ __forceinline__ void read_all(float (&x)[4], const float* p) { to_floats(x, *reinterpret_cast<const f4_any*>(p)); }
__device__ __forceinline__ void read_all(float (&x)[8], const bf16* p) { to_floats(x, *reinterpret_cast<const b8_any*>(p)); }
__device__ __forceinline__ void read_all(float (&x)[8], const float* p) {
    const f8 v = *reinterpret_cast<const f8_any*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = v[e];
}
__device__ __forceinline__ void write_all(float* p, const float (&x)[4]) { *reinterpret_cast<f4_any*>(p) = from_floats(x); }
__device__ __forceinline__ void write_all(bf16* p, const float (&x)[8]) { *reinterpret_cast<b8_any*>(p) = from_floats(x); }
__device__ __forceinline__ void write_all(float* p, const float (&x)[8]) {
    *reinterpret_cast<f8_any*>(p) = f8{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]};
}
template <typename T, int W> __device__ __forceinline__ void read(float (&x)[W], const T* row, const Own& own) {
    if (own.hi == W) {
        read_all(x, row + own.from);
        if (own.lo > 0)
#pragma unroll
            for (int e = 0; e < W; ++e) x[e] = e < own.lo ? 0.f : x[e];
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e) x[e] = e < own.hi ? (float)row[own.from + e] : 0.f;
    }
}
template <typename T, int W> __device__ __forceinline__ void write(T* row, const float (&x)[W], const Own& own) {
    if (own.lo == 0 && own.hi == W) {
        write_all(row + own.from, x);
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
            if (e >= own.lo && e < own.hi) row[own.from + e] = (T)x[e];
    }
}
template <int W> __device__ __forceinline__ void parameters(float (&x)[W], const float* p, const Own& own, float factor = 1.f) {
    if (p) read(x, p, own);
#pragma unroll
    for (int e = 0; e < W; ++e) x[e] = p ? x[e] * factor : factor;
}

// T: x, gate and y.  R: the residual stream.  LANES threads a row, IT accesses of 16 bytes of x each.  The loop over the rows is the same for
// all threads of a workgroup.
template <int LANES> constexpr int rows_of() { return LANES <= 64 ? 256 / LANES : 1; }
template <typename T, typename R, int LANES, int IT>
__global__ __launch_bounds__(LANES <= 64 ? 256 : LANES) void residual_fwd_kernel(ResidualArgs a) {
    constexpr int W = Elements<T>::kVec, kRows = rows_of<LANES>();
    __shared__ float shared[16];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float inv = 1.f / (float)a.channels;
    Own own[IT];
    float inner[IT][W], outer[IT][W], scale[IT][W];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        own[i] = own_of<W>((i * LANES + lane) * W, a.channels);
        parameters(inner[i], a.inner, own[i]);
        parameters(outer[i], a.outer, own[i]);
        parameters(scale[i], a.scale, own[i], a.factor);
    }
    for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.rows; base += (int64_t)gridDim.x * kRows) {
        const int64_t row = base + sub;
        const bool on = row < a.rows;
        float b[IT][W], r[IT][W], z[IT][W], sum = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
#pragma unroll
            for (int e = 0; e < W; ++e) b[i][e] = r[i][e] = z[i][e] = 0;
            if (on && own[i].hi > 0) {
                read(b[i], (const T*)a.in + row * a.in_stride, own[i]);
                if (a.activation != GATE_NONE) read(z[i], (const T*)a.gate + row * a.gate_stride, own[i]);
                if (a.residual) read(r[i], (const R*)a.residual + row * a.residual_stride, own[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < W; ++e) sum = fmaf(b[i][e], b[i][e], sum);
        float r1 = 1.f;
        if (a.inner) r1 = 1.f / sqrtf(sum_row<LANES>(sum, shared) * inv + a.eps);
        sum = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                float v = b[i][e] * r1 * inner[i][e];
                if (a.activation != GATE_NONE) v *= gate_of<T>(a.activation, z[i][e]).value;
                b[i][e] = fmaf(scale[i][e], v, r[i][e]);
                sum = fmaf(b[i][e], b[i][e], sum);
            }
            if (a.total && on && own[i].hi > 0) write((R*)a.total + row * a.channels, b[i], own[i]);
        }
        float r2 = 1.f;
        if (a.outer) {
            r2 = 1.f / sqrtf(sum_row<LANES>(sum, shared) * inv + a.eps);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
#pragma unroll
                for (int e = 0; e < W; ++e) b[i][e] = b[i][e] * r2 * outer[i][e];
                if (on && own[i].hi > 0) write((T*)a.out + row * a.channels, b[i], own[i]);
            }
        }
        if (a.stats && lane == 0 && on) {
            a.stats[2 * row] = r1;
            a.stats[2 * row + 1] = r2;
        }
    }
}

// One workgroup's part of a parameter's gradient: the sums of its rows' threads, into parts[workgroup][channels].
template <int LANES, int IT, int W>
__device__ __forceinline__ void write_part(float* part, const float (&x)[IT][W], const Own (&own)[IT], int channels, float* shared) {
    if (!part) return;
    part += (int64_t)blockIdx.x * channels;
    if (rows_of<LANES>() == 1) {
#pragma unroll
        for (int i = 0; i < IT; ++i)
            if (own[i].hi > 0) write(part, x[i], own[i]);
        return;
    }
    constexpr int kRows = rows_of<LANES>(), kWidth = LANES * IT * W;
    const int sub = threadIdx.x / LANES;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e)
            if (e >= own[i].lo && e < own[i].hi) shared[sub * kWidth + own[i].from + e] = x[i][e];
    __syncthreads();
    for (int c = threadIdx.x; c < channels; c += 256) {
        float sum = 0;
        for (int s = 0; s < kRows; ++s) sum += shared[s * kWidth + c];
        part[c] = sum;
    }
}

template <typename T, typename R, int LANES, int IT>
__global__ __launch_bounds__(LANES <= 64 ? 256 : LANES) void residual_bwd_kernel(ResidualArgs a) {
    constexpr int W = Elements<T>::kVec, kRows = rows_of<LANES>();
    constexpr bool kAgain = LANES == 1024;     // parameters are read for every row: of 128 registers there are none to keep them in
    __shared__ float shared[kRows > 1 ? 256 * IT * W : 16];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float inv = 1.f / (float)a.channels;
    const bool outwards = a.outer && a.grad_out;
    Own own[IT];
    float inner[IT][W], outer[IT][W], scale[IT][W], dinner[IT][W], douter[IT][W], dscale[IT][W];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        own[i] = own_of<W>((i * LANES + lane) * W, a.channels);
        if (!kAgain) {
            parameters(inner[i], a.inner, own[i]);
            parameters(outer[i], a.outer, own[i]);
            parameters(scale[i], a.scale, own[i], a.factor);
        }
#pragma unroll
        for (int e = 0; e < W; ++e) dinner[i][e] = douter[i][e] = dscale[i][e] = 0;
    }
    for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.rows; base += (int64_t)gridDim.x * kRows) {
        const int64_t row = base + sub;
        const bool on = row < a.rows;
        float u[IT][W], z[IT][W], hat[IT][W], dt[IT][W], dy[IT][W], r1 = 0, r2 = 0, sum = 0;
        if (on) {
            r1 = a.stats[2 * row];
            r2 = a.stats[2 * row + 1];
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
#pragma unroll
            for (int e = 0; e < W; ++e) u[i][e] = z[i][e] = hat[i][e] = dt[i][e] = dy[i][e] = 0;
            if (on && own[i].hi > 0) {
                read(u[i], (const T*)a.in + row * a.in_stride, own[i]);
                if (a.activation != GATE_NONE) read(z[i], (const T*)a.gate + row * a.gate_stride, own[i]);
                if (a.grad_total) read(dt[i], (const R*)a.grad_total + row * a.grad_total_stride, own[i]);
                if (outwards) {
                    if (a.residual) read(hat[i], (const R*)a.residual + row * a.residual_stride, own[i]);
                    read(dy[i], (const T*)a.grad_out + row * a.grad_out_stride, own[i]);
                }
            }
        }
        Gate gate[IT][W];
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                u[i][e] *= r1;
                gate[i][e] = {1.f, 0.f};
                if (a.activation != GATE_NONE) gate[i][e] = gate_of<T>(a.activation, z[i][e]);
            }
        if (outwards) {
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                if (kAgain) {
                    parameters(inner[i], a.inner, own[i]);
                    parameters(outer[i], a.outer, own[i]);
                    parameters(scale[i], a.scale, own[i], a.factor);
                }
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    hat[i][e] = fmaf(scale[i][e], u[i][e] * inner[i][e] * gate[i][e].value, hat[i][e]) * r2;
                    douter[i][e] = fmaf(dy[i][e], hat[i][e], douter[i][e]);
                    const float d = dy[i][e] * outer[i][e];
                    sum = fmaf(d, hat[i][e], sum);
                    dt[i][e] = fmaf(r2, d, dt[i][e]);
                }
            }
            const float m = sum_row<LANES>(sum, shared) * inv * r2;
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int e = 0; e < W; ++e) dt[i][e] = fmaf(-m, hat[i][e], dt[i][e]);
        }
        sum = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const bool here = on && own[i].hi > 0;
            if (a.grad_residual && here) write((R*)a.grad_residual + row * a.channels, dt[i], own[i]);
            if (kAgain) {
                parameters(inner[i], a.inner, own[i]);
                parameters(scale[i], a.scale, own[i], a.factor);
            }
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float n = u[i][e] * inner[i][e], db = dt[i][e] * scale[i][e], d = db * gate[i][e].value;
                dscale[i][e] = fmaf(dt[i][e], gate[i][e].value * n, dscale[i][e]);          // (times the factor, in the end)
                dinner[i][e] = fmaf(d, u[i][e], dinner[i][e]);
                z[i][e] = db * n * gate[i][e].slope;
                dt[i][e] = d * inner[i][e];
                sum = fmaf(dt[i][e], u[i][e], sum);
            }
            if (a.grad_gate && here) write((T*)a.grad_gate + row * a.channels, z[i], own[i]);
        }
        float m = 0;
        if (a.inner) m = sum_row<LANES>(sum, shared) * inv;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
#pragma unroll
            for (int e = 0; e < W; ++e) dt[i][e] = (dt[i][e] - u[i][e] * m) * r1;
            if (a.grad_in && on && own[i].hi > 0) write((T*)a.grad_in + row * a.channels, dt[i], own[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e) dscale[i][e] *= a.factor;
    write_part<LANES>(a.part_inner, dinner, own, a.channels, shared);
    write_part<LANES>(a.part_outer, douter, own, a.channels, shared);
    write_part<LANES>(a.part_scale, dscale, own, a.channels, shared);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
constexpr int64_t kMostChannels = 8192;

// Threads of a row and accesses of a thread: eight channels a thread.  Four in float32 rows of up to 256 channels, which leaves fewer threads idle and
// less to do before a row's sum: forward / forward and backward, us, four and eight: [800,128] 3.4 / 11.4 and 4.4 / 13.7, [20000,128] 9.8 / 30.5 and
// 10.5 / 33.3, [60000,256] 51.1 / 155 and 51.0 / 159.  Forward passes over more than the last-level cache holds take eight: [250000,100] 106 and 103,
// [250000,128] 129 and 125.
struct Shape { int lanes, its; int64_t blocks; };
Shape shape_of(const slayer_residual_norm* p, bool backward) {
    const bool four = p->dtype == SLAYER_FLOAT32 && p->channels <= 256 && (backward || p->rows * p->channels < 20000000);
    const int each = four ? 4 : 8;
    Shape s;
    s.its = p->dtype == SLAYER_FLOAT32 && !four ? 2 : 1;
    s.lanes = 8;
    while (s.lanes * each < p->channels) s.lanes *= 2;
    const int together = s.lanes <= 64 ? 256 / s.lanes : 1;        // rows of a workgroup at a time
    const int64_t groups = (p->rows + together - 1) / together;
    // as many workgroups as run at a time; of the backward kernel, which leaves a part of each sum for every one of them, twelve waves a
    // compute unit
    const int64_t most = backward ? (s.lanes <= 64 ? 768 : s.lanes < 512 ? 196608 / s.lanes : 256) : s.lanes <= 64 ? 2048 : 524288 / s.lanes;
    s.blocks = groups < most ? groups : most;
    return s;
}

int check_residual(const slayer_residual_norm* p) {
    if (!p) return SLAYER_ENULL;
    if (p->rows < 0 || p->channels < 1) return SLAYER_EINVAL;
    if (p->dtype != SLAYER_FLOAT32 && p->dtype != SLAYER_BFLOAT16) return SLAYER_EINVAL;
    if (p->residual_dtype != SLAYER_FLOAT32 && p->residual_dtype != p->dtype) return SLAYER_EINVAL;
    if (p->activation < GATE_NONE || p->activation > GATE_SILU) return SLAYER_EINVAL;
    if (p->channels > kMostChannels || p->rows > kMaxNumel / p->channels) return SLAYER_ERANGE;
    return 0;
}

ResidualArgs args_of(const slayer_residual_norm* p) {
    ResidualArgs a = {};
    a.inner = p->inner; a.outer = p->outer; a.scale = p->scale;
    a.rows = p->rows; a.channels = (int)p->channels; a.activation = p->activation; a.eps = p->eps; a.factor = p->factor;
    a.in_stride = p->input_stride; a.residual_stride = p->residual_stride; a.gate_stride = p->gate_stride;
    a.grad_out_stride = p->grad_out_stride; a.grad_total_stride = p->grad_total_stride;
    return a;
}

#define SHORT(T, R, IT, LAUNCH)                 \
    switch (s.lanes) {                          \
        case 8: LAUNCH(T, R, 8, IT); break;     \
        case 16: LAUNCH(T, R, 16, IT); break;   \
        case 32: LAUNCH(T, R, 32, IT); break;   \
        default: LAUNCH(T, R, 64, IT);          \
    }
#define LONG(T, R, IT, LAUNCH)                  \
    switch (s.lanes) {                          \
        case 128: LAUNCH(T, R, 128, IT); break; \
        case 256: LAUNCH(T, R, 256, IT); break; \
        case 512: LAUNCH(T, R, 512, IT); break; \
        default: LAUNCH(T, R, 1024, IT);        \
    }
#define BY_TYPE(LAUNCH)                                                       \
    if (p->dtype == SLAYER_FLOAT32) {                                         \
        if (s.its == 1) SHORT(float, float, 1, LAUNCH)                        \
        else if (s.lanes <= 64) SHORT(float, float, 2, LAUNCH)                \
        else LONG(float, float, 2, LAUNCH)                                    \
    } else if (p->residual_dtype == SLAYER_FLOAT32) {                         \
        if (s.lanes <= 64) SHORT(bf16, float, 1, LAUNCH)                      \
        else LONG(bf16, float, 1, LAUNCH)                                     \
    } else {                                                                  \
        if (s.lanes <= 64) SHORT(bf16, bf16, 1, LAUNCH)                       \
        else LONG(bf16, bf16, 1, LAUNCH)                                      \
    }

}  // namespace
}  // namespace slayer

using namespace slayer;

extern "C" int64_t slayer_residual_norm_workspace(const slayer_residual_norm* p) {
    if (int e = check_residual(p)) return e;
    return 3 * shape_of(p, true).blocks * p->channels;
}

extern "C" int slayer_residual_norm_fwd(void* out, void* total, float* stats, const void* input, const void* residual, const void* gate,
                                        const slayer_residual_norm* p, void* stream) {
    if (int e = check_residual(p)) return e;
    if (p->rows == 0) return 0;
    if (!input || (p->activation != GATE_NONE) != (gate != nullptr) || (p->outer != nullptr) != (out != nullptr) || (!out && !total))
        return SLAYER_ENULL;
    ResidualArgs a = args_of(p);
    a.out = out; a.total = total; a.stats = stats; a.in = input; a.residual = residual; a.gate = gate;
    const Shape s = shape_of(p, false);
#define LAUNCH(T, R, LANES, IT) \
    hipLaunchKernelGGL((residual_fwd_kernel<T, R, LANES, IT>), dim3((unsigned)s.blocks), dim3(LANES <= 64 ? 256 : LANES), 0, \
                       (hipStream_t)stream, a)
    BY_TYPE(LAUNCH)
#undef LAUNCH
    return (int)hipGetLastError();
}

extern "C" int slayer_residual_norm_bwd(void* grad_input, void* grad_residual, void* grad_gate, float* grad_inner, float* grad_outer,
                                        float* grad_scale, const void* grad_out, const void* grad_total, const float* stats,
                                        const void* input, const void* residual, const void* gate, const slayer_residual_norm* p,
                                        float* workspace, int64_t floats, void* stream) {
    if (int e = check_residual(p)) return e;
    float* const wanted[3] = {grad_inner, grad_outer, grad_scale};
    if (p->rows == 0) {
        for (float* w : wanted)
            if (w)
                if (int e = launch_zero_fill(w, p->channels, (hipStream_t)stream)) return e;
        return 0;
    }
    if (!input || !stats || (p->activation != GATE_NONE) != (gate != nullptr)) return SLAYER_ENULL;
    if ((grad_inner && !p->inner) || (grad_scale && !p->scale) || (grad_outer && !p->outer) || (grad_gate && !gate) ||
        (grad_residual && !residual))
        return SLAYER_ENULL;
    const bool sums = grad_inner || grad_outer || grad_scale;
    const int64_t need = sums ? slayer_residual_norm_workspace(p) : 0;
    if (need > 0 && !workspace) return SLAYER_ENULL;
    if (floats < need) return SLAYER_EINVAL;
    ResidualArgs a = args_of(p);
    a.grad_in = grad_input; a.grad_residual = grad_residual; a.grad_gate = grad_gate; a.grad_out = grad_out; a.grad_total = grad_total;
    a.stats = (float*)stats; a.in = input; a.residual = residual; a.gate = gate;
    const Shape s = shape_of(p, true);
    const int64_t size = s.blocks * p->channels;
    a.part_inner = grad_inner ? workspace : nullptr;
    a.part_outer = grad_outer ? workspace + size : nullptr;
    a.part_scale = grad_scale ? workspace + 2 * size : nullptr;
#define LAUNCH(T, R, LANES, IT) \
    hipLaunchKernelGGL((residual_bwd_kernel<T, R, LANES, IT>), dim3((unsigned)s.blocks), dim3(LANES <= 64 ? 256 : LANES), 0, \
                       (hipStream_t)stream, a)
    BY_TYPE(LAUNCH)
#undef LAUNCH
    if (int e = (int)hipGetLastError()) return e;
    ColumnSums c = {};
    int count = 0;
    for (int i = 0; i < 3; ++i)
        if (wanted[i]) {
            c.out[count] = wanted[i];
            c.parts[count++] = workspace + i * size;
        }
    c.rows = s.blocks; c.columns = c.pitch = p->channels; c.factor = 1.f;
    return launch_column_sums(c, count, (hipStream_t)stream);
}

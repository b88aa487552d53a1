// A norm behind a block and one in front of the next, with the block's gate and residual scale, in one operator.  Rows x (the block's
// result), r (the residual stream) and z (the gate) of `channels`:
//     u = x / rms(x),  b = act(z) * inner * u,  total = r + factor * scale * b,  hat = total / rms(total),  y = outer * hat,
// rms(v) = sqrt(mean(v^2) + eps).  Without an inner norm u = x, without an outer one there is no y; gate, scale, r may be missing.
// Backwards, with dt the derivative with respect to total, means over the row:
//     dt = dtotal + (dy outer - hat mean(dy outer hat)) / rms(total),  dr = dt,  db = dt factor scale,  dz = db inner u act'(z),
//     d = db act(z) inner,  dx = (d - u mean(d u)) / rms(x);  sums over the rows: dscale of dt factor b, dinner of db act(z) u, douter of dy hat.
//   The norms see the sum as it is, not the one that is rounded to the stream's type.  A row lies in the registers of a wave, or of a
// workgroup where it is longer, so that each tensor is read or written once; the backward pass makes the row again and takes the
// reciprocals of the two rms from the forward pass.
//   Bound: memory.
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

// Sum over the LANES threads of a row (a workgroup of one row, or one to four waves with a row each).
template <int LANES> __device__ __forceinline__ float sum_row(float v, float* shared) {
    v = sum_lanes(v, LANES < 64 ? LANES : 64);
    if (LANES <= 64) return v;
    __syncthreads();                                               // who reads the sum before
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = v;
    __syncthreads();
    float sum = shared[0];
#pragma unroll
    for (int w = 1; w < LANES / 64; ++w) sum += shared[w];
    return sum;
}

__device__ __forceinline__ f4 parameters(const float* p, int c, int left) {
    f4 v = {1.f, 1.f, 1.f, 1.f};
    if (p)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) v[e] = p[c + e];
    return v;
}

// T: x, gate and y.  R: the residual stream.  LANES threads a row, IT times four channels each; the loop over the rows is the same for all
// threads of a workgroup.
template <typename T, typename R, int LANES, int IT>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void residual_fwd_kernel(ResidualArgs a) {
    constexpr int kThreads = LANES < 256 ? 256 : LANES, kRows = kThreads / LANES;
    __shared__ float shared[16];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float inv = 1.f / (float)a.channels;
    for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.rows; base += (int64_t)gridDim.x * kRows) {
        const int64_t row = base + sub;
        const bool on = row < a.rows;
        f4 b[IT], g[IT];
        float sum = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * LANES + lane) * 4, left = on ? a.channels - c : 0;
            b[i] = g[i] = f4{};
            if (left > 0) {
                b[i] = __builtin_convertvector(load_four((const T*)a.in + row * a.in_stride + c, left), f4);
                if (a.residual) g[i] = __builtin_convertvector(load_four((const R*)a.residual + row * a.residual_stride + c, left), f4);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = fmaf(b[i][e], b[i][e], sum);
        }
        float r1 = 1.f;
        if (a.inner) r1 = 1.f / sqrtf(sum_row<LANES>(sum, shared) * inv + a.eps);
        sum = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * LANES + lane) * 4, left = on ? a.channels - c : 0;
            if (left <= 0) continue;
            const f4 inner = parameters(a.inner, c, left), scale = parameters(a.scale, c, left) * a.factor;
            typename Four<T>::Vec z = {};
            if (a.activation != GATE_NONE) z = load_four((const T*)a.gate + row * a.gate_stride + c, left);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = b[i][e] * r1 * inner[e];
                if (a.activation != GATE_NONE) v *= gate_of<T>(a.activation, (float)z[e]).value;
                b[i][e] = fmaf(scale[e], v, g[i][e]);
                sum = fmaf(b[i][e], b[i][e], sum);
            }
            if (a.total) store_four((R*)a.total + row * a.channels + c, b[i], left);
        }
        float r2 = 1.f;
        if (a.outer) {
            r2 = 1.f / sqrtf(sum_row<LANES>(sum, shared) * inv + a.eps);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int c = (i * LANES + lane) * 4, left = on ? a.channels - c : 0;
                if (left > 0) store_four((T*)a.out + row * a.channels + c, b[i] * r2 * parameters(a.outer, c, left), left);
            }
        }
        if (a.stats && lane == 0 && on) {
            a.stats[2 * row] = r1;
            a.stats[2 * row + 1] = r2;
        }
    }
}

template <typename T, typename R, int LANES, int IT>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void residual_bwd_kernel(ResidualArgs a) {
    constexpr int kThreads = LANES < 256 ? 256 : LANES, kRows = kThreads / LANES;
    __shared__ float shared[16];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float inv = 1.f / (float)a.channels;
    f4 dinner[IT], douter[IT], dscale[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) dinner[i] = douter[i] = dscale[i] = f4{};
    for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.rows; base += (int64_t)gridDim.x * kRows) {
        const int64_t row = base + sub;
        const bool on = row < a.rows;
        const float r1 = on ? a.stats[2 * row] : 0.f, r2 = on ? a.stats[2 * row + 1] : 0.f;
        f4 u[IT], hat[IT], dt[IT];
        typename Four<T>::Vec z[IT];
        float sum = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * LANES + lane) * 4, left = on ? a.channels - c : 0;
            u[i] = hat[i] = dt[i] = f4{};
            z[i] = {};
            if (left <= 0) continue;
            u[i] = __builtin_convertvector(load_four((const T*)a.in + row * a.in_stride + c, left), f4) * r1;
            if (a.activation != GATE_NONE) z[i] = load_four((const T*)a.gate + row * a.gate_stride + c, left);
            if (a.grad_total) dt[i] = __builtin_convertvector(load_four((const R*)a.grad_total + row * a.grad_total_stride + c, left), f4);
            if (a.outer && a.grad_out) {
                f4 total = {};
                if (a.residual) total = __builtin_convertvector(load_four((const R*)a.residual + row * a.residual_stride + c, left), f4);
                const f4 dy = __builtin_convertvector(load_four((const T*)a.grad_out + row * a.grad_out_stride + c, left), f4);
                const f4 inner = parameters(a.inner, c, left), scale = parameters(a.scale, c, left) * a.factor, outer = parameters(a.outer, c, left);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = u[i][e] * inner[e];
                    if (a.activation != GATE_NONE) v *= gate_of<T>(a.activation, (float)z[i][e]).value;
                    hat[i][e] = fmaf(scale[e], v, total[e]) * r2;
                    douter[i][e] = fmaf(dy[e], hat[i][e], douter[i][e]);
                    const float d = dy[e] * outer[e];
                    sum = fmaf(d, hat[i][e], sum);
                    dt[i][e] = fmaf(r2, d, dt[i][e]);
                }
            }
        }
        if (a.outer && a.grad_out) {
            const float m = sum_row<LANES>(sum, shared) * inv * r2;
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) dt[i][e] = fmaf(-m, hat[i][e], dt[i][e]);
        }
        sum = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * LANES + lane) * 4, left = on ? a.channels - c : 0;
            if (left <= 0) continue;
            if (a.grad_residual) store_four((R*)a.grad_residual + row * a.channels + c, dt[i], left);
            const f4 inner = parameters(a.inner, c, left), scale = parameters(a.scale, c, left) * a.factor;
            f4 dz;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float n = u[i][e] * inner[e];
                Gate gate = {1.f, 0.f};
                if (a.activation != GATE_NONE) gate = gate_of<T>(a.activation, (float)z[i][e]);
                dscale[i][e] = fmaf(dt[i][e], gate.value * n, dscale[i][e]);      // (times the factor, in the end)
                const float db = dt[i][e] * scale[e];
                dz[e] = db * n * gate.slope;
                const float d = db * gate.value;
                dinner[i][e] = fmaf(d, u[i][e], dinner[i][e]);
                dt[i][e] = d * inner[e];
                sum = fmaf(dt[i][e], u[i][e], sum);
            }
            if (a.grad_gate) store_four((T*)a.grad_gate + row * a.channels + c, dz, left);
        }
        float m = 0;
        if (a.inner) m = sum_row<LANES>(sum, shared) * inv;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = (i * LANES + lane) * 4, left = on ? a.channels - c : 0;
            if (left > 0 && a.grad_in) store_four((T*)a.grad_in + row * a.channels + c, (dt[i] - u[i] * m) * r1, left);
        }
    }
    // this workgroup's rows: [slot][channels]
    const int64_t slot = (int64_t)blockIdx.x * kRows + sub;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = (i * LANES + lane) * 4, left = a.channels - c;
        if (left <= 0) continue;
        if (a.part_inner) store_four(a.part_inner + slot * a.channels + c, dinner[i], left);
        if (a.part_outer) store_four(a.part_outer + slot * a.channels + c, douter[i], left);
        if (a.part_scale) store_four(a.part_scale + slot * a.channels + c, dscale[i] * a.factor, left);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
constexpr int64_t kMostChannels = 16384;

struct Shape { int lanes, its, rows; int64_t fwd_blocks, bwd_blocks; };     // rows: of a workgroup at a time
Shape shape_of(int64_t rows, int64_t channels) {
    const int64_t quads = (channels + 3) / 4;
    Shape s;
    s.lanes = quads <= 8 ? 8 : quads <= 16 ? 16 : quads <= 32 ? 32 : quads <= 256 ? 64 : quads <= 1024 ? 256 : 1024;
    s.its = quads <= s.lanes ? 1 : quads <= 2 * s.lanes ? 2 : 4;
    s.rows = s.lanes < 256 ? 256 / s.lanes : 1;
    const int64_t all = (rows + s.rows - 1) / s.rows;
    s.fwd_blocks = all < 4096 ? all : 4096;
    s.bwd_blocks = all < 512 ? all : 512;
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

#define BY_SHAPE(T, R, LAUNCH)                                       \
    switch (s.lanes) {                                               \
        case 8: LAUNCH(T, R, 8, 1); break;                           \
        case 16: LAUNCH(T, R, 16, 1); break;                         \
        case 32: LAUNCH(T, R, 32, 1); break;                         \
        case 64:                                                     \
            if (s.its == 1) LAUNCH(T, R, 64, 1);                     \
            else if (s.its == 2) LAUNCH(T, R, 64, 2);                \
            else LAUNCH(T, R, 64, 4);                                \
            break;                                                   \
        case 256:                                                    \
            if (s.its == 2) LAUNCH(T, R, 256, 2);                    \
            else LAUNCH(T, R, 256, 4);                               \
            break;                                                   \
        default:                                                     \
            if (s.its == 2) LAUNCH(T, R, 1024, 2);                   \
            else LAUNCH(T, R, 1024, 4);                              \
    }
#define BY_TYPE(LAUNCH)                                              \
    if (p->dtype == SLAYER_FLOAT32) BY_SHAPE(float, float, LAUNCH)   \
    else if (p->residual_dtype == SLAYER_FLOAT32) BY_SHAPE(bf16, float, LAUNCH) \
    else BY_SHAPE(bf16, bf16, LAUNCH)

}  // namespace
}  // namespace slayer

using namespace slayer;

extern "C" int64_t slayer_residual_norm_workspace(const slayer_residual_norm* p) {
    if (int e = check_residual(p)) return e;
    const Shape s = shape_of(p->rows, p->channels);
    return 3 * s.bwd_blocks * s.rows * p->channels;
}

extern "C" int slayer_residual_norm_fwd(void* out, void* total, float* stats, const void* input, const void* residual, const void* gate,
                                        const slayer_residual_norm* p, void* stream) {
    if (int e = check_residual(p)) return e;
    if (p->rows == 0) return 0;
    if (!input || (p->activation != GATE_NONE) != (gate != nullptr) || (p->outer != nullptr) != (out != nullptr) || (!out && !total))
        return SLAYER_ENULL;
    ResidualArgs a = args_of(p);
    a.out = out; a.total = total; a.stats = stats; a.in = input; a.residual = residual; a.gate = gate;
    const Shape s = shape_of(p->rows, p->channels);
#define LAUNCH(T, R, LANES, IT) \
    hipLaunchKernelGGL((residual_fwd_kernel<T, R, LANES, IT>), dim3((unsigned)s.fwd_blocks), dim3(LANES < 256 ? 256 : LANES), 0, \
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
    const Shape s = shape_of(p->rows, p->channels);
    const int64_t slots = s.bwd_blocks * s.rows, size = slots * p->channels;
    a.part_inner = grad_inner ? workspace : nullptr;
    a.part_outer = grad_outer ? workspace + size : nullptr;
    a.part_scale = grad_scale ? workspace + 2 * size : nullptr;
#define LAUNCH(T, R, LANES, IT) \
    hipLaunchKernelGGL((residual_bwd_kernel<T, R, LANES, IT>), dim3((unsigned)s.bwd_blocks), dim3(LANES < 256 ? 256 : LANES), 0, \
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
    c.rows = slots; c.columns = c.pitch = p->channels; c.factor = 1.f;
    return launch_column_sums(c, count, (hipStream_t)stream);
}

// Sums of the columns of a matrix of partial sums, in one fixed order: the last step of the gradients of parameters that many rows share.
//   Sixteen columns and 64 shares of the rows a workgroup: rows are few thousands and columns few hundreds, so a workgroup for each
// sixteen (64 bytes, half a cache line) is what brings enough of them.  A share adds up its rows in float64: there may be thousands, and
// rows that are alike are off by the same amount each.
#include "common.h"
#include "elements.h"

namespace slayer {

__global__ __launch_bounds__(1024) void column_sums_kernel(ColumnSums a) {
    __shared__ float sums[64][17];
    const int i = threadIdx.x % 16, share = threadIdx.x / 16, which = blockIdx.y;
    const int64_t c = (int64_t)blockIdx.x * 16 + i;
    const float* parts = a.parts[which];
    double rows = 0;
    if (c < a.columns) {
#pragma unroll 8
        for (int64_t row = share; row < a.rows; row += 64) rows += parts[row * a.pitch + c];
    }
    sums[share][i] = (float)rows;
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int column = threadIdx.x / 16;                            // sixteen sums, sixteen lanes each
    float sum = (sums[i][column] + sums[i + 16][column]) + (sums[i + 32][column] + sums[i + 48][column]);
    sum = sum_lanes(sum, 16);
    const int64_t to = (int64_t)blockIdx.x * 16 + column;
    if (i == 0 && to < a.columns) a.out[which][to] = sum * a.factor;
}

int launch_column_sums(const ColumnSums& a, int count, hipStream_t stream) {
    if (count == 0 || a.columns == 0) return 0;
    const int64_t blocks = (a.columns + 15) / 16;
    if (blocks > (1 << 20)) return SLAYER_ERANGE;
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)blocks, (unsigned)count), dim3(1024), 0, stream, a);
    return (int)hipGetLastError();
}

}  // namespace slayer

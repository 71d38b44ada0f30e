// Column sums of the partial rows that the sequence-layer backward kernels leave (see seq_common.h).  5 us for 512 rows of
// 10240 columns (21 MB, 4 TB/s out of the L2): little more than a launch.
#include "seq_common.h"

namespace {

constexpr long kMostGroups = 1 << 20;  // (a launch holds less than 2^32 threads: 2^28 columns would be too many at once)

__global__ void __launch_bounds__(1024)
column_sums_kernel(const float* __restrict__ part, long rows, int cols, const afd::ColumnOuts outs) {
    __shared__ float lds[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (long c0 = (long)blockIdx.x * 64; c0 < cols; c0 += (long)gridDim.x * 64) {
        const bool live = c0 + lane < cols;
        const int col = (int)(live ? c0 + lane : 0);
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        if (live) {
            long r = w;
            for (; r + 48 < rows; r += 64) {
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[u] += part[(size_t)(r + 16 * u) * cols + col];
            }
            for (; r < rows; r += 16) acc[0] += part[(size_t)r * cols + col];
        }
        lds[w][lane] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
        __syncthreads();
        if (w == 0 && live) {
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) v += lds[i][lane];
            for (int k = 0; k < outs.n; ++k) {
                const afd::ColumnOut o = outs.o[k];
                if (col < o.begin || col >= o.end || !o.out) continue;
                const int i = col - o.begin, g = i / o.width, j = i - g * o.width;
                if (j >= o.keep) continue;
                const size_t at = (size_t)g * o.gs + (size_t)j * o.js;
                if (o.dtype == AFD_T_F32) static_cast<float*>(o.out)[at] = v;
                else if (o.dtype == AFD_T_BF16) static_cast<afd::bf16_t*>(o.out)[at] = afd::from_f32<afd::bf16_t>(v);
                else static_cast<afd::f16_t*>(o.out)[at] = afd::from_f32<afd::f16_t>(v);
            }
        }
        __syncthreads();  // (the next columns' sums go to the same places)
    }
}

}  // namespace

int afd::launch_column_sums(const float* part, long rows, int cols, const ColumnOuts& outs, hipStream_t s) {
    const long groups = ((long)cols + 63) / 64;
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)(groups < kMostGroups ? groups : kMostGroups)), dim3(1024), 0, s, part, rows, cols, outs);
    return check_launch("column_sums_kernel");
}

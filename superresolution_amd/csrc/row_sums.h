// The join of partial sums: workgroups leave rows of partial column sums, one launch adds the rows in a fixed order.
#pragma once
#include "common.h"

namespace srmi {

// dst[k][c] = scale_k * sum over rows of part[row][k][c]; blockIdx.y = k (or the image of a per-image gate, whose rows are its own)
struct SumRows {
    const float* part;
    long long outer_stride;  // floats between two blockIdx.y
    long long row_stride;
    unsigned rows;
    int c;
    int n_dst;               // > 0: dst[blockIdx.y] pointers; 0: dst[0] + blockIdx.y * c
    float* dst[5];
    float scale[5];
};
static __global__ __launch_bounds__(1024) void sum_rows_kernel(const SumRows p) {
    __shared__ float red[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), grp = threadIdx.x >> 5;
    const float* src = p.part + (long long)blockIdx.y * p.outer_stride + col;
    float s = 0.f;
    if (col < p.c) {
#pragma unroll 8
        for (unsigned r = grp; r < p.rows; r += 32) s += src[(long long)r * p.row_stride];
    }
    red[grp][threadIdx.x & 31] = s;
    __syncthreads();
    if (grp == 0 && col < p.c) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += red[i][threadIdx.x];
        const int k = p.n_dst ? blockIdx.y : 0;
        (p.n_dst ? p.dst[k] : p.dst[0] + (long long)blockIdx.y * p.c)[col] = p.scale[k] * t;
    }
}

}  // namespace srmi

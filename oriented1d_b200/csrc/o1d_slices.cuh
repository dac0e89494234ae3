// Last step of the column sums: partial sums of slices of rows, added in a fixed order (no atomics: bit-reproducible).
#pragma once

#include "o1d_common.cuh"

namespace o1d {

// out[c] = sum over slices of partial[slice][c] for na + nb columns, the first na of which go to `a` and the others to `b`.
// Block (32, 32): thread (x, y) adds the slices congruent to y modulo 32 for one column, the 32 sums are then added in
// order of y.  In fp64: thousands of slices may cancel.  A few
// microseconds, most of them latency: hence 32 short chains of loads and not one.
static __global__ void __launch_bounds__(1024)
sum_slices_kernel(const float *__restrict__ partial, void *__restrict__ a, int na, void *__restrict__ b, int nb, int bf16, int slices) {
    __shared__ double part[32][33];
    const int n = na + nb, c = blockIdx.x * 32 + threadIdx.x;
    double s = 0.;
    if (c < n)
#pragma unroll 4
        for (int k = threadIdx.y; k < slices; k += 32) s += partial[(size_t)k * n + c];
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < n) {
        double t = 0.;
#pragma unroll
        for (int y = 0; y < 32; y++) t += part[y][threadIdx.x];
        if (c < na) st_param(a, c, bf16, (float)t); else st_param(b, c - na, bf16, (float)t);
    }
}
inline cudaError_t sum_slices(const float *partial, void *a, int na, void *b, int nb, int bf16, int slices, cudaStream_t st) {
    sum_slices_kernel<<<ceil_div(na + nb, 32), dim3(32, 32), 0, st>>>(partial, a, na, b, nb, bf16, slices);
    return cudaGetLastError();
}

}  // namespace o1d

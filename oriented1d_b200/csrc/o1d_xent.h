// Host-callable interface of the linear cross entropy kernels (o1d_xent.cuh), compiled in their own translation unit.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace o1d {

// Rows, classes and features, each: kernels hold their indices in 32 bits and step past an end by up to a grid's worth of classes (10^4).
constexpr int kXentMost = 0x7fff0000;

struct XentArgs {
    const void *x, *w, *bias;                 // [N, D], [V, D], [V] or null
    const long long *target;                  // [N]
    long long N;
    int D, V;
    bool bf16;                                // x, w and their gradients
    int bias_bf16;                            // bias and its gradient
    long long ignore;
    float smoothing;
    int reduction;                            // O1D_XENT_*
    // forward
    float *loss, *lse, *count;                // lse [3, N], null: no backward pass will follow
    // backward (lse and count are read)
    const float *dloss;
    void *dx, *dw, *db;                       // any may be null
    void *workspace;
    size_t workspace_bytes;
};

size_t xent_workspace(const XentArgs &a, bool backward, int sms);
// 0: launched.  > 0: an O1D_ERR_* code; *cuda holds the CUDA error where there is one, *encode the driver's answer.
int xent_forward(const XentArgs &a, int sms, int *err_flag, cudaStream_t st, cudaError_t *cuda, int *encode);
int xent_backward(const XentArgs &a, int sms, int *err_flag, cudaStream_t st, cudaError_t *cuda, int *encode);

}  // namespace o1d

// Host-callable interface of the 8-bit checkpoint kernels (o1d_keep8.cuh), compiled in their own translation unit.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace o1d {

constexpr int kKeepGroup = 128;          // columns that share a range
constexpr int kKeepMaxRow = 8192;        // longest row of the LayerNorm kernels
constexpr int kKeepMaxColumns = 1 << 24; // and of the elementwise ones (32-bit offsets within a block of rows)

enum : int { KEEP_FWD = 0, KEEP_RESTORE, KEEP_GELU_FWD, KEEP_GELU_BWD };

struct KeepArgs {
    const void *x;           // forward: the values; GELU backward: dy
    const void *bias;        // GELU forward, may be null
    uint8_t *codes;          // written by the forward kinds (null: not kept), read by the others
    float *ranges;           // [rows][groups][2]: least value, step
    void *y;                 // GELU: the activation (backward: may be null); restore: the values
    void *dx;                // GELU backward
    void *dbias;             // GELU backward, may be null
    float *partial;          // GELU backward with dbias: keep_partials() slices of C floats
    long long rows;
    int C;
    int pbf16;               // bias / dbias are bf16
};
// Slices of column sums that the GELU backward writes for this shape.
int keep_slices(long long rows, int C, int sms);
cudaError_t keep_launch(int kind, bool bf16, const KeepArgs &a, int sms, cudaStream_t st);

struct LnKeepArgs {
    const void *x;           // forward: the input; backward: dy
    const void *gamma, *beta;
    uint8_t *codes;          // forward: null, nothing is kept
    float *ranges, *stats;   // stats [rows][2]: mean, 1 / standard deviation (forward: null with codes)
    void *y;                 // forward: the output; backward: may be null, else the output once more, from the codes
    void *dx, *dgamma, *dbeta;
    float *partial;          // backward: ln_keep_ctas() x 2 x C floats
    long long rows;
    int C;
    float eps;
    int pbf16;
};
int ln_keep_ctas(long long rows, int C, int sms);
cudaError_t ln_keep_launch(bool backward, bool bf16, const LnKeepArgs &a, int sms, cudaStream_t st);

}  // namespace o1d

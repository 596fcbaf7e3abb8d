// Affine layer norm, forward and backward (launch interface).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace ctu {
namespace norm {

struct AffineArgs {
    const void *x;       // [rows, hidden]
    const void *weight;  // [hidden] or null (1)
    const void *bias;    // [hidden] or null (0)
    void *out;           // forward
    float *mean;         // [rows]
    float *rstd;         // [rows]
    const void *grad;    // backward: [rows, hidden]
    void *dx;            // or null
    void *dweight;       // or null
    void *dbias;         // or null
    float *workspace;    // backward: 2 * slices * hidden
    int64_t rows;
    int hidden;
    float epsilon;
    int dtype;         // CTU_DTYPE_* of x, out, grad, dx
    int weight_dtype;  // CTU_DTYPE_* of weight, bias and their gradients
    int num_sms;
    uint32_t *err;     // the device's error word (bounded waits)
};

// Limit of the backward pass's waits.  Test hook: wait `never` (counted from 0) of the first team is on a barrier that
// nothing arrives on; -1: none.
struct WaitLimit {
    uint64_t ns;
    int never;
};

// Row slices whose partial sums of the weight's and bias's gradients are joined at the end.
int64_t backward_slices(int64_t rows, int64_t hidden);

cudaError_t launch_layer_norm(const AffineArgs &a, cudaStream_t stream);
// One storage type's backward pass (layer_norm_backward_*.cu).
template <typename T>
cudaError_t backward_as(const AffineArgs &a, const WaitLimit &wait, cudaStream_t stream);
constexpr int kSlices = 148;  // backward CTAs that leave partial sums: one an SM of a B200

cudaError_t launch_layer_norm_backward(const AffineArgs &a, const WaitLimit &wait, cudaStream_t stream);

}  // namespace norm
}  // namespace ctu

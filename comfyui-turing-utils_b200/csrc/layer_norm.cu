// Affine layer norm, forward and backward.
//
//   xhat = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   y    = xhat * w + b
//   g    = dy * w
//   dx   = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dw   = sum over rows of dy * xhat,   db = sum over rows of dy
//
// Statistics, sums and gradients are fp32 whatever the storage type; each result is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../../include/ctu_b200.h"
#include "layer_norm.cuh"

namespace ctu {
namespace norm {

namespace {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

constexpr int kThreads = 256;

// Sum of two values over the block, in every thread.
__device__ __forceinline__ float2 block_sum(float2 v) {
    __shared__ float2 part[kThreads / 32];
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float2 s = make_float2(0.0f, 0.0f);
    for (int i = 0; i < kThreads / 32; ++i) {
        s.x += part[i].x;
        s.y += part[i].y;
    }
    return s;
}

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) forward_kernel(const AffineArgs a) {
    const int h = a.hidden;
    const W *w = static_cast<const W *>(a.weight);
    const W *b = static_cast<const W *>(a.bias);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * h;
        T *y = static_cast<T *>(a.out) + r * h;
        float s = 0.0f;
        for (int c = threadIdx.x; c < h; c += kThreads) s += to_f(x[c]);
        const float mean = block_sum(make_float2(s, 0.0f)).x / static_cast<float>(h);
        float q = 0.0f;
        for (int c = threadIdx.x; c < h; c += kThreads) {
            const float d = to_f(x[c]) - mean;
            q += d * d;
        }
        const float var = block_sum(make_float2(q, 0.0f)).x / static_cast<float>(h);
        const float rstd = 1.0f / sqrtf(var + a.epsilon);
        if (threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int c = threadIdx.x; c < h; c += kThreads) {
            const float n = (to_f(x[c]) - mean) * rstd;
            y[c] = from_f<T>(n * (w ? to_f(w[c]) : 1.0f) + (b ? to_f(b[c]) : 0.0f));
        }
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) input_gradient_kernel(const AffineArgs a) {
    const int h = a.hidden;
    const W *w = static_cast<const W *>(a.weight);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * h;
        const T *dy = static_cast<const T *>(a.grad) + r * h;
        T *dx = static_cast<T *>(a.dx) + r * h;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float2 s = make_float2(0.0f, 0.0f);
        for (int c = threadIdx.x; c < h; c += kThreads) {
            const float n = (to_f(x[c]) - mean) * rstd;
            const float g = to_f(dy[c]) * (w ? to_f(w[c]) : 1.0f);
            s.x += g;
            s.y += g * n;
        }
        s = block_sum(s);
        s.x /= static_cast<float>(h);
        s.y /= static_cast<float>(h);
        for (int c = threadIdx.x; c < h; c += kThreads) {
            const float n = (to_f(x[c]) - mean) * rstd;
            const float g = to_f(dy[c]) * (w ? to_f(w[c]) : 1.0f);
            dx[c] = from_f<T>(rstd * (g - s.x - n * s.y));
        }
    }
}

// Partial sums of one slice of rows: workspace [slice][0: dw, 1: db][hidden].
template <typename T>
__global__ void __launch_bounds__(256) parameter_partial_kernel(const AffineArgs a, int slices) {
    __shared__ float2 part[8][33];
    const int h = a.hidden;
    const int c = blockIdx.x * 32 + threadIdx.x;
    const int slice = blockIdx.y;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < h) {
        for (int64_t r = slice * 8 + threadIdx.y; r < a.rows; r += static_cast<int64_t>(slices) * 8) {
            const float dy = to_f(static_cast<const T *>(a.grad)[r * h + c]);
            s.x += dy * ((to_f(static_cast<const T *>(a.x)[r * h + c]) - a.mean[r]) * a.rstd[r]);
            s.y += dy;
        }
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < h) {
        for (int i = 1; i < 8; ++i) {
            s.x += part[i][threadIdx.x].x;
            s.y += part[i][threadIdx.x].y;
        }
        a.workspace[(static_cast<int64_t>(slice) * 2) * h + c] = s.x;
        a.workspace[(static_cast<int64_t>(slice) * 2 + 1) * h + c] = s.y;
    }
}

template <typename W>
__global__ void __launch_bounds__(256) parameter_join_kernel(const AffineArgs a, int slices) {
    const int h = a.hidden;
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= h) return;
    float dw = 0.0f, db = 0.0f;
    for (int s = 0; s < slices; ++s) {
        dw += a.workspace[(static_cast<int64_t>(s) * 2) * h + c];
        db += a.workspace[(static_cast<int64_t>(s) * 2 + 1) * h + c];
    }
    if (a.dweight) static_cast<W *>(a.dweight)[c] = from_f<W>(dw);
    if (a.dbias) static_cast<W *>(a.dbias)[c] = from_f<W>(db);
}

template <typename F>
cudaError_t with_type(int dtype, F f) {
    switch (dtype) {
    case CTU_DTYPE_BF16: return f(__nv_bfloat16());
    case CTU_DTYPE_FP16: return f(__half());
    default: return f(float());
    }
}

}  // namespace

int64_t backward_slices(int64_t rows, int64_t) { return std::max<int64_t>(1, std::min<int64_t>(64, (rows + 31) / 32)); }

cudaError_t launch_layer_norm(const AffineArgs &a, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, a.num_sms * 8));
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return with_type(a.weight_dtype, [&](auto w) {
            forward_kernel<T, decltype(w)><<<grid, kThreads, 0, stream>>>(a);
            return cudaGetLastError();
        });
    });
}

cudaError_t launch_layer_norm_backward(const AffineArgs &a, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, a.num_sms * 8));
    const int slices = static_cast<int>(backward_slices(a.rows, a.hidden));
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        return with_type(a.weight_dtype, [&](auto w) {
            using W = decltype(w);
            if (a.dx && a.rows > 0) input_gradient_kernel<T, W><<<grid, kThreads, 0, stream>>>(a);
            if (a.dweight || a.dbias) {
                parameter_partial_kernel<T>
                    <<<dim3((a.hidden + 31) / 32, slices), dim3(32, 8), 0, stream>>>(a, slices);
                parameter_join_kernel<W><<<(a.hidden + 255) / 256, 256, 0, stream>>>(a, slices);
            }
            return cudaGetLastError();
        });
    });
}

}  // namespace norm
}  // namespace ctu

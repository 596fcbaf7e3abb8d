// Rows to 4-bit floating point with block scales, and back.
//
// One CTA takes a row: the values (rotated, if asked, in blocks of 256) stay in shared memory as
// fp32 between the pass that finds the row's largest magnitude and the one that writes codes.
//
// Row scale (nvfp4): 2^ceil(log2(amax / 2688)), 2688 = 6 * 448, so that the largest block scale
// lies in (224, 448]; a power of two keeps every division by it exact.  Block scale: nvfp4
// e4m3(block amax / 6 / row scale); mxfp4 2^(floor(log2(block amax)) - 2), the OCP rule.  Code:
// e2m1(v / block scale / row scale) to nearest, ties to even, saturating at 6.  A row that holds a
// NaN or an infinity gets a NaN row scale and zero codes and block scales.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "../../include/ctu_b200.h"
#include "fp4.cuh"

namespace ctu {
namespace fp4 {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float load_value(const void *x, int64_t i, int dtype) {
    return dtype == CTU_DTYPE_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(x)[i])
                                   : __half2float(static_cast<const __half *>(x)[i]);
}

// Two values to one byte of e2m1 codes, `lo` in the low nibble.
__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n\tcvt.u32.u8 %0, t;\n\t}"
        : "=r"(r)
        : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ float e2m1_value(uint32_t code) {
    const uint32_t e = (code >> 1) & 3u, m = code & 1u;
    const float v = e == 0 ? 0.5f * m : __uint_as_float(((e + 126u) << 23) | (m << 22));
    return (code & 8u) ? -v : v;
}

__device__ __forceinline__ float block_scale_value(uint32_t byte, int format) {
    if (format == kNvfp4) {
        const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
        return __half2float(__half(h));
    }
    if (byte == 255u) return __uint_as_float(0x7fc00000u);
    return byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);  // 2^-127 is subnormal
}

__device__ __forceinline__ float pow2_row_scale(float amax) {
    if (amax == 0.0f) return 1.0f;
    const uint32_t t = __float_as_uint(__fdiv_rn(amax, 2688.0f));
    const uint32_t e = (t >> 23) + ((t & 0x7fffffu) != 0 ? 1u : 0u);
    return __uint_as_float(max(e, 1u) << 23);
}

template <int kFormat>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const QuantArgs a) {
    extern __shared__ float v[];
    __shared__ float red[kThreads / 32];
    constexpr int kBlock = block_of(kFormat);
    const int k = a.k;
    const int64_t col_tiles = scale_col_tiles(k, kFormat);
    const int blocks = k / kBlock;
    for (int64_t r = blockIdx.x; r < scale_row_tiles(a.rows) * 128; r += gridDim.x) {
        if (r >= a.rows) {
            for (int b = threadIdx.x; b < col_tiles * 4; b += kThreads)
                a.block_scales[scale_offset(r, b, col_tiles)] = 0;
            continue;
        }
        __syncthreads();
        const float pre = a.rotation ? 0.0625f : 1.0f;
        for (int c = threadIdx.x; c < k; c += kThreads) v[c] = __fmul_rn(load_value(a.x, r * k + c, a.dtype), pre);
        __syncthreads();
        if (a.rotation) {
            for (int stride = 1; stride <= 64; stride *= 4) {
                for (int q = threadIdx.x; q < k / 4; q += kThreads) {
                    const int base = (q / stride) * stride * 4 + q % stride;
                    const float x0 = v[base], x1 = v[base + stride], x2 = v[base + 2 * stride], x3 = v[base + 3 * stride];
                    const float t = __fadd_rn(x0, x1), b = __fsub_rn(x0, x1);
                    v[base] = __fsub_rn(__fadd_rn(t, x2), x3);
                    v[base + stride] = __fadd_rn(__fsub_rn(t, x2), x3);
                    v[base + 2 * stride] = __fadd_rn(__fadd_rn(b, x2), x3);
                    v[base + 3 * stride] = __fadd_rn(__fsub_rn(x2, b), x3);
                }
                __syncthreads();
            }
        }
        // Largest magnitude as an unsigned integer: infinities and NaN come out above all else.
        uint32_t top = 0;
        for (int c = threadIdx.x; c < k; c += kThreads) top = max(top, __float_as_uint(v[c]) & 0x7fffffffu);
        top = __reduce_max_sync(0xffffffffu, top);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(top);
        __syncthreads();
        for (int i = 0; i < kThreads / 32; ++i) top = max(top, __float_as_uint(red[i]));
        const bool bad = top >= 0x7f800000u;
        const float row = kFormat == kNvfp4 && !bad ? pow2_row_scale(__uint_as_float(top)) : 1.0f;
        if (threadIdx.x == 0) a.row_scales[r] = bad ? __uint_as_float(0x7fc00000u) : row;
        const float inv_row = 1.0f / row;
        for (int b = threadIdx.x; b < col_tiles * 4; b += kThreads) {
            uint32_t scale_byte = 0;
            if (b < blocks) {
                uint32_t *out = reinterpret_cast<uint32_t *>(a.codes + r * (k / 2) + b * (kBlock / 2));
                if (bad) {
                    for (int i = 0; i < kBlock / 8; ++i) out[i] = 0;
                } else {
                    float amax = 0.0f;
                    for (int i = 0; i < kBlock; ++i) amax = fmaxf(amax, fabsf(v[b * kBlock + i]));
                    float divisor;
                    if (kFormat == kNvfp4) {
                        scale_byte = __nv_cvt_float_to_fp8(__fdiv_rn(amax * inv_row, 6.0f), __NV_SATFINITE, __NV_E4M3);
                        divisor = block_scale_value(scale_byte, kFormat);
                    } else {
                        const uint32_t e = __float_as_uint(amax) >> 23;
                        scale_byte = e > 2 ? e - 2 : 0;
                        divisor = block_scale_value(scale_byte, kFormat);
                    }
                    for (int i = 0; i < kBlock / 8; ++i) {
                        uint32_t word = 0;
                        for (int j = 0; j < 4; ++j) {
                            const float x0 = v[b * kBlock + 8 * i + 2 * j] * inv_row;
                            const float x1 = v[b * kBlock + 8 * i + 2 * j + 1] * inv_row;
                            const float q0 = divisor == 0.0f ? copysignf(0.0f, x0) : __fdiv_rn(x0, divisor);
                            const float q1 = divisor == 0.0f ? copysignf(0.0f, x1) : __fdiv_rn(x1, divisor);
                            word |= e2m1x2(q0, q1) << (8 * j);
                        }
                        out[i] = word;
                    }
                }
            }
            a.block_scales[scale_offset(r, b, col_tiles)] = static_cast<uint8_t>(scale_byte);
        }
    }
}

template <typename T>
__device__ __forceinline__ T store_as(float v);
template <>
__device__ __forceinline__ float store_as(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 store_as(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half store_as(float v) { return __float2half_rn(v); }

template <int kFormat, typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantArgs a) {
    const int64_t half = a.k / 2;
    const int64_t col_tiles = scale_col_tiles(a.k, kFormat);
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < a.rows * half; i += gridDim.x * 256ll) {
        const int64_t r = i / half;
        const int c = static_cast<int>(i - r * half) * 2;
        const float s = block_scale_value(a.block_scales[scale_offset(r, c / block_of(kFormat), col_tiles)], kFormat);
        const float rs = a.row_scales[a.row_scale_count == 1 ? 0 : r];
        const uint32_t byte = a.codes[i];
        T *out = static_cast<T *>(a.out) + r * a.k + c;
        out[0] = store_as<T>(e2m1_value(byte & 15u) * s * rs);
        out[1] = store_as<T>(e2m1_value(byte >> 4) * s * rs);
    }
}

// 32 x 32 tiles through shared memory: reads run along k, writes along n.
template <int kFormat>
__global__ void __launch_bounds__(256) decode_transposed_kernel(const DequantArgs a) {
    __shared__ float tile[32][33];
    const int64_t n0 = blockIdx.y * 32ll;
    const int k0 = blockIdx.x * 32;
    const int64_t col_tiles = scale_col_tiles(a.k, kFormat);
    for (int i = threadIdx.x; i < 32 * 16; i += 256) {
        const int64_t r = n0 + i / 16;
        const int c = k0 + 2 * (i % 16);
        float v0 = 0.0f, v1 = 0.0f;
        if (r < a.rows && c < a.k) {
            const uint32_t byte = a.codes[r * (a.k / 2) + c / 2];
            const float s = block_scale_value(a.block_scales[scale_offset(r, c / block_of(kFormat), col_tiles)], kFormat);
            const float rs = a.row_scales[a.row_scale_count == 1 ? 0 : r];
            v0 = e2m1_value(byte & 15u) * s * rs;
            v1 = e2m1_value(byte >> 4) * s * rs;
        }
        tile[i / 16][2 * (i % 16)] = v0;
        tile[i / 16][2 * (i % 16) + 1] = v1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * 32; i += 256) {
        const int c = k0 + i / 32;
        const int64_t r = n0 + i % 32;
        if (c < a.k && r < a.rows)
            static_cast<__nv_bfloat16 *>(a.out)[c * a.rows + r] = __float2bfloat16_rn(tile[i % 32][i / 32]);
    }
}

}  // namespace

cudaError_t launch_quantize(const QuantArgs &a, cudaStream_t stream) {
    const int smem = a.k * static_cast<int>(sizeof(float));
    const unsigned grid =
        static_cast<unsigned>(std::min<int64_t>(scale_row_tiles(a.rows) * 128, static_cast<int64_t>(a.num_sms) * 8));
    auto kernel = a.format == kNvfp4 ? quantize_kernel<kNvfp4> : quantize_kernel<kMxfp4>;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return e;
    kernel<<<grid, kThreads, smem, stream>>>(a);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t dequantize_as(const DequantArgs &a, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(
        std::min<int64_t>((a.rows * (a.k / 2) + 255) / 256, static_cast<int64_t>(a.num_sms) * 16));
    if (a.format == kNvfp4)
        dequantize_kernel<kNvfp4, T><<<grid, 256, 0, stream>>>(a);
    else
        dequantize_kernel<kMxfp4, T><<<grid, 256, 0, stream>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_dequantize(const DequantArgs &a, cudaStream_t stream) {
    if (a.dtype == CTU_DTYPE_BF16) return dequantize_as<__nv_bfloat16>(a, stream);
    if (a.dtype == CTU_DTYPE_FP16) return dequantize_as<__half>(a, stream);
    return dequantize_as<float>(a, stream);
}

cudaError_t launch_decode_transposed(const DequantArgs &a, cudaStream_t stream) {
    const dim3 grid((a.k + 31) / 32, static_cast<unsigned>((a.rows + 31) / 32));
    if (a.format == kNvfp4)
        decode_transposed_kernel<kNvfp4><<<grid, 256, 0, stream>>>(a);
    else
        decode_transposed_kernel<kMxfp4><<<grid, 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace fp4
}  // namespace ctu

// 4-bit floating point (e2m1) with block scales: formats, layouts and launch interfaces.
//
// A quantized matrix [rows, k] stands for  code[r, c] * block_scale[r, c / block] * row_scale[r]:
//   nvfp4  block 16, e4m3 block scales, a power-of-two fp32 scale per row;
//   mxfp4  block 32, e8m0 (power-of-two) block scales, row scale 1.
// Codes: [rows, k / 2] bytes, the even column in the low nibble.  Block scales lie in tiles of 128
// rows x 4 blocks, 512 bytes each, tile order [rows / 128][blocks / 4]: row 32 j + l, block b of a
// tile at byte 16 l + 4 j + b.  That is the order in which one tcgen05.cp (32 lanes x 128 bits)
// puts a tile into tensor memory, so the product copies tiles without touching a byte of them.
// Bytes of a tile beyond the matrix are zero.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace ctu {
namespace fp4 {

constexpr int kNvfp4 = 0;
constexpr int kMxfp4 = 1;

__host__ __device__ constexpr int block_of(int format) { return format == kNvfp4 ? 16 : 32; }
__host__ __device__ constexpr int64_t scale_row_tiles(int64_t rows) { return (rows + 127) / 128; }
__host__ __device__ constexpr int64_t scale_col_tiles(int64_t k, int format) {
    return (k / block_of(format) + 3) / 4;
}
// Byte of row r, block b of a matrix with `col_tiles` tiles to a row of tiles.
__host__ __device__ constexpr int64_t scale_offset(int64_t r, int64_t b, int64_t col_tiles) {
    return ((r >> 7) * col_tiles + (b >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}

// Limit of a kernel's waits.  Test hook: wait `never` (counted from 0) of the first CTA for a copy is on a barrier
// that nothing arrives on; -1: none.
struct WaitLimit {
    uint64_t ns;
    int never;
};

struct QuantArgs {
    const void *x;          // [rows, k]
    uint8_t *codes;         // [rows, k / 2]
    uint8_t *block_scales;  // tiles
    float *row_scales;      // [rows]
    int64_t rows;
    int k;
    int format;
    int rotation;  // 0 or 256
    int dtype;     // CTU_DTYPE_BF16 / FP16
    int num_sms;
    uint32_t *err;
    WaitLimit wait;
    // Rows side by side: up to eight groups of 256 columns, in a warp (8, 4 or 2 of one, two or four groups,
    // else 1); beyond, in a CTA.
    int side_by_side;
    int load_groups;    // groups of 256 columns per tile load (rotation)
};
// `map` (rotation only): x as lines of 64 values, 4 * load_groups of them to a box, 128-byte swizzle.
cudaError_t launch_quantize(const QuantArgs &a, const CUtensorMap &map, cudaStream_t stream);

struct DequantArgs {
    const uint8_t *codes;
    const uint8_t *block_scales;
    const float *row_scales;
    void *out;  // [rows, k]
    int64_t rows;
    int k;
    int format;
    int row_scale_count;  // rows or 1
    int dtype;            // CTU_DTYPE_*
    int num_sms;
};
cudaError_t launch_dequantize(const DequantArgs &a, cudaStream_t stream);
// out[m, n] = bf16(fma(acc * a_scale[m], w_scale[n], bias[n]))
struct LinearArgs {
    const float *a_scale;  // [m]
    const float *w_scale;  // [n] or scalar
    const float *bias;     // [n] or null
    void *out;             // bf16 [m, n]
    uint32_t *err;
    int m, n, k;
    int w_scale_count;
    int format;
    int split;  // CTAs of a cluster that share K (the kernel for few rows)
    WaitLimit wait;
};

// Kernel for few rows: a strip of 128 weight rows per CTA, `tokens` activation rows at a time.
struct SmallKernel {
    const void *kernel;
    int smem;
    int threads;
    int tokens;
    int per_sm;  // CTAs resident on an SM
};
constexpr int kStripRows = 128;
SmallKernel linear_small_kernel(int format, int64_t m);

// CTA-pair product (tcgen05 block-scaled MMA).
constexpr int kPairRows = 256;  // output rows of a pair tile
constexpr int kPairCols = 256;
int linear_pair_smem();
const void *linear_pair_kernel(int format);
int linear_pair_threads(bool few_tiles, int64_t n, int64_t k);

// Gradient with respect to the input: dx[m, k] = grad[m, n] w[n, k], rotated back.
struct GradArgs {
    void *out;        // bf16 [m, k]
    float *partials;  // sums of the split tiles' parts: [tile][part][256 columns][256 rows]
    uint32_t *err;
    int m, n, k;
    int rotation;
    int whole;  // tiles that are not split, the first ones
    int split;  // parts of the others' sums over n
    WaitLimit wait;
};
constexpr int kGradCols = 256;
int grad_pair_smem();
const void *grad_pair_kernel(int rotation);
int grad_pair_threads();
// Joins the partial sums of a split product: sum over parts in order, one rounding.
cudaError_t launch_grad_join(const GradArgs &a, cudaStream_t stream);

}  // namespace fp4
}  // namespace ctu

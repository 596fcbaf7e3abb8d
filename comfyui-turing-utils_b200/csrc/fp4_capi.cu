// C ABI of the 4-bit floating point linear layer and the affine layer norm (include/ctu_b200.h):
// argument checks, tensor maps and launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <mutex>

#include "../../include/ctu_b200.h"
#include "fp4.cuh"
#include "host.cuh"
#include "layer_norm.cuh"
#include "ptx.cuh"

namespace {

using ctu::host::aligned16;
using ctu::host::cuda_fail;
using ctu::host::DeviceQuery;
using ctu::host::encode_tiled;
using ctu::host::fail;
using ctu::host::kernel_device;
namespace fp4 = ctu::fp4;

#define CTU_CUDA(call)                                      \
    do {                                                    \
        cudaError_t e_ = (call);                            \
        if (e_ != cudaSuccess) return cuda_fail(e_, #call); \
    } while (0)

constexpr int64_t kMaxDim = int64_t(1) << 30;

int check_format(const char *what, int format) {
    if (format != CTU_FP4_NVFP4 && format != CTU_FP4_MXFP4)
        return fail(CTU_ERR_INVALID_ARGUMENT, "%s format must be nvfp4 or mxfp4", what);
    return CTU_OK;
}

int check_matrix(const char *what, int64_t rows, int64_t k, int format) {
    if (int rc = check_format(what, format)) return rc;
    if (rows < 0 || k <= 0 || k % 32 != 0)
        return fail(CTU_ERR_INVALID_ARGUMENT, "%s requires K%%32=0 (rows=%lld K=%lld)", what,
                    static_cast<long long>(rows), static_cast<long long>(k));
    if (rows > kMaxDim || k > kMaxDim)
        return fail(CTU_ERR_INVALID_ARGUMENT, "%s dimensions exceed the CUDA kernel range", what);
    return CTU_OK;
}

// Launch plan of a CTA-pair kernel on a device: shared memory opted in and the number of resident
// pairs, found once.
struct PairPlan {
    std::mutex mutex;
    int clusters[64] = {};
};

int pair_clusters(PairPlan &plan, const void *kernel, int threads, int smem, const DeviceQuery &q, int *clusters) {
    std::lock_guard<std::mutex> lock(plan.mutex);
    if (plan.clusters[q.device] == 0) {
        CTU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {2, 1, 1};
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(2 * (q.num_sms / 2), 1, 1);
        cfg.blockDim = dim3(threads, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        CTU_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
        if (n <= 0) return fail(CTU_ERR_UNSUPPORTED, "no CTA pair of the kernel fits on device %d", q.device);
        plan.clusters[q.device] = n;
    }
    *clusters = plan.clusters[q.device];
    return CTU_OK;
}

// Opts a kernel in to its shared memory, once per device.
struct SmemPlan {
    std::mutex mutex;
    bool set[64] = {};
};

int opt_in_smem(SmemPlan &plan, const void *kernel, int smem, int device) {
    std::lock_guard<std::mutex> lock(plan.mutex);
    if (!plan.set[device]) {
        CTU_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        plan.set[device] = true;
    }
    return CTU_OK;
}

int launch_clusters(const void *kernel, int threads, int smem, int64_t ctas, int cluster, void **params,
                    cudaStream_t stream) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CTU_CUDA(cudaLaunchKernelExC(&cfg, kernel, params));
    return CTU_OK;
}

int launch_pairs(const void *kernel, int threads, int smem, int64_t pairs, void **params, cudaStream_t stream) {
    return launch_clusters(kernel, threads, smem, 2 * pairs, 2, params, stream);
}

// Code rows of 128 bytes, `box_rows` of them, and whole scale tiles.
int encode_codes(CUtensorMap *map, const void *codes, int64_t rows, int64_t k, int box_rows) {
    const uint64_t dims[2] = {static_cast<uint64_t>(k / 2), static_cast<uint64_t>(rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(k / 2)};
    const uint32_t box[2] = {128, static_cast<uint32_t>(box_rows)};
    return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int encode_scales(CUtensorMap *map, const void *scales, int64_t rows, int64_t k, int format, int box_cols,
                  int box_rows) {
    const uint64_t cols = static_cast<uint64_t>(fp4::scale_col_tiles(k, format));
    const uint64_t dims[3] = {128, cols, static_cast<uint64_t>(fp4::scale_row_tiles(rows))};
    const uint64_t strides[2] = {512, 512 * cols};
    const uint32_t box[3] = {128, static_cast<uint32_t>(box_cols), static_cast<uint32_t>(box_rows)};
    return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, scales, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Forces a product kernel for tests: 0 by size, 1 the pair kernel, 2 the kernel for few rows.
std::atomic<int> g_fp4_kernel{0};

// The kernel for few rows up to 64 of them, and up to 128 where its strips leave half of the SMs to split
// K over.  us with the weights in the L2, it against the pair kernel: 64 x 5120 x 5120 8.8 / 13.1, 64 x 13824 x 5120 14.0 / 13.5,
// 128 x 5120 x 5120 11.1 / 13.7, 128 x 13824 x 5120 19.4 / 14.3, 128 x 512 x 512 11.0 / 8.2.
bool few_rows(int64_t m, int64_t n, int64_t k, int num_sms) {
    const int64_t strips = (n + fp4::kStripRows - 1) / fp4::kStripRows;
    return m <= 64 || (m <= 128 && 2 * strips <= num_sms && k >= 1024);
}

// Limit of the kernels' waits, and one that a test makes run out.
std::atomic<uint64_t> g_wait_ns{ctu::kWaitLimitNs};
std::atomic<int> g_wait_never{-1};
fp4::WaitLimit wait_limit() {
    return {g_wait_ns.load(std::memory_order_relaxed), g_wait_never.load(std::memory_order_relaxed)};
}

SmemPlan g_small_plan[8];

PairPlan g_linear_plan[2];
PairPlan g_grad_plan[2];

// The gradient's tiles beyond the last full round of pairs (74 on a B200) are split along n, into as many
// parts as lower the time of that round: stages of 64 rows (0.28 us) over the rounds that the parts need,
// plus the write and read of their fp32 sums at 5 TB/s (256 KB a part) and of a launch.  4096 x 5120 x 5120
// is 320 tiles, four rounds and 24 tiles in three parts each; 333 x 13824 x 5120 is 40 tiles of 216 stages in
// three parts.  Depends on the sizes alone, so that the workspace and the sums' order do.
struct GradPlan {
    int64_t tiles, whole, split;
};

GradPlan grad_plan(int64_t m, int64_t n, int64_t k) {
    constexpr int64_t kPairs = 74;
    GradPlan p{};
    p.tiles = ((m + fp4::kPairRows - 1) / fp4::kPairRows) * ((k + fp4::kGradCols - 1) / fp4::kGradCols);
    const int64_t stages = (n + 63) / 64;
    p.whole = p.tiles / kPairs * kPairs;
    p.split = 1;
    const int64_t tail = p.tiles - p.whole;
    double cost = static_cast<double>(stages);
    for (int64_t s = 2; tail > 0 && s <= 16 && 2 * s <= stages; ++s) {
        const double rounds = static_cast<double>((tail * s + kPairs - 1) / kPairs * ((stages + s - 1) / s));
        const double c = rounds + 12.0 + 0.374 * static_cast<double>(s * tail);
        if (c < cost) {
            cost = c;
            p.split = s;
        }
    }
    if (p.split == 1) p.whole = p.tiles;
    return p;
}

}  // namespace

extern "C" {

int64_t ctu_fp4_block_scale_bytes(int64_t rows, int64_t k, int format) {
    if (rows <= 0 || k <= 0 || (format != CTU_FP4_NVFP4 && format != CTU_FP4_MXFP4)) return 0;
    return fp4::scale_row_tiles(rows) * fp4::scale_col_tiles(k, format) * 512;
}

int ctu_fp4_quantize(const void *x, int64_t rows, int64_t k, int dtype, int format, int rotation, uint8_t *codes,
                     uint8_t *block_scales, float *row_scales, void *stream) {
    if (int rc = check_matrix("FP4 quantizer", rows, k, format)) return rc;
    if (dtype != CTU_DTYPE_BF16 && dtype != CTU_DTYPE_FP16)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 quantizer input must be float16 or bfloat16");
    if (rotation != 0 && rotation != 256)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 quantizer rotation must be 0 or 256");
    if (rotation != 0 && k % rotation != 0)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 quantizer width must be divisible by the rotation block (%d)", rotation);
    if (k > CTU_FP4_MAX_QUANTIZE_K)
        return fail(CTU_ERR_UNSUPPORTED, "FP4 quantizer takes rows of at most %d columns", CTU_FP4_MAX_QUANTIZE_K);
    if (rows == 0) return CTU_OK;
    if (!x || !codes || !block_scales || !row_scales) return fail(CTU_ERR_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned16(x) || !aligned16(codes) || !aligned16(block_scales))
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 quantizer tensors must be 16-byte aligned");
    DeviceQuery q;
    uint32_t *err;
    if (int rc = kernel_device(&q, &err)) return rc;
    fp4::QuantArgs a{x, codes, block_scales, row_scales, rows, static_cast<int>(k), format, rotation, dtype, q.num_sms, err, wait_limit()};
    const int groups = static_cast<int>((k + 255) / 256);
    a.side_by_side = groups == 1 ? 8 : groups == 2 ? 4 : groups <= 4 ? 2 : 1;
    // A CTA's warps hold eight groups each: two rows where one would leave more than a tenth of the lanes
    // idle and two leave fewer (20 groups: 2.5 warps a row, five for two).
    if (groups > 8) {
        auto idle = [&](int rows) { return static_cast<double>((groups * rows + 7) / 8 * 8) / (groups * rows) - 1.0; };
        a.side_by_side = groups <= 64 && idle(1) > 0.1 && idle(2) < idle(1) ? 2 : 1;
    }
    CUtensorMap map{};
    if (rotation != 0) {
        // Rows of three groups do not lie side by side: one to a warp.
        if (groups == 3) a.side_by_side = 1;
        const int held = groups * a.side_by_side;
        a.load_groups = held % 8 == 0 ? 8 : held % 4 == 0 ? 4 : 2;
        const uint64_t lines = static_cast<uint64_t>(rows) * static_cast<uint64_t>(k / 64);
        if (lines > INT32_MAX) return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 quantizer dimensions exceed the CUDA kernel range");
        const uint64_t dims[2] = {64, lines};
        const uint64_t strides[1] = {128};
        const uint32_t box[2] = {64, static_cast<uint32_t>(4 * a.load_groups)};
        if (int rc = encode_tiled(&map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, x, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
            return rc;
    }
    CTU_CUDA(fp4::launch_quantize(a, map, static_cast<cudaStream_t>(stream)));
    return CTU_OK;
}

int ctu_fp4_dequantize(const uint8_t *codes, const uint8_t *block_scales, const float *row_scales,
                       int64_t row_scale_count, int64_t rows, int64_t k, int format, int dtype, void *out,
                       void *stream) {
    if (int rc = check_matrix("FP4 dequantizer", rows, k, format)) return rc;
    if (dtype < CTU_DTYPE_BF16 || dtype > CTU_DTYPE_FP32)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 dequantizer output must be float16, bfloat16, or float32");
    if (rows * ((k + 1023) / 1024) > INT32_MAX)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 dequantizer dimensions exceed the CUDA kernel range");
    if (row_scale_count != 1 && row_scale_count != rows)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 dequantizer requires one row scale or one per row");
    if (rows == 0) return CTU_OK;
    if (!codes || !block_scales || !row_scales || !out) return fail(CTU_ERR_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned16(codes) || !aligned16(block_scales) || !aligned16(out))
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 dequantizer tensors must be 16-byte aligned");
    DeviceQuery q;
    uint32_t *err;
    if (int rc = kernel_device(&q, &err)) return rc;
    fp4::DequantArgs a{codes, block_scales, row_scales, out, rows, static_cast<int>(k), format,
                       row_scale_count == 1 ? 1 : 0, dtype, q.num_sms};
    CTU_CUDA(fp4::launch_dequantize(a, static_cast<cudaStream_t>(stream)));
    return CTU_OK;
}

int ctu_fp4_linear(const uint8_t *a, const uint8_t *w, const uint8_t *a_block_scales, const uint8_t *w_block_scales,
                   const float *a_scale, const float *w_scale, int64_t w_scale_count, const float *bias, void *out,
                   int64_t m, int64_t n, int64_t k, int format, void *stream) {
    if (int rc = check_matrix("FP4 linear", m, k, format)) return rc;
    if (int rc = check_matrix("FP4 linear", n, k, format)) return rc;
    if (w_scale_count != 1 && w_scale_count != n)
        return fail(CTU_ERR_INVALID_ARGUMENT, "weight scale must be scalar or one per output channel");
    if (m == 0 || n == 0) return CTU_OK;
    if (!a || !w || !a_block_scales || !w_block_scales || !a_scale || !w_scale || !out)
        return fail(CTU_ERR_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned16(a) || !aligned16(w) || !aligned16(a_block_scales) || !aligned16(w_block_scales) || !aligned16(out))
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 linear tensors must be 16-byte aligned");
    const int64_t tiles = ((m + fp4::kPairRows - 1) / fp4::kPairRows) * ((n + fp4::kPairCols - 1) / fp4::kPairCols);
    if (tiles > INT32_MAX / 2) return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 linear dimensions exceed the CUDA kernel range");
    DeviceQuery q;
    uint32_t *err;
    if (int rc = kernel_device(&q, &err)) return rc;
    const int col_tiles = format == CTU_FP4_NVFP4 ? 4 : 2;
    fp4::LinearArgs args{a_scale, w_scale, bias, out, err, static_cast<int>(m), static_cast<int>(n),
                         static_cast<int>(k), w_scale_count == 1 ? 1 : 0, format, 1, wait_limit()};
    const int forced = g_fp4_kernel.load(std::memory_order_relaxed);
    if (forced == 2 || (forced == 0 && few_rows(m, n, k, q.num_sms))) {
        const fp4::SmallKernel sk = fp4::linear_small_kernel(format, m);
        const int64_t strips =
            ((m + sk.tokens - 1) / sk.tokens) * ((n + fp4::kStripRows - 1) / fp4::kStripRows);
        const int64_t slots = static_cast<int64_t>(q.num_sms) * sk.per_sm;
        const int64_t stages = (k + 255) / 256;
        if (strips > INT32_MAX / 8)
            return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 linear dimensions exceed the CUDA kernel range");
        args.split = static_cast<int>(std::max<int64_t>(1, std::min({int64_t(8), slots / strips, stages})));
        CUtensorMap map_w, map_a, map_ws, map_as;
        if (int rc = encode_codes(&map_w, w, n, k, fp4::kStripRows)) return rc;
        if (int rc = encode_codes(&map_a, a, m, k, sk.tokens)) return rc;
        if (int rc = encode_scales(&map_ws, w_block_scales, n, k, format, col_tiles, 1)) return rc;
        if (int rc = encode_scales(&map_as, a_block_scales, m, k, format, col_tiles, 1)) return rc;
        const int which = (sk.tokens == 16 ? 0 : sk.tokens == 32 ? 1 : sk.tokens == 64 ? 2 : 3) + 4 * format;
        if (int rc = opt_in_smem(g_small_plan[which], sk.kernel, sk.smem, q.device)) return rc;
        void *params[] = {&map_w, &map_a, &map_ws, &map_as, &args};
        return launch_clusters(sk.kernel, sk.threads, sk.smem, strips * args.split, args.split, params,
                               static_cast<cudaStream_t>(stream));
    }
    CUtensorMap map_a, map_b, map_as, map_bs;
    if (int rc = encode_codes(&map_a, a, m, k, 128)) return rc;
    if (int rc = encode_codes(&map_b, w, n, k, fp4::kPairCols / 2)) return rc;
    if (int rc = encode_scales(&map_as, a_block_scales, m, k, format, col_tiles, 1)) return rc;
    if (int rc = encode_scales(&map_bs, w_block_scales, n, k, format, col_tiles, 2)) return rc;
    // The output's tile stores need rows on 16 bytes; others are written by the kernel's warps.
    CUtensorMap map_out = map_a;
    if (n % 8 == 0) {
        const uint64_t dims[2] = {static_cast<uint64_t>(n), static_cast<uint64_t>(m)};
        const uint64_t strides[1] = {static_cast<uint64_t>(2 * n)};
        const uint32_t box[2] = {64, 32};
        if (int rc = encode_tiled(&map_out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out, dims, strides, box,
                                  CU_TENSOR_MAP_SWIZZLE_128B))
            return rc;
    }
    const void *kernel = fp4::linear_pair_kernel(format);
    int clusters = 0;
    if (int rc = pair_clusters(g_linear_plan[format], kernel, fp4::linear_pair_threads(true, n, k),
                               fp4::linear_pair_smem(), q, &clusters))
        return rc;
    void *params[] = {&map_a, &map_b, &map_as, &map_bs, &map_out, &args};
    return launch_pairs(kernel, fp4::linear_pair_threads(tiles <= 2 * clusters, n, k), fp4::linear_pair_smem(),
                        std::min<int64_t>(tiles, clusters), params, static_cast<cudaStream_t>(stream));
}

int ctu_debug_set_fp4_kernel(int which) {
    if (which < 0 || which > 2) return fail(CTU_ERR_INVALID_ARGUMENT, "unknown FP4 product kernel %d", which);
    return g_fp4_kernel.exchange(which);
}

int ctu_debug_inject_timeout(int which, uint64_t limit_ns) {
    if (which >= 0 && (limit_ns == 0 || limit_ns > 5000000000ull))
        return fail(CTU_ERR_INVALID_ARGUMENT, "wait limit must be in (0, 5 s]");
    g_wait_ns.store(which < 0 ? ctu::kWaitLimitNs : limit_ns, std::memory_order_relaxed);
    g_wait_never.store(which < 0 ? -1 : which, std::memory_order_relaxed);
    return CTU_OK;
}

int64_t ctu_fp4_grad_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    const GradPlan p = grad_plan(m, n, k);
    return 2 * n * k + (p.tiles - p.whole) * p.split * fp4::kPairRows * fp4::kGradCols * 4;
}

int ctu_fp4_linear_grad_input(const void *grad, const uint8_t *w, const uint8_t *w_block_scales, const float *w_scale,
                              int64_t w_scale_count, int rotation, void *workspace, void *dx, int64_t m, int64_t n,
                              int64_t k, int format, void *stream) {
    if (int rc = check_matrix("FP4 linear gradient", m, k, format)) return rc;
    if (n <= 0 || n % 8 != 0 || n > kMaxDim)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 linear gradient requires N%%8=0 (N=%lld)", static_cast<long long>(n));
    if (rotation != 0 && rotation != 256)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 linear gradient rotation must be 0 or 256");
    if (rotation != 0 && k % rotation != 0)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 linear gradient width must be divisible by the rotation block (%d)",
                    rotation);
    if (w_scale_count != 1 && w_scale_count != n)
        return fail(CTU_ERR_INVALID_ARGUMENT, "weight scale must be scalar or one per output channel");
    if (m == 0) return CTU_OK;
    if (!grad || !w || !w_block_scales || !w_scale || !workspace || !dx)
        return fail(CTU_ERR_INVALID_ARGUMENT, "null tensor pointer");
    if (!aligned16(grad) || !aligned16(w) || !aligned16(w_block_scales) || !aligned16(workspace) || !aligned16(dx))
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 linear gradient tensors must be 16-byte aligned");
    const int64_t tiles = ((m + fp4::kPairRows - 1) / fp4::kPairRows) * ((k + fp4::kGradCols - 1) / fp4::kGradCols);
    if (tiles > INT32_MAX / 16 || n * ((k + 1023) / 1024) > INT32_MAX)
        return fail(CTU_ERR_INVALID_ARGUMENT, "FP4 linear gradient dimensions exceed the CUDA kernel range");
    DeviceQuery q;
    uint32_t *err;
    if (int rc = kernel_device(&q, &err)) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    fp4::DequantArgs d{w, w_block_scales, w_scale, workspace, n, static_cast<int>(k), format, w_scale_count == 1 ? 1 : 0,
                       CTU_DTYPE_BF16, q.num_sms};
    CUtensorMap map_a, map_b, map_out;
    const uint32_t box_a[2] = {64, 128}, box_b[2] = {64, 64};
    const uint64_t dims_a[2] = {static_cast<uint64_t>(n), static_cast<uint64_t>(m)};
    const uint64_t dims_b[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(n)};
    const uint64_t stride_a[1] = {static_cast<uint64_t>(2 * n)}, stride_b[1] = {static_cast<uint64_t>(2 * k)};
    if (int rc = encode_tiled(&map_a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, grad, dims_a, stride_a, box_a,
                              CU_TENSOR_MAP_SWIZZLE_128B))
        return rc;
    if (int rc = encode_tiled(&map_b, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, workspace, dims_b, stride_b, box_b,
                              CU_TENSOR_MAP_SWIZZLE_128B))
        return rc;
    const uint32_t box_out[2] = {64, 32};
    const uint64_t dims_out[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(m)};
    if (int rc = encode_tiled(&map_out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, dx, dims_out, stride_b, box_out,
                              CU_TENSOR_MAP_SWIZZLE_128B))
        return rc;
    const void *kernel = fp4::grad_pair_kernel(rotation);
    int clusters = 0;
    if (int rc = pair_clusters(g_grad_plan[rotation ? 1 : 0], kernel, fp4::grad_pair_threads(), fp4::grad_pair_smem(), q,
                               &clusters))
        return rc;
    CTU_CUDA(fp4::launch_dequantize(d, s));
    const GradPlan plan = grad_plan(m, n, k);
    fp4::GradArgs args{dx, reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + 2 * n * k), err,
                       static_cast<int>(m), static_cast<int>(n), static_cast<int>(k), rotation, static_cast<int>(plan.whole),
                       static_cast<int>(plan.split), wait_limit()};
    void *params[] = {&map_a, &map_b, &map_out, &args};
    if (int rc = launch_pairs(kernel, fp4::grad_pair_threads(), fp4::grad_pair_smem(),
                              std::min<int64_t>(plan.whole + (plan.tiles - plan.whole) * plan.split, clusters), params, s))
        return rc;
    if (plan.whole < plan.tiles) CTU_CUDA(fp4::launch_grad_join(args, s));
    return CTU_OK;
}

// ---------------------------------------------------------------------------- affine layer norm
static int check_layer_norm(int64_t rows, int64_t hidden, int dtype, int weight_dtype) {
    if (dtype < CTU_DTYPE_BF16 || dtype > CTU_DTYPE_FP32)
        return fail(CTU_ERR_INVALID_ARGUMENT, "LayerNorm input must be float16, bfloat16, or float32");
    if (weight_dtype != dtype && weight_dtype != CTU_DTYPE_FP32)
        return fail(CTU_ERR_INVALID_ARGUMENT, "LayerNorm weight and bias must have the input's type or float32");
    if (rows < 0 || hidden <= 0) return fail(CTU_ERR_INVALID_ARGUMENT, "LayerNorm dimensions must be positive");
    if (rows > kMaxDim || hidden > kMaxDim)
        return fail(CTU_ERR_INVALID_ARGUMENT, "LayerNorm dimensions exceed the CUDA kernel range");
    return CTU_OK;
}

int ctu_layer_norm(const void *x, const void *weight, const void *bias, void *out, float *mean, float *rstd,
                   int64_t rows, int64_t hidden, float epsilon, int dtype, int weight_dtype, void *stream) {
    if (int rc = check_layer_norm(rows, hidden, dtype, weight_dtype)) return rc;
    if (!(std::isfinite(epsilon) && epsilon > 0.0f))
        return fail(CTU_ERR_INVALID_ARGUMENT, "LayerNorm epsilon must be finite and positive");
    if (rows == 0) return CTU_OK;
    if (!x || !out || !mean || !rstd) return fail(CTU_ERR_INVALID_ARGUMENT, "null tensor pointer");
    DeviceQuery q;
    uint32_t *err;
    if (int rc = kernel_device(&q, &err)) return rc;
    ctu::norm::AffineArgs a{};
    a.x = x;
    a.weight = weight;
    a.bias = bias;
    a.out = out;
    a.mean = mean;
    a.rstd = rstd;
    a.rows = rows;
    a.hidden = static_cast<int>(hidden);
    a.epsilon = epsilon;
    a.dtype = dtype;
    a.weight_dtype = weight_dtype;
    a.num_sms = q.num_sms;
    CTU_CUDA(ctu::norm::launch_layer_norm(a, static_cast<cudaStream_t>(stream)));
    return CTU_OK;
}

int64_t ctu_layer_norm_backward_workspace_bytes(int64_t rows, int64_t hidden) {
    if (rows < 0 || hidden <= 0) return 0;
    return 2 * ctu::norm::backward_slices(rows, hidden) * hidden * static_cast<int64_t>(sizeof(float));
}

int ctu_layer_norm_backward(const void *grad, const void *x, const void *weight, const float *mean, const float *rstd,
                            void *dx, void *dweight, void *dbias, void *workspace, int64_t rows, int64_t hidden,
                            int dtype, int weight_dtype, void *stream) {
    if (int rc = check_layer_norm(rows, hidden, dtype, weight_dtype)) return rc;
    if (!dx && !dweight && !dbias) return CTU_OK;
    if (rows == 0 && !dweight && !dbias) return CTU_OK;
    if (rows > 0 && (!grad || !x || !mean || !rstd)) return fail(CTU_ERR_INVALID_ARGUMENT, "null tensor pointer");
    if ((dweight || dbias) && !workspace) return fail(CTU_ERR_INVALID_ARGUMENT, "null workspace pointer");
    DeviceQuery q;
    uint32_t *err;
    if (int rc = kernel_device(&q, &err)) return rc;
    ctu::norm::AffineArgs a{};
    a.x = x;
    a.weight = weight;
    a.mean = const_cast<float *>(mean);
    a.rstd = const_cast<float *>(rstd);
    a.grad = grad;
    a.dx = dx;
    a.dweight = dweight;
    a.dbias = dbias;
    a.workspace = static_cast<float *>(workspace);
    a.rows = rows;
    a.hidden = static_cast<int>(hidden);
    a.dtype = dtype;
    a.weight_dtype = weight_dtype;
    a.num_sms = q.num_sms;
    a.err = err;
    const fp4::WaitLimit wait = wait_limit();
    CTU_CUDA(ctu::norm::launch_layer_norm_backward(a, {wait.ns, wait.never}, static_cast<cudaStream_t>(stream)));
    return CTU_OK;
}

}  // extern "C"

// Gradient of the 4-bit linear layer with respect to its input (CTA pair, tcgen05 bf16 MMA):
//
//   dx[m, k] = sum_n grad[m, n] * w[n, k],  then rotated back (the rotation is its own inverse)
//
// The weights arrive decoded to bf16 [k, n] (code * block scale has six significant bits, a
// power-of-two channel scale adds none, so the decoding of this library's own weights is exact).
// A pair of CTAs owns a 256 x 256 tile of dx; accumulators are fp32, and a rotation block of 256
// columns lies inside one tile, so the rotation runs on the fp32 sums: an epilogue thread holds one
// row and takes the strides 1, 4 and 16 in registers, 64 columns at a time, writes them back to
// tensor memory, and takes stride 64 from there.  Rounded once, to bf16.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "fp4.cuh"
#include "fp4_mma.cuh"
#include "ptx.cuh"

namespace ctu {
namespace fp4 {

namespace {

constexpr int kStages = 6;
constexpr int kStageK = 64;  // bf16 values of the contraction per stage: 128 bytes
constexpr int kABytes = 128 * 128;
constexpr int kBBytes = 128 * 128;
constexpr int kBOffset = kStages * kABytes;
constexpr int kStructOffset = kBOffset + kStages * kBBytes;
constexpr int kEpilogueWarps = 4;
constexpr int kThreadCount = 32 * (2 + kEpilogueWarps);
constexpr int kTmemCols = 512;

struct Shared {
    uint64_t full[kStages];
    uint64_t empty[kStages];
    uint64_t acc_full[2];
    uint64_t acc_empty[2];
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
};

constexpr int kSmem = kStructOffset + static_cast<int>(sizeof(Shared)) + 1024;
static_assert(kSmem <= 232448, "shared memory of one CTA");

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

__device__ __forceinline__ void radix4(uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    const float x0 = __uint_as_float(r0), x1 = __uint_as_float(r1), x2 = __uint_as_float(r2), x3 = __uint_as_float(r3);
    const float t = x0 + x1, b = x0 - x1;
    r0 = __float_as_uint((t + x2) - x3);
    r1 = __float_as_uint((t - x2) + x3);
    r2 = __float_as_uint((b + x2) + x3);
    r3 = __float_as_uint((x2 - b) + x3);
}

__device__ __forceinline__ void store_row16(__nv_bfloat16 *dst, const uint32_t *r) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            p[j] = pack_bf16x2(__uint_as_float(r[8 * q + 2 * j]), __uint_as_float(r[8 * q + 2 * j + 1]));
        reinterpret_cast<uint4 *>(dst)[q] = make_uint4(p[0], p[1], p[2], p[3]);
    }
}

}  // namespace

template <bool kRotate>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreadCount, 1)
    fp4_grad_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                         const GradArgs args) {
    constexpr uint32_t kStageTx = 2 * (kABytes + kBBytes);
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Shared &S = *reinterpret_cast<Shared *>(smem + kStructOffset);

    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int pair = blockIdx.x >> 1;
    const int num_pairs = gridDim.x >> 1;
    const int num_n = (args.k + kGradCols - 1) / kGradCols;
    const int num_m = (args.m + kPairRows - 1) / kPairRows;
    const int num_tiles = num_m * num_n;
    const int nk = (args.n + kStageK - 1) / kStageK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&S.acc_full[b], 1);
            mbar_init(&S.acc_empty[b], 2 * kEpilogueWarps);
        }
        mbar_init(&S.drain, 1);
        S.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(&S.tmem_base, kTmemCols);
        tmem_relinquish_pair();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = S.tmem_base;
    const PairAbort guard{&S.abort_flag, mapa_shared(smem_u32(&S.abort_flag), rank ^ 1u), args.err};
    volatile int *abort_flag = &S.abort_flag;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = pair; t < num_tiles && ok; t += num_pairs) {
                const int m0 = (t / num_n) * kPairRows + static_cast<int>(rank) * 128;
                const int n0 = (t % num_n) * kGradCols + static_cast<int>(rank) * 128;
                for (int kb = 0; kb < nk; ++kb) {
                    if (!guard.wait(&S.empty[s], ph ^ 1u, kErrTimeoutEmpty)) {
                        ok = false;
                        break;
                    }
                    const uint32_t full = mapa_shared(smem_u32(&S.full[s]), 0u);
                    if (leader) mbar_arrive_expect_tx(&S.full[s], kStageTx);
                    tma_load_2d_pair(smem + s * kABytes, &tmap_a, kb * kStageK, m0, full);
                    tma_load_2d_pair(smem + kBOffset + s * kBBytes, &tmap_b, kb * kStageK, n0, full);
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            if (!ok || *abort_flag) settle_inflight_copies();
        }
    } else if (warp == 1) {
        if (leader && lane == 0) {
            constexpr uint32_t idesc = idesc_bf16(kPairRows, kGradCols);
            int s = 0;
            uint32_t ph = 0;
            int local = 0;
            bool ok = true;
            for (int t = pair; t < num_tiles && ok; t += num_pairs, ++local) {
                const int ab = local & 1;
                if (!guard.wait_cluster(&S.acc_empty[ab], ((local >> 1) & 1) ^ 1u, kErrTimeoutAccumFree)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem_base + static_cast<uint32_t>(ab * kGradCols);
                for (int kb = 0; kb < nk; ++kb) {
                    if (!guard.wait(&S.full[s], ph, kErrTimeoutFull)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem + s * kABytes);
                    const uint32_t b = smem_u32(smem + kBOffset + s * kBBytes);
#pragma unroll
                    for (int c = 0; c < kStageK / 16; ++c)
                        mma_bf16_pair(d, smem_desc_sw128(a + 32 * c), smem_desc_sw128(b + 32 * c), idesc,
                                      (kb | c) != 0 ? 1u : 0u);
                    mma_commit_pair_both(&S.empty[s]);
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                if (!ok) break;
                mma_commit_pair_both(&S.acc_full[ab]);
            }
            mma_commit_pair_local(&S.drain);
            mbar_wait(&S.drain, 0u, nullptr, args.err, kErrTimeoutDrain);
        }
    } else {
        const int quad = warp & 3;
        const uint32_t leader_empty = mapa_shared(smem_u32(&S.acc_empty[0]), 0u);
        bool alive = true;
        int local = 0;
        for (int t = pair; t < num_tiles; t += num_pairs, ++local) {
            const int ab = local & 1;
            if (alive) {
                int ok = 1;
                if (lane == 0) ok = guard.wait(&S.acc_full[ab], (local >> 1) & 1, kErrTimeoutAccum) ? 1 : 0;
                alive = __shfl_sync(0xffffffffu, ok, 0) != 0;
            }
            if (!alive) continue;
            tc_fence_after();
            const int m = (t / num_n) * kPairRows + static_cast<int>(rank) * 128 + quad * 32 + lane;
            const int n0 = (t % num_n) * kGradCols;
            const bool row_ok = m < args.m;
            const uint32_t acc = tmem_base + static_cast<uint32_t>(ab * kGradCols) + (static_cast<uint32_t>(quad * 32) << 16);
            __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(args.out) + static_cast<int64_t>(m) * args.k + n0;
            if constexpr (kRotate) {
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t lo[32], hi[32];
                    tmem_ld_32x32b_x32(acc + c * 64, lo);
                    tmem_ld_32x32b_x32(acc + c * 64 + 32, hi);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        lo[j] = __float_as_uint(__uint_as_float(lo[j]) * 0.0625f);
                        hi[j] = __float_as_uint(__uint_as_float(hi[j]) * 0.0625f);
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        radix4(lo[j], lo[j + 1], lo[j + 2], lo[j + 3]);
                        radix4(hi[j], hi[j + 1], hi[j + 2], hi[j + 3]);
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 16) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            radix4(lo[j + i], lo[j + i + 4], lo[j + i + 8], lo[j + i + 12]);
                            radix4(hi[j + i], hi[j + i + 4], hi[j + i + 8], hi[j + i + 12]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) radix4(lo[i], lo[i + 16], hi[i], hi[i + 16]);
                    tmem_st_32x32b_x32(acc + c * 64, lo);
                    tmem_st_32x32b_x32(acc + c * 64 + 32, hi);
                }
                tmem_st_wait();
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t r[4][16];
#pragma unroll
                    for (int q = 0; q < 4; ++q) tmem_ld_32x32b_x16(acc + q * 64 + c * 16, r[q]);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; ++i) radix4(r[0][i], r[1][i], r[2][i], r[3][i]);
                    if (row_ok) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) store_row16(dst + q * 64 + c * 16, r[q]);
                    }
                }
            } else {
#pragma unroll 1
                for (int c = 0; c < 16; ++c) {
                    uint32_t r[16];
                    tmem_ld_32x32b_x16(acc + c * 16, r);
                    tmem_ld_wait();
                    if (row_ok && n0 + c * 16 < args.k) store_row16(dst + c * 16, r);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(leader_empty + static_cast<uint32_t>(ab * sizeof(uint64_t)));
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

int grad_pair_smem() { return kSmem; }
int grad_pair_threads() { return kThreadCount; }
const void *grad_pair_kernel(int rotation) {
    return rotation ? reinterpret_cast<const void *>(&fp4_grad_pair_kernel<true>)
                    : reinterpret_cast<const void *>(&fp4_grad_pair_kernel<false>);
}

}  // namespace fp4
}  // namespace ctu

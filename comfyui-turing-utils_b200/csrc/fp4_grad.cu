// Gradient of the 4-bit linear layer with respect to its input (CTA pair, tcgen05 bf16 MMA):
//
//   dx[m, k] = sum_n grad[m, n] * w[n, k],  then rotated back (the rotation is its own inverse)
//
// The weights arrive decoded to bf16 [n, k] (code * block scale has six significant bits, a
// power-of-two channel scale adds none, so the decoding of this library's own weights is exact).  The
// sum runs over their rows, so the MMA reads them with k as the contiguous dimension (MN-major B).
// A pair of CTAs owns a 256 x 256 tile of dx; accumulators are fp32, and a rotation block of 256
// columns lies inside one tile, so the rotation runs on the fp32 sums: an epilogue thread holds one
// row and takes the strides 1, 4 and 16 in registers, 64 columns at a time, writes them back to
// tensor memory, and takes stride 64 from there.  Rounded once, to bf16.
//
// Tiles beyond the last full round of pairs are split along n; each part leaves its fp32 sums (rotated: the
// rotation is linear), tile by tile and a column's rows together, so that a warp's store is 128 contiguous
// bytes; a second kernel adds the parts in order, transposes and rounds.  Whole tiles go out through staged
// tile stores.
//
// Measured: 4096 x 5120 x 5120 134 us (1.60 PFLOP/s, bound by the tensor pipe), 11 for decoding and 4 for
// joining; 149 us without the split of the last round.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>

#include "fp4.cuh"
#include "fp4_mma.cuh"
#include "ptx.cuh"

namespace ctu {
namespace fp4 {

namespace {

constexpr int kStages = 5;
constexpr int kStageK = 64;  // bf16 values of the contraction per stage: 128 bytes
constexpr int kABytes = 128 * 128;
constexpr int kBBytes = 128 * 128;
constexpr int kBOffset = kStages * kABytes;
constexpr int kStageOutOffset = kBOffset + kStages * kBBytes;
constexpr int kEpilogueWarps = 4;
constexpr int kPieceBytes = 32 * 128;  // a warp's 32 rows of 64 output columns
constexpr int kStructOffset = kStageOutOffset + kEpilogueWarps * 4 * kPieceBytes;
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

// 16 columns of a staged row (128-byte swizzle), `c` the quarter of the piece's 64.
__device__ __forceinline__ void stage16(uint32_t piece, int c, uint32_t lane, const uint32_t *r) {
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q) {
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            p[j] = pack_bf16x2(__uint_as_float(r[8 * q + 2 * j]), __uint_as_float(r[8 * q + 2 * j + 1]));
        st_shared_v4(piece + 128u * lane + (((2u * c + q) ^ (lane & 7u)) << 4), p);
    }
}
// 16 columns of a part's sums: a column's 256 rows lie together.
__device__ __forceinline__ void store_sums16(float *dst, const uint32_t *r) {
#pragma unroll
    for (int j = 0; j < 16; ++j) dst[j * 256] = __uint_as_float(r[j]);
}

}  // namespace

template <bool kRotate>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreadCount, 1)
    fp4_grad_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                         const __grid_constant__ CUtensorMap tmap_out, const GradArgs args) {
    constexpr uint32_t kStageTx = 2 * (kABytes + kBBytes);
    // B: 64 rows of n by 128 columns of k, as two pieces of 64 columns; eight rows 1024 bytes apart.
    constexpr uint32_t kDescBHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
    constexpr uint32_t kDescBLow = (8192u >> 4) << 16;
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
    const int tiles = num_m * num_n;
    const int num_tiles = args.whole + (tiles - args.whole) * args.split;  // work items
    const int nk_all = (args.n + kStageK - 1) / kStageK;
    // Work items: the first `whole` tiles, then the parts of the others.  Item t sums stages [first, last) of
    // its tile; `part` counts the parts' sums, -1 for a whole tile.
    auto work_item = [&](int t, int &m_tile, int &n_tile, int &part, int &first, int &last) {
        int tile = t;
        part = -1;
        first = 0;
        last = nk_all;
        if (t >= args.whole) {
            part = t - args.whole;
            tile = args.whole + part / args.split;
            const int i = part % args.split;
            first = static_cast<int>(static_cast<int64_t>(nk_all) * i / args.split);
            last = static_cast<int>(static_cast<int64_t>(nk_all) * (i + 1) / args.split);
        }
        n_tile = tile / num_m;  // down the rows first: pairs at work share panels of the weights
        m_tile = tile - n_tile * num_m;
    };

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
        prefetch_tmap(&tmap_out);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = S.tmem_base;
    const PairAbort guard{&S.abort_flag, mapa_shared(smem_u32(&S.abort_flag), rank ^ 1u), args.err, args.wait.ns};
    volatile int *abort_flag = &S.abort_flag;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = pair; t < num_tiles && ok; t += num_pairs) {
                int m_tile, n_tile, part, first, last;
                work_item(t, m_tile, n_tile, part, first, last);
                const int m0 = m_tile * kPairRows + static_cast<int>(rank) * 128;
                const int n0 = n_tile * kGradCols + static_cast<int>(rank) * 128;
                for (int kb = first; kb < last; ++kb) {
                    if (!guard.wait(&S.empty[s], ph ^ 1u, kErrTimeoutEmpty)) {
                        ok = false;
                        break;
                    }
                    const uint32_t full = mapa_shared(smem_u32(&S.full[s]), 0u);
                    if (leader) mbar_arrive_expect_tx(&S.full[s], kStageTx);
                    tma_load_2d_pair(smem + s * kABytes, &tmap_a, kb * kStageK, m0, full);
                    tma_load_2d_pair(smem + kBOffset + s * kBBytes, &tmap_b, n0, kb * kStageK, full);
                    tma_load_2d_pair(smem + kBOffset + s * kBBytes + 8192, &tmap_b, n0 + 64, kb * kStageK, full);
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (leader) {
            // Warp-uniform, one elected lane issues (see the 4-bit product).
            constexpr uint32_t idesc = idesc_bf16(kPairRows, kGradCols) | (1u << 16);  // B is MN-major
            int s = 0;
            uint32_t ph = 0;
            int local = 0;
            bool ok = true;
            const uint32_t a0 = smem_desc_low(smem_u32(smem));
            const uint32_t b0 = ((smem_u32(smem + kBOffset) & 0x3FFFFu) >> 4) | kDescBLow;
            const uint32_t empty0 = smem_u32(&S.empty[0]);
            int left = pair == 0 && args.wait.never >= 0 ? args.wait.never : INT_MAX;  // stages until the test's wait
            for (int t = pair; t < num_tiles && ok; t += num_pairs, ++local) {
                int m_tile, n_tile, part, first, last;
                work_item(t, m_tile, n_tile, part, first, last);
                const uint32_t ab = local & 1;
                ok = __all_sync(0xffffffffu, guard.wait_cluster(&S.acc_empty[ab], ((local >> 1) & 1) ^ 1u, kErrTimeoutAccumFree));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem_base + ab * kGradCols;
                const int stop = first + min(last - first, left);
                left -= stop - first;
                for (int kb = first; kb < stop; ++kb) {
                    ok = __all_sync(0xffffffffu, guard.wait(&S.full[s], ph, kErrTimeoutFull));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t a = a0 + s * (kABytes >> 4);
                    const uint32_t b = b0 + s * (kBBytes >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int c = 0; c < kStageK / 16; ++c)
                            mma_bf16_pair(d, desc64(a + 2 * c, kDescSw128High), desc64(b + 128 * c, kDescBHigh), idesc,
                                          (kb != first || c != 0) ? 1u : 0u);
                        mma_commit_pair_both_at(empty0 + 8 * s);
                        if (kb == last - 1) mma_commit_pair_both(&S.acc_full[ab]);
                    }
                    __syncwarp();
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                if (ok && stop < last) ok = __all_sync(0xffffffffu, guard.wait(&S.drain, 0u, kErrTimeoutFull));
            }
            if (elect_one()) {
                mma_commit_pair_local(&S.drain);
                mbar_wait(&S.drain, 0u, nullptr, args.err, kErrTimeoutDrain, args.wait.ns);
            }
            __syncwarp();
        }
    } else {
        const int quad = warp & 3;
        const uint32_t leader_empty = mapa_shared(smem_u32(&S.acc_empty[0]), 0u);
        const uint32_t staged = smem_u32(smem + kStageOutOffset + (warp - 2) * 4 * kPieceBytes);
        const uint64_t policy = evict_first_policy();
        bool alive = true;
        int local = 0;
        for (int t = pair; t < num_tiles; t += num_pairs, ++local) {
            const int ab = local & 1;
            if (alive) alive = __all_sync(0xffffffffu, guard.wait(&S.acc_full[ab], (local >> 1) & 1, kErrTimeoutAccum));
            tc_fence_after();
            int m_tile, n_tile, part, first, last;
            work_item(t, m_tile, n_tile, part, first, last);
            const int row = static_cast<int>(rank) * 128 + quad * 32;
            const int m = m_tile * kPairRows + row;
            const int n0 = n_tile * kGradCols;
            const uint32_t acc = tmem_base + static_cast<uint32_t>(ab * kGradCols) + (static_cast<uint32_t>(quad * 32) << 16);
            float *sums = args.partials + static_cast<int64_t>(max(part, 0)) * (kPairRows * kGradCols) + row + lane;
            if (part < 0) {  // the staged pieces are free once the last stores out of them have read them
                if (lane == 0) bulk_wait_read_all();
                __syncwarp();
            }
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
            }
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {  // 16 columns of each piece of 64
                uint32_t r[4][16];
#pragma unroll
                for (int q = 0; q < 4; ++q) tmem_ld_32x32b_x16(acc + q * 64 + c * 16, r[q]);
                tmem_ld_wait();
                if (!alive) {  // after a wait that gave up every output and sum of the pair is NaN
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int i = 0; i < 16; ++i) r[q][i] = 0x7fc00000u;
                }
                if constexpr (kRotate) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) radix4(r[0][i], r[1][i], r[2][i], r[3][i]);
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (part < 0)
                        stage16(staged + q * kPieceBytes, c, lane, r[q]);
                    else
                        store_sums16(sums + (q * 64 + c * 16) * kPairRows, r[q]);
                }
            }
            if (part < 0) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0 && m < args.m) {
#pragma unroll 1
                    for (int q = 0; q < 4; ++q)
                        if (n0 + q * 64 < args.k) tma_store_2d(&tmap_out, staged + q * kPieceBytes, n0 + q * 64, m, policy);
                    bulk_commit();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(leader_empty + static_cast<uint32_t>(ab * sizeof(uint64_t)));
        }
        if (lane == 0) bulk_wait_all();  // the staged rows leave shared memory before the CTA does
    }

    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && *abort_flag) settle_inflight_copies();  // whichever wait gave up
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// Sums of a tile's parts, in order, rounded: 64 columns by 32 rows a block, through shared memory.
__global__ void __launch_bounds__(256) grad_join_kernel(const GradArgs a) {
    __shared__ float block[64][33];
    const int num_m = (a.m + kPairRows - 1) / kPairRows;
    const int tile = blockIdx.x >> 5;  // of the split ones
    const int col0 = (blockIdx.x & 3) * 64, row0 = (blockIdx.x >> 2 & 7) * 32;
    const int m = (a.whole + tile) % num_m * kPairRows + row0;
    const int k = (a.whole + tile) / num_m * kGradCols + col0;
    if (m >= a.m || k >= a.k) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int64_t kTile = kPairRows * kGradCols;
    const float *src = a.partials + tile * a.split * kTile + col0 * kPairRows + row0 + lane;
    float sum[8] = {};
#pragma unroll 2
    for (int p = 0; p < a.split; ++p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += __ldcs(src + p * kTile + (warp * 8 + i) * kPairRows);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) block[warp * 8 + i][lane] = sum[i];
    __syncthreads();
    const int c = 2 * lane;
    if (k + c >= a.k) return;  // K is even
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = warp * 4 + i;
        if (m + r < a.m)
            *reinterpret_cast<uint32_t *>(static_cast<__nv_bfloat16 *>(a.out) + static_cast<int64_t>(m + r) * a.k + k + c) =
                pack_bf16x2(block[c][r], block[c + 1][r]);
    }
}

cudaError_t launch_grad_join(const GradArgs &a, cudaStream_t stream) {
    const int tiles = ((a.m + kPairRows - 1) / kPairRows) * ((a.k + kGradCols - 1) / kGradCols) - a.whole;
    grad_join_kernel<<<static_cast<unsigned>(tiles) * 32u, 256, 0, stream>>>(a);
    return cudaGetLastError();
}

int grad_pair_smem() { return kSmem; }
int grad_pair_threads() { return kThreadCount; }
const void *grad_pair_kernel(int rotation) {
    return rotation ? reinterpret_cast<const void *>(&fp4_grad_pair_kernel<true>)
                    : reinterpret_cast<const void *>(&fp4_grad_pair_kernel<false>);
}

}  // namespace fp4
}  // namespace ctu

// Product of two 4-bit floating point matrices (CTA pair, tcgen05 block-scaled MMA):
//
//   out[m, n] = bf16( fma( (sum_k A[m, k] B[n, k]) * a_scale[m], w_scale[n], bias[n] ) )
//
// A and B are e2m1 codes times their block scales; the tensor cores apply both and accumulate in
// fp32.  A pair of CTAs owns a 256 x 256 tile: CTA r stages rows [128 r, 128 r + 128) of A and as many of
// B, the scales of its own A rows and those of all 256 B rows; one M = 256, N = 256, K = 64 instruction of
// the leader reads both CTAs' halves.
//
// The tile is as large as tensor memory allows: each column more is an operand row read once for more MMAs
// (32760 x 13824 x 5120: 951 us with 192 columns and two separate accumulators, 891 so).  Two accumulators of
// 256 columns and the scales need 560 of the 512 columns: the second accumulator starts 48 columns before
// the first one's end, and the epilogue of a tile reads the shared columns first and then lets the next
// tile's MMAs start.
//
// What bounds it is the tensor pipe and the way from tile to tile.  Four MMAs of a stage take 512 cycles; a stage of 76 KB
// takes 526 (18944 x 1024 with K = 5120 and 10240), so the scale copies are nearly hidden, and a tile 2500 more
// whatever its K (with 47 rounds of tiles against four).  16384 x 13824 x 5120 is 667 cycles a stage in all, the
// pipe 76 % busy, the L2 52 % (14 TB/s).
//
// Roles: warp 0 loads (TMA), warp 1 of the leader copies scales into tensor memory and issues the
// MMAs, warps 2..9 write the output.  Every wait is bounded.
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
constexpr int kStageK = 256;  // values of K per stage: 128 bytes of codes
constexpr int kChunks = 4;    // MMAs per stage
constexpr int kABytes = 128 * 128;
constexpr int kHalfCols = kPairCols / 2;
constexpr int kBBytes = kHalfCols * 128;
constexpr int kAScaleBytes = 4 * 512;
constexpr int kBScaleBytes = 2 * 4 * 512;
constexpr int kAOffset = 0;
constexpr int kBOffset = kStages * kABytes;
constexpr int kAScaleOffset = kBOffset + kStages * kBBytes;
constexpr int kBScaleOffset = kAScaleOffset + kStages * kAScaleBytes;
constexpr int kStageOutOffset = kBScaleOffset + kStages * kBScaleBytes;
constexpr int kEpilogueWarps = 8;         // at most; the launch chooses 4 or 8
constexpr int kOutCols = 64;             // columns a warp stages at a time: 128 bytes a row
constexpr int kOutBytes = 32 * 128;      // its 32 rows
constexpr int kStructOffset = kStageOutOffset + kEpilogueWarps * kOutBytes;
constexpr int kThreadCount = 32 * (2 + kEpilogueWarps);
constexpr int kTmemCols = 512;
constexpr int kScaleCols = 48;                             // 4 chunks x (4 of A + 8 of B)
constexpr int kScaleCol = kTmemCols - kScaleCols;          // first of them
constexpr int kSecondAcc = kScaleCol - kPairCols;          // first column of the second accumulator: 208
static_assert(kPairCols - kSecondAcc <= kOutCols, "the shared columns are within the epilogue's first piece");

struct Shared {
    uint64_t full[kStages];
    uint64_t empty[kStages];
    uint64_t acc_full[2];
    uint64_t acc_free;  // a tile's shared columns have been read (leader)
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
    alignas(16) float col_scale[kPairCols];
    alignas(16) float col_bias[kPairCols];
};

constexpr int kSmem = kStructOffset + static_cast<int>(sizeof(Shared)) + 1024;
static_assert(kSmem <= 232448, "shared memory of one CTA");

}  // namespace

template <int kFormat>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreadCount, 1)
    fp4_linear_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                           const __grid_constant__ CUtensorMap tmap_as, const __grid_constant__ CUtensorMap tmap_bs,
                           const __grid_constant__ CUtensorMap tmap_out, const LinearArgs args) {
    // Scale tiles of 128 rows per stage: 64 values of K per tile (nvfp4) or 128 (mxfp4).
    constexpr int kTiles = kFormat == kNvfp4 ? 4 : 2;
    constexpr uint32_t kStageTx = 2 * (kABytes + kBBytes + 3 * kTiles * 512);
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Shared &S = *reinterpret_cast<Shared *>(smem + kStructOffset);

    const int epilogue_warps = static_cast<int>(blockDim.x >> 5) - 2;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int pair = blockIdx.x >> 1;
    const int num_pairs = gridDim.x >> 1;
    const int num_n = (args.n + kPairCols - 1) / kPairCols;
    const int num_m = (args.m + kPairRows - 1) / kPairRows;
    const int num_tiles = num_m * num_n;
    const int nk = (args.k + kStageK - 1) / kStageK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) mbar_init(&S.acc_full[b], 1);
        mbar_init(&S.acc_free, 2 * epilogue_warps);
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
        prefetch_tmap(&tmap_as);
        prefetch_tmap(&tmap_bs);
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
                const int m0 = (t / num_n) * kPairRows + static_cast<int>(rank) * 128;
                const int n0 = (t % num_n) * kPairCols;
                for (int kb = 0; kb < nk; ++kb) {
                    if (!guard.wait(&S.empty[s], ph ^ 1u, kErrTimeoutEmpty)) {
                        ok = false;
                        break;
                    }
                    const uint32_t full = mapa_shared(smem_u32(&S.full[s]), 0u);
                    if (leader) mbar_arrive_expect_tx(&S.full[s], kStageTx);
                    tma_load_2d_pair(smem + kAOffset + s * kABytes, &tmap_a, kb * 128, m0, full);
                    tma_load_2d_pair(smem + kBOffset + s * kBBytes, &tmap_b, kb * 128,
                                     n0 + static_cast<int>(rank) * kHalfCols, full);
                    tma_load_3d_pair(smem + kAScaleOffset + s * kAScaleBytes, &tmap_as, 0, kb * kTiles, m0 / 128, full);
                    tma_load_3d_pair(smem + kBScaleOffset + s * kBScaleBytes, &tmap_bs, 0, kb * kTiles, n0 / 128, full);
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (leader) {
            // The whole warp runs this loop on warp-uniform values and one elected lane issues: the
            // operands then sit in uniform registers already (a single-lane loop moves each of them
            // there first, which costs more than an MMA of this width takes).
            int s = 0;
            uint32_t ph = 0;
            int local = 0;
            bool ok = true;
            const uint32_t a0 = smem_desc_low(smem_u32(smem + kAOffset));
            const uint32_t b0 = smem_desc_low(smem_u32(smem + kBOffset));
            const uint32_t as0 = smem_desc_low(smem_u32(smem + kAScaleOffset));
            const uint32_t bs0 = smem_desc_low(smem_u32(smem + kBScaleOffset));
            const uint32_t empty0 = smem_u32(&S.empty[0]);
            int left = pair == 0 && args.wait.never >= 0 ? args.wait.never : INT_MAX;  // stages until the test's wait
            for (int t = pair; t < num_tiles && ok; t += num_pairs, ++local) {
                const uint32_t ab = local & 1;
                // A warp's first piece of a tile read: its part of the tile before is, and the shared columns.
                if (local > 0)
                    ok = __all_sync(0xffffffffu, guard.wait_cluster(&S.acc_free, (local - 1) & 1, kErrTimeoutAccumFree));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem_base + ab * kSecondAcc;
                const int stop = min(nk, left);
                left -= stop;
                for (int kb = 0; kb < stop; ++kb) {
                    ok = __all_sync(0xffffffffu, guard.wait(&S.full[s], ph, kErrTimeoutFull));
                    if (!ok) break;
                    tc_fence_after();
                    // Scale copies and MMAs of one thread execute in order, so one set of columns serves
                    // every stage.
                    const uint32_t sa = tmem_base + kScaleCol;
                    const uint32_t sb = sa + 16;
                    const uint32_t a = a0 + s * (kABytes >> 4);
                    const uint32_t b = b0 + s * (kBBytes >> 4);
                    const uint32_t as = as0 + s * (kAScaleBytes >> 4);
                    const uint32_t bs = bs0 + s * (kBScaleBytes >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int c = 0; c < kTiles; ++c) {
                            copy_scales_pair(sa + 4 * c, desc64(as + c * 32, kDescScalesHigh));
                            copy_scales_pair(sb + 8 * c, desc64(bs + c * 32, kDescScalesHigh));
                            copy_scales_pair(sb + 8 * c + 4, desc64(bs + (kTiles + c) * 32, kDescScalesHigh));
                        }
#pragma unroll
                        for (int c = 0; c < kChunks; ++c) {
                            const int tile = kFormat == kNvfp4 ? c : c / 2;
                            const uint32_t idesc = kFormat == kNvfp4
                                                       ? idesc_fp4(kFormat, kPairRows, kPairCols, 0)
                                                       : idesc_fp4(kFormat, kPairRows, kPairCols, 2 * (c & 1));
                            mma_fp4_pair<kFormat>(d, desc64(a + 2 * c, kDescSw128High), desc64(b + 2 * c, kDescSw128High),
                                                  idesc, sa + 4 * tile, sb + 8 * tile, (kb | c) != 0 ? 1u : 0u);
                        }
                        mma_commit_pair_both_at(empty0 + 8 * s);
                        if (kb == nk - 1) mma_commit_pair_both(&S.acc_full[ab]);
                    }
                    __syncwarp();
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                if (ok && stop < nk) ok = __all_sync(0xffffffffu, guard.wait(&S.drain, 0u, kErrTimeoutFull));
            }
            if (elect_one()) {
                mma_commit_pair_local(&S.drain);
                mbar_wait(&S.drain, 0u, nullptr, args.err, kErrTimeoutDrain, args.wait.ns);
            }
            __syncwarp();
        }
    } else {
        const int quad = warp & 3;
        const int sharers = epilogue_warps >> 2;  // warps to each 32 rows, and this one's place among them
        const int share = (warp - 2) >> 2;
        const int ethread = threadIdx.x - 64;
        const uint32_t leader_free = mapa_shared(smem_u32(&S.acc_free), 0u);
        const uint32_t staged = smem_u32(smem + kStageOutOffset + (warp - 2) * kOutBytes);
        const bool tma_out = (args.n & 7) == 0;  // rows of the output start on 16 bytes
        const uint64_t policy = evict_first_policy();
        bool alive = true;
        int local = 0;
        for (int t = pair; t < num_tiles; t += num_pairs, ++local) {
            const int ab = local & 1;
            const int m0 = (t / num_n) * kPairRows + static_cast<int>(rank) * 128;
            const int n0 = (t % num_n) * kPairCols;
            named_barrier(1, 32 * epilogue_warps);
            for (int c = ethread; c < kPairCols; c += 32 * epilogue_warps) {
                const int n = n0 + c;
                const bool in = n < args.n;
                S.col_scale[c] = in ? args.w_scale[args.w_scale_count == 1 ? 0 : n] : 0.0f;
                S.col_bias[c] = in && args.bias != nullptr ? args.bias[n] : 0.0f;
            }
            named_barrier(1, 32 * epilogue_warps);
            if (alive) {
                alive = __all_sync(0xffffffffu, guard.wait(&S.acc_full[ab], (local >> 1) & 1, kErrTimeoutAccum));
            }
            tc_fence_after();
            const int m_warp = m0 + quad * 32;
            // After a wait that gave up every output of the pair is NaN.
            float a_s = m_warp + lane < args.m ? args.a_scale[m_warp + lane] : 0.0f;
            if (!alive) a_s = __uint_as_float(0x7fc00000u);
            const f32x2 a_s2 = pk2(a_s, a_s);
#pragma unroll 1
            for (int i = share; i < kPairCols / kOutCols; i += sharers) {
                // The piece with the shared columns first: the last one of the first accumulator, the first
                // one of the second.
                const int c = ab == 0 ? (i + kPairCols / kOutCols - 1) % (kPairCols / kOutCols) : i;
                const int n = n0 + c * kOutCols;
                const bool inside = n < args.n && m_warp < args.m;
                uint32_t acc[2][32];
                const uint32_t src = tmem_base + static_cast<uint32_t>(ab * kSecondAcc + c * kOutCols) +
                                     (static_cast<uint32_t>(quad * 32) << 16);
                tmem_ld_32x32b_x32(src, acc[0]);
                tmem_ld_32x32b_x32(src + 32, acc[1]);
                // The staging rows are free once the last copy out of them has read them.
                if (lane == 0) bulk_wait_read_all();
                tmem_ld_wait();
                if (i == share) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_remote(leader_free);
                }
                __syncwarp();
                if (!inside) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int col = c * kOutCols + 32 * h + 8 * q;
                        uint32_t p[4];
#pragma unroll
                        for (int j = 0; j < 4; j += 2) {
                            const ulonglong2 scale = *reinterpret_cast<const ulonglong2 *>(&S.col_scale[col + 2 * j]);
                            const ulonglong2 bias = *reinterpret_cast<const ulonglong2 *>(&S.col_bias[col + 2 * j]);
                            const uint32_t *from = acc[h] + 8 * q + 2 * j;
                            float v[4];
                            const f32x2 lo = fmul2(pk2(__uint_as_float(from[0]), __uint_as_float(from[1])), a_s2);
                            const f32x2 hi = fmul2(pk2(__uint_as_float(from[2]), __uint_as_float(from[3])), a_s2);
                            unpk2(ffma2(lo, scale.x, bias.x), v[0], v[1]);
                            unpk2(ffma2(hi, scale.y, bias.y), v[2], v[3]);
                            p[j] = pack_bf16x2(v[0], v[1]);
                            p[j + 1] = pack_bf16x2(v[2], v[3]);
                        }
                        st_shared_v4(staged + 128u * lane + ((static_cast<uint32_t>(4 * h + q) ^ (lane & 7u)) << 4), p);
                    }
                }
                if (tma_out) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmap_out, staged, n, m_warp, policy);
                        bulk_commit();
                    }
                } else {
                    __syncwarp();
                    store_rows(static_cast<__nv_bfloat16 *>(args.out), staged, m_warp, n, args.m, args.n, lane);
                    __syncwarp();
                }
            }
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

int linear_pair_smem() { return kSmem; }
// Eight epilogue warps shorten the way from a tile's last MMA to its output, which is what few tiles wait
// for (1025 x 1537 x 1568: 12.7 us against 14.8 with four), what short tiles do (13679 x 1856 x 2304: 35 against
// 39) and what rows off 16 bytes need, which warps write themselves (8894 x 8395 x 1888: 125 against 160).  Four
// leave more to the MMAs of long tiles that follow one another (32760 x 13824 x 5120: 3 % less time).
int linear_pair_threads(bool few_tiles, int64_t n, int64_t k) {
    return few_tiles || n % 8 != 0 || k < 4096 ? kThreadCount : 32 * (2 + 4);
}
const void *linear_pair_kernel(int format) {
    return format == kNvfp4 ? reinterpret_cast<const void *>(&fp4_linear_pair_kernel<kNvfp4>)
                            : reinterpret_cast<const void *>(&fp4_linear_pair_kernel<kMxfp4>);
}

}  // namespace fp4
}  // namespace ctu

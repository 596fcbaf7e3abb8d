// Product of 4-bit floating point matrices with few rows: one to a few hundred tokens against the
// weights, whose bytes bound it.  Same arithmetic and epilogue as the pair kernel, operands swapped:
// 128 weight rows are the MMA's M, kTokens (16, 32, 64 or 128) activation rows its N, so one token
// still fills the tensor core's rows with weights, and each CTA streams a 128-row strip of them.
//
// K is split over the CTAs of a cluster, so that all SMs load at once however few strips there are.
// Each CTA leaves its fp32 partial sums in its shared memory; after a cluster barrier the CTAs share
// out the tokens, add the partials in rank order (equal calls give equal bits) and write the output, a
// warp 256 contiguous bytes of a token.
//
// Measured: 1 x 5120 x 5120 6.1 us and 17 x 13824 x 5120 10.4 us with the weights in the L2, as in a loop over one
// layer; 7.6 and 11.7 us with weights from HBM, as a model's layers in turn have them.  Latencies of launch, load, MMA and
// cluster barriers bound it, not the 2.3 and 5.9 us that the weights' bytes take from HBM.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "fp4.cuh"
#include "fp4_mma.cuh"
#include "ptx.cuh"

namespace ctu {
namespace fp4 {

namespace {

constexpr int kStageK = 256;
constexpr int kChunks = 4;
constexpr int kStrip = 128;  // weight rows of a CTA
constexpr int kABytes = kStrip * 128;
constexpr int kScaleBytes = 4 * 512;
constexpr int kEpilogueWarps = 4;
constexpr int kThreadCount = 32 * (2 + kEpilogueWarps);

// One CTA an SM with as deep a ring as fits: what bounds a strip is bytes in flight (1 x 5120 x 5120: 9.3 us with
// four stages of 24 KB and two CTAs an SM, 6.4 so; 17 x 13824 x 5120 takes as long either way).
template <int kTokens>
struct Small {
    static constexpr int kStages = kTokens <= 32 ? 9 : kTokens == 64 ? 8 : 6;
    static constexpr int kBBytes = kTokens * 128;
    static constexpr int kBOffset = kStages * kABytes;
    static constexpr int kAScaleOffset = kBOffset + kStages * kBBytes;
    static constexpr int kBScaleOffset = kAScaleOffset + kStages * kScaleBytes;
    static constexpr int kStructOffset = kBScaleOffset + kStages * kScaleBytes;
    static constexpr int kSmem = kStructOffset + 256 + 1024;
    static constexpr int kScaleCol = kTokens;
    static constexpr int kTmemCols = kTokens + 64 <= 128 ? 128 : 256;
    static_assert(kTokens * kStrip * 4 <= kBOffset, "partial sums fit the weights' ring");
    static_assert(kSmem <= 232448, "shared memory of one CTA");
};

struct Shared {
    uint64_t full[9];
    uint64_t empty[9];
    uint64_t acc_full;
    uint64_t drain;
    uint64_t issued;  // `copies` is final
    uint32_t tmem_base;
    int abort_flag;
    int copies;
};

__device__ __forceinline__ void tma_load_3d(void *smem_dst, const void *tmap, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_u32(smem_dst)),
        "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

template <int kFormat>
__device__ __forceinline__ void mma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t a_scale, uint32_t b_scale, uint32_t accumulate) {
    if constexpr (kFormat == 0) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
                d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(a_scale), "r"(b_scale)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
                d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(a_scale), "r"(b_scale)
            : "memory");
    }
}

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t cluster_addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(cluster_addr)
                 : "memory");
    return v;
}

}  // namespace

template <int kFormat, int kTokens>
__global__ void __launch_bounds__(kThreadCount)
    fp4_linear_small_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                            const __grid_constant__ CUtensorMap tmap_ws, const __grid_constant__ CUtensorMap tmap_as,
                            const LinearArgs args) {
    using L = Small<kTokens>;
    constexpr int kStages = L::kStages;
    constexpr int kTiles = kFormat == kNvfp4 ? 4 : 2;
    constexpr uint32_t kStageTx = kABytes + L::kBBytes + 2 * kTiles * 512;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Shared &S = *reinterpret_cast<Shared *>(smem + L::kStructOffset);

    const uint32_t rank = cluster_ctarank();
    const int split = args.split;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int tile = blockIdx.x / split;
    const int num_m = (args.m + kTokens - 1) / kTokens;
    const int m0 = (tile % num_m) * kTokens;
    const int n0 = (tile / num_m) * kStrip;
    const int nk_all = (args.k + kStageK - 1) / kStageK;
    const int k_begin = static_cast<int>(static_cast<int64_t>(nk_all) * rank / split);
    const int nk = static_cast<int>(static_cast<int64_t>(nk_all) * (rank + 1) / split) - k_begin;  // at least one

    // The thread that loads sets the barriers up and starts at once; the others meet below.
    if (threadIdx.x == 0) {
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_ws);
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_as);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&S.full[s], 1);
            mbar_init(&S.empty[s], 1);
        }
        mbar_init(&S.acc_full, 1);
        mbar_init(&S.drain, 1);
        mbar_init(&S.issued, 1);
        S.abort_flag = 0;
        fence_mbar_init();
    }
    volatile int *abort_flag = &S.abort_flag;
    const uint64_t limit = args.wait.ns;
    auto load = [&](int s, int kb) {
        mbar_arrive_expect_tx(&S.full[s], kStageTx);
        tma_load_2d(smem + s * kABytes, &tmap_w, kb * 128, n0, &S.full[s]);
        tma_load_3d(smem + L::kAScaleOffset + s * kScaleBytes, &tmap_ws, 0, kb * kTiles, n0 / 128, &S.full[s]);
        tma_load_2d(smem + L::kBOffset + s * L::kBBytes, &tmap_a, kb * 128, m0, &S.full[s]);
        tma_load_3d(smem + L::kBScaleOffset + s * kScaleBytes, &tmap_as, 0, kb * kTiles, m0 / 128, &S.full[s]);
    };
    const int first = min(nk, kStages);  // stages that are free to begin with
    if (threadIdx.x == 0) {
        for (int s = 0; s < first; ++s) load(s, k_begin + s);
    }
    if (warp == 1) {
        tmem_alloc(&S.tmem_base, L::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = S.tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 1;
            int fills = first;
            for (; fills < nk; ++fills) {
                if (!mbar_wait(&S.empty[s], ph ^ 1u, abort_flag, args.err, kErrTimeoutEmpty, limit)) break;
                load(s, k_begin + fills);
                if (++s == kStages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
            S.copies = fills;
            mbar_arrive(&S.issued);
        }
    } else if (warp == 1) {
        int s = 0;
        uint32_t ph = 0;
        uint32_t set = 0;
        const uint32_t a0 = smem_desc_low(smem_u32(smem));
        const uint32_t b0 = smem_desc_low(smem_u32(smem + L::kBOffset));
        const uint32_t as0 = smem_desc_low(smem_u32(smem + L::kAScaleOffset));
        const uint32_t bs0 = smem_desc_low(smem_u32(smem + L::kBScaleOffset));
        bool ok = true;
        const int never = blockIdx.x == 0 ? args.wait.never : -1;
        const int stop = never >= 0 ? min(nk, never) : nk;
        for (int kb = 0; kb < stop; ++kb) {
            ok = __all_sync(0xffffffffu, mbar_wait(&S.full[s], ph, abort_flag, args.err, kErrTimeoutFull, limit));
            if (!ok) break;
            tc_fence_after();
            const uint32_t sa = tmem_base + L::kScaleCol + set * 32;
            const uint32_t sb = sa + 16;
            const uint32_t a = a0 + s * (kABytes >> 4);
            const uint32_t b = b0 + s * (L::kBBytes >> 4);
            const uint32_t as = as0 + s * (kScaleBytes >> 4);
            const uint32_t bs = bs0 + s * (kScaleBytes >> 4);
            if (elect_one()) {
#pragma unroll
                for (int c = 0; c < kTiles; ++c) {
                    copy_scales(sa + 4 * c, desc64(as + c * 32, kDescScalesHigh));
                    copy_scales(sb + 4 * c, desc64(bs + c * 32, kDescScalesHigh));
                }
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int t = kFormat == kNvfp4 ? c : c / 2;
                    const uint32_t idesc =
                        kFormat == kNvfp4 ? idesc_fp4(kFormat, 128, kTokens, 0) : idesc_fp4(kFormat, 128, kTokens, 2 * (c & 1));
                    mma_fp4<kFormat>(tmem_base, desc64(a + 2 * c, kDescSw128High), desc64(b + 2 * c, kDescSw128High), idesc,
                                     sa + 4 * t, sb + 4 * t, (kb | c) != 0 ? 1u : 0u);
                }
                mma_commit(&S.empty[s]);
                if (kb == nk - 1) mma_commit(&S.acc_full);
            }
            __syncwarp();
            set ^= 1u;
            if (++s == kStages) {
                s = 0;
                ph ^= 1u;
            }
        }
        if (stop < nk) ok = __all_sync(0xffffffffu, mbar_wait(&S.drain, 0u, abort_flag, args.err, kErrTimeoutFull, limit));
        if (!ok) {  // no last commit comes: wait for what was issued
            if (elect_one()) mma_commit(&S.drain);
            __syncwarp();
            mbar_wait(&S.drain, 0u, nullptr, args.err, kErrTimeoutDrain, limit);
        }
    }
    // Everything issued has completed before shared and tensor memory are used otherwise or freed: the
    // last commit covers all MMAs, and each MMA's stage had landed.
    bool alive = true;
    if (warp >= 1)
        alive = __all_sync(0xffffffffu, mbar_wait(&S.acc_full, 0u, abort_flag, args.err, kErrTimeoutAccum, limit));
    tc_fence_after();

    const int valid = min(kTokens, args.m - m0);
    if (warp >= 2) {
        // Partial sums to shared memory, [token][column of the strip]; the lanes are columns here.  Where a wait
        // gave up they are NaN, and so is what the cluster makes of them.
        float *part = reinterpret_cast<float *>(smem);
        const int row = (warp & 3) * 32 + lane;
        if (!alive && mbar_wait(&S.issued, 0u, nullptr, args.err, kErrTimeoutDrain, limit)) {
            // Copies in flight land before shared memory is used otherwise and before the CTA leaves.
            for (int f = max(0, S.copies - kStages); f < S.copies; ++f)
                if (!mbar_wait(&S.full[f % kStages], (f / kStages) & 1, nullptr, args.err, kErrTimeoutDrain, limit)) break;
        }
#pragma unroll 1
        for (int c = 0; c < valid; c += 16) {
            uint32_t acc[16];
            tmem_ld_32x32b_x16(tmem_base + c + (static_cast<uint32_t>((warp & 3) * 32) << 16), acc);
            tmem_ld_wait();
            if (!alive) {
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[j] = 0x7fc00000u;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (c + j < valid) part[(c + j) * kStrip + row] = __uint_as_float(acc[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (split > 1)
            cluster_sync();
        else
            named_barrier(1, 32 * kEpilogueWarps);
        // A warp takes a token, a lane four columns of it.
        const int n = n0 + 4 * lane;
        if (n < args.n) {
            float w_s[4], bias[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = n + i < args.n;
                w_s[i] = in ? args.w_scale[args.w_scale_count == 1 ? 0 : n + i] : 0.0f;
                bias[i] = in && args.bias != nullptr ? args.bias[n + i] : 0.0f;
            }
            const bool wide = (args.n & 3) == 0;
            for (int t = static_cast<int>(rank) + split * (warp - 2); t < valid; t += split * kEpilogueWarps) {
                const uint32_t src = smem_u32(smem) + 4u * (kStrip * t + 4 * lane);
                float4 p[8];
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < split) p[r] = ld_cluster_f32x4(mapa_shared(src, r));
                const float a_s = args.a_scale[m0 + t];
                float4 sum = p[0];
#pragma unroll
                for (int r = 1; r < 8; ++r) {
                    if (r < split) {
                        sum.x += p[r].x;
                        sum.y += p[r].y;
                        sum.z += p[r].z;
                        sum.w += p[r].w;
                    }
                }
                const float v[4] = {__fmaf_rn(__fmul_rn(sum.x, a_s), w_s[0], bias[0]), __fmaf_rn(__fmul_rn(sum.y, a_s), w_s[1], bias[1]),
                                    __fmaf_rn(__fmul_rn(sum.z, a_s), w_s[2], bias[2]), __fmaf_rn(__fmul_rn(sum.w, a_s), w_s[3], bias[3])};
                __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(args.out) + static_cast<int64_t>(m0 + t) * args.n + n;
                if (wide) {
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < args.n) dst[i] = __float2bfloat16_rn(v[i]);
                }
            }
        }
        __syncwarp();
        if (split > 1) cluster_sync();  // no CTA leaves while another reads its partial sums
    } else if (split > 1) {
        __syncwarp();
        cluster_sync();
        cluster_sync();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, L::kTmemCols);
    }
}

namespace {
template <int kTokens>
SmallKernel small_of(int format) {
    return {format == kNvfp4 ? reinterpret_cast<const void *>(&fp4_linear_small_kernel<kNvfp4, kTokens>)
                             : reinterpret_cast<const void *>(&fp4_linear_small_kernel<kMxfp4, kTokens>),
            Small<kTokens>::kSmem, kThreadCount, kTokens, 1};
}
}  // namespace

SmallKernel linear_small_kernel(int format, int64_t m) {
    if (m <= 16) return small_of<16>(format);
    if (m <= 32) return small_of<32>(format);
    if (m <= 64) return small_of<64>(format);
    return small_of<128>(format);
}

}  // namespace fp4
}  // namespace ctu

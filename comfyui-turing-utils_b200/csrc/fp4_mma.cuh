// tcgen05 pieces of the 4-bit products: block-scaled MMA, scale copies into tensor memory, 3D tile
// loads, and the abort protocol of a CTA pair.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx.cuh"

namespace ctu {
namespace fp4 {

__device__ __forceinline__ void named_barrier(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// 3D tile load whose bytes are counted on a barrier of the pair's leader (no multicast).
__device__ __forceinline__ void tma_load_3d_pair(void *smem_dst, const void *tmap, int x, int y, int z,
                                                 uint32_t leader_bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4}], [%5];" ::"r"(smem_u32(smem_dst)),
        "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(leader_bar)
        : "memory");
}

// Operand descriptors: 128-byte-swizzled tiles (8-row groups 1024 bytes apart) and 512-byte scale tiles
// (32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart).
// The two halves of a descriptor: the low word holds the address (and a constant), so a step through
// shared memory is one addition; the high words are constants.
__device__ __forceinline__ uint32_t smem_desc_low(uint32_t smem_addr) {
    return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16);
}
constexpr uint32_t kDescSw128High = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kDescScalesHigh = (128u >> 4) | (1u << 14);
__device__ __forceinline__ uint64_t desc64(uint32_t low, uint32_t high) {
    return (static_cast<uint64_t>(high) << 32) | low;
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r)::"memory");
    return r != 0;
}

__device__ __forceinline__ void mma_commit_pair_both_at(uint32_t bar) {
    const uint16_t mask = 0x3;
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(mask)
        : "memory");
}

// One scale tile into four columns of tensor memory, repeated for the four groups of 32 lanes; in
// both CTAs, each from its own shared memory.
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// D (+)= (A * scale A) (B * scale B)^T over K = 64 e2m1 values of both operands.  kFormat 0: a scale
// for 16 values (four to a row, e4m3); 1: for 32 (two, e8m0).
template <int kFormat>
__device__ __forceinline__ void mma_fp4_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t a_scale, uint32_t b_scale, uint32_t accumulate) {
    if constexpr (kFormat == 0) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
                d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(a_scale), "r"(b_scale)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
                d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(a_scale), "r"(b_scale)
            : "memory");
    }
}

// Instruction descriptor of the block-scaled product: e2m1 x e2m1 -> fp32, both K-major.  `scale_id`
// is the byte of a 32-bit scale column where a row's scales start (mxfp4: 0 or 2).
__host__ __device__ constexpr uint32_t idesc_fp4(int format, int m, int n, int scale_id) {
    return (static_cast<uint32_t>(scale_id) << 4)     // B scale byte
           | (1u << 7)                                // A: e2m1
           | (1u << 10)                               // B: e2m1
           | (static_cast<uint32_t>(n >> 3) << 17)    // N / 8
           | (static_cast<uint32_t>(format) << 23)    // scales: 0 e4m3, 1 e8m0
           | (static_cast<uint32_t>(m >> 7) << 27)    // M / 128
           | (static_cast<uint32_t>(scale_id) << 29); // A scale byte
}

// bf16 x bf16 -> fp32 over K = 16, both K-major, CTA pair.
__device__ __forceinline__ void mma_bf16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__host__ __device__ constexpr uint32_t idesc_bf16(int m, int n) {
    return (1u << 4)                                  // D: f32
           | (1u << 7)                                // A: bf16
           | (1u << 10)                               // B: bf16
           | (static_cast<uint32_t>(n >> 3) << 17)    // N / 8
           | (static_cast<uint32_t>(m >> 4) << 24);   // M / 16
}

// 2D tile store from shared memory; what lies beyond the tensor is not written.  Output lines are the
// first to leave the L2, which the operands' tiles are read from many times.
__device__ __forceinline__ uint64_t evict_first_policy() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void tma_store_2d(const void *tmap, uint32_t smem_src, int x, int y, uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group.L2::cache_hint [%0, {%1, %2}], [%3], %4;" ::"l"(
                     tmap),
                 "r"(x), "r"(y), "r"(smem_src), "l"(policy)
                 : "memory");
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                 : "memory");
}

__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// 32 staged rows of 64 bf16 values (128-byte swizzle) to an output whose rows need not start on 16
// bytes: a warp writes a row in aligned pairs, eight rows' loads in flight.  Where a row starts on an odd
// element, a lane pairs its neighbour's second value with its own first, and the row's ends go out alone.
__device__ __forceinline__ void store_rows(__nv_bfloat16 *out, uint32_t staged, int m0, int n0, int rows, int cols,
                                           int lane) {
    const int valid = min(64, cols - n0);
    const int count = min(32, rows - m0);
    uint16_t *dst = reinterpret_cast<uint16_t *>(out) + static_cast<int64_t>(m0) * cols + n0;
    bool odd = (static_cast<int64_t>(m0) * cols + n0) & 1;
    for (int r0 = 0; r0 < count; r0 += 8) {
        uint32_t own[8], before[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            own[i] = ld_shared_u32(staged + 128u * (r0 + i) + (((static_cast<uint32_t>(lane) >> 2) ^ static_cast<uint32_t>(i)) << 4) +
                                   (lane & 3u) * 4u);
#pragma unroll
        for (int i = 0; i < 8; ++i) before[i] = __shfl_up_sync(0xffffffffu, own[i], 1);
        if (valid == 64 && r0 + 8 <= count) {  // no lane leaves the others' path
            const bool edge = lane == 0 || lane == 31;
#pragma unroll
            for (int i = 0; i < 8; ++i, dst += cols, odd ^= (cols & 1) != 0) {
                const uint32_t word = odd ? __byte_perm(before[i], own[i], 0x5432) : own[i];
                uint16_t *at = dst + 2 * lane - (odd ? 1 : 0);
                if (!odd || lane > 0) *reinterpret_cast<uint32_t *>(at) = word;
                if (odd && edge) dst[lane == 0 ? 0 : 63] = static_cast<uint16_t>(lane == 0 ? own[i] : own[i] >> 16);
            }
            continue;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i, dst += cols, odd ^= (cols & 1) != 0) {
            if (r0 + i >= count) break;
            if (!odd) {
                if (2 * lane + 1 < valid)
                    *reinterpret_cast<uint32_t *>(dst + 2 * lane) = own[i];
                else if (2 * lane < valid)
                    dst[2 * lane] = static_cast<uint16_t>(own[i]);
            } else {
                if (lane == 0)
                    dst[0] = static_cast<uint16_t>(own[i]);
                else if (2 * lane < valid)
                    *reinterpret_cast<uint32_t *>(dst + 2 * lane - 1) = __byte_perm(before[i], own[i], 0x5432);
                else if (2 * lane - 1 < valid)
                    dst[2 * lane - 1] = static_cast<uint16_t>(before[i] >> 16);
                if (lane == 31 && valid == 64) dst[63] = static_cast<uint16_t>(own[i] >> 16);
            }
        }
    }
}

__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

// Abort state of one CTA of a pair: its own flag, the peer's flag (cluster address), error word.  A
// wait that gives up stops both CTAs.
struct PairAbort {
    volatile int *flag;
    uint32_t peer_flag;
    uint32_t *err;
    uint64_t limit;  // of a wait, ns

    __device__ __forceinline__ void raise() const {
        *flag = 1;
        st_cluster_u32(peer_flag, 1u);
    }
    __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, uint32_t code) const {
        if (mbar_wait(bar, parity, flag, err, code, limit)) return true;
        raise();
        return false;
    }
    __device__ __forceinline__ bool wait_cluster(uint64_t *bar, uint32_t parity, uint32_t code) const {
        if (mbar_wait_cluster(bar, parity, flag, err, code, limit)) return true;
        raise();
        return false;
    }
};

// Bounded pause that lets copies already issued land before a CTA that gave up leaves (their bytes
// are counted on the other CTA's barrier and cannot be waited for one by one).
__device__ __forceinline__ void settle_inflight_copies() {
    const uint64_t start = globaltimer();
    while (globaltimer() - start < 1000000ull) __nanosleep(1000);
}

}  // namespace fp4
}  // namespace ctu

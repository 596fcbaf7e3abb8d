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

// Descriptor of one 512-byte scale tile: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>(128 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    return d;
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

__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

// Abort state of one CTA of a pair: its own flag, the peer's flag (cluster address), error word.  A
// wait that gives up stops both CTAs.
struct PairAbort {
    volatile int *flag;
    uint32_t peer_flag;
    uint32_t *err;

    __device__ __forceinline__ void raise() const {
        *flag = 1;
        st_cluster_u32(peer_flag, 1u);
    }
    __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, uint32_t code) const {
        if (mbar_wait(bar, parity, flag, err, code)) return true;
        raise();
        return false;
    }
    __device__ __forceinline__ bool wait_cluster(uint64_t *bar, uint32_t parity, uint32_t code) const {
        if (mbar_wait_cluster(bar, parity, flag, err, code)) return true;
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

// Rows to 4-bit floating point with block scales, and back.
//
// Row scale (nvfp4): 2^ceil(log2(amax / 2688)), 2688 = 6 * 448, so that the largest block scale
// lies in (224, 448]; a power of two keeps every division by it exact.  Block scale: nvfp4
// e4m3(block amax / 6 / row scale); mxfp4 2^(floor(log2(block amax)) - 2), the OCP rule.  Code:
// e2m1(v / block scale / row scale) to nearest, ties to even, saturating at 6.  A row that holds a
// NaN or an infinity gets a NaN row scale and zero codes and block scales.
//
// Four lanes share 256 columns: lane q holds columns 64 j + 16 q .. + 15 for j = 0..3, so a block of 16
// lies in one lane and a block of 32 in two.  A warp covers 2048 columns, or several short rows; a
// longer row takes several warps, which meet once, for the row's largest magnitude.  Values stay in
// registers from the load to the codes.
//
// Measured, 32760 x 5120 rotated: nvfp4 157 us, mxfp4 138 (one row at a time in shared memory 535).  No pipe is full:
// the fp32 pipe is 48 % busy, the issue slots 53 %, DRAM 29 %; the 15 warps that 128 registers leave an SM do not hide
// the latencies of a chain of 16 fp32 operations an element and the row's barrier.  Unrotated: nvfp4 32760 x 5120 89 us (4.8
// TB/s), mxfp4 4097 x 13824 fp16 29 us (5.0 TB/s).  The dequantizer 79 us at 32760 x 5120 (5.4 TB/s; 102 with a
// division for each eight values).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>

#include "../../include/ctu_b200.h"
#include "fp4.cuh"
#include "ptx.cuh"

namespace ctu {
namespace fp4 {

namespace {

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

// max(a, |b|, |c|); a NaN among them comes out as NaN.
__device__ __forceinline__ float max_abs3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Eight values (four pairs) to a word of e2m1 codes, the first in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x8(const f32x2 (&q)[4]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) unpk2(q[i], v[2 * i], v[2 * i + 1]);
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Where a lane's columns are.  A team of lanes owns a row: some lanes of a warp, a warp, or several warps
// of a CTA, which may hold `rows_per_cta` rows side by side.
struct Place {
    int64_t row;
    int group;    // of 256 columns in the row
    int q;        // lane of the group
    bool active;  // the row and the group exist
};

// Largest magnitude over a row.  Within a warp `span` lanes hold a row.  kMulti: a warp's lanes belong to
// the CTA's row `first_row` and, from lane `border` on, to the next one; red[2 * warp] and the next are
// their maxima, and a row's warps are those of its groups.
template <bool kMulti>
__device__ __forceinline__ float row_max(float amax, int span, float *red, int groups, int slot) {
    if (!kMulti) {
        for (int o = 1; o < span; o <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        return amax;
    }
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int first_row = warp * 8 / groups;  // of the CTA
    const bool later = slot != first_row;
    float lo = later ? 0.0f : amax, hi = later ? amax : 0.0f;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) lo = max_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    if (__any_sync(0xffffffffu, later)) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (lane == 0) *reinterpret_cast<float2 *>(red + 2 * warp) = make_float2(lo, hi);
    __syncthreads();
    const int from = slot * groups / 8, to = min((slot * groups + groups - 1) / 8, static_cast<int>(blockDim.x >> 5) - 1);
    amax = 0.0f;
    for (int w = from; w <= to; ++w) amax = max_nan(amax, red[2 * w + (slot != w * 8 / groups ? 1 : 0)]);
    return amax;
}

// t / 6 to nearest, for t in the range where the e4m3 rounding that follows can tell: a product with the reciprocal,
// corrected by its exact remainder (Markstein's step, IBM J. Res. Dev. 34(1), 1990).  This, the reciprocal and the
// quotient below are checked against IEEE division for every significand, and for every scale on the GPU.
__device__ __forceinline__ float sixth(float t) {
    const float c = 1.0f / 6.0f;
    const float q = __fmul_rn(t, c);
    return __fmaf_rn(__fmaf_rn(q, -6.0f, t), c, q);
}

// 1 / s of a block scale: the hardware's approximation, within one unit in the last place, and one step of Newton's
// iteration.  With s of four significant bits the result is the nearest fp32 value.
__device__ __forceinline__ float scale_reciprocal(float s) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
    return __fmaf_rn(y, __fmaf_rn(-s, y, 1.0f), y);
}

// Codes and scales of one lane's four blocks of 16; pair(j, p) is columns 2p, 2p + 1 of block j and
// amax[j] its largest magnitude.  kWhole: K is a multiple of 256, so a group has all its columns.
template <int kFormat, bool kMulti, bool kWhole, typename Pair>
__device__ __forceinline__ void finish(const QuantArgs &a, const Place &at, float (&amax)[4], int span, float *red,
                                       int slot, Pair pair) {
    float row_amax = max_nan(max_nan(amax[0], amax[1]), max_nan(amax[2], amax[3]));
    row_amax = row_max<kMulti>(at.active ? row_amax : 0.0f, span, red, (a.k + 255) / 256, slot);
    const bool bad = !(row_amax <= 3.402823466e38f);
    float row = 1.0f;
    if (kFormat == kNvfp4 && !bad) row = pow2_row_scale(row_amax);
    if (kFormat == kMxfp4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) amax[j] = fmaxf(amax[j], __shfl_xor_sync(0xffffffffu, amax[j], 1));
    }
    // 1 / row: a power of two, whose exponent is negated (2^-126 has its reciprocal, 2^126, in range).
    const float inv_row = __uint_as_float(0x7f000000u - __float_as_uint(row));
    const f32x2 minus_row = pk2(-inv_row, -inv_row);
    if (at.active && at.group == 0 && at.q == 0) a.row_scales[at.row] = bad ? __uint_as_float(0x7fc00000u) : row;
    uint8_t *codes = a.codes + at.row * (a.k / 2) + at.group * 128 + at.q * 8;

    uint32_t bytes = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t byte;
        uint32_t word[2];
        if (kFormat == kNvfp4) {
            byte = __nv_cvt_float_to_fp8(sixth(amax[j] * inv_row), __NV_SATFINITE, __NV_E4M3);
            const float s = block_scale_value(byte, kNvfp4);
            // v / s rounded to nearest by Markstein's step, so that ties of the code grid stay ties.
            // The signs are placed so that a zero keeps its own; a zero scale leaves such zeros.
            const float inv = byte == 0 ? 0.0f : scale_reciprocal(s);
            const f32x2 minus_inv = pk2(-inv, -inv), s2 = pk2(s, s);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f32x2 q[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x2 minus_v = fmul2(pair(j, 4 * h + i), minus_row);
                    const f32x2 q0 = fmul2(minus_v, minus_inv);
                    q[i] = ffma2(ffma2(q0, s2, minus_v), minus_inv, q0);
                }
                word[h] = e2m1x8(q);
            }
        } else {
            const uint32_t e = __float_as_uint(amax[j]) >> 23;
            byte = e > 2 ? e - 2 : 0;
            const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte), exact
            const f32x2 inv2 = pk2(inv, inv);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f32x2 q[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) q[i] = fmul2(pair(j, 4 * h + i), inv2);
                word[h] = e2m1x8(q);
            }
        }
        const bool in = kWhole || at.group * 256 + j * 64 + at.q * 16 < a.k;
        if (in) bytes |= byte << (8 * j);
        if (in && at.active)
            *reinterpret_cast<uint2 *>(codes + j * 32) = bad ? make_uint2(0u, 0u) : make_uint2(word[0], word[1]);
    }
    if (bad) bytes = 0;
    // The group's scale bytes to whole words of its tiles: a byte transpose among the four lanes.
    const int64_t col_tiles = scale_col_tiles(a.k, kFormat);
    uint32_t word;
    int64_t tile;
    if (kFormat == kNvfp4) {
        uint32_t p = __shfl_xor_sync(0xffffffffu, bytes, 1);
        bytes = __byte_perm(bytes, p, (at.q & 1) ? 0x3715 : 0x6240);
        p = __shfl_xor_sync(0xffffffffu, bytes, 2);
        word = __byte_perm(bytes, p, (at.q & 2) ? 0x3276 : 0x5410);
        tile = at.group * 4 + at.q;
    } else {
        const uint32_t p = __shfl_xor_sync(0xffffffffu, bytes, 2);
        word = __byte_perm(bytes, p, (at.q & 1) ? 0x7362 : 0x5140);
        tile = at.q < 2 ? at.group * 2 + at.q : col_tiles;
    }
    if (at.active && tile < col_tiles)
        *reinterpret_cast<uint32_t *>(a.block_scales + ((at.row >> 7) * col_tiles + tile) * 512 + (at.row & 31) * 16 +
                                      ((at.row >> 5) & 3) * 4) = word;
}

// Scale bytes of the last tile's rows beyond the matrix.
__device__ __forceinline__ void clear_padding(const QuantArgs &a, int format) {
    const int col_tiles = static_cast<int>(scale_col_tiles(a.k, format));
    const int first = static_cast<int>(a.rows & 127);
    if (first == 0) return;
    uint32_t *tiles = reinterpret_cast<uint32_t *>(a.block_scales) + (a.rows >> 7) * col_tiles * 128;
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < col_tiles * 128; i += gridDim.x * blockDim.x) {
        const int word = i & 127;  // row 32 (word & 3) + word / 4 of the tile
        if (32 * (word & 3) + (word >> 2) >= first) tiles[i] = 0u;
    }
}

template <bool kHalf>
__device__ __forceinline__ float low_value(uint32_t w) {
    return kHalf ? __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xffffu))) : bf16lo(w);
}
template <bool kHalf>
__device__ __forceinline__ float high_value(uint32_t w) {
    return kHalf ? __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16))) : bf16hi(w);
}

// Without rotation: loads go straight to registers, and magnitudes are compared as 16-bit integers,
// where infinities and NaN rank above every finite value.
template <int kFormat, bool kHalf, bool kMulti>
__global__ void __launch_bounds__(kMulti ? 768 : 128) quantize_kernel(const QuantArgs a) {
    __shared__ float red[2][48];
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int groups = (a.k + 255) / 256;
    const int slots = a.side_by_side;  // rows of a warp, or (kMulti) of the CTA
    const int span = kMulti ? 32 : 32 / slots;
    const int64_t teams = kMulti ? gridDim.x : static_cast<int64_t>(gridDim.x) * 4;
    const int64_t team = kMulti ? blockIdx.x : blockIdx.x * 4ll + warp;
    const int place = warp * 8 + (lane >> 2);  // kMulti: group of the CTA's rows
    const int slot = kMulti ? place / groups : lane / span;
    Place at;
    at.q = lane & 3;
    at.group = kMulti ? place - slot * groups : (lane % span) >> 2;
    int flip = 0;
    for (int64_t r0 = team * slots; r0 < a.rows; r0 += teams * slots, flip ^= 1) {
        at.row = r0 + slot;
        at.active = slot < slots && at.row < a.rows && at.group < groups;
        uint4 w[4][2];
        float amax[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = at.group * 256 + j * 64 + at.q * 16;
            w[j][0] = w[j][1] = make_uint4(0u, 0u, 0u, 0u);
            if (at.active && col < a.k) {
                const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.x) + at.row * a.k + col);
                w[j][0] = __ldcs(src);
                w[j][1] = __ldcs(src + 1);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t *p = &w[j][0].x;
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = __vmaxu2(m, p[i] & 0x7fff7fffu);
            m = max(m & 0xffffu, m >> 16);
            if (kHalf)
                amax[j] = __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
            else
                amax[j] = __uint_as_float(m << 16);
        }
        finish<kFormat, kMulti, false>(a, at, amax, span, red[flip], slot, [&](int j, int p) {
            const uint32_t v = (&w[j][0].x)[p];
            return pk2(low_value<kHalf>(v), high_value<kHalf>(v));
        });
    }
    clear_padding(a, kFormat);
}

// Radix-4 butterfly of two tuples at once, in the rotation's order of sums; halvings are taken before
// the first stage (exact: a 16-bit input over 16 is a fp32 value).
__device__ __forceinline__ void radix4_pair(f32x2 &x0, f32x2 &x1, f32x2 &x2, f32x2 &x3) {
    const f32x2 t = fadd2(x0, x1), b = fsub2(x0, x1);
    x0 = fsub2(fadd2(t, x2), x3);
    x1 = fadd2(fsub2(t, x2), x3);
    const f32x2 y2 = fadd2(fadd2(b, x2), x3);
    x3 = fadd2(fsub2(x2, b), x3);
    x2 = y2;
}

// With rotation.  A warp's 2048 columns arrive by tile loads (128-byte swizzle) in 4 KB of its 8 KB of
// shared memory.  A lane first holds 64 columns in a row (lane q: 64 q ..) and takes the strides 1, 4
// and 16 in registers, two tuples to an instruction where the pairing allows; then the four lanes
// exchange 16-column pieces through the same 8 KB, and stride 64 is in registers too, with whole blocks
// of 16 left in each lane.  The next row's load runs under the codes of this one.  After a wait that gave up a
// warp loads no more, and its rows come out as those that hold a NaN.
template <int kFormat, bool kHalf, bool kMulti, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads)
    rotate_quantize_kernel(const __grid_constant__ CUtensorMap tmap, const QuantArgs a) {
    __shared__ float red[2][48];
    __shared__ uint64_t bars[24], dead;  // dead: nothing arrives on it (test hook)
    extern __shared__ uint8_t smem_raw[];
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023)) + warp * 8192;
    const uint32_t base = smem_u32(smem);
    uint64_t *bar = &bars[warp];
    const uint64_t limit = a.wait.ns;
    const int slots = a.side_by_side;
    const int span = kMulti ? 32 : 32 / slots;
    const int groups = a.k / 256;
    // Rows are counted in 32 bits: x has fewer than 2^31 lines of 64 values.
    const int rows = static_cast<int>(a.rows), step = static_cast<int>(gridDim.x) * (kMulti ? 1 : 4) * slots;
    const int first = static_cast<int>(kMulti ? blockIdx.x : blockIdx.x * 4 + warp) * slots;
    const int place = warp * 8 + (lane >> 2);
    const int slot = kMulti ? place / groups : lane / span;
    Place at;
    at.q = lane & 3;
    at.group = kMulti ? place - slot * groups : (lane % span) >> 2;
    // Copies of `load_groups` groups each: this warp's part of the CTA's rows (they follow one another), or
    // several whole rows.
    const int mine = kMulti ? min(8, groups * slots - warp * 8) : slots > 1 ? 8 : groups;
    const int copies = (mine + a.load_groups - 1) / a.load_groups;
    auto load = [&](int r0) {  // lane 0
        mbar_arrive_expect_tx(bar, static_cast<uint32_t>(copies * a.load_groups * 512));
        const int line = r0 * (a.k / 64) + (kMulti ? warp * 32 : 0);
        for (int c = 0; c < copies; ++c)
            tma_load_2d(smem + c * a.load_groups * 512, &tmap, 0, line + c * a.load_groups * 4, bar);
    };
    if (lane == 0) {
        mbar_init(bar, 1);
        if (warp == 0) mbar_init(&dead, 1);
        fence_mbar_init();
        if (first < rows) load(first);
    }
    __syncwarp();
    // 16-byte chunk c of (column digit d3, d2) of this lane's group in the exchange: the address bits are
    // mixed so that eight lanes of a store or load touch eight different 16-byte banks.
    const uint32_t area = base + (lane >> 2) * 1024u;
    const uint32_t gp = ((lane >> 2) & 1) * 4u;
    auto chunk = [&](uint32_t d3, uint32_t d2, uint32_t c) {
        const uint32_t low = c ^ gp ^ d3 ^ ((d2 & 1u) * 5u) ^ (d2 & 2u);
        return area + ((d3 * 16u + (d2 >> 1) * 8u + low) << 4);
    };
    uint32_t phase = 0;
    bool alive = true;
    int it = 0;
    for (int r0 = first; r0 < rows; r0 += step, ++it) {
        at.row = r0 + slot;
        at.active = slot < slots && at.row < a.rows && at.group < groups;
        const bool never = it == a.wait.never && blockIdx.x == 0 && warp == 0;
        if (alive)
            alive = __all_sync(0xffffffffu, mbar_wait(never ? &dead : bar, never ? 0u : phase, nullptr, a.err, kErrTimeoutFull, limit));
        if (alive) phase ^= 1u;  // else the phase of the copy that may be in flight
        // x[h][i]: column 16 h + i in the low half, 16 (h + 2) + i in the high half.
        f32x2 x[2][16];
        {
            const uint32_t line = static_cast<uint32_t>(lane);
            const f32x2 pre = pk2(0.0625f, 0.0625f);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 lo = *reinterpret_cast<const uint4 *>(smem + line * 128 + (((2 * h + half) ^ (line & 7)) << 4));
                    const uint4 hi = *reinterpret_cast<const uint4 *>(smem + line * 128 + (((2 * h + 4 + half) ^ (line & 7)) << 4));
                    const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, u[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[h][8 * half + 2 * i] = fmul2(pk2(low_value<kHalf>(l[i]), low_value<kHalf>(u[i])), pre);
                        x[h][8 * half + 2 * i + 1] = fmul2(pk2(high_value<kHalf>(l[i]), high_value<kHalf>(u[i])), pre);
                    }
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) radix4_pair(x[h][i], x[h][i + 1], x[h][i + 2], x[h][i + 3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) radix4_pair(x[h][i], x[h][i + 4], x[h][i + 8], x[h][i + 12]);
        }
        __syncwarp();  // the load's bytes are in registers everywhere
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float o[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x0, x1, x2, x3;
                unpk2(x[0][4 * c + i], x0, x2);
                unpk2(x[1][4 * c + i], x1, x3);
                const float t = __fadd_rn(x0, x1), b = __fsub_rn(x0, x1);
                o[0][i] = __fsub_rn(__fadd_rn(t, x2), x3);
                o[1][i] = __fadd_rn(__fsub_rn(t, x2), x3);
                o[2][i] = __fadd_rn(__fadd_rn(b, x2), x3);
                o[3][i] = __fadd_rn(__fsub_rn(x2, b), x3);
            }
#pragma unroll
            for (uint32_t d2 = 0; d2 < 4; ++d2)
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(chunk(at.q, d2, c)), "f"(o[d2][0]),
                             "f"(o[d2][1]), "f"(o[d2][2]), "f"(o[d2][3])
                             : "memory");
        }
        __syncwarp();
        f32x2 v[4][8];
#pragma unroll
        for (uint32_t d3 = 0; d3 < 4; ++d3) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];"
                             : "=l"(v[d3][2 * c]), "=l"(v[d3][2 * c + 1])
                             : "r"(chunk(d3, at.q, c))
                             : "memory");
        }
        fence_proxy_async_smem();  // the exchange is over before the next load writes here
        __syncwarp();
        if (lane == 0 && alive && r0 + step < rows) load(r0 + step);
        float amax[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            radix4_pair(v[0][p], v[1][p], v[2][p], v[3][p]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float lo, hi;
                unpk2(v[j][p], lo, hi);
                amax[j] = max_abs3_nan(amax[j], lo, hi);
            }
        }
        if (!alive) amax[0] = __uint_as_float(0x7fc00000u);
        finish<kFormat, kMulti, true>(a, at, amax, span, red[it & 1], slot, [&](int j, int p) { return v[j][p]; });
    }
    if (!alive) mbar_wait(bar, phase, nullptr, a.err, kErrTimeoutDrain, limit);  // it lands before the CTA leaves
    clear_padding(a, kFormat);
}

template <typename T>
__device__ __forceinline__ T store_as(float v);
template <>
__device__ __forceinline__ float store_as(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 store_as(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half store_as(float v) { return __float2half_rn(v); }

// Four bytes of codes to four pairs of fp16, exact.
__device__ __forceinline__ void decode8(uint32_t w, __half2 (&h)[4]) {
    uint32_t r[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
        : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<__half2 *>(&r[i]);
}

// A warp takes up to 2048 columns of a row, eight to a lane and step, all steps' loads in flight.
// code * block scale is exact (in fp16 for nvfp4: six significant bits, 2^-10 .. 2688); the product with
// the row scale rounds to fp32 unless that is a power of two.
template <int kFormat, typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const DequantArgs a) {
    constexpr int kSteps = sizeof(T) == 4 ? 4 : 8;
    const int lane = threadIdx.x & 31;
    const int parts = (a.k + 256 * kSteps - 1) / (256 * kSteps);
    const uint32_t total = static_cast<uint32_t>(a.rows) * parts;
    const int64_t col_tiles = scale_col_tiles(a.k, kFormat);
    for (uint32_t i = blockIdx.x * 8u + (threadIdx.x >> 5); i < total; i += gridDim.x * 8u) {
        const uint32_t r = i / parts;
        const int c0 = static_cast<int>(i - r * parts) * (256 * kSteps) + 8 * lane;
        const int64_t at = static_cast<int64_t>(r) * a.k + c0;
        const uint32_t *codes = reinterpret_cast<const uint32_t *>(a.codes + at / 2);
        const uint8_t *scales = a.block_scales + scale_offset(r, c0 / block_of(kFormat), col_tiles);
        constexpr int kScaleStep = 256 / (4 * block_of(kFormat)) * 512;  // tiles a step, in bytes
        uint32_t w[kSteps], byte[kSteps];
#pragma unroll
        for (int p = 0; p < kSteps; ++p) {
            w[p] = byte[p] = 0;
            if (c0 + 256 * p < a.k) {
                w[p] = __ldcs(codes + 32 * p);
                byte[p] = scales[p * kScaleStep];
            }
        }
        const float row = a.row_scales[a.row_scale_count == 1 ? 0 : r];
        const f32x2 row2 = pk2(row, row);
        T *out = static_cast<T *>(a.out) + at;
#pragma unroll
        for (int p = 0; p < kSteps; ++p) {
            if (c0 + 256 * p >= a.k) break;
            __half2 h[4];
            decode8(w[p], h);
            f32x2 v[4];
            if (kFormat == kNvfp4) {
                const __half s = __half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte[p]), __NV_E4M3));
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float2 f = __half22float2(__hmul2(h[q], __half2half2(s)));
                    v[q] = fmul2(pk2(f.x, f.y), row2);
                }
            } else {
                const float s = block_scale_value(byte[p], kMxfp4);
                const f32x2 s2 = pk2(s, s);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float2 f = __half22float2(h[q]);
                    v[q] = fmul2(fmul2(pk2(f.x, f.y), s2), row2);
                }
            }
            alignas(16) T o[8];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float lo, hi;
                unpk2(v[q], lo, hi);
                o[2 * q] = store_as<T>(lo);
                o[2 * q + 1] = store_as<T>(hi);
            }
            uint4 *dst = reinterpret_cast<uint4 *>(out + 256 * p);
#pragma unroll
            for (int q = 0; q < static_cast<int>(sizeof(T)) / 2; ++q) dst[q] = reinterpret_cast<const uint4 *>(o)[q];
        }
    }
}

}  // namespace

namespace {

template <int kFormat, bool kHalf>
cudaError_t quantize_as(const QuantArgs &a, const CUtensorMap &map, cudaStream_t stream) {
    const int groups = (a.k + 255) / 256;
    const bool multi = groups > 8;
    const int warps = multi ? (groups * a.side_by_side + 7) / 8 : 4;
    const int per_cta = multi ? a.side_by_side : 4 * a.side_by_side;
    int64_t rows = (a.rows + per_cta - 1) / per_cta;
    // Enough CTAs to clear the last tile's padding at once, however few rows there are.
    if (a.rows & 127) rows = std::max<int64_t>(rows, (scale_col_tiles(a.k, kFormat) * 128 + warps * 32 - 1) / (warps * 32));
    if (a.rotation == 0) {
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(rows, a.num_sms * static_cast<int64_t>(64 / warps)));
        if (multi)
            quantize_kernel<kFormat, kHalf, true><<<grid, warps * 32, 0, stream>>>(a);
        else
            quantize_kernel<kFormat, kHalf, false><<<grid, warps * 32, 0, stream>>>(a);
        return cudaGetLastError();
    }
    const int smem = warps * 8192 + 1024;
    const int variant = !multi ? 0 : warps <= 16 ? 1 : 2;
    auto kernel = variant == 0   ? rotate_quantize_kernel<kFormat, kHalf, false, 128>
                  : variant == 1 ? rotate_quantize_kernel<kFormat, kHalf, true, 512>
                                 : rotate_quantize_kernel<kFormat, kHalf, true, 768>;
    // CTAs an SM by warps a CTA, asked once a device (a call's host time is most of a small call's).
    static std::atomic<int> resident[64][3][25];
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    std::atomic<int> &known = resident[dev][variant][warps];
    int per_sm = known.load(std::memory_order_acquire);
    if (per_sm == 0) {
        if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 24 * 8192 + 1024)) return e;
        if (cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, warps * 32, smem)) return e;
        per_sm = std::max(1, per_sm);
        known.store(per_sm, std::memory_order_release);
    }
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(rows, a.num_sms * static_cast<int64_t>(per_sm)));
    kernel<<<grid, warps * 32, smem, stream>>>(map, a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_quantize(const QuantArgs &a, const CUtensorMap &map, cudaStream_t stream) {
    const bool half = a.dtype == CTU_DTYPE_FP16;
    if (a.format == kNvfp4)
        return half ? quantize_as<kNvfp4, true>(a, map, stream) : quantize_as<kNvfp4, false>(a, map, stream);
    return half ? quantize_as<kMxfp4, true>(a, map, stream) : quantize_as<kMxfp4, false>(a, map, stream);
}

template <typename T>
static cudaError_t dequantize_as(const DequantArgs &a, cudaStream_t stream) {
    const unsigned grid = static_cast<unsigned>(
        std::min<int64_t>((a.rows * ((a.k + 1023) / 1024) + 7) / 8, static_cast<int64_t>(a.num_sms) * 8));
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

}  // namespace fp4
}  // namespace ctu

// What the affine layer norm's forward and backward kernels share: a thread's part of a row, sums over a
// team, and the choice of a kernel by shape.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "../../include/ctu_b200.h"
#include "layer_norm.cuh"
#include "ptx.cuh"

namespace ctu {
namespace norm {
namespace {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }


constexpr int kThreads = 256;  // of the looping kernels, for rows wider than a team holds

// Sum of two values over the block, in every thread.
__device__ __forceinline__ float2 block_sum(float2 v) {
    __shared__ float2 part[kThreads / 32];
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float2 s = make_float2(0.0f, 0.0f);
    for (int i = 0; i < kThreads / 32; ++i) {
        s.x += part[i].x;
        s.y += part[i].y;
    }
    return s;
}

// A thread's part of a row: kPieces loads of kVec elements (16 bytes), or of single elements where the tensors
// start differently within 16 bytes.  Elements are handled in pairs; a group is the pairs that share a load (or
// two single loads).
// kThreads: of the team, 0 where only the launch knows.  A team is no larger than its row needs, so of wide
// loads only the last one can lie beyond the row.
template <typename T, int kVec, int kPieces, int kThreads>
struct Part {
    static constexpr bool kWide = kVec > 1;
    static constexpr int kGroups = kWide ? kPieces : kPieces / 2;
    static constexpr int kPairs = kWide ? kVec / 2 : 1;  // of a group
    uint4 wide[kWide ? kPieces : 1];
    T single[kWide ? 1 : kPieces];

    static __device__ __forceinline__ int column(int piece) {
        return threadIdx.x * kVec + piece * (kThreads ? kThreads : static_cast<int>(blockDim.x)) * kVec;
    }
    // Whether a group's first element (all of them, with wide loads) and second element exist.
    static __device__ __forceinline__ bool first(int g, int h) {
        return kWide ? g + 1 < kPieces || column(g) < h : column(2 * g) < h;
    }
    static __device__ __forceinline__ bool second(int g, int h) { return kWide ? first(g, h) : column(2 * g + 1) < h; }

    // What does not exist reads as zero.
    __device__ __forceinline__ void load(const T *row, int h) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int c = column(p);
            if constexpr (kWide)
                wide[p] = first(p, h) ? __ldcs(reinterpret_cast<const uint4 *>(row + c)) : make_uint4(0u, 0u, 0u, 0u);
            else
                single[p] = c < h ? row[c] : from_f<T>(0.0f);
        }
    }
    __device__ __forceinline__ f32x2 pair(int g, int i) const {
        if constexpr (!kWide) return pk2(to_f(single[2 * g]), to_f(single[2 * g + 1]));
        const uint32_t w[4] = {wide[g].x, wide[g].y, wide[g].z, wide[g].w};
        if constexpr (sizeof(T) == 4) return pk2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return pk2(bf16lo(w[i]), bf16hi(w[i]));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        return pk2(f.x, f.y);
    }
    // One group of results.
    static __device__ __forceinline__ void store(T *row, int g, int h, const f32x2 (&v)[kPairs]) {
        float e[2 * kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; ++i) unpk2(v[i], e[2 * i], e[2 * i + 1]);
        if constexpr (kWide) {
            alignas(16) T out[kVec];
#pragma unroll
            for (int i = 0; i < kVec; ++i) out[i] = from_f<T>(e[i]);
            *reinterpret_cast<uint4 *>(row + column(g)) = *reinterpret_cast<const uint4 *>(out);
        } else {
            row[column(2 * g)] = from_f<T>(e[0]);
            if (second(g, h)) row[column(2 * g + 1)] = from_f<T>(e[1]);
        }
    }
    // One group of weights (of the input's type or fp32), `fill` where there are none.
    static __device__ __forceinline__ void weights(const void *p, bool fp32, int g, int h, float fill,
                                                   f32x2 (&out)[kPairs]) {
        if (p == nullptr) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) out[i] = pk2(fill, fill);
        } else if constexpr (!kWide) {
            const int c0 = column(2 * g), c1 = column(2 * g + 1);
            const bool two = second(g, h);
            if (fp32)
                out[0] = pk2(static_cast<const float *>(p)[c0], two ? static_cast<const float *>(p)[c1] : 0.0f);
            else
                out[0] = pk2(to_f(static_cast<const T *>(p)[c0]), two ? to_f(static_cast<const T *>(p)[c1]) : 0.0f);
        } else if (fp32) {
            const float *f = static_cast<const float *>(p) + column(g);
            if constexpr (kVec == 8) {
                // 32 bytes a lane as one load where they are aligned: two loads 32 bytes apart take twice the
                // passes of the L1, which bounds the forward pass with fp32 weights (16384 x 5120: 72 us, 59 so).
                // volatile: an asm that is not may be executed ahead of the test for a null pointer.
                if ((reinterpret_cast<uintptr_t>(p) & 31u) == 0) {
                    asm volatile("ld.global.nc.v4.b64 {%0, %1, %2, %3}, [%4];"
                                 : "=l"(out[0]), "=l"(out[1]), "=l"(out[2]), "=l"(out[3])
                                 : "l"(f)
                                 : "memory");
                    return;
                }
            }
#pragma unroll
            for (int i = 0; i < kPairs / 2; ++i) {
                const ulonglong2 u = __ldg(reinterpret_cast<const ulonglong2 *>(f) + i);
                out[2 * i] = u.x;
                out[2 * i + 1] = u.y;
            }
        } else {
            Part one;
            one.wide[0] = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p) + column(g)));
#pragma unroll
            for (int i = 0; i < kPairs; ++i) out[i] = one.pair(0, i);
        }
    }
};

// Sum of two values over a team of `warps` warps, in every thread, in a fixed order.  Two buffers in
// turn: a team's threads are past a buffer's last reads when its barrier after next is passed.
// kNamed: several teams of warps in a CTA meet at barriers of their own (which reserves all sixteen of a
// CTA, so not where occupancy counts); otherwise the CTA is one team, or every team one warp.
template <bool kNamed>
struct TeamSum {
    float2 (*part)[20];  // [2][20] of this team
    int warps;
    int barrier;
    int flip = 0;

    __device__ __forceinline__ float2 operator()(float2 v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
            v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
        }
        if (warps == 1) return v;
        float2 *buf = part[flip];
        flip ^= 1;
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) buf[warp] = v;
        if (kNamed)
            asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
        else
            __syncthreads();
        v = buf[0];
#pragma unroll
        for (int i = 1; i < 20; ++i) {
            if (i >= warps) break;
            v.x += buf[i].x;
            v.y += buf[i].y;
        }
        return v;
    }
};

__device__ __forceinline__ float both(f32x2 v) {
    float lo, hi;
    unpk2(v, lo, hi);
    return lo + hi;
}

// Rows that do not start on 16 bytes, in tensors that start alike within 16 bytes: what lies on 16 bytes (inner)
// is handled as in aligned rows, and each element before it (head) and behind it (tail) by a thread of its own:
// threads 0 to 7 of a team take the head's, 8 to 15 the tail's, in every row the same.  For that a CTA's rows
// start alike: row r starts as row r + kVec does, so CTAs take every kVec-th row.
template <int kVec>
struct Ragged {
    int head, inner, column;  // inner: a multiple of kVec; column: of the thread's own element
    bool own;

    template <typename T>
    __device__ __forceinline__ Ragged(const T *row, int h) {
        head = (-static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T))) & (kVec - 1);
        inner = (h - head) / kVec * kVec;
        const int slot = threadIdx.x, tail = h - head - inner;
        own = slot < 8 ? slot < head : slot < 8 + tail;
        column = slot < 8 ? slot : head + inner + slot - 8;
    }
};

// The rows of a team: every kPeriod-th one's from blockIdx.x % kPeriod on are shared among the CTAs of that
// remainder.  The grid is a multiple of kPeriod, or smaller than it.
template <int kPeriod>
struct TeamRows {
    int64_t first, stride;

    __device__ __forceinline__ TeamRows(int teams, int team) {
        const int64_t groups = gridDim.x < kPeriod ? 1 : gridDim.x / kPeriod;
        first = blockIdx.x % kPeriod + kPeriod * (static_cast<int64_t>(blockIdx.x / kPeriod) * teams + team);
        stride = kPeriod * groups * teams;
    }
};

inline int64_t ragged_grid(int64_t rows, int64_t ctas, int period) {
    return rows < period ? rows : std::max<int64_t>(1, ctas / period) * period;
}

template <typename T>
__device__ __forceinline__ float weight_at(const void *p, bool fp32, int c, float fill) {
    return p == nullptr ? fill : fp32 ? static_cast<const float *>(p)[c] : to_f(static_cast<const T *>(p)[c]);
}

// Weights in shared memory as fp32, a piece of eight as two fours, the first ones of all pieces together and
// the second ones: lanes then read 16 bytes 16 bytes apart, without bank conflicts.
template <typename T, int kVec>
__device__ __forceinline__ void stage_weights(float *to, const void *p, bool fp32, float fill, int head, int inner) {
    const int second_half = kVec == 8 ? inner / 2 : 0;
    const int step = blockDim.x * blockDim.y;
#pragma unroll 8
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < inner; c += step) {
        const int at = kVec == 8 ? (c & 4 ? second_half : 0) + (c >> 3) * 4 + (c & 3) : c;
        to[at] = weight_at<T>(p, fp32, head + c, fill);
    }
}
template <int kVec>
__device__ __forceinline__ void staged_weights(const float *from, int inner, int column, f32x2 (&w)[kVec / 2]) {
    const int second_half = kVec == 8 ? inner / 2 : 0;
#pragma unroll
    for (int i = 0; i < kVec / 2; i += 2) {
        const ulonglong2 u = *reinterpret_cast<const ulonglong2 *>(
            kVec == 8 ? from + (i ? second_half : 0) + column / 2 : from + column);
        w[i] = u.x;
        w[i + 1] = u.y;
    }
}

constexpr int kMaxSmem = 220 * 1024;

// Opts a kernel in to the most it may ask for, once a device.
template <typename K>
cudaError_t allow_smem(K kernel, std::atomic<bool> (&done)[64]) {
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem)) return e;
    done[dev].store(true, std::memory_order_release);
    return cudaSuccess;
}

// blockDim = (threads of a team, teams).

template <typename F>
cudaError_t with_type(int dtype, F f) {
    switch (dtype) {
    case CTU_DTYPE_BF16: return f(__nv_bfloat16());
    case CTU_DTYPE_FP16: return f(__half());
    default: return f(float());
    }
}

// Weights have the input's type or fp32.
template <typename T, typename F>
cudaError_t with_weight(const AffineArgs &a, F f) {
    return a.weight_dtype == CTU_DTYPE_FP32 ? f(float()) : f(T());
}

// How a row is held: `vec` elements a piece, `pieces` pieces a thread (0: wider than a team holds),
// `threads` of a team, `teams` a CTA.  Depends on the sizes and the alignment of rows alone.
struct TeamPlan {
    int vec, pieces, threads, teams;
};

// Five wide pieces (sixteen single elements; seven of four fp32 values where five do not hold the row) a thread
// at most, and as few threads as hold the row that way: more rows are in flight, and what a row costs a warp
// besides its elements is spread over more of them.
// With wide pieces the kernels know the team's size: a power of two up to `block`, or `block`.
inline TeamPlan team_plan(int64_t hidden, int bytes, bool wide, int block) {
    TeamPlan p{};
    p.vec = wide ? 16 / bytes : 1;
    const int64_t count = hidden / p.vec;
    const int most = p.vec == 1 ? 16 : 5;
    int64_t threads = ((count + most - 1) / most + 31) / 32 * 32;
    if (threads > block) {
        if (!wide || bytes != 4 || count > 7 * block) return p;
        threads = block;
    }
    if (p.vec > 1) {
        int64_t t = 32;
        while (t < threads) t *= 2;
        threads = std::min<int64_t>(t, block);
    }
    p.pieces = static_cast<int>((count + threads - 1) / threads);
    if (p.vec == 1) p.pieces = p.pieces <= 2 ? 2 : p.pieces <= 4 ? 4 : p.pieces <= 8 ? 8 : 16;
    p.threads = static_cast<int>(threads);
    p.teams = 1;
    return p;
}

inline bool row_aligned(const void *p) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// The same place within 16 bytes; a gradient that is not asked for counts as on 16 bytes, as those that are do:
// the others then have the same bits with it and without it.
inline bool start_alike(const void *p, const void *q) {
    return ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(q)) & 15u) == 0;
}
// Shorter rows than this are not split into a head, an inner part and a tail.
inline bool ragged_length(int64_t hidden, int bytes) { return hidden * bytes >= 64; }

// Calls f(vec, pieces, threads) with the plan's values as constants (threads 0 with single elements).  With
// wide loads that is 32 threads and one to five pieces, or more threads and what fewer do not hold: three to
// five; with kSeven also six and seven, of `block` threads, or of half as many with 16-bit values.
template <int kBlock, int kVec, int kPieces, typename F>
cudaError_t with_threads(int threads, F f) {
    using std::integral_constant;
    constexpr integral_constant<int, kVec> vec{};
    constexpr integral_constant<int, kPieces> pieces{};
    if constexpr (kVec == 1) {
        return f(vec, pieces, integral_constant<int, 0>());
    } else {
        if constexpr (kPieces <= 5)
            if (threads == 32) return f(vec, pieces, integral_constant<int, 32>());
        if constexpr (kPieces > 5) {
            constexpr int kWidest = kVec == 8 ? kBlock / 2 : kBlock;
            if (threads == kWidest) return f(vec, pieces, integral_constant<int, kWidest>());
        } else if constexpr (kPieces >= 3) {
            switch (threads) {
            case 64: return f(vec, pieces, integral_constant<int, 64>());
            case 128: return f(vec, pieces, integral_constant<int, 128>());
            case 256: return f(vec, pieces, integral_constant<int, 256>());
            case kBlock: return f(vec, pieces, integral_constant<int, kBlock>());
            default: break;
            }
        }
        return cudaErrorInvalidValue;
    }
}

template <typename T, int kBlock, bool kSeven, typename F>
cudaError_t with_shape(const TeamPlan &p, F f) {
    constexpr int kFull = 16 / sizeof(T);
    if (p.vec == 1) {
        switch (p.pieces) {
        case 2: return with_threads<kBlock, 1, 2>(p.threads, f);
        case 4: return with_threads<kBlock, 1, 4>(p.threads, f);
        case 8: return with_threads<kBlock, 1, 8>(p.threads, f);
        default: return with_threads<kBlock, 1, 16>(p.threads, f);
        }
    }
    switch (p.pieces) {
    case 1: return with_threads<kBlock, kFull, 1>(p.threads, f);
    case 2: return with_threads<kBlock, kFull, 2>(p.threads, f);
    case 3: return with_threads<kBlock, kFull, 3>(p.threads, f);
    case 4: return with_threads<kBlock, kFull, 4>(p.threads, f);
    case 5: return with_threads<kBlock, kFull, 5>(p.threads, f);
    default: break;
    }
    if constexpr (kSeven) {
        if (p.pieces == 6) return with_threads<kBlock, kFull, 6>(p.threads, f);
        if (p.pieces == 7) return with_threads<kBlock, kFull, 7>(p.threads, f);
    }
    return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace norm
}  // namespace ctu

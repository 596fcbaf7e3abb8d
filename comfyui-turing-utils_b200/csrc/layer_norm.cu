// Affine layer norm, forward and backward.
//
//   xhat = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   y    = xhat * w + b
//   g    = dy * w
//   dx   = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dw   = sum over rows of dy * xhat,   db = sum over rows of dy
//
// Statistics, sums and gradients are fp32 whatever the storage type; each result is rounded once.
//
// All passes are bound by memory: a team of lanes (a warp, or several with a named barrier) keeps a row
// in registers, as loaded, from its load to the result, so x (and dy) are read once; arithmetic is on
// packed fp32 pairs.  In the backward pass a thread keeps the same columns for every row its team takes
// and holds their sums of dw and db in registers; one CTA an SM leaves one partial sum per column, joined
// in order by a second kernel (equal shapes add in equal order).  Rows wider than a team holds take the
// looping kernels at the end.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
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

constexpr int kThreads = 256;  // of the looping kernels
constexpr int kSlices = 148;   // CTAs of the backward pass: one an SM of a B200
constexpr int kForwardBlock = 512;
constexpr int kBackwardBlock = 640;  // times 96 registers: an SM's register file

// A thread's part of a row: kPieces loads of kVec elements (16 bytes), or of single elements where rows
// do not start on 16 bytes.  Elements are handled in pairs; a group is the pairs that share a load (or
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
    static __device__ __forceinline__ void weights(const void *p, bool fp32, int g, int h, float fill, f32x2 (&out)[kPairs]) {
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
            const ulonglong2 *f = reinterpret_cast<const ulonglong2 *>(static_cast<const float *>(p) + column(g));
#pragma unroll
            for (int i = 0; i < kPairs / 2; ++i) {
                const ulonglong2 u = __ldg(f + i);
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

// blockDim = (threads of a team, teams).
// One team a CTA, or four teams of one warp.
template <typename T, int kVec, int kPieces, int kThreads>
__global__ void __maxnreg__(64) team_forward_kernel(const AffineArgs a) {
    using P = Part<T, kVec, kPieces, kThreads>;
    constexpr int kTeams = kThreads == 32 ? 4 : 1;
    __shared__ float2 part[2][20];
    const int h = a.hidden;
    const int team = kTeams > 1 ? threadIdx.y : 0;
    TeamSum<false> sum{part, kThreads ? kThreads / 32 : static_cast<int>(blockDim.x >> 5), 0};
    const bool fp32 = a.weight_dtype == CTU_DTYPE_FP32;
    const void *weight = a.weight, *bias = a.bias;
    const float epsilon = a.epsilon;
    const int64_t rows = a.rows, stride = static_cast<int64_t>(gridDim.x) * kTeams;
    const float inv_h = 1.0f / static_cast<float>(h);
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kTeams + team; r < rows; r += stride) {
        P x;
        x.load(static_cast<const T *>(a.x) + r * h, h);
        f32x2 s = pk2(0.0f, 0.0f);
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g)
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) s = fadd2(s, x.pair(g, i));
        const float mean = sum(make_float2(both(s), 0.0f)).x * inv_h;
        const f32x2 mean2 = pk2(mean, mean);
        f32x2 q = pk2(0.0f, 0.0f);
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g) {
            if (!P::first(g, h)) continue;
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) {
                f32x2 d = fsub2(x.pair(g, i), mean2);
                if (!P::kWide && !P::second(g, h)) {
                    float lo, hi;
                    unpk2(d, lo, hi);
                    d = pk2(lo, 0.0f);
                }
                q = ffma2(d, d, q);
            }
        }
        const float var = sum(make_float2(both(q), 0.0f)).x * inv_h;
        const float rstd = 1.0f / sqrtf(var + epsilon);
        if (threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        const f32x2 rstd2 = pk2(rstd, rstd);
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g) {
            if (!P::first(g, h)) continue;
            f32x2 w[P::kPairs], b[P::kPairs], y[P::kPairs];
            P::weights(weight, fp32, g, h, 1.0f, w);
            P::weights(bias, fp32, g, h, 0.0f, b);
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) y[i] = ffma2(fmul2(fsub2(x.pair(g, i), mean2), rstd2), w[i], b[i]);
            P::store(static_cast<T *>(a.out) + r * h, g, h, y);
        }
    }
}

template <typename T, int kVec, int kPieces, bool kParams>
__global__ void __launch_bounds__(kBackwardBlock) team_backward_kernel(const AffineArgs a) {
    using P = Part<T, kVec, kPieces, 0>;
    __shared__ float2 part[15][2][20];
    extern __shared__ float joined[];  // [teams - 1][2 sums][elements of a thread][threads of a team]
    const int h = a.hidden;
    const int team = threadIdx.y;
    TeamSum<true> sum{part[team], static_cast<int>(blockDim.x >> 5), 1 + team};
    const bool fp32 = a.weight_dtype == CTU_DTYPE_FP32;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.y;
    const float inv_h = 1.0f / static_cast<float>(h);
    f32x2 dw[P::kGroups][P::kPairs], db[P::kGroups][P::kPairs];
#pragma unroll
    for (int g = 0; g < P::kGroups; ++g)
#pragma unroll
        for (int i = 0; i < P::kPairs; ++i) dw[g][i] = db[g][i] = pk2(0.0f, 0.0f);
    // The next row's loads in flight, where registers allow it.
    constexpr bool kAhead = kPieces * kVec <= (sizeof(T) == 4 ? 8 : 16);
    P next_x, next_dy;
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto load = [&](int64_t r) {
        next_x.load(static_cast<const T *>(a.x) + r * h, h);
        next_dy.load(static_cast<const T *>(a.grad) + r * h, h);
        next_mean = a.mean[r];
        next_rstd = a.rstd[r];
    };
    int64_t r = static_cast<int64_t>(blockIdx.x) * blockDim.y + team;
    if (kAhead && r < a.rows) load(r);
    for (; r < a.rows; r += stride) {
        if (!kAhead) load(r);
        const P x = next_x, dy = next_dy;
        const float mean = next_mean, rstd = next_rstd;
        if (kAhead && r + stride < a.rows) load(r + stride);
        const f32x2 mean2 = pk2(mean, mean), rstd2 = pk2(rstd, rstd);
        f32x2 s = pk2(0.0f, 0.0f), t = s;
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g) {
            if (!P::first(g, h)) continue;
            f32x2 w[P::kPairs];
            if (a.dx) P::weights(a.weight, fp32, g, h, 1.0f, w);
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) {
                const f32x2 n = fmul2(fsub2(x.pair(g, i), mean2), rstd2);
                const f32x2 d = dy.pair(g, i);
                if (kParams) {
                    dw[g][i] = ffma2(d, n, dw[g][i]);
                    db[g][i] = fadd2(db[g][i], d);
                }
                if (a.dx) {
                    const f32x2 gw = fmul2(d, w[i]);
                    s = fadd2(s, gw);
                    t = ffma2(gw, n, t);
                }
            }
        }
        if (a.dx == nullptr) continue;
        const float2 st = sum(make_float2(both(s), both(t)));
        const f32x2 minus_s = pk2(-st.x * inv_h, -st.x * inv_h), minus_t = pk2(-st.y * inv_h, -st.y * inv_h);
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g) {
            if (!P::first(g, h)) continue;
            f32x2 w[P::kPairs], out[P::kPairs];
            P::weights(a.weight, fp32, g, h, 1.0f, w);
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) {
                const f32x2 n = fmul2(fsub2(x.pair(g, i), mean2), rstd2);
                out[i] = fmul2(rstd2, ffma2(n, minus_t, ffma2(dy.pair(g, i), w[i], minus_s)));
            }
            P::store(static_cast<T *>(a.dx) + r * h, g, h, out);
        }
    }
    if (!kParams) return;
    // The teams' sums, then the CTA's slice of the workspace.
    constexpr int kEach = P::kGroups * P::kPairs * 2;
    const int step = blockDim.x;
    if (team > 0) {
        float *mine = joined + static_cast<int64_t>(team - 1) * 2 * kEach * step + threadIdx.x;
#pragma unroll
        for (int e = 0; e < kEach; e += 2) {
            unpk2(dw[e / 2 / P::kPairs][e / 2 % P::kPairs], mine[e * step], mine[(e + 1) * step]);
            unpk2(db[e / 2 / P::kPairs][e / 2 % P::kPairs], mine[(kEach + e) * step], mine[(kEach + e + 1) * step]);
        }
    }
    __syncthreads();
    if (team > 0) return;
    float *out = a.workspace + static_cast<int64_t>(blockIdx.x) * 2 * h;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        float lo, hi;
        unpk2(dw[e / 2 / P::kPairs][e / 2 % P::kPairs], lo, hi);
        float sw = e & 1 ? hi : lo;
        unpk2(db[e / 2 / P::kPairs][e / 2 % P::kPairs], lo, hi);
        float sb = e & 1 ? hi : lo;
        for (int t = 0; t + 1 < static_cast<int>(blockDim.y); ++t) {
            sw += joined[(t * 2 * kEach + e) * step + threadIdx.x];
            sb += joined[((t * 2 + 1) * kEach + e) * step + threadIdx.x];
        }
        const int c = P::kWide ? P::column(e / kVec) + e % kVec : P::column(e);
        if (c < h) {
            out[c] = sw;
            out[h + c] = sb;
        }
    }
}

// Slices of partial sums joined: 32 columns by 8 runs of slices a block.
template <typename W>
__global__ void __launch_bounds__(256) team_join_kernel(const AffineArgs a, int slices) {
    __shared__ float part[8][33];
    const int c = blockIdx.x * 32 + threadIdx.x;  // of 2 * hidden: dw, then db
    const int total = 2 * a.hidden;
    float s = 0.0f;
    if (c < total) {
        const int first = slices * threadIdx.y / 8, last = slices * (threadIdx.y + 1) / 8;
#pragma unroll 4
        for (int i = first; i < last; ++i) s += a.workspace[static_cast<int64_t>(i) * total + c];
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y != 0 || c >= total) return;
    for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
    if (c < a.hidden) {
        if (a.dweight) static_cast<W *>(a.dweight)[c] = from_f<W>(s);
    } else if (a.dbias) {
        static_cast<W *>(a.dbias)[c - a.hidden] = from_f<W>(s);
    }
}

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

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) forward_kernel(const AffineArgs a) {
    const int h = a.hidden;
    const W *w = static_cast<const W *>(a.weight);
    const W *b = static_cast<const W *>(a.bias);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * h;
        T *y = static_cast<T *>(a.out) + r * h;
        float s = 0.0f;
        for (int c = threadIdx.x; c < h; c += kThreads) s += to_f(x[c]);
        const float mean = block_sum(make_float2(s, 0.0f)).x / static_cast<float>(h);
        float q = 0.0f;
        for (int c = threadIdx.x; c < h; c += kThreads) {
            const float d = to_f(x[c]) - mean;
            q += d * d;
        }
        const float var = block_sum(make_float2(q, 0.0f)).x / static_cast<float>(h);
        const float rstd = 1.0f / sqrtf(var + a.epsilon);
        if (threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int c = threadIdx.x; c < h; c += kThreads) {
            const float n = (to_f(x[c]) - mean) * rstd;
            y[c] = from_f<T>(n * (w ? to_f(w[c]) : 1.0f) + (b ? to_f(b[c]) : 0.0f));
        }
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) input_gradient_kernel(const AffineArgs a) {
    const int h = a.hidden;
    const W *w = static_cast<const W *>(a.weight);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * h;
        const T *dy = static_cast<const T *>(a.grad) + r * h;
        T *dx = static_cast<T *>(a.dx) + r * h;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float2 s = make_float2(0.0f, 0.0f);
        for (int c = threadIdx.x; c < h; c += kThreads) {
            const float n = (to_f(x[c]) - mean) * rstd;
            const float g = to_f(dy[c]) * (w ? to_f(w[c]) : 1.0f);
            s.x += g;
            s.y += g * n;
        }
        s = block_sum(s);
        s.x /= static_cast<float>(h);
        s.y /= static_cast<float>(h);
        for (int c = threadIdx.x; c < h; c += kThreads) {
            const float n = (to_f(x[c]) - mean) * rstd;
            const float g = to_f(dy[c]) * (w ? to_f(w[c]) : 1.0f);
            dx[c] = from_f<T>(rstd * (g - s.x - n * s.y));
        }
    }
}

// Partial sums of one slice of rows: workspace [slice][0: dw, 1: db][hidden].
template <typename T>
__global__ void __launch_bounds__(256) parameter_partial_kernel(const AffineArgs a, int slices) {
    __shared__ float2 part[8][33];
    const int h = a.hidden;
    const int c = blockIdx.x * 32 + threadIdx.x;
    const int slice = blockIdx.y;
    float2 s = make_float2(0.0f, 0.0f);
    if (c < h) {
        for (int64_t r = slice * 8 + threadIdx.y; r < a.rows; r += static_cast<int64_t>(slices) * 8) {
            const float dy = to_f(static_cast<const T *>(a.grad)[r * h + c]);
            s.x += dy * ((to_f(static_cast<const T *>(a.x)[r * h + c]) - a.mean[r]) * a.rstd[r]);
            s.y += dy;
        }
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && c < h) {
        for (int i = 1; i < 8; ++i) {
            s.x += part[i][threadIdx.x].x;
            s.y += part[i][threadIdx.x].y;
        }
        a.workspace[(static_cast<int64_t>(slice) * 2) * h + c] = s.x;
        a.workspace[(static_cast<int64_t>(slice) * 2 + 1) * h + c] = s.y;
    }
}

template <typename F>
cudaError_t with_type(int dtype, F f) {
    switch (dtype) {
    case CTU_DTYPE_BF16: return f(__nv_bfloat16());
    case CTU_DTYPE_FP16: return f(__half());
    default: return f(float());
    }
}

}  // namespace

namespace {
// Weights have the input's type or fp32.
template <typename T, typename F>
cudaError_t with_weight(const AffineArgs &a, F f) {
    return a.weight_dtype == CTU_DTYPE_FP32 ? f(float()) : f(T());
}
}  // namespace

// How a row is held: `vec` elements a piece, `pieces` pieces a thread (0: wider than a team holds),
// `threads` of a team, `teams` a CTA.  Depends on the sizes and the alignment of rows alone.
namespace {
struct TeamPlan {
    int vec, pieces, threads, teams;
};

TeamPlan team_plan(int64_t hidden, int bytes, bool aligned, bool backward) {
    TeamPlan p{};
    p.vec = aligned && hidden * bytes % 16 == 0 ? 16 / bytes : 1;
    const int64_t count = hidden / p.vec;
    const int block = backward ? kBackwardBlock : kForwardBlock;
    // Pieces a thread, as many as its registers hold.  Forward (64): x alone.  Backward (96): two fp32 sums
    // an element, x, dy and the next row's x and dy; more pieces, without the next row, only for rows that
    // the CTA would not hold otherwise.
    int most = p.vec == 1 ? (backward ? 8 : 16) : backward ? 2 : 5;
    if (backward && (count + most - 1) / most > block) most = p.vec == 1 ? 16 : p.vec == 4 ? 4 : 3;
    int64_t threads = ((count + most - 1) / most + 31) / 32 * 32;
    if (threads > block) return p;
    if (!backward && p.vec > 1) {  // a power of two, which the kernels know
        int64_t t = 32;
        while (t < threads) t *= 2;
        threads = t;
    }
    p.pieces = static_cast<int>((count + threads - 1) / threads);
    if (p.vec == 1) p.pieces = p.pieces <= 2 ? 2 : p.pieces <= 4 ? 4 : p.pieces <= 8 ? 8 : 16;
    p.threads = static_cast<int>(threads);
    // Forward CTAs are small (a team, or four of a warp) and many; a backward CTA fills an SM, with at most
    // fifteen teams (named barriers).
    p.teams = static_cast<int>(backward ? std::min<int64_t>(15, block / threads) : p.vec > 1 && threads == 32 ? 4 : 1);
    return p;
}

bool row_aligned(const void *p) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int kVec, bool kBackward, typename F>
cudaError_t with_pieces(int pieces, F f) {
    if constexpr (kVec == 1) {
        switch (pieces) {
        case 2: return f(std::integral_constant<int, 2>());
        case 4: return f(std::integral_constant<int, 4>());
        case 8: return f(std::integral_constant<int, 8>());
        case 16: return f(std::integral_constant<int, 16>());
        default: return cudaErrorInvalidValue;
        }
    } else {
        switch (pieces) {
        case 1: return f(std::integral_constant<int, 1>());
        case 2: return f(std::integral_constant<int, 2>());
        case 3: return f(std::integral_constant<int, 3>());
        default: break;
        }
        if constexpr (!kBackward || kVec == 4) {
            if (pieces == 4) return f(std::integral_constant<int, 4>());
        }
        if constexpr (!kBackward) {
            if (pieces == 5) return f(std::integral_constant<int, 5>());
        }
        return cudaErrorInvalidValue;
    }
}

// Forward teams of wide loads: 32 threads and one to five pieces, or 64 to 512 and what those do not hold,
// three to five.
template <int kVec, int kPieces, typename F>
cudaError_t with_threads(int threads, F f) {
    if constexpr (kVec == 1) {
        return f(std::integral_constant<int, 0>());
    } else {
        if (threads == 32) return f(std::integral_constant<int, 32>());
        if constexpr (kPieces >= 3) {
            switch (threads) {
            case 64: return f(std::integral_constant<int, 64>());
            case 128: return f(std::integral_constant<int, 128>());
            case 256: return f(std::integral_constant<int, 256>());
            case 512: return f(std::integral_constant<int, 512>());
            default: break;
            }
        }
        return cudaErrorInvalidValue;
    }
}

template <typename T, bool kBackward, typename F>
cudaError_t with_shape(const TeamPlan &p, F f) {
    constexpr int kFull = 16 / sizeof(T);
    if (p.vec == kFull)
        return with_pieces<kFull, kBackward>(p.pieces, [&](auto n) { return f(std::integral_constant<int, kFull>(), n); });
    return with_pieces<1, kBackward>(p.pieces, [&](auto n) { return f(std::integral_constant<int, 1>(), n); });
}
}  // namespace

int64_t backward_slices(int64_t rows, int64_t) { return std::max<int64_t>(1, std::min<int64_t>(kSlices, rows)); }

cudaError_t launch_layer_norm(const AffineArgs &a, cudaStream_t stream) {
    const bool aligned = row_aligned(a.x) && row_aligned(a.out) && row_aligned(a.weight) && row_aligned(a.bias);
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const TeamPlan plan = team_plan(a.hidden, sizeof(T), aligned, false);
        if (plan.pieces == 0) {
            const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, a.num_sms * 8));
            return with_weight<T>(a, [&](auto w) {
                forward_kernel<T, decltype(w)><<<grid, kThreads, 0, stream>>>(a);
                return cudaGetLastError();
            });
        }
        const unsigned grid = static_cast<unsigned>(
            std::min<int64_t>((a.rows + plan.teams - 1) / plan.teams, static_cast<int64_t>(a.num_sms) * 16));
        return with_shape<T, false>(plan, [&](auto vec, auto pieces) {
            return with_threads<vec, pieces>(plan.threads, [&](auto threads) {
                team_forward_kernel<T, vec, pieces, threads>
                    <<<grid, dim3(plan.threads, plan.teams), 0, stream>>>(a);
                return cudaGetLastError();
            });
        });
    });
}

cudaError_t launch_layer_norm_backward(const AffineArgs &a, cudaStream_t stream) {
    const bool aligned = row_aligned(a.x) && row_aligned(a.grad) && row_aligned(a.dx) && row_aligned(a.weight);
    const bool params = a.dweight || a.dbias;
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const TeamPlan plan = team_plan(a.hidden, sizeof(T), aligned, true);
        if (plan.pieces == 0) {
            const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, a.num_sms * 8));
            const int slices = static_cast<int>(std::min<int64_t>(64, backward_slices(a.rows, a.hidden)));
            return with_weight<T>(a, [&](auto w) {
                using W = decltype(w);
                if (a.dx && a.rows > 0) input_gradient_kernel<T, W><<<grid, kThreads, 0, stream>>>(a);
                if (params) {
                    parameter_partial_kernel<T>
                        <<<dim3((a.hidden + 31) / 32, slices), dim3(32, 8), 0, stream>>>(a, slices);
                    team_join_kernel<W><<<(2 * a.hidden + 31) / 32, dim3(32, 8), 0, stream>>>(a, slices);
                }
                return cudaGetLastError();
            });
        }
        const int64_t ctas = std::min<int64_t>((a.rows + plan.teams - 1) / plan.teams, kSlices);
        const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, ctas));
        const cudaError_t e = with_shape<T, true>(plan, [&](auto vec, auto pieces) {
            const dim3 block(plan.threads, plan.teams);
            if (!params) {
                team_backward_kernel<T, vec, pieces, false><<<grid, block, 0, stream>>>(a);
                return cudaGetLastError();
            }
            auto kernel = team_backward_kernel<T, vec, pieces, true>;
            const int smem = (plan.teams - 1) * 2 * vec * pieces * plan.threads * static_cast<int>(sizeof(float));
            if (smem > 32768)
                if (cudaError_t f = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))
                    return f;
            kernel<<<grid, block, smem, stream>>>(a);
            return cudaGetLastError();
        });
        if (e != cudaSuccess || !params) return e;
        return with_weight<T>(a, [&](auto w) {
            team_join_kernel<decltype(w)>
                <<<(2 * a.hidden + 31) / 32, dim3(32, 8), 0, stream>>>(a, static_cast<int>(grid));
            return cudaGetLastError();
        });
    });
}

}  // namespace norm
}  // namespace ctu

// Affine layer norm, forward pass:
//
//   xhat = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = xhat * w + b
//
// Statistics and sums are fp32 whatever the storage type; each result is rounded once.  Bound by memory:
// a team of lanes (a warp, or a CTA of several) keeps a row in registers, as loaded, so x is read once;
// arithmetic is on packed fp32 pairs.  32760 x 5120 bf16: 114 us, 5.9 TB/s (0.91 of a copy's rate); with the
// team's size a launch parameter, so that each access computed its address and bounds, 154 us.  Rows off 16
// bytes: 32760 x 5121 119 us (with loads of single elements 540 us).  Rows wider than a team holds take the
// looping kernel.
#include "layer_norm_parts.cuh"

namespace ctu {
namespace norm {

namespace {

constexpr int kForwardBlock = 512;

// One team a CTA, or four teams of one warp.
template <typename T, int kVec, int kPieces, int kThreads>
__global__ void __maxnreg__(kPieces > 5 && sizeof(T) == 2 && kVec > 1 ? 80 : 64) team_forward_kernel(const AffineArgs a) {
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

// Threads of a CTA and CTAs of an SM in the kernel below.
template <typename T, int kPieces>
constexpr int kRaggedCtas = kPieces > 5 && sizeof(T) == 2 ? 1 : 2;
template <typename T, int kPieces>
constexpr int kRaggedBlock = kPieces > 5 && sizeof(T) == 2 ? 768 : kForwardBlock;

// Rows that do not start on 16 bytes.  Neither do their weights, so those are in shared memory, shifted as the
// CTA's rows are; CTAs are large, so that they are copied there once for many rows.  blockDim = (threads of a
// team, teams).
template <typename T, int kPieces, int kThreads>
__global__ void __launch_bounds__(kRaggedBlock<T, kPieces>, kRaggedCtas<T, kPieces>) ragged_forward_kernel(const AffineArgs a) {
    constexpr int kVec = 16 / sizeof(T);
    using P = Part<T, kVec, kPieces, kThreads>;
    __shared__ float2 part[kThreads > 32 ? kRaggedBlock<T, kPieces> / kThreads : 1][2][20];
    __shared__ float ends[2][16];
    extern __shared__ __align__(16) float weights[];
    const int h = a.hidden;
    const int team = threadIdx.y;
    const TeamRows<kVec> mine(blockDim.y, team);
    const T *const from = static_cast<const T *>(a.x);
    const Ragged<kVec> at(from + mine.first * h, h);
    const int inner = at.inner;
    TeamSum<true> sum{part[kThreads > 32 ? team : 0], kThreads / 32, 1 + team};
    const bool fp32 = a.weight_dtype == CTU_DTYPE_FP32;
    const float inv_h = 1.0f / static_cast<float>(h);
    P x;
    float own = 0.0f;
    stage_weights<T, kVec>(weights, a.weight, fp32, 1.0f, at.head, inner);
    stage_weights<T, kVec>(weights + inner, a.bias, fp32, 0.0f, at.head, inner);
    if (at.own && team == 0) {
        ends[0][threadIdx.x] = weight_at<T>(a.weight, fp32, at.column, 1.0f);
        ends[1][threadIdx.x] = weight_at<T>(a.bias, fp32, at.column, 0.0f);
    }
    __syncthreads();
    const int rows = static_cast<int>(a.rows), stride = static_cast<int>(mine.stride);
    for (int r = static_cast<int>(mine.first); r < rows; r += stride) {
        const T *const row = from + static_cast<int64_t>(r) * h;
        x.load(row + at.head, inner);
        if (at.own) own = to_f(row[at.column]);
        f32x2 s = pk2(own, 0.0f);
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g)
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) s = fadd2(s, x.pair(g, i));
        const float mean = sum(make_float2(both(s), 0.0f)).x * inv_h;
        const f32x2 mean2 = pk2(mean, mean);
        const float own_d = at.own ? own - mean : 0.0f;
        f32x2 q = pk2(own_d * own_d, 0.0f);
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g) {
            if (!P::first(g, inner)) continue;
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) {
                const f32x2 d = fsub2(x.pair(g, i), mean2);
                q = ffma2(d, d, q);
            }
        }
        const float var = sum(make_float2(both(q), 0.0f)).x * inv_h;
        const float rstd = 1.0f / sqrtf(var + a.epsilon);
        if (threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        const f32x2 rstd2 = pk2(rstd, rstd);
        T *const out = static_cast<T *>(a.out) + static_cast<int64_t>(r) * h;
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g) {
            if (!P::first(g, inner)) continue;
            f32x2 w[P::kPairs], b[P::kPairs], y[P::kPairs];
            staged_weights<kVec>(weights, inner, P::column(g), w);
            staged_weights<kVec>(weights + inner, inner, P::column(g), b);
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) y[i] = ffma2(fmul2(fsub2(x.pair(g, i), mean2), rstd2), w[i], b[i]);
            P::store(out + at.head, g, inner, y);
        }
        if (at.own) out[at.column] = from_f<T>(fmaf((own - mean) * rstd, ends[0][threadIdx.x], ends[1][threadIdx.x]));
    }
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

}  // namespace

cudaError_t launch_layer_norm(const AffineArgs &a, cudaStream_t stream) {
    const bool aligned = row_aligned(a.x) && row_aligned(a.out) && row_aligned(a.weight) && row_aligned(a.bias);
    return with_type(a.dtype, [&](auto t) {
        using T = decltype(t);
        const bool whole = aligned && a.hidden * static_cast<int64_t>(sizeof(T)) % 16 == 0;
        const bool ragged = !whole && start_alike(a.x, a.out) && ragged_length(a.hidden, sizeof(T)) &&
                            a.rows < (int64_t{1} << 30);  // counted in 32 bits
        TeamPlan plan = team_plan(a.hidden, sizeof(T), whole || ragged, kForwardBlock);
        // Wide rows of 16-bit values: up to seven pieces in half the threads keep more bytes in flight than four in
        // all (6000 x 13824 bf16: 81 us, 68 so; 6000 x 13823: 104, 75).
        if (sizeof(T) == 2 && plan.vec > 1 && plan.threads == kForwardBlock &&
            a.hidden / plan.vec <= 7 * (kForwardBlock / 2)) {
            plan.threads = kForwardBlock / 2;
            plan.pieces = (a.hidden / plan.vec + plan.threads - 1) / plan.threads;
        }
        if (plan.pieces == 0) {
            const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, a.num_sms * 8));
            return with_weight<T>(a, [&](auto w) {
                forward_kernel<T, decltype(w)><<<grid, kThreads, 0, stream>>>(a);
                return cudaGetLastError();
            });
        }
        // CTAs are small and many: a team, or four of a warp.
        if (plan.vec > 1 && plan.threads == 32) plan.teams = 4;
        const unsigned grid = static_cast<unsigned>(
            std::min<int64_t>((a.rows + plan.teams - 1) / plan.teams, static_cast<int64_t>(a.num_sms) * 16));
        return with_shape<T, kForwardBlock, true>(plan, [&](auto vec, auto pieces, auto threads) {
            if constexpr (vec > 1) {
                if (ragged) {
                    // As many teams as the rows give every SM two CTAs of, and as many CTAs as run at once.
                    const int smem = 2 * a.hidden * static_cast<int>(sizeof(float));
                    const int each = smem + 4096 <= 114 * 1024 ? kRaggedCtas<T, pieces> : 1;
                    plan.teams = static_cast<int>(std::min<int64_t>(
                        kRaggedBlock<T, pieces> / threads, (a.rows + each * a.num_sms - 1) / (each * a.num_sms)));
                    auto kernel = ragged_forward_kernel<T, pieces, threads>;
                    static std::atomic<bool> done[64];
                    if (cudaError_t e = allow_smem(kernel, done)) return e;
                    const int64_t ctas = (a.rows + plan.teams - 1) / plan.teams;
                    const int64_t some = ragged_grid(a.rows, std::min<int64_t>(ctas + vec - 1, a.num_sms * each), vec);
                    kernel<<<static_cast<unsigned>(some), dim3(plan.threads, plan.teams), smem, stream>>>(a);
                    return cudaGetLastError();
                }
            }
            team_forward_kernel<T, vec, pieces, threads><<<grid, dim3(plan.threads, plan.teams), 0, stream>>>(a);
            return cudaGetLastError();
        });
    });
}

int64_t backward_slices(int64_t rows, int64_t) { return std::max<int64_t>(1, std::min<int64_t>(kSlices, rows)); }

cudaError_t launch_layer_norm_backward(const AffineArgs &a, const WaitLimit &wait, cudaStream_t stream) {
    return with_type(a.dtype, [&](auto t) { return backward_as<decltype(t)>(a, wait, stream); });
}

}  // namespace norm
}  // namespace ctu

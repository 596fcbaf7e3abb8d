// Affine layer norm, backward pass (xhat as in the forward pass):
//
//   g  = dy * w,  dx = rstd * (g - mean(g) - xhat * mean(g * xhat))
//   dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// A thread keeps the same columns for every row its team takes and holds their sums of dw and db in
// registers; one CTA an SM leaves one partial sum per column, joined in order by a second kernel (equal
// shapes that start alike within 16 bytes add in equal order).  Sums are fp32; each result is rounded once.
//
// Bytes in flight bound it: a team's next rows of x and dy are copied into shared memory (bulk copies, two
// rows deep; fp32 rows beyond 10240 values, one deep) while it works on one, and the weights are there as fp32,
// so registers hold the sums alone.  Of rows off 16 bytes that is the inner part.  Where x, dy and dx do not
// start alike within 16 bytes, rows are kept in registers, loaded by single elements; rows wider than a team
// holds take the looping kernels.
//
// Measured: 4096 x 5120 bf16 36 us and 5 for the join (54 us with rows in registers); 32760 x 5120 173 us (5.8
// TB/s), 5121 wide 210; 6000 x 13823 fp32 195 us, 5.1 TB/s (looping 486); one row of 5120 11.7 us, two launches.
#pragma once

#include "layer_norm_parts.cuh"

namespace ctu {
namespace norm {

namespace {

constexpr int kBackwardBlock = 512;  // times 128 registers: an SM's register file

// Sums of an element of its own that a thread may have, and where the inner part starts: see Ragged.
struct OwnSums {
    int head, inner, column;
    bool own;
    float dw, db;
};

// The teams' sums to the CTA's slice of the workspace: through shared memory ([teams][dw, db][hidden]),
// added over the teams in order, written 128 bytes a warp (one team gathering the others' by element took 5 us
// longer at 5120 columns).  Every team has left its last row when this is called.
template <typename P>
__device__ __forceinline__ void leave_sums(const AffineArgs &a, const f32x2 (&dw)[P::kGroups][P::kPairs],
                                           const f32x2 (&db)[P::kGroups][P::kPairs], const OwnSums &own,
                                           float *sums) {
    if (!a.dweight && !a.dbias) return;
    const int h = a.hidden;
    __syncthreads();
    float *mine = sums + static_cast<int64_t>(threadIdx.y) * 2 * h;
    if (own.own) {
        mine[own.column] = own.dw;
        mine[h + own.column] = own.db;
    }
#pragma unroll
    for (int g = 0; g < P::kGroups; ++g) {
        if (!P::first(g, own.inner)) continue;
        const int c0 = own.head + P::column(P::kWide ? g : 2 * g);
        const int c1 = P::kWide ? c0 + 1 : P::column(2 * g + 1);
        const bool two = P::second(g, own.inner);
#pragma unroll
        for (int i = 0; i < P::kPairs; ++i) {
            float lo, hi;
            unpk2(dw[g][i], lo, hi);
            mine[c0 + 2 * i] = lo;
            if (two) mine[c1 + 2 * i] = hi;
            unpk2(db[g][i], lo, hi);
            mine[h + c0 + 2 * i] = lo;
            if (two) mine[h + c1 + 2 * i] = hi;
        }
    }
    __syncthreads();
    float *out = a.workspace + static_cast<int64_t>(blockIdx.x) * 2 * h;
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < 2 * h; c += blockDim.x * blockDim.y) {
        float v = sums[c];
        for (int t = 1; t < static_cast<int>(blockDim.y); ++t) v += sums[t * 2 * h + c];
        out[c] = v;
    }
}

// Rows of single elements, in registers.  blockDim = (threads of a team, teams).
template <typename T, int kPieces>
__global__ void __launch_bounds__(kBackwardBlock) team_backward_kernel(const AffineArgs a) {
    using P = Part<T, 1, kPieces, 0>;
    __shared__ float2 part[15][2][20];
    extern __shared__ float joined[];
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
    const void *weight = a.weight;
    T *const dx = static_cast<T *>(a.dx);
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * blockDim.y + team; r < a.rows; r += stride) {
        P x, dy;
        x.load(static_cast<const T *>(a.x) + r * h, h);
        dy.load(static_cast<const T *>(a.grad) + r * h, h);
        const float mean = a.mean[r], rstd = a.rstd[r];
        const f32x2 mean2 = pk2(mean, mean), rstd2 = pk2(rstd, rstd);
        f32x2 s = pk2(0.0f, 0.0f), t = s;
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g) {
            if (!P::first(g, h)) continue;
            f32x2 w[P::kPairs];
            if (dx) P::weights(weight, fp32, g, h, 1.0f, w);
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) {
                const f32x2 n = fmul2(fsub2(x.pair(g, i), mean2), rstd2);
                const f32x2 d = dy.pair(g, i);
                dw[g][i] = ffma2(d, n, dw[g][i]);
                db[g][i] = fadd2(db[g][i], d);
                if (dx) {
                    const f32x2 gw = fmul2(d, w[i]);
                    s = fadd2(s, gw);
                    t = ffma2(gw, n, t);
                }
            }
        }
        if (dx == nullptr) continue;
        const float2 st = sum(make_float2(both(s), both(t)));
        const f32x2 minus_s = pk2(-st.x * inv_h, -st.x * inv_h), minus_t = pk2(-st.y * inv_h, -st.y * inv_h);
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g) {
            if (!P::first(g, h)) continue;
            f32x2 w[P::kPairs], out[P::kPairs];
            P::weights(weight, fp32, g, h, 1.0f, w);
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) {
                const f32x2 n = fmul2(fsub2(x.pair(g, i), mean2), rstd2);
                out[i] = fmul2(rstd2, ffma2(n, minus_t, ffma2(dy.pair(g, i), w[i], minus_s)));
            }
            P::store(dx + r * h, g, h, out);
        }
    }
    leave_sums<P>(a, dw, db, OwnSums{0, h, 0, false, 0.0f, 0.0f}, joined);
}

// Wide rows through shared memory.  blockDim = (kTeam, teams); dynamic shared memory holds the weights as
// fp32, then [teams][2 buffers][x, dy] rows, and the teams' sums at the end.
template <typename T, int kPieces, int kTeam, bool kRagged>
__global__ void __launch_bounds__(kBackwardBlock) staged_backward_kernel(const AffineArgs a, const WaitLimit wait) {
    constexpr int kVec = 16 / sizeof(T);
    using P = Part<T, kVec, kPieces, kTeam>;
    constexpr int kTeams = kBackwardBlock / kTeam;
    constexpr bool kNamed = kTeam > 32 && kTeams > 1;
    constexpr int kDepth = kPieces > 5 ? 1 : 2;  // rows in shared memory: of the widest, one
    static_assert(kDepth == 2 || kTeams == 1, "the barrier below is the CTA's");
    __shared__ float2 part[kTeams][2][20];
    __shared__ uint64_t bars[kTeams][2], dead;  // dead: nothing arrives on it (test hook)
    // Whether a wait of a team gave up (its other waits then do at once), and rows whose copies were issued.
    __shared__ int gave_up[kTeams], issued[kTeams];
    // Of a thread's own element, in shared memory as registers are short (32760 x 5121 bf16: 246 us with them in
    // registers and rows counted in 64 bits, 210 so): weight, sums of dw and db, and the row's dy * w and xhat.
    enum { kOwnW, kOwnDw, kOwnDb, kOwnGw, kOwnN };
    __shared__ float ends[kRagged ? kTeams : 1][5][16];
    extern __shared__ __align__(16) uint8_t smem[];
    const int team = threadIdx.y;
    const TeamRows<kRagged ? kVec : 1> mine(kTeams, team);
    // Rows are counted in 32 bits: backward_as sees to it that they can be.
    const int stride = static_cast<int>(mine.stride), first = static_cast<int>(mine.first);
    const int rows_end = static_cast<int>(a.rows);
    const Ragged<kVec> at(static_cast<const T *>(a.x) + static_cast<int64_t>(first) * a.hidden, a.hidden);
    const int head = kRagged ? at.head : 0;
    const int h = kRagged ? at.inner : a.hidden;  // of a row's part on 16 bytes
    const bool has_own = kRagged && at.own;
    const uint32_t row_bytes = static_cast<uint32_t>(h) * sizeof(T);
    float *const weights = reinterpret_cast<float *>(smem);
    uint8_t *const rows = smem + h * 4 + team * 4 * row_bytes;
    TeamSum<kNamed> sum{part[team], kTeam / 32, 1 + team};
    const float inv_h = 1.0f / static_cast<float>(a.hidden);
    T *const dx = static_cast<T *>(a.dx);

    auto load = [&](int r, int buf) {  // one thread of the team
        uint8_t *dst = rows + buf * 2 * row_bytes;
        uint64_t *bar = &bars[team][buf];
        const int64_t from = static_cast<int64_t>(r) * a.hidden + head;
        mbar_arrive_expect_tx(bar, 2 * row_bytes);
        bulk_load(dst, static_cast<const T *>(a.x) + from, row_bytes, bar);
        bulk_load(dst + row_bytes, static_cast<const T *>(a.grad) + from, row_bytes, bar);
        ++issued[team];
    };
    if (threadIdx.x == 0) {
        mbar_init(&bars[team][0], 1);
        mbar_init(&bars[team][1], 1);
        if (team == 0) mbar_init(&dead, 1);
        gave_up[team] = issued[team] = 0;
        fence_mbar_init();
        if (first < rows_end) load(first, 0);
        if (kDepth == 2 && first + stride < rows_end) load(first + stride, 1);
    }
    const bool fp32 = a.weight_dtype == CTU_DTYPE_FP32;
    stage_weights<T, kVec>(weights, a.weight, fp32, 1.0f, head, h);
    float own_x = 0.0f, own_dy = 0.0f;
    auto own = [&](int what) -> float & { return ends[kRagged ? team : 0][what][threadIdx.x]; };
    auto load_own = [&](int r) {
        const int64_t from = static_cast<int64_t>(r) * a.hidden + at.column;
        own_x = to_f(static_cast<const T *>(a.x)[from]);
        own_dy = to_f(static_cast<const T *>(a.grad)[from]);
    };
    if (has_own) {
        own(kOwnW) = weight_at<T>(a.weight, fp32, at.column, 1.0f);
        own(kOwnDw) = own(kOwnDb) = 0.0f;
        if (first < rows_end) load_own(first);
    }
    __syncthreads();

    f32x2 dw[P::kGroups][P::kPairs], db[P::kGroups][P::kPairs];
#pragma unroll
    for (int g = 0; g < P::kGroups; ++g)
#pragma unroll
        for (int i = 0; i < P::kPairs; ++i) dw[g][i] = db[g][i] = pk2(0.0f, 0.0f);
    // One piece of x, dy and the weights.
    auto piece = [&](const uint8_t *row, int g, Part<T, kVec, 1, kTeam> &x, Part<T, kVec, 1, kTeam> &dy,
                     f32x2 (&w)[P::kPairs]) {
        const int c = P::column(g);
        x.wide[0] = *reinterpret_cast<const uint4 *>(row + c * sizeof(T));
        dy.wide[0] = *reinterpret_cast<const uint4 *>(row + row_bytes + c * sizeof(T));
        staged_weights<kVec>(weights, h, c, w);
    };
    float next_mean = 0.0f, next_rstd = 0.0f;
    if (first < rows_end) {
        next_mean = a.mean[first];
        next_rstd = a.rstd[first];
    }
    // After a wait that gave up the team's rows and its columns' sums are NaN, and no more is loaded.
    const float nan = __uint_as_float(0x7fc00000u);
    volatile int *const lost = &gave_up[team];
    int buf = 0;
    uint32_t phase = 0;
    for (int r = first; r < rows_end; r += stride) {
        const float mean = next_mean, rstd = next_rstd;
        const f32x2 mean2 = pk2(mean, mean), rstd2 = pk2(rstd, rstd);
        if (r + stride < rows_end) {
            next_mean = a.mean[r + stride];
            next_rstd = a.rstd[r + stride];
        }
        const bool never = r == first + wait.never * stride && blockIdx.x == 0 && team == 0;
        mbar_wait(never ? &dead : &bars[team][buf], never ? 0u : phase, lost, a.err, kErrTimeoutFull, wait.ns);
        const float start = *lost ? nan : 0.0f;
        const uint8_t *row = rows + buf * 2 * row_bytes;
        f32x2 s = pk2(0.0f, start), t = pk2(0.0f, 0.0f);
        if (has_own) {
            const float n = (own_x - mean) * rstd, gw = own_dy * own(kOwnW);
            own(kOwnDw) = fmaf(own_dy, n, own(kOwnDw));
            own(kOwnDb) += own_dy;
            own(kOwnGw) = gw;
            own(kOwnN) = n;
            s = pk2(gw, start);
            t = pk2(gw * n, 0.0f);
            if (r + stride < rows_end) load_own(r + stride);
        }
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g) {
            if (!P::first(g, h)) continue;
            Part<T, kVec, 1, kTeam> x, dy;
            f32x2 w[P::kPairs];
            piece(row, g, x, dy, w);
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) {
                const f32x2 n = fmul2(fsub2(x.pair(0, i), mean2), rstd2);
                const f32x2 d = dy.pair(0, i);
                dw[g][i] = ffma2(d, n, dw[g][i]);
                db[g][i] = fadd2(db[g][i], d);
                const f32x2 gw = fmul2(d, w[i]);
                s = fadd2(s, gw);
                t = ffma2(gw, n, t);
            }
        }
        const float2 st = sum(make_float2(both(s), both(t)));
        // Every thread of the team is past the row before: its buffer takes the row after the next.
        if (kTeam == 32) __syncwarp();
        if (kDepth == 2 && threadIdx.x == 0 && !*lost && r != first && r + stride < rows_end) {
            fence_proxy_async_smem();
            load(r + stride, buf ^ 1);
        }
        const f32x2 minus_s = pk2(-st.x * inv_h, -st.x * inv_h), minus_t = pk2(-st.y * inv_h, -st.y * inv_h);
        if (dx != nullptr) {
            if (has_own)
                dx[static_cast<int64_t>(r) * a.hidden + at.column] =
                    from_f<T>(rstd * (own(kOwnGw) - st.x * inv_h - own(kOwnN) * (st.y * inv_h)));
#pragma unroll
            for (int g = 0; g < P::kGroups; ++g) {
                if (!P::first(g, h)) continue;
                Part<T, kVec, 1, kTeam> x, dy;
                f32x2 w[P::kPairs], out[P::kPairs];
                piece(row, g, x, dy, w);
#pragma unroll
                for (int i = 0; i < P::kPairs; ++i) {
                    const f32x2 n = fmul2(fsub2(x.pair(0, i), mean2), rstd2);
                    out[i] = fmul2(rstd2, ffma2(n, minus_t, ffma2(dy.pair(0, i), w[i], minus_s)));
                }
                P::store(dx + static_cast<int64_t>(r) * a.hidden + head, g, h, out);
            }
        }
        if (kDepth == 2) {
            buf ^= 1;
            if (buf == 0) phase ^= 1u;
        } else {
            __syncthreads();
            if (threadIdx.x == 0 && !*lost && r + stride < rows_end) {
                fence_proxy_async_smem();
                load(r + stride, 0);
            }
            phase ^= 1u;
        }
    }
    const bool whole = !*lost;
    if (!whole) {
        if (threadIdx.x == 0) {
            // Copies in flight land before shared memory is used otherwise.
            for (int i = max(0, issued[team] - kDepth); i < issued[team]; ++i)
                if (!mbar_wait(&bars[team][i & (kDepth - 1)], (kDepth == 2 ? i >> 1 : i) & 1, nullptr, a.err, kErrTimeoutDrain, wait.ns))
                    break;
        }
#pragma unroll
        for (int g = 0; g < P::kGroups; ++g)
#pragma unroll
            for (int i = 0; i < P::kPairs; ++i) dw[g][i] = db[g][i] = pk2(nan, nan);
    }
    const bool own_sums = has_own && whole;
    leave_sums<P>(a, dw, db,
                  OwnSums{head, h, at.column, has_own, own_sums ? own(kOwnDw) : nan, own_sums ? own(kOwnDb) : nan},
                  reinterpret_cast<float *>(smem));
}

// Slices of partial sums joined: 32 columns by 8 runs of slices a block.
template <typename W>
__global__ void __launch_bounds__(256) team_join_kernel(const AffineArgs a, int slices) {
    __shared__ float part[8][33];
    // Columns of 2 * hidden, dw's and then db's: more than 31 bits count at the widest row.
    const int64_t total = 2 * static_cast<int64_t>(a.hidden), c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
    float s = 0.0f;
    if (c < total) {
        const int first = slices * threadIdx.y / 8, last = slices * (threadIdx.y + 1) / 8;
#pragma unroll 10
        for (int i = first; i < last; ++i) s += a.workspace[i * total + c];
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

}  // namespace

namespace {
int staged_smem(int hidden, int bytes, int teams, int depth) {
    return hidden / 4 * 16 + teams * 2 * depth * (hidden * bytes / 16 * 16);
}
}  // namespace

static unsigned join_blocks(int hidden) { return static_cast<unsigned>((2 * static_cast<int64_t>(hidden) + 31) / 32); }

template <typename T>
cudaError_t backward_as(const AffineArgs &a, const WaitLimit &wait, cudaStream_t stream) {
    const bool aligned = row_aligned(a.x) && row_aligned(a.grad) && row_aligned(a.dx);
    const bool whole = aligned && a.hidden * static_cast<int64_t>(sizeof(T)) % 16 == 0;
    const bool ragged =
        !whole && start_alike(a.x, a.grad) && start_alike(a.x, a.dx) && ragged_length(a.hidden, sizeof(T));
    const bool params = a.dweight || a.dbias;
    const bool counted = a.rows < (int64_t{1} << 30);
    TeamPlan plan = team_plan(a.hidden, sizeof(T), counted && (whole || ragged), kBackwardBlock);
    const int depth = plan.pieces > 5 ? 1 : 2;
    if (plan.pieces != 0 && plan.vec > 1 &&
        staged_smem(a.hidden, sizeof(T), kBackwardBlock / plan.threads, depth) > kMaxSmem)
        plan.pieces = 0;
    if (plan.pieces == 0) {
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(a.rows, a.num_sms * 8));
        const int slices = static_cast<int>(std::min<int64_t>(64, backward_slices(a.rows, a.hidden)));
        return with_weight<T>(a, [&](auto w) {
            using W = decltype(w);
            if (a.dx && a.rows > 0) input_gradient_kernel<T, W><<<grid, kThreads, 0, stream>>>(a);
            if (params) {
                parameter_partial_kernel<T>
                    <<<dim3((a.hidden + 31) / 32, slices), dim3(32, 8), 0, stream>>>(a, slices);
                team_join_kernel<W><<<join_blocks(a.hidden), dim3(32, 8), 0, stream>>>(a, slices);
            }
            return cudaGetLastError();
        });
    }
    plan.teams = plan.vec > 1 ? kBackwardBlock / plan.threads : std::min(15, kBackwardBlock / plan.threads);
    const int64_t ctas = std::min<int64_t>((a.rows + plan.teams - 1) / plan.teams, kSlices);
    const int period = ragged ? plan.vec : 1;  // vec 1: of single elements
    const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, ragged_grid(a.rows, ctas, period)));
    const cudaError_t e = with_shape<T, kBackwardBlock, sizeof(T) == 4>(plan, [&](auto vec, auto pieces, auto threads) {
        const dim3 block(plan.threads, plan.teams);
        const int sums = params ? plan.teams * 2 * a.hidden * static_cast<int>(sizeof(float)) : 0;
        if constexpr (vec == 1) {
            auto kernel = team_backward_kernel<T, pieces>;
            static std::atomic<bool> done[64];
                if (cudaError_t f = allow_smem(kernel, done)) return f;
            kernel<<<grid, block, sums, stream>>>(a);
        } else {
            const int smem = std::max(sums, staged_smem(a.hidden, sizeof(T), plan.teams, depth));
            auto launch = [&](auto kernel, std::atomic<bool>(&done)[64]) {
                if (cudaError_t f = allow_smem(kernel, done)) return f;
                kernel<<<grid, block, smem, stream>>>(a, wait);
                return cudaSuccess;
            };
            static std::atomic<bool> done[2][64];
            const cudaError_t f = ragged ? launch(staged_backward_kernel<T, pieces, threads, true>, done[1])
                                         : launch(staged_backward_kernel<T, pieces, threads, false>, done[0]);
            if (f) return f;
        }
        return cudaGetLastError();
    });
    if (e != cudaSuccess || !params) return e;
    return with_weight<T>(a, [&](auto w) {
        team_join_kernel<decltype(w)>
            <<<join_blocks(a.hidden), dim3(32, 8), 0, stream>>>(a, static_cast<int>(grid));
        return cudaGetLastError();
    });
}

}  // namespace norm
}  // namespace ctu

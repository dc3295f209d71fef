// The gradients of layer norm -> ReLU -> dropout (norm_forward.hip).  With h = (x - m) r and g = the gradient of the output
// where the element was kept and the ReLU open, times the dropout's scale:
//
//   dw = sum over rows of g h, db = sum over rows of g
//   dx = r (g w - mean(g w) - h mean(g w h)), means over the row
#include "rows.h"

namespace cgnn {
namespace {

constexpr int64_t kChain = 1024;  // rows at most that a lane adds up one after the other, in float
constexpr int kLongRows = 64;     // rows longer than the registers: rows per part of the parameters' sums, at least
constexpr int kLongParts = 512;   // ... parts, as long as no lane's chain grows too long for that
constexpr int kLanes = 64;        // ... lanes side by side, a pack each
constexpr int kLongGroups = kBlock / kLanes;

int64_t long_rows(int64_t rows) { return std::min(std::max<int64_t>(kLongRows, ceil_div(rows, kLongParts)), kLongGroups * kChain); }

// Workgroups of norm_gradients_kernel, each of which leaves a part of the parameters' sums.  A part is two rows of floats: it is to stand for
// sixteen rows or more (4,096 rows of 4,096 float16 features: 32 us with 256 parts, 35 with 512), if half the chip is not to be idle for that.
// A few rows are one workgroup's, which then needs no second launch for the sums.
constexpr int64_t kPartRows = 16, kFewestParts = 256, kAloneRounds = 4;

int64_t row_parts(int64_t rows, const RowShape &s, size_t element) {
    const int64_t groups = s.threads / s.lanes;
    if (rows <= groups * kAloneRounds) return 1;
    const int64_t most = std::min(row_workgroups(rows, s, element, true), std::max(kFewestParts, rows / kPartRows));
    return std::max(most, ceil_div(rows, groups * kChain));
}

int64_t long_parts(int64_t rows) { return ceil_div(rows, long_rows(rows)); }

int64_t parts_of(int64_t rows, const RowShape &s, size_t element) { return s.lanes ? row_parts(rows, s, element) : long_parts(rows); }

// A sum of column j: to the part's place, or, where there is one part, to the result, of float or of the rows' type.
template <typename T>
__device__ __forceinline__ void leave_sum(compute_t<T> *part, void *whole, bool wide, int64_t j, compute_t<T> sum) {
    if (part) part[j] = sum;
    else if (whole && wide) static_cast<float *>(whole)[j] = (float)sum;
    else if (whole) static_cast<T *>(whole)[j] = (T)sum;
}

// Rows that fit the registers of their lanes, as in the forward pass: x and the gradient are read once for dx and for
// the parameters' sums, which every lane holds for its own columns until its rows are through.  Bound as the forward pass is:
// 2,449,029 rows of 256 float32 features with ReLU and dropout 1,438 us, 5.2 of the 6.0 TB/s that two matrices in and one out reach;
// 325,557 of 257 float16 features 147 us, ALU 75 % busy.
template <typename T, int LANES, int K, int THREADS, bool RELU, bool DROP>
__global__ __launch_bounds__(THREADS) void norm_gradients_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    constexpr int N = 16 / (int)sizeof(T), GROUPS = THREADS / LANES, WAVES = THREADS / kWave;
    constexpr int COLUMNS = LANES * K * N;  // that the lanes have room for
    __shared__ C scratch[LANES > kWave ? WAVES * 4 : WAVES * COLUMNS];
    bool odd = false;
    const int lane = threadIdx.x % LANES, F = (int)a.F;
    const int64_t extent_x = (a.rows - 1) * a.ldx + F, extent_g = (a.rows - 1) * a.ldg + F;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    // the dropout's scale is a factor of all sums and of dx: taken where those are done
    const C inverse_F = (C)a.inverse_F, dropped = DROP ? (C)a.drop.scale : C(1);
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t r = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;

    words_t next_x[K], next_g[K];
    double next_mean = 0, next_rstd = 0;
    auto ask = [&](int64_t row) {
        next_mean = a.stats[2 * row];
        next_rstd = a.stats[2 * row + 1];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int j = (lane + k * LANES) * N, from = j < F ? j : 0;
            next_x[k] = ask_within<T>(a.x, row * a.ldx + from, extent_x);
            next_g[k] = ask_within<T>(a.grad, row * a.ldg + from, extent_g);
        }
    };
    if (r < a.rows) ask(r);
    C w[K][N], b[K][N], dw[K][N], db[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        a.weight.template read<N>((lane + k * LANES) * N, F, C(1), w[k]);
        if constexpr (RELU) a.bias.template read<N>((lane + k * LANES) * N, F, C(0), b[k]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (!RELU) b[k][i] = C(0);
            dw[k][i] = db[k][i] = C(0);
        }
    }
    arrived(next_x);
    arrived(next_g);
    arrived(next_mean);
    arrived(next_rstd);
    arrived(w);
    arrived(b);
    for (; r < a.rows; r += step) {
        C h[K][N], g[K][N];
        Pack<T, N> x[K], d[K];
        const Centre<C> centre(next_mean, next_rstd);
        row_arrived<T, LANES, K>(next_x, a.x, r * a.ldx, extent_x, lane, F, x);
        row_arrived<T, LANES, K>(next_g, a.grad, r * a.ldg, extent_g, lane, F, d);
        ask(r + step < a.rows ? r + step : r);
        C sum = 0, product = 0;
        Draws drawn[K];
        if constexpr (DROP) draw_row<N, LANES>(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks), lane, drawn);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            C v[N];
            normalised<RELU>(x[k], centre, w[k], b[k], h[k], v);
            if constexpr (DROP) d[k] = masked<T, N>(d[k], drawn[k], a.drop.kept);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                g[k][i] = (C)d[k].v[i];
                if constexpr (RELU) g[k][i] = v[i] <= 0 ? C(0) : g[k][i];
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
            if ((lane + k * LANES) * N + N > F)  // behind the row's end lies what the next one holds
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if ((lane + k * LANES) * N + i >= F) h[k][i] = g[k][i] = C(0);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                dw[k][i] = fused(g[k][i], h[k][i], dw[k][i]);
                db[k][i] += g[k][i];
                g[k][i] *= w[k][i];
                sum += g[k][i];
                product = fused(g[k][i], h[k][i], product);
            }
        if (a.dx) {
            row_sums<LANES, THREADS>(sum, product, scratch, odd);
            const C c1 = sum * inverse_F, c2 = product * inverse_F, scale = centre.scale * dropped;
            Pack<T, N> dx[K];
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < N; ++i) g[k][i] = scale * (fused(-h[k][i], c2, g[k][i]) - c1);
                dx[k] = rounded<T, N>(g[k]);
            }
            arrived(next_x);
            arrived(next_g);
            arrived(next_mean);
            arrived(next_rstd);
#pragma unroll
            for (int k = 0; k < K; ++k) store_columns<T, N>(a.dx + r * a.F, (lane + k * LANES) * N, F, dx[k], a.streamed);
        }
    }
    if (a.partial == nullptr && a.dweight == nullptr && a.dbias == nullptr) return;
    // the lane groups of a wave, then its waves in their order
    auto leave = [&](C(&acc)[K][N], C *part, void *whole) {
        if constexpr (LANES > kWave) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int j = (lane + k * LANES) * N + i;
                    if (j < F) leave_sum<T>(part, whole, a.weight.wide, j, acc[k][i] * dropped);
                }
        } else {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const C total = sum_over_groups<LANES>(acc[k][i]);
                    if (threadIdx.x % kWave < LANES) scratch[threadIdx.x / kWave * COLUMNS + (lane + k * LANES) * N + i] = total;
                }
            __syncthreads();
            for (int j = threadIdx.x; j < F; j += THREADS) {
                C total = scratch[j];
#pragma unroll
                for (int wave = 1; wave < WAVES; ++wave) total += scratch[wave * COLUMNS + j];
                leave_sum<T>(part, whole, a.weight.wide, j, total * dropped);
            }
        }
    };
    C *part = a.partial ? a.partial + (int64_t)blockIdx.x * 2 * a.F : nullptr;
    leave(dw, part, a.dweight);
    leave(db, part ? part + a.F : nullptr, a.dbias);
}

// A pack of a row as the gradient sees it: h, and g as described above but for the dropout's scale; zeros behind the row's end.
template <typename T, bool RELU, bool DROP, int N>
__device__ __forceinline__ void taken(const NormArgs<T> &a, const Pack<T, N> &x, Pack<T, N> d, int64_t r, int64_t j, const Centre<compute_t<T>> &centre,
                                      const compute_t<T> (&w)[N], const compute_t<T> (&b)[N], uint64_t offset, compute_t<T> (&h)[N],
                                      compute_t<T> (&g)[N]) {
    using C = compute_t<T>;
    C v[N];
    normalised<RELU>(x, centre, w, b, h, v);
    if constexpr (DROP) {
        Draws drawn = draw(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks + j / kDrawn));
        drawn.from<N>((int)(j % kDrawn));
        d = masked<T, N>(d, drawn, a.drop.kept);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        g[i] = (C)d.v[i];
        if constexpr (RELU) g[i] = v[i] <= 0 ? C(0) : g[i];
        if (j + i >= a.F) h[i] = g[i] = C(0);
    }
}

// dx of longer rows: a workgroup per row, which reads it twice.  A pack's terms are added up in float and the packs in 64 bits: a lane's chain
// grows with the row (20,000,003 features, a gradient of 0.1 everywhere, of which its mean leaves nothing: 1.7e-5 was left in float).
template <typename T, bool RELU, bool DROP>
__global__ __launch_bounds__(kLongThreads) void norm_long_dx_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    constexpr int N = 16 / (int)sizeof(T), PACKS = sizeof(T) == 2 ? 1 : 2;  // as many as the registers hold
    constexpr int64_t kStride = (int64_t)kLongThreads * N;
    __shared__ double scratch[kLongThreads / kWave * 4];
    bool odd = false;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const int64_t extent_x = (a.rows - 1) * a.ldx + a.F, extent_g = (a.rows - 1) * a.ldg + a.F;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const Centre<C> centre(a.stats[2 * r], a.stats[2 * r + 1]);
        double sum = 0, product = 0;
        C w[PACKS][N], b[PACKS][N], h[N], g[N];
        words_t asked_x[PACKS], asked_g[PACKS];
        auto ask = [&](int64_t j0) {
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                const int64_t j = std::min(j0 + k * kStride, a.F - 1);
                asked_x[k] = ask_within<T>(a.x, r * a.ldx + j, extent_x);
                asked_g[k] = ask_within<T>(a.grad, r * a.ldg + j, extent_g);
            }
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                a.weight.template read<N>(j0 + k * kStride, a.F, C(1), w[k]);
                if constexpr (RELU) a.bias.template read<N>(j0 + k * kStride, a.F, C(0), b[k]);
                if constexpr (!RELU)
#pragma unroll
                    for (int i = 0; i < N; ++i) b[k][i] = C(0);
            }
        };
        auto take = [&](int64_t j0, int k) {
            const int64_t j = std::min(j0 + k * kStride, a.F - 1);
            taken<T, RELU, DROP, N>(a, settled<T>(asked_x[k], a.x, r * a.ldx + j, extent_x), settled<T>(asked_g[k], a.grad, r * a.ldg + j, extent_g), r,
                                    j0 + k * kStride, centre, w[k], b[k], offset, h, g);
        };
        for (int64_t j0 = (int64_t)threadIdx.x * N; j0 < a.F; j0 += PACKS * kStride) {
            ask(j0);
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                take(j0, k);
                C pack_sum = 0, pack_product = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const C gw = g[i] * w[k][i];
                    pack_sum += gw;
                    pack_product = fused(gw, h[i], pack_product);
                }
                sum += (double)pack_sum;
                product += (double)pack_product;
            }
        }
        row_sums<kLongThreads, kLongThreads>(sum, product, scratch, odd);
        const C c1 = (C)(sum * a.inverse_F), c2 = (C)(product * a.inverse_F), scale = centre.scale * (DROP ? (C)a.drop.scale : C(1));
        for (int64_t j0 = (int64_t)threadIdx.x * N; j0 < a.F; j0 += PACKS * kStride) {
            ask(j0);
#pragma unroll
            for (int k = 0; k < PACKS; ++k) {
                take(j0, k);
                C dx[N];
#pragma unroll
                for (int i = 0; i < N; ++i) dx[i] = scale * (fused(-h[i], c2, g[i] * w[k][i]) - c1);
                store_columns<T, N>(a.dx + r * a.F, j0 + k * kStride, a.F, rounded<T, N>(dx), false);
            }
        }
    }
}

// Their dw and db: blockIdx.y names the part, `part` rows each, blockIdx.x the columns.  A lane keeps its columns and goes down the rows.
template <typename T, bool RELU, bool DROP>
__global__ __launch_bounds__(kBlock) void norm_long_parts_kernel(NormArgs<T> a, int64_t part) {
    using C = compute_t<T>;
    constexpr int N = 16 / (int)sizeof(T), GROUPS = kLongGroups;
    __shared__ C sums[GROUPS][2][N][kLanes];
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const int64_t extent_x = (a.rows - 1) * a.ldx + a.F, extent_g = (a.rows - 1) * a.ldg + a.F;
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const int64_t j = ((int64_t)blockIdx.x * kLanes + lane) * N, from = std::min(j, a.F - 1);
    const int64_t last = std::min(a.rows, (int64_t)(blockIdx.y + 1) * part);
    int64_t r = (int64_t)blockIdx.y * part + group;
    words_t next_x[1] = {}, next_g[1] = {};
    double next_mean = 0, next_rstd = 0;
    auto ask = [&](int64_t row) {
        next_mean = a.stats[2 * row];
        next_rstd = a.stats[2 * row + 1];
        next_x[0] = ask_within<T>(a.x, row * a.ldx + from, extent_x);
        next_g[0] = ask_within<T>(a.grad, row * a.ldg + from, extent_g);
    };
    if (r < last) ask(r);
    C w[N], b[N] = {}, dw[N] = {}, db[N] = {};
    a.weight.template read<N>(j, a.F, C(1), w);
    if constexpr (RELU) a.bias.template read<N>(j, a.F, C(0), b);
    for (; r < last; r += GROUPS) {
        const Centre<C> centre(next_mean, next_rstd);
        const auto x = settled<T>(next_x[0], a.x, r * a.ldx + from, extent_x);
        const auto d = settled<T>(next_g[0], a.grad, r * a.ldg + from, extent_g);
        ask(r + GROUPS < last ? r + GROUPS : r);
        C h[N], g[N];
        taken<T, RELU, DROP, N>(a, x, d, r, j, centre, w, b, offset, h, g);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            dw[i] = fused(g[i], h[i], dw[i]);
            db[i] += g[i];
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        sums[group][0][i][lane] = dw[i];
        sums[group][1][i][lane] = db[i];
    }
    __syncthreads();
    if (group == 0)
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (j + i < a.F) {
                const C dropped = DROP ? (C)a.drop.scale : C(1);
                C weight = 0, bias = 0;
#pragma unroll
                for (int k = 0; k < GROUPS; ++k) {
                    weight += sums[k][0][i][lane];
                    bias += sums[k][1][i][lane];
                }
                C *to = a.partial ? a.partial + (int64_t)blockIdx.y * 2 * a.F : nullptr;
                leave_sum<T>(to, a.dweight, a.weight.wide, j + i, weight * dropped);
                leave_sum<T>(to ? to + a.F : nullptr, a.dbias, a.weight.wide, j + i, bias * dropped);
            }
}

// Matrices of less than 16 bytes: a lane a row for dx, then a lane a column for the sums.
template <typename T, bool RELU, bool DROP>
__global__ __launch_bounds__(kWave) void norm_few_gradients_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    auto one = [&](int64_t r, int64_t j, C &h, C &g, C &weight) {
        C w[1], b[1] = {}, hh[1], v[1];
        a.weight.template read<1>(j, a.F, C(1), w);
        if constexpr (RELU) a.bias.template read<1>(j, a.F, C(0), b);
        const Pack<T, 1> x = {{a.x[r * a.ldx + j]}};
        normalised<RELU>(x, Centre<C>(a.stats[2 * r], a.stats[2 * r + 1]), w, b, hh, v);
        h = hh[0];
        weight = w[0];
        g = (C)a.grad[r * a.ldg + j];
        if constexpr (DROP) g = draw(a.drop.seed, offset, (uint64_t)r).keeps((int)j, a.drop.kept) ? g * (C)a.drop.scale : C(0);
        if constexpr (RELU) g = v[0] <= 0 ? C(0) : g;
    };
    C h, g, w;
    const int64_t lane = threadIdx.x;
    if (a.dx && lane < a.rows) {
        C sum = 0, product = 0;
        for (int64_t j = 0; j < a.F; ++j) {
            one(lane, j, h, g, w);
            sum += g * w;
            product = fused(g * w, h, product);
        }
        const C c1 = sum * (C)a.inverse_F, c2 = product * (C)a.inverse_F, scale = (C)a.stats[2 * lane + 1];
        for (int64_t j = 0; j < a.F; ++j) {
            one(lane, j, h, g, w);
            a.dx[lane * a.F + j] = (T)(scale * (fused(-h, c2, g * w) - c1));
        }
    }
    if (lane < a.F) {
        C dw = 0, db = 0;
        for (int64_t r = 0; r < a.rows; ++r) {
            one(r, lane, h, g, w);
            dw = fused(g, h, dw);
            db += g;
        }
        leave_sum<T>((C *)nullptr, a.dweight, a.weight.wide, lane, dw);
        leave_sum<T>((C *)nullptr, a.dbias, a.weight.wide, lane, db);
    }
}

// The parts' sums, added up in 64 bits in an order that the number of parts fixes: column c < F of the weight's gradient, then
// the bias's.  Sixteen columns a workgroup: as many lines of 64 bytes in flight as it has lane groups (256 to 768 parts of up to
// 602 columns: 4 to 7 us; with a quarter of the threads and a load at a time 20 to 32).  Of rows of more than half a million columns a workgroup takes
// several sixteens: a launch has fewer than 2^32 threads a dimension.
constexpr int kSumColumns = 16, kSumThreads = 1024, kSumUnroll = 4, kSumWorkgroups = 1 << 16;

template <typename C, typename P>
__global__ __launch_bounds__(kSumThreads) void norm_sum_parts_kernel(const C *partial, int64_t parts, int64_t F, P *dweight, P *dbias) {
    constexpr int GROUPS = kSumThreads / kSumColumns;
    __shared__ double sums[GROUPS][kSumColumns];
    const int lane = threadIdx.x % kSumColumns, group = threadIdx.x / kSumColumns;
    for (int64_t first = (int64_t)blockIdx.x * kSumColumns; first < 2 * F; first += (int64_t)gridDim.x * kSumColumns) {
        const int64_t c = first + lane;
        double sum = 0;
        if (c < 2 * F)
            for (int64_t k = group; k < parts; k += GROUPS * kSumUnroll) {
                C part[kSumUnroll];
#pragma unroll
                for (int u = 0; u < kSumUnroll; ++u) part[u] = k + u * GROUPS < parts ? partial[(k + u * GROUPS) * 2 * F + c] : C(0);
#pragma unroll
                for (int u = 0; u < kSumUnroll; ++u) sum += (double)part[u];
            }
        sums[group][lane] = sum;
#pragma unroll
        for (int half = GROUPS / 2; half > 0; half /= 2) {
            __syncthreads();
            if (group < half) sums[group][lane] += sums[group + half][lane];
        }
        P *to = c < F ? dweight : dbias;
        if (group == 0 && c < 2 * F && to) to[c < F ? c : c - F] = (P)(compute_t<P>)sums[0][lane];
        __syncthreads();  // the places are written again
    }
}

template <typename T, bool RELU, bool DROP>
int gradients_launch(const NormArgs<T> &a, const RowShape &shape, int64_t parts, hipStream_t stream) {
    if (a.rows * a.F * (int64_t)sizeof(T) < 16) {
        hipLaunchKernelGGL((norm_few_gradients_kernel<T, RELU, DROP>), dim3(1), dim3(kWave), 0, stream, a);
        return check_launch("layer_norm_backward");
    }
    if (shape.lanes)
        return with_row_shape<T, true>(shape, [&](auto tag) {
            using S = decltype(tag);
            hipLaunchKernelGGL((norm_gradients_kernel<T, S::lanes, S::packs, S::threads, RELU, DROP>), dim3((unsigned)parts), dim3(S::threads),
                               0, stream, a);
            return check_launch("layer_norm_backward");
        });
    if (a.dx) {
        hipLaunchKernelGGL((norm_long_dx_kernel<T, RELU, DROP>), dim3((unsigned)std::min<int64_t>(a.rows, 1024)), dim3(kLongThreads), 0, stream, a);
        if (int rc = check_launch("layer_norm_backward")) return rc;
    }
    if (a.partial || a.dweight || a.dbias) {
        const dim3 grid((unsigned)ceil_div(a.F, (int64_t)kLanes * 16 / (int64_t)sizeof(T)), (unsigned)parts);
        hipLaunchKernelGGL((norm_long_parts_kernel<T, RELU, DROP>), grid, dim3(kBlock), 0, stream, a, ceil_div(a.rows, parts));
    }
    return check_launch("layer_norm_backward");
}

template <typename T>
int norm_backward_typed(NormArgs<T> a, bool drops, void *dweight, void *dbias, hipStream_t stream) {
    using C = compute_t<T>;
    const RowShape shape = row_shape(a.rows, a.F, sizeof(T), true);
    const int64_t parts = parts_of(a.rows, shape, sizeof(T));
    if (shape.lanes) a.streamed = streams(a.rows, a.F * (int64_t)sizeof(T), shape.lanes * 16, 3);
    const bool sums = dweight != nullptr || dbias != nullptr, alone = parts == 1;
    if (!sums || alone) a.partial = nullptr;
    if (alone) {
        a.dweight = dweight;
        a.dbias = dbias;
    }
    const int rc = drops ? (a.relu ? gradients_launch<T, true, true>(a, shape, parts, stream) : gradients_launch<T, false, true>(a, shape, parts, stream))
                         : (a.relu ? gradients_launch<T, true, false>(a, shape, parts, stream) : gradients_launch<T, false, false>(a, shape, parts, stream));
    if (rc != CGNN_OK || !sums || alone) return rc;
    const dim3 columns((unsigned)std::min<int64_t>(ceil_div(2 * a.F, kSumColumns), kSumWorkgroups));
    auto add = [&](auto tag) {
        using P = typename decltype(tag)::type;
        hipLaunchKernelGGL((norm_sum_parts_kernel<C, P>), columns, dim3(kSumThreads), 0, stream, a.partial, parts, a.F, static_cast<P *>(dweight),
                           static_cast<P *>(dbias));
        return check_launch("layer_norm_backward");
    };
    if constexpr (sizeof(T) == 2)
        if (a.weight.wide) return add(TypeTag<float>());
    return add(TypeTag<T>());
}

}  // namespace
}  // namespace cgnn

using namespace cgnn;

extern "C" size_t cgnn_layer_norm_backward_workspace_bytes(int64_t rows, int64_t F, int dtype) {
    if (rows <= 0 || F <= 0) return 0;
    const RowShape shape = row_shape(rows, F, row_type_bytes(dtype), true);
    const int64_t parts = parts_of(rows, shape, row_type_bytes(dtype));
    return parts == 1 ? 0 : (size_t)parts * 2 * (size_t)F * (dtype == CGNN_F64 ? 8 : 4);
}

extern "C" int cgnn_layer_norm_backward(int64_t rows, int64_t F, int dtype, int param_dtype, const void *grad, int64_t ldg,
                                        const void *x, int64_t ldx, const double *stats, const void *weight, const void *bias,
                                        int relu, const cgnn_drop *drop, void *dx, void *dweight, void *dbias, void *workspace,
                                        size_t workspace_bytes, cgnn_stream_t stream) {
    CGNN_REQUIRE(rows > 0 && F > 0 && (rows <= 1 || (ldx >= F && ldg >= F)), "cgnn_layer_norm_backward: bad size");
    CGNN_REQUIRE(F < ((int64_t)1 << 31) - 65536, "cgnn_layer_norm_backward: a row must be shorter than 2^31 elements");
    CGNN_REQUIRE(param_dtype == dtype || (param_dtype == CGNN_F32 && dtype != CGNN_F64),
                 "cgnn_layer_norm_backward: parameters have the type of the rows, or f32 for 16-bit rows");
    if (drop) CGNN_REQUIRE_DROP("cgnn_layer_norm_backward", drop);
    return with_row_type(dtype, "cgnn_layer_norm_backward: dtype must be f32, f64, f16 or bf16", [&](auto tag) {
        using T = typename decltype(tag)::type;
        if (dx == nullptr && dweight == nullptr && dbias == nullptr) return (int)CGNN_OK;
        CGNN_REQUIRE(grad && x && stats, "cgnn_layer_norm_backward: null array");
        if ((dweight || dbias) &&
            (workspace_bytes < cgnn_layer_norm_backward_workspace_bytes(rows, F, dtype) || (workspace == nullptr && workspace_bytes)))
            return fail(CGNN_EWORKSPACE, "cgnn_layer_norm_backward: workspace too small");
        NormArgs<T> a{};
        a.x = static_cast<const T *>(x);
        a.ldx = ldx;
        a.grad = static_cast<const T *>(grad);
        a.ldg = ldg;
        a.stats = const_cast<double *>(stats);
        a.weight = {weight, param_dtype != dtype};
        a.bias = {bias, param_dtype != dtype};
        a.relu = relu;
        a.drop = drop_of(drop, F);
        a.dx = static_cast<T *>(dx);
        a.partial = static_cast<compute_t<T> *>(workspace);
        a.rows = rows;
        a.F = F;
        a.inverse_F = 1.0 / (double)F;
        return norm_backward_typed<T>(a, a.drop.kept < kAllKept, dweight, dbias, stream);
    });
}

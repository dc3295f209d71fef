// Layer norm of node rows, with the ReLU and the dropout behind it in the same pass:
//
//   m = sum x / F, v = sum (x - m)^2 / F, r = 1 / sqrt(v + eps), out = drop(relu((x - m) r w + b))
#include <limits>

#include "rows.h"

namespace cgnn {
namespace {

// Rows that fit the registers of their lanes: LANES of them hold K packs of 16 bytes each, so a row is read once and
// written once.  The packs of the next row are asked for before this one's are used.  Bound by memory for whole packs of
// four-byte elements (2,449,029 rows of 256 float32 features with ReLU and dropout: 905 us, 5.5 TB/s of the 6.2 that a copy
// reaches), by the vector ALU for 16-bit rows of odd widths (325,557 of 257 float16 features, the same: 125 us, 2.7 TB/s, ALU
// 72 % busy: conversions, sums in 64 bits and the generator cost an element of two bytes what they cost one of four).
template <typename T, int LANES, int K, int THREADS, bool RELU, bool DROP>
__global__ __launch_bounds__(THREADS) void norm_rows_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    constexpr int N = 16 / (int)sizeof(T);
    __shared__ double scratch[LANES > kWave ? THREADS / kWave * 4 : 1];
    bool odd = false;
    const int lane = threadIdx.x % LANES, F = (int)a.F;
    const int64_t step = a.walk.step, extent = (a.rows - 1) * a.ldx + F;
    const int64_t end = std::min(a.rows, (int64_t)blockIdx.x * a.walk.first + step * a.walk.rounds);
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    int64_t r = (int64_t)blockIdx.x * a.walk.first + threadIdx.x / LANES;

    words_t next[K];
    T next_first = T(0);
    auto ask = [&](int64_t row) {
        const int64_t at = row * a.ldx;
        next_first = a.x[at];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int j = (lane + k * LANES) * N;
            next[k] = ask_within<T>(a.x, at + (j < F ? j : 0), extent);
        }
    };
    if (r < end) ask(r);
    C w[K][N], b[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        a.weight.template read<N>((lane + k * LANES) * N, F, C(1), w[k]);
        a.bias.template read<N>((lane + k * LANES) * N, F, C(0), b[k]);
    }
    arrived(next);
    arrived(next_first);
    arrived(w);
    arrived(b);
    for (; r < end; r += step) {
        Pack<T, N> x[K];
        const T first = next_first;
        row_arrived<T, LANES, K>(next, a.x, r * a.ldx, extent, lane, F, x);
        ask(r + step < end ? r + step : r);
        auto about = [&](T pivot) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if ((lane + k * LANES) * N + N > F)  // what lies behind the row's end adds nothing to its sums
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if ((lane + k * LANES) * N + i >= F) x[k].v[i] = pivot;
            double sum = 0, squares = 0;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const double d = (double)x[k].v[i] - (double)pivot;
                    sum += d;
                    squares = __builtin_fma(d, d, squares);
                }
            row_sums<LANES, THREADS>(sum, squares, scratch, odd);
            return moments((double)pivot, sum, squares, a.inverse_F);
        };
        Moments m = about(first);
        if constexpr (sizeof(T) == 8) m = about(m.mean);
        const Centre<C> centre(m.mean, reciprocal_root(m.variance + a.eps));
        Pack<T, N> y[K];
        Draws drawn[K];
        if constexpr (DROP) draw_row<N, LANES>(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks), lane, drawn);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            C h[N], v[N];
            normalised<RELU>(x[k], centre, w[k], b[k], h, v);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (RELU) v[i] = rectified(v[i]);
                if constexpr (DROP) v[i] *= (C)a.drop.scale;
            }
            y[k] = rounded<T, N>(v);
            if constexpr (DROP) y[k] = masked<T, N>(y[k], drawn[k], a.drop.kept);
        }
        arrived(next);
        arrived(next_first);
        if (a.stats && lane == 0) {
            a.stats[2 * r] = centre.mean;
            a.stats[2 * r + 1] = centre.rstd;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) store_columns<T, N>(a.out + r * a.F, (lane + k * LANES) * N, F, y[k], a.streamed);
    }
}

// Longer rows: a workgroup a row, which reads it twice (float64: three times), kLongPacks packs a lane at a time.  Bound by the latency of the
// readings, one workgroup a compute unit (3,000 rows of 20,000 float32 features: 206 us, 2.3 TB/s; a pack at a time 299; float64 278 us, 3.5 TB/s).
template <typename T, bool RELU, bool DROP>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    constexpr int N = 16 / (int)sizeof(T);
    constexpr int64_t kStride = (int64_t)kLongThreads * N;
    __shared__ double scratch[kLongThreads / kWave * 4];
    bool odd = false;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const int64_t extent = (a.rows - 1) * a.ldx + a.F;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int64_t at = r * a.ldx;
        words_t asked[kLongPacks];
        auto ask = [&](int64_t j0) {
#pragma unroll
            for (int k = 0; k < kLongPacks; ++k) asked[k] = ask_within<T>(a.x, at + std::min(j0 + k * kStride, a.F - 1), extent);
        };
        auto about = [&](T pivot) {
            double sum = 0, squares = 0;
            for (int64_t j0 = (int64_t)threadIdx.x * N; j0 < a.F; j0 += kLongPacks * kStride) {
                ask(j0);
#pragma unroll
                for (int k = 0; k < kLongPacks; ++k) {
                    const int64_t j = j0 + k * kStride;
                    const auto x = settled<T>(asked[k], a.x, at + std::min(j, a.F - 1), extent);
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const double d = j + i < a.F ? (double)x.v[i] - (double)pivot : 0.0;
                        sum += d;
                        squares = __builtin_fma(d, d, squares);
                    }
                }
            }
            row_sums<kLongThreads, kLongThreads>(sum, squares, scratch, odd);
            return moments((double)pivot, sum, squares, a.inverse_F);
        };
        Moments m = about(a.x[at]);
        if constexpr (sizeof(T) == 8) m = about(m.mean);
        const Centre<C> centre(m.mean, reciprocal_root(m.variance + a.eps));
        if (a.stats && threadIdx.x == 0) {
            a.stats[2 * r] = centre.mean;
            a.stats[2 * r + 1] = centre.rstd;
        }
        for (int64_t j0 = (int64_t)threadIdx.x * N; j0 < a.F; j0 += kLongPacks * kStride) {
            C w[kLongPacks][N], b[kLongPacks][N];
            ask(j0);
#pragma unroll
            for (int k = 0; k < kLongPacks; ++k) {
                a.weight.template read<N>(j0 + k * kStride, a.F, C(1), w[k]);
                a.bias.template read<N>(j0 + k * kStride, a.F, C(0), b[k]);
            }
#pragma unroll
            for (int k = 0; k < kLongPacks; ++k) {
                const int64_t j = j0 + k * kStride;
                const auto x = settled<T>(asked[k], a.x, at + std::min(j, a.F - 1), extent);
                C h[N], v[N];
                normalised<RELU>(x, centre, w[k], b[k], h, v);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if constexpr (RELU) v[i] = rectified(v[i]);
                    if constexpr (DROP) v[i] *= (C)a.drop.scale;
                }
                auto y = rounded<T, N>(v);
                if constexpr (DROP) {
                    Draws drawn = draw(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks + j / kDrawn));
                    drawn.from<N>((int)(j % kDrawn));
                    y = masked<T, N>(y, drawn, a.drop.kept);
                }
                store_columns<T, N>(a.out + r * a.F, j, a.F, y, false);
            }
        }
    }
}

// Matrices of less than 16 bytes: a lane a row.
template <typename T, bool RELU, bool DROP>
__global__ __launch_bounds__(kWave) void norm_few_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    const int64_t r = threadIdx.x;
    if (r >= a.rows) return;
    const T *x = a.x + r * a.ldx;
    auto about = [&](T pivot) {
        double sum = 0, squares = 0;
        for (int64_t j = 0; j < a.F; ++j) {
            const double d = (double)x[j] - (double)pivot;
            sum += d;
            squares = __builtin_fma(d, d, squares);
        }
        return moments((double)pivot, sum, squares, a.inverse_F);
    };
    Moments m = about(x[0]);
    if constexpr (sizeof(T) == 8) m = about(m.mean);
    const Centre<C> centre(m.mean, reciprocal_root(m.variance + a.eps));
    if (a.stats) {
        a.stats[2 * r] = centre.mean;
        a.stats[2 * r + 1] = centre.rstd;
    }
    const Draws drawn = DROP ? draw(a.drop.seed, drop_offset(a.drop), (uint64_t)r) : Draws{};  // F < 8: one call a row
    for (int64_t j = 0; j < a.F; ++j) {
        const Pack<T, 1> one = {{x[j]}};
        C w[1], b[1], h[1], v[1];
        a.weight.template read<1>(j, a.F, C(1), w);
        a.bias.template read<1>(j, a.F, C(0), b);
        normalised<RELU>(one, centre, w, b, h, v);
        if constexpr (RELU) v[0] = rectified(v[0]);
        if constexpr (DROP) v[0] = drawn.keeps((int)j, a.drop.kept) ? v[0] * (C)a.drop.scale : C(0);
        a.out[r * a.F + j] = (T)v[0];
    }
}

constexpr int64_t kLargeRounds = 8;

template <typename T, bool RELU, bool DROP>
int norm_launch(NormArgs<T> a, hipStream_t stream) {
    const RowShape shape = row_shape(a.rows, a.F, sizeof(T), false, a.weight.wide);
    if (a.rows * a.F * (int64_t)sizeof(T) < 16) {
        hipLaunchKernelGGL((norm_few_kernel<T, RELU, DROP>), dim3(1), dim3(kWave), 0, stream, a);
        return check_launch("layer_norm");
    }
    if (shape.lanes == 0) {
        hipLaunchKernelGGL((norm_long_kernel<T, RELU, DROP>), dim3((unsigned)std::min<int64_t>(a.rows, 1024)), dim3(kLongThreads), 0, stream, a);
        return check_launch("layer_norm");
    }
    // Over and over the chip's width, or, from a gigabyte on, a few rounds of neighbouring rows for each of more workgroups, so that none gets
    // far ahead of the others (2,449,029 rows of 256 features with ReLU and dropout, float32: 909 us, 1,026 the other way, bfloat16:
    // 492 and 548; 300,000 of 602, bfloat16: 171 and 150).  Below the limit (float32, no ReLU, no dropout) the width tells more than the bytes: 100, 128
    // and 256 features cross at 0.7 GB (0.5 GB: 2 % lost, 0.95 GB: 1 to 2 % gained), 47 lose 9 % from 0.5 to 0.95 GB, 300 and 602 gain 9 to 15 % there.
    const int64_t bytes = a.rows * a.F * (int64_t)sizeof(T), groups = shape.threads / shape.lanes, tiles = ceil_div(a.rows, groups);
    int64_t workgroups = row_workgroups(a.rows, shape, sizeof(T), false);
    a.walk = {groups, groups * workgroups, ceil_div(tiles, workgroups)};
    if (bytes >= (int64_t)1 << 30) {
        // more rounds where a launch, which has fewer than 2^32 threads a dimension, would not hold the workgroups
        const int64_t rounds = std::max(kLargeRounds, ceil_div(tiles, ((int64_t)1 << 31) / shape.threads));
        a.walk = {groups * rounds, groups, rounds};
        workgroups = ceil_div(tiles, rounds);
    }
    a.streamed = streams(a.rows, a.F * (int64_t)sizeof(T), shape.lanes * 16, 2);
    return with_row_shape<T, false>(shape, [&](auto tag) {
        using S = decltype(tag);
        const dim3 grid((unsigned)workgroups);
        hipLaunchKernelGGL((norm_rows_kernel<T, S::lanes, S::packs, S::threads, RELU, DROP>), grid, dim3(S::threads), 0, stream, a);
        return check_launch("layer_norm");
    });
}

}  // namespace
}  // namespace cgnn

using namespace cgnn;

extern "C" int cgnn_layer_norm(int64_t rows, int64_t F, int dtype, int param_dtype, const void *x, int64_t ldx,
                               const void *weight, const void *bias, double eps, int relu, const cgnn_drop *drop, void *out,
                               double *stats, cgnn_stream_t stream) {
    CGNN_REQUIRE(rows >= 0 && F >= 0 && (rows <= 1 || ldx >= F), "cgnn_layer_norm: bad size");
    CGNN_REQUIRE(F < ((int64_t)1 << 31) - 65536, "cgnn_layer_norm: a row must be shorter than 2^31 elements");
    CGNN_REQUIRE(eps >= 0 && eps <= std::numeric_limits<double>::max(), "cgnn_layer_norm: eps must be finite and not negative");
    CGNN_REQUIRE(param_dtype == dtype || (param_dtype == CGNN_F32 && dtype != CGNN_F64),
                 "cgnn_layer_norm: parameters have the type of the rows, or f32 for 16-bit rows");
    if (drop) CGNN_REQUIRE_DROP("cgnn_layer_norm", drop);
    return with_row_type(dtype, "cgnn_layer_norm: dtype must be f32, f64, f16 or bf16", [&](auto tag) {
        using T = typename decltype(tag)::type;
        if (rows == 0 || F == 0) return (int)CGNN_OK;
        CGNN_REQUIRE(x && out, "cgnn_layer_norm: null array");
        NormArgs<T> a{};
        a.x = static_cast<const T *>(x);
        a.ldx = ldx;
        a.weight = {weight, param_dtype != dtype};
        a.bias = {bias, param_dtype != dtype};
        a.eps = eps;
        a.drop = drop_of(drop, F);
        a.out = static_cast<T *>(out);
        a.stats = stats;
        a.rows = rows;
        a.F = F;
        a.inverse_F = 1.0 / (double)F;
        if (a.drop.kept < kAllKept) return relu ? norm_launch<T, true, true>(a, stream) : norm_launch<T, false, true>(a, stream);
        return relu ? norm_launch<T, true, false>(a, stream) : norm_launch<T, false, false>(a, stream);
    });
}

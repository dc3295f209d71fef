// Layer norm of node rows, with the ReLU and the dropout behind it in the same pass:
//
//   m = sum x / F, v = sum (x - m)^2 / F, r = 1 / sqrt(v + eps), out = drop(relu((x - m) r w + b))
#include "rows.h"

namespace cgnn {
namespace {

// Rows that fit the registers of their lanes: LANES of them hold K packs of 16 bytes each, so a row is read once and
// written once.  The packs of the next row are asked for before this one's are used.
template <typename T, int LANES, int K, int THREADS, bool DROP>
__global__ __launch_bounds__(THREADS) void norm_rows_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    constexpr int N = 16 / (int)sizeof(T), GROUPS = THREADS / LANES;
    __shared__ double scratch[LANES > kWave ? THREADS / kWave * 2 : 1];
    const int lane = threadIdx.x % LANES, F = (int)a.F;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const double inverse_F = 1.0 / (double)F;
    int64_t r = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;

    Pack<T, N> next[K];
    T next_first = T(0);
    auto ask = [&](int64_t row) {
        const T *x = a.x + row * a.ldx;
        next_first = x[0];
#pragma unroll
        for (int k = 0; k < K; ++k) next[k] = load_pack<T, N>(x, (lane + k * LANES) * N, F);
    };
    if (r < a.rows) ask(r);
    C w[K][N], b[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (lane + k * LANES) * N + i;
            w[k][i] = j < F ? a.weight.at(j, C(1)) : C(0);
            b[k][i] = j < F ? a.bias.at(j, C(0)) : C(0);
        }
    for (; r < a.rows; r += step) {
        Pack<T, N> x[K];
        const double pivot = (double)next_first;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            x[k] = next[k];
            const int j = (lane + k * LANES) * N;
            if (j + N > F)  // what lies behind the row's end adds nothing to its sums
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (j + i >= F) x[k].v[i] = next_first;
        }
        if (r + step < a.rows) ask(r + step);
        double sum = 0, squares = 0;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const double d = (double)x[k].v[i] - pivot;
                sum += d;
                squares = __builtin_fma(d, d, squares);
            }
        row_sums<LANES, THREADS>(sum, squares, scratch);
        const Moments m = moments(pivot, sum, squares, inverse_F);
        const double rstd = reciprocal_root(m.variance + a.eps);
        if (a.stats && lane == 0) {
            a.stats[2 * r] = m.mean;
            a.stats[2 * r + 1] = rstd;
        }
        T *out = a.out + r * a.F;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int j = (lane + k * LANES) * N;
            Pack<T, N> y;
            C h[N], v[N];
            normalised<N>(x[k].v, m.mean, rstd, w[k], b[k], a.relu, h, v);
            Draws drawn;
            if constexpr (DROP) {
                drawn = draw(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks + j / kDrawn));
                drawn.from<N>(j);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                C c = a.relu && v[i] <= 0 ? C(0) : v[i];
                if constexpr (DROP) c = drawn.keeps(i, a.drop.kept) ? c * (C)a.drop.scale : C(0);
                y.v[i] = (T)c;
            }
            if (j < F) store_pack<T, N>(out, j, F, y);
        }
    }
}

// Longer rows: a workgroup a row, which reads it twice.
constexpr int kLongThreads = 1024;

template <typename T, bool DROP>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    __shared__ double scratch[kLongThreads / kWave * 2];
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = a.x + r * a.ldx;
        T *out = a.out + r * a.F;
        const double pivot = (double)x[0];
        double sum = 0, squares = 0;
        for (int64_t j = (int64_t)threadIdx.x * kDrawn; j < a.F; j += (int64_t)kLongThreads * kDrawn) {
            const auto p = load_pack<T, kDrawn>(x, j, a.F);
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                const double d = j + i < a.F ? (double)p.v[i] - pivot : 0.0;
                sum += d;
                squares = __builtin_fma(d, d, squares);
            }
        }
        row_sums<kLongThreads, kLongThreads>(sum, squares, scratch);
        const Moments m = moments(pivot, sum, squares, 1.0 / (double)a.F);
        const double rstd = reciprocal_root(m.variance + a.eps);
        if (a.stats && threadIdx.x == 0) {
            a.stats[2 * r] = m.mean;
            a.stats[2 * r + 1] = rstd;
        }
        for (int64_t j = (int64_t)threadIdx.x * kDrawn; j < a.F; j += (int64_t)kLongThreads * kDrawn) {
            const auto p = load_pack<T, kDrawn>(x, j, a.F);
            Pack<T, kDrawn> y;
            C w[kDrawn], b[kDrawn], h[kDrawn], v[kDrawn];
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                w[i] = j + i < a.F ? a.weight.at(j + i, C(1)) : C(0);
                b[i] = j + i < a.F ? a.bias.at(j + i, C(0)) : C(0);
            }
            normalised<kDrawn>(p.v, m.mean, rstd, w, b, a.relu, h, v);
            Draws drawn;
            if constexpr (DROP) drawn = draw(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks + j / kDrawn));
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                C c = a.relu && v[i] <= 0 ? C(0) : v[i];
                if constexpr (DROP) c = drawn.keeps(i, a.drop.kept) ? c * (C)a.drop.scale : C(0);
                y.v[i] = (T)c;
            }
            store_pack<T, kDrawn>(out, j, a.F, y);
        }
    }
}

template <typename T>
int norm_typed(const NormArgs<T> &a, bool drops, hipStream_t stream) {
    const RowShape shape = row_shape(a.F, sizeof(T), kMostPacks);
    if (shape.lanes == 0) {
        const dim3 grid((unsigned)std::min<int64_t>(a.rows, 1024));
        if (drops)
            hipLaunchKernelGGL((norm_long_kernel<T, true>), grid, dim3(kLongThreads), 0, stream, a);
        else
            hipLaunchKernelGGL((norm_long_kernel<T, false>), grid, dim3(kLongThreads), 0, stream, a);
        return check_launch("layer_norm");
    }
    return with_row_shape(shape, [&](auto tag) {
        using S = decltype(tag);
        const dim3 grid((unsigned)std::min<int64_t>(ceil_div(a.rows, S::threads / S::lanes), 256 * 2048 / S::threads));
        if (drops)
            hipLaunchKernelGGL((norm_rows_kernel<T, S::lanes, S::packs, S::threads, true>), grid, dim3(S::threads), 0, stream, a);
        else
            hipLaunchKernelGGL((norm_rows_kernel<T, S::lanes, S::packs, S::threads, false>), grid, dim3(S::threads), 0, stream, a);
        return check_launch("layer_norm");
    });
}

}  // namespace
}  // namespace cgnn

using namespace cgnn;

extern "C" int cgnn_layer_norm(int64_t rows, int64_t F, int dtype, int param_dtype, const void *x, int64_t ldx,
                               const void *weight, const void *bias, double eps, int relu, const cgnn_drop *drop, void *out,
                               double *stats, cgnn_stream_t stream) {
    CGNN_REQUIRE(rows >= 0 && F >= 0 && ldx >= 0, "cgnn_layer_norm: bad size");
    CGNN_REQUIRE(eps >= 0, "cgnn_layer_norm: eps must not be negative");
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
        a.relu = relu;
        a.drop = drop_of(drop, F);
        a.out = static_cast<T *>(out);
        a.stats = stats;
        a.rows = rows;
        a.F = F;
        return norm_typed<T>(a, a.drop.kept < kAllKept, stream);
    });
}

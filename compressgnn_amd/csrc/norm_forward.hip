// Layer norm of node rows, with the ReLU and the dropout behind it in the same pass:
//
//   m = sum x / F, v = sum (x - m)^2 / F, r = 1 / sqrt(v + eps), out = drop(relu((x - m) r w + b))
#include "rows.h"

namespace cgnn {
namespace {

// A workgroup per row, which reads it three times: for the mean, for the squares around it, for the output.
template <typename T, bool DROP>
__global__ __launch_bounds__(kBlock) void norm_long_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    __shared__ double scratch[kBlock / kWave];
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = a.x + r * a.ldx;
        T *out = a.out + r * a.F;
        double sum = 0;
        for (int64_t j = (int64_t)threadIdx.x * kDrawn; j < a.F; j += (int64_t)kBlock * kDrawn) {
            const auto p = load_pack<T, kDrawn>(x, j, a.F);
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) sum += (double)p.v[i];
        }
        const double mean = workgroup_sum<double, kBlock>(sum, scratch) / (double)a.F;
        double squares = 0;
        for (int64_t j = (int64_t)threadIdx.x * kDrawn; j < a.F; j += (int64_t)kBlock * kDrawn) {
            const auto p = load_pack<T, kDrawn>(x, j, a.F);
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                const double d = j + i < a.F ? (double)p.v[i] - mean : 0.0;
                squares = __builtin_fma(d, d, squares);
            }
        }
        const double rstd = reciprocal_root(workgroup_sum<double, kBlock>(squares, scratch) / (double)a.F + a.eps);
        if (a.stats && threadIdx.x == 0) {
            a.stats[2 * r] = mean;
            a.stats[2 * r + 1] = rstd;
        }
        for (int64_t j = (int64_t)threadIdx.x * kDrawn; j < a.F; j += (int64_t)kBlock * kDrawn) {
            const auto p = load_pack<T, kDrawn>(x, j, a.F);
            Pack<T, kDrawn> y;
            Draws drawn;
            if constexpr (DROP) drawn = draw(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks + j / kDrawn));
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                const bool in = j + i < a.F;
                const double w = in ? (double)a.weight.at(j + i, C(1)) : 0.0, b = in ? (double)a.bias.at(j + i, C(0)) : 0.0;
                double v = before_relu((double)p.v[i], mean, rstd, w, b);
                if (a.relu && v <= 0) v = 0;
                C c = (C)v;
                if constexpr (DROP) c = drawn.keeps(i, a.drop.kept) ? c * (C)a.drop.scale : C(0);
                y.v[i] = (T)c;
            }
            store_pack<T, kDrawn>(out, j, a.F, y);
        }
    }
}

template <typename T>
int norm_typed(const NormArgs<T> &a, bool drops, hipStream_t stream) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 4096);
    if (drops)
        hipLaunchKernelGGL((norm_long_kernel<T, true>), dim3(grid), dim3(kBlock), 0, stream, a);
    else
        hipLaunchKernelGGL((norm_long_kernel<T, false>), dim3(grid), dim3(kBlock), 0, stream, a);
    return check_launch("layer_norm");
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

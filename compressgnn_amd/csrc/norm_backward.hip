// The gradients of layer norm -> ReLU -> dropout (norm_forward.hip).  With h = (x - m) r and g = the gradient of the output
// where the element was kept and the ReLU open, times the dropout's scale:
//
//   dw = sum over rows of g h, db = sum over rows of g
//   dx = r (g w - mean(g w) - h mean(g w h)), means over the row
#include "rows.h"

namespace cgnn {
namespace {

constexpr int kPartRows = 64;   // rows per part of the parameters' sums, at least
constexpr int kMostParts = 512;
constexpr int kLanes = 64;      // column_parts_kernel: lanes side by side, kDrawn columns each

int64_t part_rows(int64_t rows) { return std::max<int64_t>(kPartRows, ceil_div(rows, kMostParts)); }
int64_t parts_of(int64_t rows) { return ceil_div(rows, part_rows(rows)); }

// Eight elements of a row as the gradient sees them: h, and g as described above.
template <typename T, bool DROP>
__device__ __forceinline__ void masked(const NormArgs<T> &a, int64_t r, int64_t j, double mean, double rstd, uint64_t offset,
                                       compute_t<T> (&h)[kDrawn], compute_t<T> (&g)[kDrawn]) {
    using C = compute_t<T>;
    const auto x = load_pack<T, kDrawn>(a.x + r * a.ldx, j, a.F);
    const auto d = load_pack<T, kDrawn>(a.grad + r * a.ldg, j, a.F);
    Draws drawn;
    if constexpr (DROP) drawn = draw(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks + j / kDrawn));
#pragma unroll
    for (int i = 0; i < kDrawn; ++i) {
        const bool in = j + i < a.F;
        h[i] = in ? (C)(((double)x.v[i] - mean) * rstd) : C(0);
        C v = (C)d.v[i];
        if constexpr (DROP) v = drawn.keeps(i, a.drop.kept) ? v * (C)a.drop.scale : C(0);
        if (a.relu && in && before_relu((double)x.v[i], mean, rstd, (double)a.weight.at(j + i, C(1)), (double)a.bias.at(j + i, C(0))) <= 0)
            v = C(0);
        g[i] = v;
    }
}

// dx: a workgroup per row, which reads it twice.
template <typename T, bool DROP>
__global__ __launch_bounds__(kBlock) void norm_long_dx_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    __shared__ C scratch[kBlock / kWave];
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const double mean = a.stats[2 * r], rstd = a.stats[2 * r + 1];
        C sum = 0, product = 0;
        for (int64_t j = (int64_t)threadIdx.x * kDrawn; j < a.F; j += (int64_t)kBlock * kDrawn) {
            C h[kDrawn], g[kDrawn];
            masked<T, DROP>(a, r, j, mean, rstd, offset, h, g);
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                const C gw = g[i] * (j + i < a.F ? a.weight.at(j + i, C(1)) : C(0));
                sum += gw;
                product += gw * h[i];
            }
        }
        const C c1 = workgroup_sum<C, kBlock>(sum, scratch) / (C)a.F;
        const C c2 = workgroup_sum<C, kBlock>(product, scratch) / (C)a.F;
        for (int64_t j = (int64_t)threadIdx.x * kDrawn; j < a.F; j += (int64_t)kBlock * kDrawn) {
            C h[kDrawn], g[kDrawn];
            masked<T, DROP>(a, r, j, mean, rstd, offset, h, g);
            Pack<T, kDrawn> dx;
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                const C gw = g[i] * (j + i < a.F ? a.weight.at(j + i, C(1)) : C(0));
                dx.v[i] = (T)((C)rstd * (gw - c1 - h[i] * c2));
            }
            store_pack<T, kDrawn>(a.dx + r * a.F, j, a.F, dx);
        }
    }
}

// dw and db over part_rows rows: blockIdx.x names the part, blockIdx.y the columns.
template <typename T, bool DROP>
__global__ __launch_bounds__(kBlock) void norm_long_parts_kernel(NormArgs<T> a, int64_t part) {
    using C = compute_t<T>;
    __shared__ C sums[kBlock / kLanes][2][kDrawn][kLanes];
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const int64_t j = ((int64_t)blockIdx.y * kLanes + lane) * kDrawn;
    const int64_t last = std::min(a.rows, (int64_t)(blockIdx.x + 1) * part);
    C dw[kDrawn] = {}, db[kDrawn] = {};
    if (j < a.F)
        for (int64_t r = (int64_t)blockIdx.x * part + group; r < last; r += kBlock / kLanes) {
            C h[kDrawn], g[kDrawn];
            masked<T, DROP>(a, r, j, a.stats[2 * r], a.stats[2 * r + 1], offset, h, g);
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                dw[i] += g[i] * h[i];
                db[i] += g[i];
            }
        }
#pragma unroll
    for (int i = 0; i < kDrawn; ++i) {
        sums[group][0][i][lane] = dw[i];
        sums[group][1][i][lane] = db[i];
    }
    __syncthreads();
    if (group == 0)
#pragma unroll
        for (int i = 0; i < kDrawn; ++i)
            if (j + i < a.F) {
                C w = 0, b = 0;
#pragma unroll
                for (int k = 0; k < kBlock / kLanes; ++k) {
                    w += sums[k][0][i][lane];
                    b += sums[k][1][i][lane];
                }
                C *to = a.partial + (int64_t)blockIdx.x * 2 * a.F + j + i;
                to[0] = w;
                to[a.F] = b;
            }
}

// The parts' sums, added up in 64 bits in the order of the parts: column c < F of the weight's gradient, then the bias's.
template <typename C, typename P>
__global__ __launch_bounds__(kBlock) void norm_sum_parts_kernel(const C *partial, int64_t parts, int64_t F, P *dweight, P *dbias) {
    constexpr int kColumns = 16, kGroups = kBlock / kColumns;
    __shared__ double sums[kGroups][kColumns];
    const int lane = threadIdx.x % kColumns, group = threadIdx.x / kColumns;
    const int64_t c = (int64_t)blockIdx.x * kColumns + lane;
    double sum = 0;
    if (c < 2 * F)
        for (int64_t k = group; k < parts; k += kGroups) sum += (double)partial[k * 2 * F + c];
    sums[group][lane] = sum;
    __syncthreads();
    if (group != 0 || c >= 2 * F) return;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) sum += sums[k][lane];
    P *to = c < F ? dweight : dbias;
    if (to) to[c < F ? c : c - F] = (P)(compute_t<P>)sum;
}

template <typename T>
int norm_backward_typed(NormArgs<T> a, bool drops, int param_dtype, void *dweight, void *dbias, hipStream_t stream) {
    using C = compute_t<T>;
    if (a.dx) {
        const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 4096);
        if (drops)
            hipLaunchKernelGGL((norm_long_dx_kernel<T, true>), dim3(grid), dim3(kBlock), 0, stream, a);
        else
            hipLaunchKernelGGL((norm_long_dx_kernel<T, false>), dim3(grid), dim3(kBlock), 0, stream, a);
        if (int rc = check_launch("layer_norm_backward")) return rc;
    }
    if (dweight == nullptr && dbias == nullptr) return CGNN_OK;
    const int64_t part = part_rows(a.rows);
    const dim3 grid((unsigned)parts_of(a.rows), (unsigned)ceil_div(a.F, (int64_t)kLanes * kDrawn));
    if (drops)
        hipLaunchKernelGGL((norm_long_parts_kernel<T, true>), grid, dim3(kBlock), 0, stream, a, part);
    else
        hipLaunchKernelGGL((norm_long_parts_kernel<T, false>), grid, dim3(kBlock), 0, stream, a, part);
    if (int rc = check_launch("layer_norm_backward")) return rc;
    const dim3 columns((unsigned)ceil_div(2 * a.F, 16));
    const int64_t parts = parts_of(a.rows);
    if (param_dtype == CGNN_F32)
        hipLaunchKernelGGL((norm_sum_parts_kernel<C, float>), columns, dim3(kBlock), 0, stream, a.partial, parts, a.F,
                           static_cast<float *>(dweight), static_cast<float *>(dbias));
    else
        hipLaunchKernelGGL((norm_sum_parts_kernel<C, T>), columns, dim3(kBlock), 0, stream, a.partial, parts, a.F,
                           static_cast<T *>(dweight), static_cast<T *>(dbias));
    return check_launch("layer_norm_backward");
}

}  // namespace
}  // namespace cgnn

using namespace cgnn;

extern "C" size_t cgnn_layer_norm_backward_workspace_bytes(int64_t rows, int64_t F, int dtype) {
    if (rows <= 0 || F <= 0) return 0;
    return (size_t)parts_of(rows) * 2 * (size_t)F * (dtype == CGNN_F64 ? 8 : 4);
}

extern "C" int cgnn_layer_norm_backward(int64_t rows, int64_t F, int dtype, int param_dtype, const void *grad, int64_t ldg,
                                        const void *x, int64_t ldx, const double *stats, const void *weight, const void *bias,
                                        int relu, const cgnn_drop *drop, void *dx, void *dweight, void *dbias, void *workspace,
                                        size_t workspace_bytes, cgnn_stream_t stream) {
    CGNN_REQUIRE(rows > 0 && F > 0 && ldx >= 0 && ldg >= 0, "cgnn_layer_norm_backward: bad size");
    CGNN_REQUIRE(F < ((int64_t)1 << 31) - 65536, "cgnn_layer_norm_backward: a row must be shorter than 2^31 elements");
    CGNN_REQUIRE(param_dtype == dtype || (param_dtype == CGNN_F32 && dtype != CGNN_F64),
                 "cgnn_layer_norm_backward: parameters have the type of the rows, or f32 for 16-bit rows");
    if (drop) CGNN_REQUIRE_DROP("cgnn_layer_norm_backward", drop);
    return with_row_type(dtype, "cgnn_layer_norm_backward: dtype must be f32, f64, f16 or bf16", [&](auto tag) {
        using T = typename decltype(tag)::type;
        if (dx == nullptr && dweight == nullptr && dbias == nullptr) return (int)CGNN_OK;
        CGNN_REQUIRE(grad && x && stats, "cgnn_layer_norm_backward: null array");
        if ((dweight || dbias) &&
            (workspace == nullptr || workspace_bytes < cgnn_layer_norm_backward_workspace_bytes(rows, F, dtype)))
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
        return norm_backward_typed<T>(a, a.drop.kept < kAllKept, param_dtype, dweight, dbias, stream);
    });
}

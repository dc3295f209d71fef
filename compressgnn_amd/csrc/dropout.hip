// Dropout of node rows: out = kept ? x * scale : 0, the mask from the positions of the elements (rows.h).  The gradient is the
// same pass over the output's gradient.
#include "rows.h"

namespace cgnn {
namespace {

template <typename T>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const T *x, int64_t ldx, int64_t rows, int64_t F, Drop drop, T *out) {
    using C = compute_t<T>;
    const uint64_t offset = drop_offset(drop);
    const int64_t blocks = rows * drop.blocks, step = (int64_t)gridDim.x * kBlock;
    for (int64_t n = (int64_t)blockIdx.x * kBlock + threadIdx.x; n < blocks; n += step) {
        const int64_t r = n / drop.blocks, j = (n - r * drop.blocks) * kDrawn;
        const Draws drawn = draw(drop.seed, offset, (uint64_t)n);
        const auto p = load_pack<T, kDrawn>(x + r * ldx, j, F);
        C v[kDrawn];
#pragma unroll
        for (int i = 0; i < kDrawn; ++i) v[i] = (C)p.v[i] * (C)drop.scale;
        auto y = rounded<T, kDrawn>(v);
        if (drop.kept < kAllKept) y = masked<T, kDrawn>(y, drawn, drop.kept);
        store_pack<T, kDrawn>(out + r * F, j, F, y);
    }
}

}  // namespace
}  // namespace cgnn

using namespace cgnn;

extern "C" int cgnn_dropout(int64_t rows, int64_t F, int dtype, const void *x, int64_t ldx, const cgnn_drop *drop, void *out,
                            cgnn_stream_t stream) {
    CGNN_REQUIRE(rows >= 0 && F >= 0 && ldx >= 0, "cgnn_dropout: bad size");
    CGNN_REQUIRE(drop, "cgnn_dropout: null drop");
    CGNN_REQUIRE_DROP("cgnn_dropout", drop);
    return with_row_type(dtype, "cgnn_dropout: dtype must be f32, f64, f16 or bf16", [&](auto tag) {
        using T = typename decltype(tag)::type;
        if (rows == 0 || F == 0) return (int)CGNN_OK;
        CGNN_REQUIRE(x && out, "cgnn_dropout: null array");
        const Drop d = drop_of(drop, F);
        const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(rows * d.blocks, kBlock), 8192);
        hipLaunchKernelGGL((dropout_kernel<T>), dim3(grid), dim3(kBlock), 0, stream, static_cast<const T *>(x), ldx, rows, F, d,
                           static_cast<T *>(out));
        return check_launch("dropout");
    });
}

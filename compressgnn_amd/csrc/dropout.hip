// Dropout of node rows: out = kept ? x * scale : 0, the mask from the positions of the elements (rows.h).  The gradient is the
// same pass over the output's gradient.
#include "rows.h"

namespace cgnn {
namespace {

template <typename T>
struct DropoutArgs {
    const T *x;
    T *out;
    int64_t rows, F, ldx;
    Drop drop;
    int64_t packs;  // of 16 bytes per row, the last ones maybe empty: as many as the row's calls of the generator serve
    int64_t first;  // workgroup of the matrix that the launch begins with
    bool streamed;
};

// A lane takes PACKS packs of 16 bytes a workgroup's width apart, and a workgroup its stretch of memory, once: so all workgroups that are
// resident read one stretch, and nothing waits for a store: 2,449,029 x 256 bfloat16 in 424 us, 5.9 of the 6.2 TB/s of a copy (540 where
// workgroups went over the matrix again and again).  FLAT: whole rows of eight or one row make one long row, whose
// packs are found without a division.
template <typename T, bool FLAT>
__global__ __launch_bounds__(kBlock) void dropout_kernel(DropoutArgs<T> a) {
    using C = compute_t<T>;
    constexpr int N = 16 / (int)sizeof(T), SHARE = kDrawn / N, PACKS = SHARE < 2 ? 2 : SHARE;
    const uint64_t offset = drop_offset(a.drop);
    const int64_t begin = (a.first + blockIdx.x) * kBlock * PACKS, extent = (a.rows - 1) * a.ldx + a.F;
    const int64_t row0 = FLAT ? 0 : begin / a.packs, pack0 = begin - row0 * a.packs;
    const float inverse = 1.0f / (float)a.packs;
    int64_t row[PACKS], pack[PACKS];
    words_t asked[PACKS];
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
        row[k] = row0;
        pack[k] = pack0 + k * kBlock + threadIdx.x;
        if constexpr (!FLAT) {
            // packs of short rows: numbers of four digits at most, whose quotient the float product hits; a long row: this one or the next
            const int64_t rows = a.packs >= kBlock * PACKS ? (pack[k] >= a.packs ? 1 : 0) : (int64_t)(((float)(int)pack[k] + 0.5f) * inverse);
            row[k] += rows;
            pack[k] -= rows * a.packs;
        }
        const bool in = row[k] < a.rows && pack[k] * N < a.F;
        asked[k] = ask_within<T>(a.x, in ? row[k] * a.ldx + pack[k] * N : 0, extent);
    }
    Draws drawn[PACKS];
    auto call = [&](int k) { return draw(a.drop.seed, offset, (uint64_t)(row[k] * a.drop.blocks + pack[k] / SHARE)); };
    if constexpr (SHARE == 1) {
#pragma unroll
        for (int k = 0; k < PACKS; ++k) drawn[k] = call(k);
    } else if constexpr (SHARE == 2) {
        const bool odd = threadIdx.x & 1;
        exchange(draw(a.drop.seed, offset, (uint64_t)(either(odd, row[1], row[0]) * a.drop.blocks + either(odd, pack[1], pack[0]) / SHARE)), odd,
                 drawn[0], drawn[1]);
    } else {
        const int lane = threadIdx.x & 3;
        int64_t r = row[0], p = pack[0];
#pragma unroll
        for (int k = 1; k < PACKS; ++k) {
            r = either(lane == k, row[k], r);
            p = either(lane == k, pack[k], p);
        }
        exchange(draw(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks + p / SHARE)), lane, drawn);
    }
#pragma unroll
    for (int k = 0; k < PACKS; ++k) {
        if (row[k] >= a.rows || pack[k] * N >= a.F) continue;
        const Pack<T, N> x = settled<T>(asked[k], a.x, row[k] * a.ldx + pack[k] * N, extent);
        C v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (C)x.v[i] * (C)a.drop.scale;
        Pack<T, N> y = rounded<T, N>(v);
        if (a.drop.kept < kAllKept) y = masked<T, N>(y, drawn[k], a.drop.kept);
        store_columns<T, N>(a.out + row[k] * a.F, pack[k] * N, a.F, y, a.streamed);
    }
}

// Matrices of less than 16 bytes.
template <typename T>
__global__ __launch_bounds__(kBlock) void dropout_few_kernel(DropoutArgs<T> a) {
    using C = compute_t<T>;
    const uint64_t offset = drop_offset(a.drop);
    for (int64_t n = threadIdx.x; n < a.rows * a.drop.blocks; n += kBlock) {
        const int64_t r = n / a.drop.blocks, j = (n - r * a.drop.blocks) * kDrawn;
        const Draws drawn = draw(a.drop.seed, offset, (uint64_t)n);
        const auto p = load_pack<T, kDrawn>(a.x + r * a.ldx, j, a.F);
        C v[kDrawn];
#pragma unroll
        for (int i = 0; i < kDrawn; ++i) v[i] = (C)p.v[i] * (C)a.drop.scale;
        auto y = rounded<T, kDrawn>(v);
        if (a.drop.kept < kAllKept) y = masked<T, kDrawn>(y, drawn, a.drop.kept);
        store_pack<T, kDrawn>(a.out + r * a.F, j, a.F, y);
    }
}

// A launch has fewer than 2^32 threads a dimension: a matrix of more (some 2^33 rows of one 16-bit feature) takes several.
constexpr int64_t kLaunched = ((int64_t)1 << 31) / kBlock;  // workgroups

template <typename T>
int dropout_launch(DropoutArgs<T> a, hipStream_t stream) {
    constexpr int N = 16 / (int)sizeof(T), SHARE = kDrawn / N, PACKS = SHARE < 2 ? 2 : SHARE;
    if (a.rows * a.F * (int64_t)sizeof(T) < 16) {
        hipLaunchKernelGGL((dropout_few_kernel<T>), dim3(1), dim3(kBlock), 0, stream, a);
        return check_launch("dropout");
    }
    a.streamed = streams(a.rows, a.F * (int64_t)sizeof(T), kBlock * 16, 2);
    const bool flat = a.rows == 1 || (a.F % kDrawn == 0 && a.ldx == a.F);
    if (flat) {
        a.F *= a.rows;
        a.rows = 1;
    }
    a.packs = a.drop.blocks * SHARE;
    const int64_t packs = flat ? ceil_div(a.F, N) : a.rows * a.packs, workgroups = ceil_div(packs, (int64_t)kBlock * PACKS);
    CGNN_REQUIRE(workgroups < (int64_t)1 << 31, "cgnn_dropout: too many elements");
    for (; a.first < workgroups; a.first += kLaunched) {
        const dim3 grid((unsigned)std::min(workgroups - a.first, kLaunched));
        if (flat)
            hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(kBlock), 0, stream, a);
        else
            hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(kBlock), 0, stream, a);
        if (int rc = check_launch("dropout")) return rc;
    }
    return CGNN_OK;
}

}  // namespace
}  // namespace cgnn

using namespace cgnn;

extern "C" int cgnn_dropout(int64_t rows, int64_t F, int dtype, const void *x, int64_t ldx, const cgnn_drop *drop, void *out,
                            cgnn_stream_t stream) {
    CGNN_REQUIRE(rows >= 0 && F >= 0 && (rows <= 1 || ldx >= F), "cgnn_dropout: bad size");
    CGNN_REQUIRE(drop, "cgnn_dropout: null drop");
    CGNN_REQUIRE_DROP("cgnn_dropout", drop);
    return with_row_type(dtype, "cgnn_dropout: dtype must be f32, f64, f16 or bf16", [&](auto tag) {
        using T = typename decltype(tag)::type;
        if (rows == 0 || F == 0) return (int)CGNN_OK;
        CGNN_REQUIRE(x && out, "cgnn_dropout: null array");
        DropoutArgs<T> a{};
        a.x = static_cast<const T *>(x);
        a.out = static_cast<T *>(out);
        a.rows = rows;
        a.F = F;
        a.ldx = ldx;
        a.drop = drop_of(drop, F);
        return dropout_launch<T>(a, stream);
    });
}

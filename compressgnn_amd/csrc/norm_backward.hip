// The gradients of layer norm -> ReLU -> dropout (norm_forward.hip).  With h = (x - m) r and g = the gradient of the output
// where the element was kept and the ReLU open, times the dropout's scale:
//
//   dw = sum over rows of g h, db = sum over rows of g
//   dx = r (g w - mean(g w) - h mean(g w h)), means over the row
#include "rows.h"

namespace cgnn {
namespace {

constexpr int kLongRows = 64;   // rows longer than the registers: rows per part of the parameters' sums, at least
constexpr int kLongParts = 512;
constexpr int kLanes = 64;      // ... lanes side by side, kDrawn columns each
constexpr int kChain = 512;     // other rows: as many of them at most are added up one after the other by a lane, in float

// Of 16-bit rows a lane has eight columns in a pack, and in float their sums, parameters and values: two packs a lane are beyond
// the 128 registers of a workgroup of 1,024.
RowShape gradient_shape(int64_t F, size_t element) { return row_shape(F, element, element == 2 ? kMostPacks / 2 : kMostPacks); }

int64_t long_rows(int64_t rows) { return std::max<int64_t>(kLongRows, ceil_div(rows, kLongParts)); }

// Workgroups of norm_gradients_kernel, each of which leaves a part of the parameters' sums: as many as are resident, more
// where the chains would get longer than kChain.
int64_t row_parts(int64_t rows, const RowShape &s) {
    const int64_t tiles = ceil_div(rows, s.threads / s.lanes);
    return std::max(std::min<int64_t>(tiles, 256 * 1024 / s.threads), ceil_div(tiles, kChain));
}

int64_t parts_of(int64_t rows, int64_t F, size_t element) {
    const RowShape shape = gradient_shape(F, element);
    return shape.lanes ? row_parts(rows, shape) : ceil_div(rows, long_rows(rows));
}

// Rows that fit the registers of their lanes, as in the forward pass: x and the gradient are read once for dx and for
// the parameters' sums, which every lane holds for its own columns until its rows are through.
template <typename T, int LANES, int K, int THREADS, bool DROP>
__global__ __launch_bounds__(THREADS) void norm_gradients_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    constexpr int N = 16 / (int)sizeof(T), GROUPS = THREADS / LANES, WAVES = THREADS / kWave;
    constexpr int COLUMNS = LANES * K * N;  // that the lanes have room for
    __shared__ C scratch[LANES > kWave ? WAVES * 2 : WAVES * COLUMNS];
    const int lane = threadIdx.x % LANES, F = (int)a.F;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const C inverse_F = C(1) / (C)F;
    int64_t r = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;

    Pack<T, N> next_x[K], next_g[K];
    double next_mean = 0, next_rstd = 0;
    auto ask = [&](int64_t row) {
        next_mean = a.stats[2 * row];
        next_rstd = a.stats[2 * row + 1];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int j = (lane + k * LANES) * N;
            next_x[k] = load_pack<T, N>(a.x + row * a.ldx, j, F);
            next_g[k] = load_pack<T, N>(a.grad + row * a.ldg, j, F);
        }
    };
    if (r < a.rows) ask(r);
    C w[K][N], b[K][N], dw[K][N], db[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (lane + k * LANES) * N + i;
            w[k][i] = j < F ? a.weight.at(j, C(1)) : C(0);
            b[k][i] = j < F && a.relu ? a.bias.at(j, C(0)) : C(0);
            dw[k][i] = db[k][i] = C(0);
        }
    for (; r < a.rows; r += step) {
        C h[K][N], g[K][N];
        const double mean = next_mean, rstd = next_rstd;
        C sum = 0, product = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int j = (lane + k * LANES) * N;
            C v[N];
            normalised<N>(next_x[k].v, mean, rstd, w[k], b[k], a.relu, h[k], v);
            Draws drawn;
            if constexpr (DROP) {
                drawn = draw(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks + j / kDrawn));
                drawn.from<N>(j);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                C d = (C)next_g[k].v[i];
                if constexpr (DROP) d = drawn.keeps(i, a.drop.kept) ? d * (C)a.drop.scale : C(0);
                g[k][i] = a.relu && v[i] <= 0 ? C(0) : d;
            }
        }
        if (r + step < a.rows) ask(r + step);
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
            row_sums<LANES, THREADS>(sum, product, scratch);
            const C c1 = sum * inverse_F, c2 = product * inverse_F;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int j = (lane + k * LANES) * N;
                Pack<T, N> dx;
#pragma unroll
                for (int i = 0; i < N; ++i) dx.v[i] = (T)((C)rstd * (fused(-h[k][i], c2, g[k][i]) - c1));
                if (j < F) store_pack<T, N>(a.dx + r * a.F, j, F, dx);
            }
        }
    }
    if (a.partial == nullptr) return;
    // the lane groups of a wave, then its waves in their order
    C *to = a.partial + (int64_t)blockIdx.x * 2 * a.F;
    auto leave = [&](C(&acc)[K][N], C *columns) {
        if constexpr (LANES > kWave) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int j = (lane + k * LANES) * N + i;
                    if (j < F) columns[j] = acc[k][i];
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
                columns[j] = total;
            }
        }
    };
    leave(dw, to);
    leave(db, to + a.F);
}

// Eight elements of a row as the gradient sees them: h, and g as described above.
template <typename T, bool DROP>
__device__ __forceinline__ void masked(const NormArgs<T> &a, int64_t r, int64_t j, double mean, double rstd, uint64_t offset,
                                       compute_t<T> (&w)[kDrawn], compute_t<T> (&h)[kDrawn], compute_t<T> (&g)[kDrawn]) {
    using C = compute_t<T>;
    const auto x = load_pack<T, kDrawn>(a.x + r * a.ldx, j, a.F);
    const auto d = load_pack<T, kDrawn>(a.grad + r * a.ldg, j, a.F);
    C b[kDrawn], v[kDrawn];
#pragma unroll
    for (int i = 0; i < kDrawn; ++i) {
        w[i] = j + i < a.F ? a.weight.at(j + i, C(1)) : C(0);
        b[i] = j + i < a.F && a.relu ? a.bias.at(j + i, C(0)) : C(0);
    }
    normalised<kDrawn>(x.v, mean, rstd, w, b, a.relu, h, v);
    Draws drawn;
    if constexpr (DROP) drawn = draw(a.drop.seed, offset, (uint64_t)(r * a.drop.blocks + j / kDrawn));
#pragma unroll
    for (int i = 0; i < kDrawn; ++i) {
        C c = (C)d.v[i];
        if constexpr (DROP) c = drawn.keeps(i, a.drop.kept) ? c * (C)a.drop.scale : C(0);
        g[i] = a.relu && v[i] <= 0 ? C(0) : c;
    }
}

constexpr int kLongThreads = 1024;

// dx of longer rows: a workgroup per row, which reads it twice.
template <typename T, bool DROP>
__global__ __launch_bounds__(kLongThreads) void norm_long_dx_kernel(NormArgs<T> a) {
    using C = compute_t<T>;
    __shared__ C scratch[kLongThreads / kWave * 2];
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const double mean = a.stats[2 * r], rstd = a.stats[2 * r + 1];
        C sum = 0, product = 0, w[kDrawn], h[kDrawn], g[kDrawn];
        for (int64_t j = (int64_t)threadIdx.x * kDrawn; j < a.F; j += (int64_t)kLongThreads * kDrawn) {
            masked<T, DROP>(a, r, j, mean, rstd, offset, w, h, g);
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                sum = fused(g[i], w[i], sum);
                product = fused(g[i] * w[i], h[i], product);
            }
        }
        row_sums<kLongThreads, kLongThreads>(sum, product, scratch);
        const C c1 = sum / (C)a.F, c2 = product / (C)a.F;
        for (int64_t j = (int64_t)threadIdx.x * kDrawn; j < a.F; j += (int64_t)kLongThreads * kDrawn) {
            masked<T, DROP>(a, r, j, mean, rstd, offset, w, h, g);
            Pack<T, kDrawn> dx;
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) dx.v[i] = (T)((C)rstd * (fused(-h[i], c2, g[i] * w[i]) - c1));
            store_pack<T, kDrawn>(a.dx + r * a.F, j, a.F, dx);
        }
    }
}

// Their dw and db: blockIdx.x names the part, `part` rows each, blockIdx.y the columns.
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
            C w[kDrawn], h[kDrawn], g[kDrawn];
            masked<T, DROP>(a, r, j, a.stats[2 * r], a.stats[2 * r + 1], offset, w, h, g);
#pragma unroll
            for (int i = 0; i < kDrawn; ++i) {
                dw[i] = fused(g[i], h[i], dw[i]);
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
    const RowShape shape = gradient_shape(a.F, sizeof(T));
    const int64_t parts = parts_of(a.rows, a.F, sizeof(T));
    const bool sums = dweight != nullptr || dbias != nullptr;
    if (!sums) a.partial = nullptr;
    int rc = CGNN_OK;
    if (shape.lanes) {
        rc = with_row_shape(shape, [&](auto tag) {
            using S = decltype(tag);
            if constexpr (S::lanes * S::packs * (int)sizeof(T) < 2 * 2048 || sizeof(T) > 2) {
                const dim3 grid((unsigned)parts);
                if (drops)
                    hipLaunchKernelGGL((norm_gradients_kernel<T, S::lanes, S::packs, S::threads, true>), grid, dim3(S::threads), 0, stream, a);
                else
                    hipLaunchKernelGGL((norm_gradients_kernel<T, S::lanes, S::packs, S::threads, false>), grid, dim3(S::threads), 0, stream, a);
            }
            return check_launch("layer_norm_backward");
        });
    } else {
        if (a.dx) {
            const dim3 grid((unsigned)std::min<int64_t>(a.rows, 1024));
            if (drops)
                hipLaunchKernelGGL((norm_long_dx_kernel<T, true>), grid, dim3(kLongThreads), 0, stream, a);
            else
                hipLaunchKernelGGL((norm_long_dx_kernel<T, false>), grid, dim3(kLongThreads), 0, stream, a);
            rc = check_launch("layer_norm_backward");
        }
        if (rc == CGNN_OK && sums) {
            const int64_t part = long_rows(a.rows);
            const dim3 grid((unsigned)parts, (unsigned)ceil_div(a.F, (int64_t)kLanes * kDrawn));
            if (drops)
                hipLaunchKernelGGL((norm_long_parts_kernel<T, true>), grid, dim3(kBlock), 0, stream, a, part);
            else
                hipLaunchKernelGGL((norm_long_parts_kernel<T, false>), grid, dim3(kBlock), 0, stream, a, part);
            rc = check_launch("layer_norm_backward");
        }
    }
    if (rc != CGNN_OK || !sums) return rc;
    const dim3 columns((unsigned)ceil_div(2 * a.F, 16));
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
    return (size_t)parts_of(rows, F, row_type_bytes(dtype)) * 2 * (size_t)F * (dtype == CGNN_F64 ? 8 : 4);
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

// What the row-wise operators on node features (norm_forward.hip, norm_backward.hip, dropout.hip) have in common: element types, the
// generator of the dropout masks, sums over lanes.
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace cgnn {

using f16_t = _Float16;
using bf16_t = __bf16;

// What values of a type are computed in.  Means, variances and everything that decides on which side of zero a
// normalised value lies are computed in 64 bits whatever the type: a float rounding there would let one pass of a step
// see a ReLU open and another see it closed, which moves a gradient by its whole size.
template <typename T> struct Compute { using type = float; };
template <> struct Compute<double> { using type = double; };
template <typename T> using compute_t = typename Compute<T>::type;

template <typename T> struct TypeTag { using type = T; };

// Calls `run(TypeTag<T>())` for the type of a cgnn_dtype.
template <typename F>
int with_row_type(int dtype, const char *unsupported, F &&run) {
    switch (dtype) {
        case CGNN_F32: return run(TypeTag<float>());
        case CGNN_F64: return run(TypeTag<double>());
        case CGNN_F16: return run(TypeTag<f16_t>());
        case CGNN_BF16: return run(TypeTag<bf16_t>());
        default: return fail(CGNN_EUNSUPPORTED, unsupported);
    }
}

inline size_t row_type_bytes(int dtype) { return dtype == CGNN_F64 ? 8 : dtype == CGNN_F32 ? 4 : 2; }

// ------------------------------------------------------------------- dropout masks ----
//
// Element (i, j) of a [rows, F] matrix is kept where a 16-bit number drawn for it lies below `kept`, the share of kept elements
// in 65,536ths.  Numbers come eight at a time from Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as
// 1, 2, 3, SC 2011) over the counter (i * ceil(F / 8) + j / 8, offset) under the key `seed`, so that every kernel
// finds the same mask again from the position alone and none is stored.  Sixteen bits an element, not 32: half the
// generator's work, for a share that is the asked one to 2^-17; the scale is the reciprocal of the share as taken, so
// that the mean stays what it was.
constexpr int kDrawn = 8;  // elements per call of the generator
constexpr uint32_t kAllKept = 65536;

struct Drop {
    uint64_t seed, offset;
    const int64_t *counter;  // added to offset when the kernel runs, or NULL
    int64_t blocks;          // generator calls per row
    uint32_t kept;
    double scale;
};

inline Drop drop_of(const cgnn_drop *d, int64_t F) {
    Drop drop{};
    drop.blocks = ceil_div(F, kDrawn);
    drop.kept = d ? (uint32_t)d->kept : kAllKept;
    drop.scale = drop.kept ? (double)kAllKept / drop.kept : 0.0;
    if (d) {
        drop.seed = d->seed;
        drop.offset = d->offset;
        drop.counter = d->counter;
    }
    return drop;
}

#define CGNN_REQUIRE_DROP(op, d) CGNN_REQUIRE((d)->kept >= 0 && (d)->kept <= (int32_t)kAllKept, op ": kept must lie in [0, 65536]")

// Eight draws of 16 bits, two a word, the low half first.
struct Draws {
    uint32_t word[4];
    __device__ __forceinline__ bool keeps(int i, uint32_t kept) const {
        const uint32_t w = word[i >> 1];
        return (i & 1 ? w >> 16 : w & 0xFFFFu) < kept;
    }
};

__device__ __forceinline__ Draws draw(uint64_t seed, uint64_t offset, uint64_t block) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        const uint32_t n0 = (uint32_t)(b >> 32) ^ c1 ^ k0, n2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        c0 = n0;
        c2 = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Draws{{c0, c1, c2, c3}};
}

__device__ __forceinline__ uint64_t drop_offset(const Drop &d) { return d.offset + (d.counter ? (uint64_t)*d.counter : 0); }

// ------------------------------------------------------------------------- reading ----

// N elements at any element's address: loads and stores of 16 bytes where they make that many.  The memory of gfx950 takes them
// at addresses that are no multiple of 16.
template <typename T, int N>
struct __attribute__((packed, aligned(alignof(T)))) Pack {
    T v[N];
};

// N elements of a row of F from column j on: those behind its end read as zero.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T *row, int64_t j, int64_t F) {
    Pack<T, N> p;
    if (j + N <= F) {
        p = *reinterpret_cast<const Pack<T, N> *>(row + j);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p.v[i] = j + i < F ? row[j + i] : T(0);
    }
    return p;
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T *row, int64_t j, int64_t F, const Pack<T, N> &p) {
    if (j + N <= F) {
        *reinterpret_cast<Pack<T, N> *>(row + j) = p;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (j + i < F) row[j + i] = p.v[i];
    }
}

// --------------------------------------------------------------------- sums of lanes ----

// The sum over the workgroup's lanes, in every lane: lanes first, then the waves in their order.  `scratch`: one
// element per wave.
template <typename A, int THREADS>
__device__ __forceinline__ A workgroup_sum(A v, A *scratch) {
#pragma unroll
    for (int step = 1; step < kWave; step <<= 1) v += __shfl_xor(v, step);
    if constexpr (THREADS > kWave) {
        __syncthreads();  // the last sum's readers are done
        if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
        __syncthreads();
        v = scratch[0];
#pragma unroll
        for (int w = 1; w < THREADS / kWave; ++w) v += scratch[w];
    }
    return v;
}

// ------------------------------------------------------------------------ layer norm ----

// 1 / sqrt(a).
__device__ __forceinline__ double reciprocal_root(double a) { return 1.0 / __builtin_sqrt(a); }

// A parameter of the rows' type or of float (`wide`); 1 or 0 where there is none.
template <typename T>
struct Params {
    const void *data;
    bool wide;
    __device__ __forceinline__ compute_t<T> at(int64_t j, compute_t<T> otherwise) const {
        if (data == nullptr) return otherwise;
        return wide ? (compute_t<T>)static_cast<const float *>(data)[j] : (compute_t<T>)static_cast<const T *>(data)[j];
    }
};

template <typename T>
struct NormArgs {
    const T *x;
    int64_t ldx;
    Params<T> weight, bias;
    double eps;
    int relu;
    Drop drop;
    T *out;         // forward
    double *stats;  // [rows, 2]: mean and reciprocal deviation (written forward where wanted, read backward)
    const T *grad;  // backward
    int64_t ldg;
    T *dx;           // or NULL
    compute_t<T> *partial;  // [parts, 2, F]: sums of g * h and of g over a part of the rows
    int64_t rows, F;
};

// h * w + b in 64 bits, by the one expression that both passes use.
__device__ __forceinline__ double before_relu(double x, double mean, double rstd, double w, double b) {
    return __builtin_fma((x - mean) * rstd, w, b);
}

}  // namespace cgnn

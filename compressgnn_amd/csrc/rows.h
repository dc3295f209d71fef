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

// By value: a choice between elements of an array would be one between addresses, and put the array into memory.
template <typename T>
__device__ __forceinline__ T either(bool first, T a, T b) {
    return first ? a : b;
}

// Eight draws of 16 bits, two a word, the low half first.
struct Draws {
    uint32_t word[4];
    __device__ __forceinline__ bool keeps(int i, uint32_t kept) const {
        const uint32_t w = word[i >> 1];
        return (i & 1 ? w >> 16 : w & 0xFFFFu) < kept;
    }
    // The N that begin at element j of a row come to the front (N divides j).
    template <int N>
    __device__ __forceinline__ void from(int j) {
        if constexpr (N <= 4) {
            word[0] = either(j & 4, word[2], word[0]);
            word[1] = either(j & 4, word[3], word[1]);
        }
        if constexpr (N == 2) word[0] = either(j & 2, word[1], word[0]);
    }
};

__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

__device__ __forceinline__ Draws draw(uint64_t seed, uint64_t offset, uint64_t block) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = xor3((uint32_t)(b >> 32), c1, k0);
        c2 = xor3((uint32_t)(a >> 32), c3, k1);
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Draws{{c0, c1, c2, c3}};
}

__device__ __forceinline__ uint32_t neighbours(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true); }
__device__ __forceinline__ uint32_t across_pairs(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true); }

// Packs of four: two lanes next to each other need half of the same eight draws.  Each makes those of one of two packs, the even
// lane the first's, and they exchange the halves that the other needs.
__device__ __forceinline__ void exchange(const Draws &own, bool odd, Draws &first, Draws &second) {
    const uint32_t got0 = neighbours(either(odd, own.word[0], own.word[2])), got1 = neighbours(either(odd, own.word[1], own.word[3]));
    first.word[0] = either(odd, got0, own.word[0]);
    first.word[1] = either(odd, got1, own.word[1]);
    second.word[0] = either(odd, own.word[2], got0);
    second.word[1] = either(odd, own.word[3], got1);
}

// Packs of two: four lanes need a word each of the same eight draws.  Lane l of the four makes those of pack l of four, and the words
// change places as rows and columns of a matrix do.
__device__ __forceinline__ void exchange(Draws own, int lane, Draws (&packs)[4]) {
    uint32_t(&w)[4] = own.word;
    const bool odd = lane & 1, high = lane & 2;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t got = neighbours(either(odd, w[i], w[i + 1]));
        w[i] = either(odd, got, w[i]);
        w[i + 1] = either(odd, w[i + 1], got);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t got = across_pairs(either(high, w[i], w[i + 2]));
        packs[i].word[0] = either(high, got, w[i]);
        packs[i + 2].word[0] = either(high, w[i + 2], got);
    }
}

// The draws of a lane's packs lane + k * LANES of a row whose numbers begin at `block`.
template <int N, int LANES, int K>
__device__ __forceinline__ void draw_row(uint64_t seed, uint64_t offset, uint64_t block, int lane, Draws (&drawn)[K]) {
    if constexpr (N == 4 && LANES == 1) {  // a lane has both halves
#pragma unroll
        for (int k = 0; k < K; k += 2) {
            drawn[k] = draw(seed, offset, block + k / 2);
            if (k + 1 < K) {
                drawn[k + 1].word[0] = drawn[k].word[2];
                drawn[k + 1].word[1] = drawn[k].word[3];
            }
        }
    } else {
        constexpr int PAIRED = N == 4 ? K / 2 * 2 : 0;
#pragma unroll
        for (int k = 0; k < PAIRED; k += 2) {
            const int pack = lane + k * LANES + (lane & 1) * LANES;
            exchange(draw(seed, offset, block + pack / 2), lane & 1, drawn[k], drawn[k + 1]);
        }
#pragma unroll
        for (int k = PAIRED; k < K; ++k) {
            const int j = (lane + k * LANES) * N;
            drawn[k] = draw(seed, offset, block + j / kDrawn);
            drawn[k].template from<N>(j);
        }
    }
}

__device__ __forceinline__ uint64_t drop_offset(const Drop &d) { return d.offset + (d.counter ? (uint64_t)*d.counter : 0); }

// --------------------------------------------------------------- reading and writing ----

// 16 bytes as they are: held this way, and not as elements, the words of a load in flight are not touched before they are used.
typedef uint32_t words_t __attribute__((ext_vector_type(4), aligned(2), may_alias));

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

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

// N elements (16 bytes) from `at` on of `extent` >= N elements: one load without a branch, so that nothing waits for it before its
// values are used.  It may run into the next row (the caller has to leave what it finds there); where it would leave the matrix it reads
// the last N elements instead, and `settled` gets the ones asked for once they are used.
template <typename T>
__device__ __forceinline__ words_t ask_within(const T *matrix, int64_t at, int64_t extent) {
    constexpr int N = 16 / (int)sizeof(T);
    return *reinterpret_cast<const words_t *>(matrix + (at < extent - N ? at : extent - N));
}

// Waits for what was asked for, here: loads and stores are counted together and in order, and a wait behind a store that not every
// lane makes has to wait for that store too.  Ahead of a row's stores this waits for the next row's loads and the last
// row's stores only, both asked for a row's work ago.  The same ahead of the loop, whose first waits would else be in every round.
template <int K>
__device__ __forceinline__ void arrived(words_t (&asked)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) asm volatile("" : "+v"(asked[k]));
}

template <typename C, int K, int N>
__device__ __forceinline__ void arrived(C (&asked)[K][N]) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) asm volatile("" : "+v"(asked[k][i]));
}

template <typename T>
__device__ __forceinline__ void arrived(T &asked) {
    if constexpr (sizeof(T) == 2) {
        uint32_t word = __builtin_bit_cast(uint16_t, asked);
        asm volatile("" : "+v"(word));
        asked = __builtin_bit_cast(T, (uint16_t)word);
    } else {
        asm volatile("" : "+v"(asked));
    }
}

// The packs of a row as `ask_within` got them, and, where the row is one of the last and they may run out of the matrix, as
// asked for.
template <typename T, int LANES, int K, int N = 16 / (int)sizeof(T)>
__device__ __forceinline__ void row_arrived(const words_t (&asked)[K], const T *matrix, int64_t at, int64_t extent, int lane, int F, Pack<T, N> (&x)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] = __builtin_bit_cast(Pack<T, N>, asked[k]);
    if (at + LANES * K * N > extent)
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int j = (lane + k * LANES) * N;
            const int64_t from = at + (j < F ? j : 0);
            if (from > extent - N)
#pragma unroll
                for (int i = 0; i < N; ++i) x[k].v[i] = matrix[from + i < extent ? from + i : extent - 1];
        }
}

template <typename T, int N = 16 / (int)sizeof(T)>
__device__ __forceinline__ Pack<T, N> settled(words_t asked, const T *matrix, int64_t at, int64_t extent) {
    Pack<T, N> p = __builtin_bit_cast(Pack<T, N>, asked);
    if (at > extent - N)
#pragma unroll
        for (int i = 0; i < N; ++i) p.v[i] = matrix[at + i < extent ? at + i : extent - 1];
    return p;
}

// The same at once, for any extent.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_within(const T *matrix, int64_t at, int64_t extent) {
    Pack<T, N> p;
    if (at + N <= extent) {
        p = *reinterpret_cast<const Pack<T, N> *>(matrix + at);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p.v[i] = matrix[at + i < extent ? at + i : extent - 1];
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

// 16 bytes, past the caches where they are not read again before they would be gone from there.  In assembly: of two stores that differ
// in nothing else the compiler makes one, the plain one; and what it knows of stores of more than 8 bytes has to be said too: gfx950
// reads their data late, and the vector ALU may write those registers again two wait states behind the store at the earliest.
template <typename T, int N>
__device__ __forceinline__ void store_whole(T *to, const Pack<T, N> &p, bool streamed) {
    if (streamed)
        asm volatile("global_store_dwordx4 %0, %1, off nt\n\ts_nop 1" : : "v"(to), "v"(__builtin_bit_cast(words_t, p)) : "memory");
    else
        *reinterpret_cast<Pack<T, N> *>(to) = p;
}

// store_pack for a column j that is a multiple of N: what is left of the row has the same length, F % N, in every row, and goes out in
// at most three pieces.
template <typename T, int N>
__device__ __forceinline__ void store_columns(T *row, int64_t j, int64_t F, const Pack<T, N> &p, bool streamed) {
    if (j + N <= F) {
        store_whole(row + j, p, streamed);
    } else if (j < F) {
        const int rest = (int)(F % N);
        T *to = row + j;
        if constexpr (N == 8) {
            const bool four = rest & 4, two = rest & 2;
            if (four) *reinterpret_cast<Pack<T, 4> *>(to) = Pack<T, 4>{{p.v[0], p.v[1], p.v[2], p.v[3]}};
            to += rest & 4;
            const T a = either(four, p.v[4], p.v[0]), b = either(four, p.v[5], p.v[1]), c = either(four, p.v[6], p.v[2]);
            if (two) *reinterpret_cast<Pack<T, 2> *>(to) = Pack<T, 2>{{a, b}};
            if (rest & 1) to[rest & 2] = either(two, c, a);
        } else if constexpr (N == 4) {
            if (rest & 2) *reinterpret_cast<Pack<T, 2> *>(to) = Pack<T, 2>{{p.v[0], p.v[1]}};
            if (rest & 1) to[rest & 2] = either(rest & 2, p.v[2], p.v[0]);
        } else {
            to[0] = p.v[0];
        }
    }
}

// p with the elements that are not kept zeroed (kept < 65536).  16-bit elements two a step: kept less the draw, not below zero, then at most one, times the
// element's bits.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> masked(const Pack<T, N> &p, const Draws &drawn, uint32_t kept) {
    if constexpr (sizeof(T) == 2) {
        struct Words {
            uint32_t v[N / 2];
        } words = __builtin_bit_cast(Words, p);
        const uint32_t share = kept * 0x10001u;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            uint32_t left;  // in assembly: the compiler makes two comparisons, two choices and a permutation of this
            asm("v_pk_sub_u16 %0, %1, %2 clamp\n\tv_pk_min_u16 %0, %0, 1 op_sel_hi:[1,0]" : "=&v"(left) : "s"(share), "v"(drawn.word[i]));
            asm("v_pk_mul_lo_u16 %0, %1, %2" : "=v"(words.v[i]) : "v"(words.v[i]), "v"(left));
        }
        return __builtin_bit_cast(Pack<T, N>, words);
    } else {
        Pack<T, N> out;
#pragma unroll
        for (int i = 0; i < N; ++i) out.v[i] = drawn.keeps(i, kept) ? p.v[i] : T(0);
        return out;
    }
}

// max(v, 0), and v where it is no number.
template <typename C>
__device__ __forceinline__ C rectified(C v) {
    if constexpr (sizeof(C) == 4) return __builtin_elementwise_maximum(v, C(0));
    return v <= 0 ? C(0) : v;
}

// Values rounded to the type of a row, two a step where the type has such a step.
template <typename T, int N, typename C>
__device__ __forceinline__ Pack<T, N> rounded(const C (&v)[N]) {
    Pack<T, N> p;
    if constexpr (sizeof(T) == 2) {
        struct Words {
            uint32_t v[N / 2];
        } words;
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
            words.v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((vec<float, 2>{v[2 * i], v[2 * i + 1]}), vec<T, 2>));
        p = __builtin_bit_cast(Pack<T, N>, words);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p.v[i] = (T)v[i];
    }
    return p;
}

// --------------------------------------------------------------------- sums of lanes ----

template <int CONTROL>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, 0xF, 0xF, true);
}

// v of the lane that the step pairs this one with, added to v.  Steps below 16 lanes go through the data-parallel moves
// of the vector ALU, those of 16 and 32 through its swaps of half rows: none through LDS.
enum { STEP_XOR1 = 0xB1, STEP_XOR2 = 0x4E, STEP_HALF_MIRROR = 0x141, STEP_MIRROR = 0x140, STEP_ROTATE = 0x120 };

template <int CONTROL>
__device__ __forceinline__ float add_moved(float v) {
    return v + __uint_as_float(moved<CONTROL>(__float_as_uint(v)));
}

template <int CONTROL>
__device__ __forceinline__ double add_moved(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint64_t other = (uint64_t)moved<CONTROL>((uint32_t)(bits >> 32)) << 32 | moved<CONTROL>((uint32_t)bits);
    return v + __builtin_bit_cast(double, other);
}

template <int LANES>  // 16 or 32
__device__ __forceinline__ uint32_t swapped(uint32_t v, uint32_t &second) {
    const auto both = LANES == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    second = both[1];
    return both[0];
}

template <int LANES>
__device__ __forceinline__ float add_swapped(float v) {
    uint32_t second;
    const uint32_t first = swapped<LANES>(__float_as_uint(v), second);
    return __uint_as_float(first) + __uint_as_float(second);
}

template <int LANES>
__device__ __forceinline__ double add_swapped(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    uint32_t low2, high2;
    const uint32_t low1 = swapped<LANES>((uint32_t)bits, low2), high1 = swapped<LANES>((uint32_t)(bits >> 32), high2);
    return __builtin_bit_cast(double, (uint64_t)high1 << 32 | low1) + __builtin_bit_cast(double, (uint64_t)high2 << 32 | low2);
}

// The sum over a lane group (LANES neighbours, a power of two up to a wave), the same bits in each of its lanes.
template <int LANES, typename A>
__device__ __forceinline__ A group_sum(A v) {
    if constexpr (LANES > 1) v = add_moved<STEP_XOR1>(v);
    if constexpr (LANES > 2) v = add_moved<STEP_XOR2>(v);
    if constexpr (LANES > 4) v = add_moved<STEP_HALF_MIRROR>(v);
    if constexpr (LANES > 8) v = add_moved<STEP_MIRROR>(v);
    if constexpr (LANES > 16) v = add_swapped<16>(v);
    if constexpr (LANES > 32) v = add_swapped<32>(v);
    return v;
}

// The sum over the lanes of a wave that have the same place in their groups of LANES.
template <int LANES, typename A>
__device__ __forceinline__ A sum_over_groups(A v) {
    if constexpr (LANES <= 32) v = add_swapped<32>(v);
    if constexpr (LANES <= 16) v = add_swapped<16>(v);
    if constexpr (LANES <= 8) v = add_moved<STEP_ROTATE + 8>(v);
    if constexpr (LANES <= 4) v = add_moved<STEP_ROTATE + 4>(v);
    if constexpr (LANES <= 2) v = add_moved<STEP_ROTATE + 2>(v);
    if constexpr (LANES <= 1) v = add_moved<STEP_ROTATE + 1>(v);
    return v;
}

// Two sums over the lanes of a row: those of a group, or of the whole workgroup (LANES == THREADS > a wave), whose waves
// leave theirs in `scratch` and add them in their order.  `scratch`: two halves of two elements a wave, of which a row takes the one that the
// row before did not: whoever writes a half has passed the barrier of the row between, and so has everyone who read it.
template <int LANES, int THREADS, typename A>
__device__ __forceinline__ void row_sums(A &first, A &second, A *scratch, bool &odd) {
    constexpr int kGroup = LANES < kWave ? LANES : kWave;
    first = group_sum<kGroup>(first);
    second = group_sum<kGroup>(second);
    if constexpr (LANES > kWave) {
        static_assert(LANES == THREADS, "a row is a lane group's or the whole workgroup's");
        A *half = scratch + (odd ? THREADS / kWave * 2 : 0);
        odd = !odd;
        if (threadIdx.x % kWave == 0) {
            half[threadIdx.x / kWave * 2] = first;
            half[threadIdx.x / kWave * 2 + 1] = second;
        }
        __syncthreads();
        first = half[0];
        second = half[1];
#pragma unroll
        for (int w = 1; w < THREADS / kWave; ++w) {
            first += half[2 * w];
            second += half[2 * w + 1];
        }
    }
}

// ------------------------------------------------------------------------ layer norm ----

// 1 / sqrt(a): the hardware's estimate of half the bits, and two steps of Newton's method for 1 / r^2 = a.
__device__ __forceinline__ double reciprocal_root(double a) {
    double r = __builtin_amdgcn_rsq(a);
#pragma unroll
    for (int step = 0; step < 2; ++step) r = __builtin_fma(0.5 * r, __builtin_fma(-a * r, r, 1.0), r);
    return a < __builtin_inf() ? r : a - a;  // of an infinite one 0 in mathematics; no row with finite differences has it
}

// Mean and variance of a row from sums over its differences to one of its own elements: that element is at most sqrt(F)
// deviations from the mean, so what the last step takes away leaves at least 1 / F of the squares.
// One reading of the row does, and nothing is lost on an offset, however large: of the 53 bits log2 F at most, which leaves float and 16-bit
// rows more than theirs.  Rows of 64 bits have none to spare: they take the same sums again about the mean found so, where nothing cancels
// (a first element 10^6 deviations off among 8,192: the variance 3e-12 off with one round, a few 2^-53 with two).
struct Moments {
    double mean, variance;
};
__device__ __forceinline__ Moments moments(double pivot, double sum, double squares, double inverse_F) {
    const double shift = sum * inverse_F, variance = __builtin_fma(-shift, shift, squares * inverse_F);
    return {pivot + shift, variance < 0 ? 0 : variance};
}

// A parameter of the rows' type or of float (`wide`); 1 or 0 where there is none.
template <typename T>
struct Params {
    const void *data;
    bool wide;
    // Columns j ... j + N - 1; zeros behind F.
    template <int N>
    __device__ __forceinline__ void read(int64_t j, int64_t F, compute_t<T> otherwise, compute_t<T> (&v)[N]) const {
        if (data == nullptr || j >= F) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = otherwise;
        } else if (wide) {
            const auto p = load_within<float, N>(static_cast<const float *>(data), j, F);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = (compute_t<T>)p.v[i];
        } else {
            const auto p = load_within<T, N>(static_cast<const T *>(data), j, F);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = (compute_t<T>)p.v[i];
        }
        if (j + N > F)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (j + i >= F) v[i] = compute_t<T>(0);
    }
};

__device__ __forceinline__ float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }

// The rows of a lane group: every step-th one from its workgroup's first on, which lies `first` behind that of the workgroup before,
// `rounds` of them at most.
struct RowWalk {
    int64_t first, step, rounds;
};

template <typename T>
struct NormArgs {
    const T *x;
    int64_t ldx;
    Params<T> weight, bias;
    double eps;
    int relu;
    Drop drop;
    RowWalk walk;
    bool streamed;  // how the rows of the result are stored
    T *out;         // forward
    double *stats;  // [rows, 2]: mean and reciprocal deviation (written forward where wanted, read backward)
    const T *grad;  // backward
    int64_t ldg;
    T *dx;           // or NULL
    compute_t<T> *partial;  // [parts, 2, F]: sums of g * h and of g over a part of the rows
    void *dweight, *dbias;  // where there is one part, which has no need of partial; parameters' type
    int64_t rows, F;
    double inverse_F;
};

// Mean and reciprocal deviation of a row as its elements meet them.  In float the mean is two numbers, the nearest float and what is left
// of it, so that a difference to it has one rounding and no offset costs bits.
template <typename C>
struct Centre {
    double mean, rstd;
    C near, scale, rest;
    __device__ __forceinline__ Centre(double m, double r) : mean(m), rstd(r), near((C)m), scale((C)r), rest(-(C)(m - (double)near) * scale) {}
    __device__ __forceinline__ C of(C x) const { return fused(x - near, scale, rest); }
};

// h = (x - m) r and v = h w + b of a pack.  Forward pass and gradient call this with the same numbers, and with RELU the
// side of zero that v is on is that of its value in 64 bits: h takes three roundings and v one more, so v is less than
// 2^-22 (|b| + |v|) off and its sign is certain where |v| > 2^-21 |b|; packs that come closer are computed again: one of
// 100,000 of those that the row fills, and in every row those that reach behind its end, where weight, bias and so v are zero (257
// features in places for 384: the third pack of each lane).  A float decision alone would let a sum over a million elements be a whole
// gradient off now and then.
template <bool RELU, int N, typename T, typename C>
__device__ __forceinline__ void normalised(const Pack<T, N> &x, const Centre<C> &centre, const C (&w)[N], const C (&b)[N], C (&h)[N], C (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        h[i] = centre.of((C)x.v[i]);
        v[i] = fused(h[i], w[i], b[i]);
    }
    if constexpr (RELU && sizeof(C) == 4) {
        float nearest = __builtin_fabsf(v[0]), largest = __builtin_fabsf(b[0]);
#pragma unroll
        for (int i = 1; i < N; ++i) {
            nearest = __builtin_fminf(nearest, __builtin_fabsf(v[i]));
            largest = __builtin_fmaxf(largest, __builtin_fabsf(b[i]));
        }
        if (nearest <= largest * 0x1p-21f) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float weight = w[i], bias = b[i];
                asm volatile("" : "+v"(weight), "+v"(bias));  // widened here: not ahead of the rows, in registers of its own
                const double exact = __builtin_fma(((double)x.v[i] - centre.mean) * centre.rstd, (double)weight, (double)bias);
                if (__builtin_fabsf(v[i]) <= largest * 0x1p-21f) v[i] = (C)exact;
            }
        }
    }
}

// How a row is spread: packs of 16 bytes over `lanes` lanes, `packs` on each; a workgroup has `threads`.  0 lanes: too long for
// registers.  The fewest places for the row's packs among powers of two with two or three packs a lane: several packs share the
// additions across the lanes and what is computed once a row, and leave loads enough in flight for a few waves a SIMD.
// Rows of 193 to 320 packs are one wave's, four or five packs a lane, in the forward pass (2,048 bfloat16 features, 43,945 rows: 75
// against 80 us with a pack a lane of four waves; 1,200 float32 features, 40,000 rows: 76 against 87 with two; beyond, 2,048 of
// float32, 4,096 rows, 19 against 14), then up to 384 packs two waves' (2,800 bfloat16 features, 40,000 rows, 90 against 99 us); in the gradient, whose sums take registers too, four waves' with a pack a lane (124
// against 144).  Of a 16-bit row a pack has eight columns, and the lanes of
// 512 have registers for two packs in the gradient, not four.
struct RowShape {
    int lanes, packs, threads;
};

// The same where the chip has lanes enough for about all packs at once, forward: there the time is that of one row's chain of loads
// and additions, and a pack a lane makes it shortest (257 bfloat16 features: one row 3.0 against 5.5 us, 8,192 rows 8.3 against 9.6;
// 1,000: one row 3.0 against 4.2, 4,096 rows 9.9 against 12.6).  16-bit rows of more than 256 packs, whose columns cost most, take it for
// more rows: under float32 parameters for four times as many (4,096 features: 2,048
// rows 15.6 against 20.4 us, 4,096 rows 21.1 against 23.8; 2,400: 4,096 rows 19.1 against 24.2; at 8,192 rows of 4,096 it loses, 35 against 33);
// under their own for three and a half times (4,096 features: 2,048 rows 12.8 against 14.2, 3,500 rows 16.6 against 17.0; 2,400: 3,500 rows 15.5
// against 17.2; at 4,096 rows it loses, among others 19.5 against 19.0, alone 22.0 against 19.9, where ReLU and dropout are behind it 24.2 and
// 24.8, from memory alone 22.4 and 23.7; 6,000 rows 23.4 against 22.4).
constexpr int64_t kAtOnce = 1 << 19;

inline RowShape spread_shape(int64_t packs) {
    if (packs > 512) return {0, 0, 0};
    return {pow2_ceil(packs), 1, std::max(pow2_ceil(packs), packs > kWave ? 128 : kBlock)};
}

inline RowShape row_shape(int64_t rows, int64_t F, size_t element, bool gradient, bool wide = false) {
    const int64_t packs = ceil_div(F, 16 / (int64_t)element);
    const RowShape spread = spread_shape(packs);
    const int64_t at_once = element == 2 && packs > 256 ? (wide ? 8 : 7) * kAtOnce / 2 : kAtOnce;
    if (!gradient && spread.lanes && rows * spread.lanes <= at_once) return spread;
    if (packs > (gradient && element == 2 ? 1024 : 2048)) return {0, 0, 0};
    if (packs <= 3) return {1, (int)packs, kBlock};
    if (packs <= 192) {
        const int lanes = pow2_ceil(ceil_div(packs, 2));  // with two packs each; or half of them with three
        if (lanes > kWave || packs <= 3 * (lanes / 2)) return {lanes / 2, 3, kBlock};
        return {lanes, 2, kBlock};
    }
    if (packs <= 320 && !gradient) return {64, packs <= 256 ? 4 : 5, 256};
    if (packs <= 384 && !gradient) return {128, 3, 128};
    if (packs <= 256) return {256, 1, 256};
    if (packs <= 768) return {256, packs <= 512 ? 2 : 3, 256};
    return {512, packs <= 1024 ? 2 : packs <= 1536 ? 3 : 4, 512};
}

// Which rows the lane groups take: neighbours within a workgroup, and workgroup by workgroup, over and over, until all are
// taken, so that the whole chip reads one stretch of memory at a time.  No more workgroups than are resident: a lane has its parameters in registers
// and, in the gradient, its sums.
inline int64_t row_workgroups(int64_t rows, const RowShape &s, size_t element, bool gradient) {
    // waves a SIMD by the registers that a lane takes for its packs
    const int64_t waves = s.packs == 1 ? 4 : s.packs > 2 ? 2 : !gradient ? 4 : s.lanes > kWave && element == 2 ? 2 : 3;
    return std::min(ceil_div(rows, s.threads / s.lanes), 256 * 256 * waves / s.threads);
}

// Whether rows of a result are stored past the caches: where a pass moves more than the 256 MB of the last one hold, and the stores fill its
// lines of 128 bytes (325,557 rows of 256 float16 features, forward: 56 us and 69 without; of 257, which fill none, 2,449,029 x 100
// float32: 412 and 401; below that size there is nothing to gain, 325,557 x 64 float32: 27 and 27, and the reader behind to lose).
inline bool streams(int64_t rows, int64_t row_bytes, int64_t store_bytes, int matrices) {
    return rows * row_bytes * matrices > ((int64_t)256 << 20) && row_bytes % 128 == 0 && store_bytes >= 128;
}

// The kernels of longer rows: a workgroup of the largest size a row, some loads of each lane in flight.
constexpr int kLongThreads = 1024, kLongPacks = 3;

template <int LANES, int PACKS, int THREADS>
struct ShapeTag {
    static constexpr int lanes = LANES, packs = PACKS, threads = THREADS;
};

// Calls `run` with the tag of a shape of at least one lane.
template <typename T, bool GRADIENT, typename F>
int with_row_shape(const RowShape &s, F &&run) {
    switch (s.lanes) {
        case 1: return s.packs == 1 ? run(ShapeTag<1, 1, 256>()) : s.packs == 2 ? run(ShapeTag<1, 2, 256>()) : run(ShapeTag<1, 3, 256>());
        case 2:
            if constexpr (!GRADIENT)
                if (s.packs == 1) return run(ShapeTag<2, 1, 256>());
            return s.packs == 2 ? run(ShapeTag<2, 2, 256>()) : run(ShapeTag<2, 3, 256>());
        case 4:
            if constexpr (!GRADIENT)
                if (s.packs == 1) return run(ShapeTag<4, 1, 256>());
            return s.packs == 2 ? run(ShapeTag<4, 2, 256>()) : run(ShapeTag<4, 3, 256>());
        case 8:
            if constexpr (!GRADIENT)
                if (s.packs == 1) return run(ShapeTag<8, 1, 256>());
            return s.packs == 2 ? run(ShapeTag<8, 2, 256>()) : run(ShapeTag<8, 3, 256>());
        case 16:
            if constexpr (!GRADIENT)
                if (s.packs == 1) return run(ShapeTag<16, 1, 256>());
            return s.packs == 2 ? run(ShapeTag<16, 2, 256>()) : run(ShapeTag<16, 3, 256>());
        case 32:
            if constexpr (!GRADIENT)
                if (s.packs == 1) return run(ShapeTag<32, 1, 256>());
            return s.packs == 2 ? run(ShapeTag<32, 2, 256>()) : run(ShapeTag<32, 3, 256>());
        case 64:
            if constexpr (!GRADIENT)
                if (s.packs == 1) return run(ShapeTag<64, 1, 256>());
            if constexpr (!GRADIENT)
                if (s.packs > 3) return s.packs == 4 ? run(ShapeTag<64, 4, 256>()) : run(ShapeTag<64, 5, 256>());
            return s.packs == 2 ? run(ShapeTag<64, 2, 256>()) : run(ShapeTag<64, 3, 256>());
        case 256:
            if (s.packs == 1) return run(ShapeTag<256, 1, 256>());
            return s.packs == 2 ? run(ShapeTag<256, 2, 256>()) : run(ShapeTag<256, 3, 256>());
        default:  // 512, and 128 in the forward pass
            if constexpr (!GRADIENT) {
                if (s.lanes == 128) return s.packs == 1 ? run(ShapeTag<128, 1, 128>()) : run(ShapeTag<128, 3, 128>());
                if (s.packs == 1) return run(ShapeTag<512, 1, 512>());
            }
            if constexpr (!GRADIENT || sizeof(T) > 2)
                if (s.packs > 2) return s.packs == 3 ? run(ShapeTag<512, 3, 512>()) : run(ShapeTag<512, 4, 512>());
            return run(ShapeTag<512, 2, 512>());
    }
}

}  // namespace cgnn

// paged_wave.hpp -- attention of one wave: query rows that share a kv head against cached positions, with the running
// maximum and sum of the softmax. First 32 rows at a time, then 16.
//
// A row is a query head of a token. The wave forms S^T = K Q^T and O^T += V^T P^T with 32x32 matrix instructions, so
// that a lane holds values of one row (lane & 31) throughout: the maximum and the sum are the lane's own but for one
// exchange with its other half (lane ^ 32), and P^T leaves the softmax in the registers that the second product reads as
// its right operand. That operand wants a run of RUN positions per half; the rows of K are read in the order that
// makes the first product leave them so (kv_row). Both left operands are 16-byte runs of memory: K pages hold a
// position's dimensions together, V pages a dimension's positions.
//
// Exponentials are powers of two: x = s * (scale * log2 e) - m. Scores, maxima, sums and O are f32. P is rounded to the
// cache's type for the second product (half a step relative, of the size of V's own rounding; below f16's normal range,
// half its smallest step); the sum l adds the unrounded values. Positions of equal scores round alike, so that what this
// takes from O does not shrink with their number: half a step (bf16 2^-8, f16 2^-11) of sum p |v| bounds it, and an f32
// result of a 16-bit cache has it too.
#pragma once

#include "paged_util.hpp"

namespace llamd {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t run4 __attribute__((ext_vector_type(4)));  // a 16-byte run of elements

template <class E> struct Mma;
template <> struct Mma<ElemF16> {
    typedef _Float16 V __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ v16f mul(run4 a, run4 b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
    static constexpr uint32_t EXP = 0x7C007C00u;
};
template <> struct Mma<ElemBF16> {
    typedef __bf16 V __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ v16f mul(run4 a, run4 b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
    }
    static constexpr uint32_t EXP = 0x7F807F80u;
};
template <> struct Mma<ElemF32> {
    static __device__ __forceinline__ v16f mul(run4 a, run4 b, v16f c) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    }
    static constexpr uint32_t EXP = 0x7F800000u;
};

constexpr float NEG_INF = -INFINITY;

// Four values at an element of `out`, rounded to the type, or f32.
template <class E> __device__ __forceinline__ void put4(void *out, size_t at, float4 x) {
    typedef typename E::T V __attribute__((ext_vector_type(4)));
    const V v = {E::put(x.x), E::put(x.y), E::put(x.z), E::put(x.w)};
    *(V *)((typename E::T *)out + at) = v;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// The maximum (sum) of a lane's value and that of its other half.
struct Halves {
    float lo, hi;
};
__device__ __forceinline__ Halves halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}
__device__ __forceinline__ float max_halves(float x) {
    const Halves v = halves(x);
    return fmaxf(v.lo, v.hi);
}
__device__ __forceinline__ float add_halves(float x) {
    const Halves v = halves(x);
    return v.lo + v.hi;
}

// The maximum that x is taken against: an empty row's is 0, so that its terms are exp2(-inf) = 0 and not NaN.
__device__ __forceinline__ float against(float m) { return m == NEG_INF ? 0.0f : m; }

// Position (0..31) that row m of the first product's left operand holds, and the one that a lane's score register i is of.
template <class E> __device__ __forceinline__ int kv_row(int m) {
    const int i = 4 * (m >> 3) + (m & 3), h = (m >> 2) & 1;
    return 2 * E::RUN * (i / E::RUN) + E::RUN * h + i % E::RUN;
}
template <class E> __device__ __forceinline__ int kv_reg(int i, int h) {
    return 2 * E::RUN * (i / E::RUN) + E::RUN * h + i % E::RUN;
}

// A run's elements whose bits are set in `keep` as they are, the others zero.
template <class E> __device__ __forceinline__ run4 keep_elements(run4 r, uint32_t keep) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (E::RUN == 4) {
            r[j] &= (keep >> j & 1) ? 0xFFFFFFFFu : 0u;
        } else {
            r[j] &= ((keep >> (2 * j) & 1) ? 0xFFFFu : 0u) | ((keep >> (2 * j + 1) & 1) ? 0xFFFF0000u : 0u);
        }
    }
    return r;
}
// Bit e: element e is an infinity or NaN.
template <class E> __device__ __forceinline__ uint32_t not_finite(run4 r) {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (E::RUN == 4) {
            bits |= (uint32_t)((r[j] & Mma<E>::EXP) == Mma<E>::EXP) << j;
        } else {
            const uint32_t lo = Mma<E>::EXP & 0xFFFFu, hi = Mma<E>::EXP & 0xFFFF0000u;
            bits |= (uint32_t)((r[j] & lo) == lo) << (2 * j) | (uint32_t)((r[j] & hi) == hi) << (2 * j + 1);
        }
    }
    return bits;
}

// Whether any element is one: its exponent's lowest bit added to an exponent of ones carries into the sign's place.
template <class E> __device__ __forceinline__ uint32_t any_not_finite(run4 r) {
    constexpr uint32_t EXP = Mma<E>::EXP, SIGN = E::RUN == 4 ? 0x80000000u : 0x80008000u;
    constexpr uint32_t ONE = E::RUN == 4 ? EXP & -EXP : (EXP & 0xFFFFu & -(EXP & 0xFFFFu)) * 0x10001u;
    return (((r[0] & EXP) + ONE) | ((r[1] & EXP) + ONE) | ((r[2] & EXP) + ONE) | ((r[3] & EXP) + ONE)) & SIGN;
}

template <class E> __device__ __forceinline__ run4 to_run(const float *x) {
    run4 r;
    if constexpr (E::RUN == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = __float_as_uint(x[j]);
    } else {
        typedef typename E::T V __attribute__((ext_vector_type(8)));
        V v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = E::put(x[j]);
        r = __builtin_bit_cast(run4, v);
    }
    return r;
}

// Scores this much above the running maximum (as powers of two) are taken against it without a new one: weights stay below
// 2^LAZY, and O is rescaled only where a row's maximum climbs further, which after the first few tiles it hardly does.
constexpr float LAZY = 8.0f;

// 32 rows' running softmax and O, over tiles of 32 * SUB positions.
template <class E, int HD> struct RowState {
    static constexpr int DB = HD / 32;             // blocks of 32 dimensions
    static constexpr int QS = HD / (2 * E::RUN);   // steps of the first product
    static constexpr int PS = 32 / (2 * E::RUN);   // steps of the second, per 32 positions
    v16f o[DB];
    float m, l;  // what x is taken against, and this half's part of the sum

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
        m = NEG_INF;
        l = 0.0f;
    }

    // The running maximum brought up to date with scores, and O and l with it.
    template <int SUB> __device__ __forceinline__ void raise(const v16f (&s)[SUB], float scale) {
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < SUB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
        top = max_halves(top) * scale;
        if (__any(top > m + LAZY)) {
            const float m1 = fmaxf(m, top), shrink = exp2_fast(m - against(m1));
            m = m1;
            l *= shrink;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= shrink;
        }
    }

    // Scores (kv_reg's order) to weights, which add to l.
    template <int SUB> __device__ __forceinline__ void weigh(v16f (&s)[SUB], float scale) {
        const float ref = against(m);
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < SUB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[b][i] = exp2_fast(__builtin_fmaf(s[b][i], scale, -ref));
                sum += s[b][i];
            }
        l += sum;
    }

    template <int SUB> __device__ __forceinline__ void softmax(v16f (&s)[SUB], float scale) {
        raise<SUB>(s, scale);
        weigh<SUB>(s, scale);
    }

    // The right operand of step c of the second product.
    static __device__ __forceinline__ run4 weights(const v16f &s, int c) {
        float x[E::RUN];
#pragma unroll
        for (int j = 0; j < E::RUN; ++j) x[j] = s[c * E::RUN + j];
        return to_run<E>(x);
    }
};

// ---- 16 rows ----------------------------------------------------------------------
// The same for up to 16 rows and 32 positions with 16x16 matrix instructions, whose four groups of 16 lanes hold a run each:
// a row's values lie in four lanes, and half the registers and columns are left unused.

typedef float v4f __attribute__((ext_vector_type(4)));

template <class E> __device__ __forceinline__ v4f mul16(run4 a, run4 b, v4f c);
template <> __device__ __forceinline__ v4f mul16<ElemF16>(run4 a, run4 b, v4f c) {
    typedef Mma<ElemF16>::V V;
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ v4f mul16<ElemBF16>(run4 a, run4 b, v4f c) {
    typedef Mma<ElemBF16>::V V;
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ v4f mul16<ElemF32>(run4 a, run4 b, v4f c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
}

// The maximum (sum) over the four groups.
__device__ __forceinline__ float max_groups(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float add_groups(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return add_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Position (0..31) of row m of block b of the first product's left operand, and of a lane's score register (b, i).
template <class E> __device__ __forceinline__ int few_row(int b, int m) {
    return E::RUN == 8 ? 8 * (m >> 2) + 4 * b + (m & 3) : 16 * b + m;
}
template <class E> __device__ __forceinline__ int few_reg(int b, int i, int g) {
    return E::RUN == 8 ? 8 * g + 4 * b + i : 16 * b + 4 * g + i;
}

template <class E, int HD> struct FewState {
    static constexpr int DB = HD / 16;            // blocks of 16 dimensions
    static constexpr int QS = HD / (4 * E::RUN);  // steps of the first product
    static constexpr int PS = 32 / (4 * E::RUN);  // steps of the second
    v4f o[DB];   // dimension 16 d + 4 group + i
    float m, l;  // what x is taken against, and this lane's part of the sum

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        m = NEG_INF;
        l = 0.0f;
    }

    __device__ __forceinline__ void softmax(v4f (&s)[2], float scale) {
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[b][i]);
        top = max_groups(top) * scale;
        if (__any(top > m + LAZY)) {
            const float m1 = fmaxf(m, top), shrink = exp2_fast(m - against(m1));
            m = m1;
            l *= shrink;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= shrink;
        }
        const float ref = against(m);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[b][i] = exp2_fast(__builtin_fmaf(s[b][i], scale, -ref));
                l += s[b][i];
            }
    }

    static __device__ __forceinline__ run4 weights(const v4f (&s)[2], int c) {
        float x[E::RUN];
#pragma unroll
        for (int j = 0; j < E::RUN; ++j) x[j] = E::RUN == 8 ? s[j / 4][j % 4] : s[c][j % 4];
        return to_run<E>(x);
    }

    // One step of the second product where some of V is not to be read as it stands: of the runs v(d, 0) of the dimension
    // blocks, the elements of `keep` can be read, the others may hold anything. An infinity or NaN at a position that
    // only some rows attend to gives the others nothing, not 0 * inf: such elements are left out of the product and
    // added one position at a time (pos0 + e) to the rows that see it.
    template <class Load>
    __device__ __forceinline__ void add_masked(Load v, uint32_t keep, run4 p, int pos0, int limit) {
        const int g = (threadIdx.x >> 4) & 3;
        uint32_t any = 0;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const run4 x = keep_elements<E>(v(d, 0u), keep);
            const uint32_t bad = not_finite<E>(x);
            any |= bad;
            asm volatile("" : "+v"(any));  // (added up here, not kept bit by bit to the end)
            o[d] = mul16<E>(keep_elements<E>(x, ~bad), p, o[d]);
            __builtin_amdgcn_sched_barrier(0);  // one d's masks at a time: registers
        }
        if (!__any(any != 0)) return;
#pragma unroll 1
        for (int e = 0; e < 4 * E::RUN; ++e) {
            const uint32_t one = (e / E::RUN == g) ? 1u << (e % E::RUN) : 0u;
            if (!__any((any & one) != 0)) continue;
            const bool seen = pos0 + e < limit;
            uint32_t none = 0;
            asm volatile("" : "+v"(none));  // the runs are read again: held in registers throughout, they would crowd out others
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const run4 x = keep_elements<E>(v(d, none), keep & one);
                const v4f t = mul16<E>(keep_elements<E>(x, not_finite<E>(x)), keep_elements<E>(p, one), o[d]);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][i] = seen ? t[i] : o[d][i];
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
};

}  // namespace llamd

// paged_util.hpp -- device helpers that the paged-cache kernels share: element types, where a token or a row of a packed
// batch belongs, and a position's page.
#pragma once

#include "common.hpp"
#include "paged.hpp"

namespace llamd {

// An element type of the pages (P): the type T of the products on them, of q and of results, elements of T in 16 bytes,
// and the rounding from f32 (to nearest, ties to even: half a unit in the last place, the one rounding of a stored value).
struct ElemF32 {
    typedef float T, P;
    static constexpr int RUN = 4;
    static __device__ __forceinline__ float put(float x) { return x; }
};
struct ElemF16 {
    typedef _Float16 T, P;
    static constexpr int RUN = 8;
    static __device__ __forceinline__ _Float16 put(float x) { return (_Float16)x; }
};
struct ElemBF16 {
    typedef __bf16 T, P;
    static constexpr int RUN = 8;
    static __device__ __forceinline__ __bf16 put(float x) { return (__bf16)x; }
};
// e4m3 numbers times a power of two for each 16 positions, which bf16 holds exactly (three bits after the point, f32's
// exponents): products are those of a bf16 cache.
struct ElemE4M3 : ElemBF16 {
    typedef uint8_t P;
};
template <class E> constexpr bool bytes_of = sizeof(typename E::P) == 1;

typedef uint32_t run4 __attribute__((ext_vector_type(4)));  // a 16-byte run of elements
typedef uint32_t run2 __attribute__((ext_vector_type(2)));  // 8 e4m3 elements

// A scale byte as the power of two that it stands for (0 is taken as 1).
__device__ __forceinline__ float unit_of(uint32_t e) { return __uint_as_float(max(e, 1u) << 23); }

// 8 e4m3 elements times a power of two (its exponent alone is looked at), exactly.
__device__ __forceinline__ run4 widen(uint32_t lo, uint32_t hi, float unit) {
    return run4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, unit, false)),
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, unit, true)),
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, unit, false)),
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, unit, true))};
}

// The page of a position (inside the table) of a table row, -1 if the id is none of the cache's.
__device__ __forceinline__ int page_of(const PagedArgs &p, const int32_t *row, int pos) {
    const int id = row[pos >> p.page_log];
    return (unsigned)id < (unsigned)p.n_page ? id : -1;
}

// Which sequence the unit (a token, or a tile of rows) number `unit` belongs to, when sequence s has units(s) of them:
// the whole wave looks at 64 sequences at a time. `unit` becomes its number within the sequence; -1: past the last.
template <class Units>
__device__ __forceinline__ int find_sequence(int n_seq, int &unit, Units units) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < n_seq; s0 += WAVE) {
        const int mine = s0 + lane < n_seq ? units(s0 + lane) : 0;
        const int sum = wave_incl_sum_i(mine);
        const unsigned long long past = __ballot(sum > unit);
        if (past) {
            const int l = __builtin_ctzll(past);
            unit -= __builtin_amdgcn_readlane(sum - mine, l);
            return s0 + l;
        }
        unit -= __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}

}  // namespace llamd

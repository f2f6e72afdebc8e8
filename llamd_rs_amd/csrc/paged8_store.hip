// paged8_store.hip -- new tokens' queries, keys and values into an 8-bit cache: norm and rotation as in paged_store.hip, then
// keys and values as e4m3 numbers times one power of two for each 16 positions of a kv head.
//
//   E = the least number (1 at least) with max |y| <= 448 * 2^(E - 127) over the block's new finite values, and at least the
//       block's E where it has positions before them
//   stored: e4m3(y * 2^(127 - E)), to nearest, ties to even: half a step, 2^-4 of a value, or 2^-10 of the unit
//
// Positions before the new ones stand where the block's E grows: their numbers are multiplied by 2^(old E - E), which is exact
// down to e4m3's normal numbers, 2^-6 units: 2^-14 of the 448 units that fit. A block that fills token by token is as exact as one
// stored at once, but below them, where the roundings add up to 2^-9 units at the most (2^-10 of the last, half as much of the one
// before, and so on). E does not shrink while the block has positions before the new ones. Infinities and NaN are stored as NaN,
// and do not count for the unit.
//
// Bound: memory, 4 (H + 2 Hkv) hd bytes read, 2 H hd + 2 Hkv hd written per token, and for a few tokens the chain of loads
// from the length to the block's scale. One launch: queries as in paged_store.hip, a wave per token; and a workgroup per 16
// positions, kv head, and K or V, since the unit is the largest of them all: HD / 8 lanes hold a token's head, the 16 tokens'
// values stay in registers between the maximum and the rounding. V's bytes are turned in LDS.
//
// Measured (one MI355X): 8000 tokens of 32 query and 4 kv heads of 128, 238 MB, 52.1 us (4.6 TB/s, a large copy's rate is 4.7); 5
// prompts of 16 and 8 heads, 52 MB, 14.1 us; one token 7.1 us, of which the kernel 5.2 (of a 16-bit cache
// 4.0). The values' loads beside the page's number, and V's old bytes before the norm: 7.3, 14.6 and 53.2. With n_rot % 8 != 0
// (pairs of single dimensions, bytes stored one by one) one token 7.6, 700 tokens 9.5 (runs 7.7), 8000 58 to 63 where the same
// call in runs takes 40 (rows already in the caches).
#include <algorithm>

#include "paged_store.hpp"

namespace llamd {
namespace {

// The scale byte for values whose largest has these bits (sign cleared, finite).
__device__ __forceinline__ uint32_t scale_of(uint32_t top) {
    return (uint32_t)max((int)(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u), 1);
}

// Four values as e4m3 (NaN for what is not finite).
__device__ __forceinline__ uint32_t narrow(f4 x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = __builtin_fabsf(x[j]) < INFINITY ? x[j] : __builtin_nanf("");
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
}

// Four e4m3 numbers times `by`, rounded again.
__device__ __forceinline__ uint32_t express(uint32_t w, float by) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return narrow(f4{a[0] * by, a[1] * by, b[0] * by, b[1] * by});
}

// Unit number `unit`: a block of 16 positions, a kv head, and K or V. RUNS: n_rot % 8 == 0, a lane's pairs are runs of four
// dimensions.
template <int HD, bool RUNS>
__device__ __forceinline__ void store_block(const PagedStoreArgs &a, int unit) {
    constexpr int LANES = HD / 8, ROWS = 256 / LANES, PASSES = (POS + ROWS - 1) / ROWS;
    __shared__ __align__(16) uint8_t turned_bytes[HD * POS];
    __shared__ uint32_t tops[4];
    const PagedArgs &p = a.p;
    const bool values = unit & 1;
    unit >>= 1;
    const int kvh = unit % p.n_kv_head;
    Block at;
    if (!block_of(p, unit / p.n_kv_head, at)) return;
    uint8_t *scale = (values ? p.v_scale : p.k_scale) + (((size_t)at.page * p.n_kv_head + kvh) << (p.page_log - SCALE_LOG)) +
                     ((at.pos0 & ((1 << p.page_log) - 1)) >> SCALE_LOG);
    const uint32_t old = at.lo ? min(max((uint32_t)*scale, 1u), 254u) : 1u;
    const int lane = threadIdx.x % LANES, row = threadIdx.x / LANES;
    // this lane's dimensions: four pairs (d[j], e[j])
    const int half = a.n_rot / 2;
    const bool apart = !values && !a.interleaved;
    int d[4], e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int pair = 4 * lane + j;
        d[j] = apart && pair < half ? pair : 2 * pair;
        e[j] = apart && pair < half ? pair + half : 2 * pair + 1;
    }
    // (as runs: four dimensions from u0, four from v0)
    const int u0 = apart && 4 * lane < half ? 4 * lane : 8 * lane, v0 = apart && 4 * lane < half ? 4 * lane + half : 8 * lane + 4;
    const float *x = a.x[values ? 2 : 1] + (size_t)kvh * HD;
    const int ld = a.ld[values ? 2 : 1];
    const float *w = values ? nullptr : a.norm[1];
    f4 y[PASSES][2];  // RUNS: dimensions u0 .. and v0 .., else d and e
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * ROWS + row, pos = at.pos0 + r;
        y[i][0] = y[i][1] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (r < at.lo || r >= at.hi) continue;
        const float *from = x + (size_t)(at.first + (pos - at.before)) * ld;
        f4 u, v;
        if constexpr (RUNS) {
            u = *(const f4 *)(from + u0);
            v = *(const f4 *)(from + v0);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = from[d[j]], v[j] = from[e[j]];
        }
        if (w) {
            const f4 q = u * u + v * v;
            const float by = 1.0f / __builtin_sqrtf(head_sum<LANES>((q[0] + q[1]) + (q[2] + q[3])) * (1.0f / HD) + a.eps);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u[j] = u[j] * w[RUNS ? u0 + j : d[j]] * by;
                v[j] = v[j] * w[RUNS ? v0 + j : e[j]] * by;
            }
        }
        if (!values) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int pair = 4 * lane + j;
                if (pair >= half) continue;
                float c, s;
                turn(a, pos, pair, c, s);
                // (interleaved runs hold their pairs side by side)
                if (RUNS && a.interleaved) {
                    f4 &z = j < 2 ? u : v;
                    const float f = z[j % 2 * 2], g = z[j % 2 * 2 + 1];
                    z[j % 2 * 2] = f * c - g * s;
                    z[j % 2 * 2 + 1] = f * s + g * c;
                } else {
                    const float f = u[j], g = v[j];
                    u[j] = f * c - g * s;
                    v[j] = f * s + g * c;
                }
            }
        }
        y[i][0] = u;
        y[i][1] = v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t f = __float_as_uint(u[j]) & 0x7FFFFFFFu, g = __float_as_uint(v[j]) & 0x7FFFFFFFu;
            top = max(top, f < 0x7F800000u ? f : 0u);
            top = max(top, g < 0x7F800000u ? g : 0u);
        }
    }
    top = (uint32_t)wave_reduce((int)top, 0, [](int m, int n) { return max(m, n); });
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
    const uint32_t unit_byte = max(scale_of(top), old);
    const float by = __uint_as_float(unit_byte < 254u ? (254u - unit_byte) << 23 : 0x00400000u);  // 2^(127 - E)
    const uint32_t grown = unit_byte - old;
    const float shrink = grown < 127u ? __uint_as_float((127u - grown) << 23) : 0.0f;
    if (threadIdx.x == 0) *scale = (uint8_t)unit_byte;
    const int slot = at.pos0 & ((1 << p.page_log) - 1);
    const size_t head = (size_t)at.page * p.n_kv_head + kvh;
    if (!values) {
        uint8_t *k = (uint8_t *)p.k + ((head << p.page_log) + slot) * HD;
        if (grown && at.lo) {
            for (int i = threadIdx.x * 4; i < at.lo * HD; i += 256 * 4) *(uint32_t *)(k + i) = express(*(uint32_t *)(k + i), shrink);
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = i * ROWS + row;
            if (r < at.lo || r >= at.hi) continue;
            const uint32_t f = narrow(y[i][0] * by), g = narrow(y[i][1] * by);
            if constexpr (RUNS) {
                *(uint32_t *)(k + r * HD + u0) = f;
                *(uint32_t *)(k + r * HD + v0) = g;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    k[r * HD + d[j]] = (uint8_t)(f >> (8 * j));
                    k[r * HD + e[j]] = (uint8_t)(g >> (8 * j));
                }
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * ROWS + row;
        if (r >= POS) continue;
        const uint32_t f = narrow(y[i][0] * by), g = narrow(y[i][1] * by);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            turned_bytes[(RUNS ? u0 + j : d[j]) * POS + r] = (uint8_t)(f >> (8 * j));
            turned_bytes[(RUNS ? v0 + j : e[j]) * POS + r] = (uint8_t)(g >> (8 * j));
        }
    }
    __syncthreads();
    uint8_t *v = (uint8_t *)p.v + (head * HD << p.page_log) + slot;
    for (int i = threadIdx.x; i < HD; i += 256) {
        run4 now = *(const run4 *)(turned_bytes + i * POS);
        run4 *to = (run4 *)(v + ((size_t)i << p.page_log));
        if (at.lo || at.hi < POS) {
            const run4 was = *to;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // bytes [lo, hi) of the 16 are new
                const int from = min(max(at.lo - 4 * j, 0), 4), end = min(max(at.hi - 4 * j, 0), 4);
                const uint32_t below = from == 4 ? ~0u : (1u << (8 * from)) - 1u, upto = end == 4 ? ~0u : (1u << (8 * end)) - 1u;
                const uint32_t kept = grown ? express(was[j], shrink) : was[j];
                now[j] = (kept & below) | (now[j] & upto & ~below) | (was[j] & ~upto);
            }
        }
        *to = now;
    }
}

// The first `tokens` workgroups: queries, WAVES waves per token (0: pairs of single dimensions); then blocks.
template <int HD, int WAVES>
__global__ __launch_bounds__(256) void paged8_store(PagedStoreArgs a, int tokens) {
    if ((int)blockIdx.x >= tokens) {
        store_block<HD, WAVES != 0>(a, blockIdx.x - tokens);
        return;
    }
    PagedStoreArgs q = a;
    q.p.n_kv_head = 0;  // queries alone
    if constexpr (WAVES) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), token = (blockIdx.x * 4 + wave) / WAVES;
        if (token < a.p.n_tok) store_token<ElemBF16, HD, WAVES>(q, token, wave % WAVES);
    } else {
        store_token_pairs<ElemBF16, HD>(q, blockIdx.x);
    }
}

template <int HD>
int store_as(const PagedStoreArgs &a, hipStream_t st) {
    const PagedArgs &p = a.p;
    // 16-position blocks of all sequences: a whole one per 16 tokens, and two that are not
    const long long blocks = std::min((long long)p.n_tok / POS + 2LL * p.n_seq, (long long)p.n_tok);
    // four waves per token while one's chain of heads takes longer than the tokens take the GPU (one and four, 4 kv heads of 128: 32
    // heads, 500 tokens 7.3 and 7.2 us, 700 7.7 and 9.0, 1900 12.9 and 16.0; 128 heads, 1 token 13.7 and 7.3, 500 16.3 and 11.0,
    // 2000 44.2 and 42.6; the wrong way at 64 heads, 1000 tokens, 12.4 and 13.5, and at 128, 2900, 63.8 and 58.8)
    const int waves = a.n_rot % 8 ? 0 : p.n_tok < p.n_head * HD / 8 ? 4 : 1;
    const int tokens = !a.x[0] ? 0 : waves == 1 ? (p.n_tok + 3) / 4 : p.n_tok;
    const long long grid = tokens + 2 * blocks * p.n_kv_head;
    if (grid > 0x7FFFFFFF / 256) return -1;
    const dim3 g((unsigned)grid), b(256);
    if (waves == 1) hipLaunchKernelGGL((paged8_store<HD, 1>), g, b, 0, st, a, tokens);
    else if (waves) hipLaunchKernelGGL((paged8_store<HD, 4>), g, b, 0, st, a, tokens);
    else hipLaunchKernelGGL((paged8_store<HD, 0>), g, b, 0, st, a, tokens);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace

int launch_paged8_store(const PagedStoreArgs &a, hipStream_t st) {
    if (a.p.hd == 64) return store_as<64>(a, st);
    if (a.p.hd == 128) return store_as<128>(a, st);
    if (a.p.hd == 256) return store_as<256>(a, st);
    return -1;
}

}  // namespace llamd

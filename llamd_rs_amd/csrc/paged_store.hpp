// paged_store.hpp -- what the stores into a paged cache share (paged_store.hip, paged8_store.hip): where a token goes, its
// rotation, and the norm and rotation of its heads.
#pragma once

#include "paged_util.hpp"

namespace llamd {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

// Where a token is: its sequence's position and page (-1: none). False: it belongs to no sequence.
struct Place {
    int pos, page;
};
__device__ __forceinline__ bool place_of(const PagedArgs &p, int token, Place &at) {
    const int lane = threadIdx.x & 63;
    int seq = -1, end = 0, len = 0;
    if (p.start) {
        // 64 sequences at a time, the lengths with the starts: one trip to memory
        for (int s0 = 0; s0 < p.n_seq && seq < 0; s0 += WAVE) {
            const int s = min(s0 + lane, p.n_seq - 1);
            const int first = max(p.start[s], 0), e = min(p.start[s + 1], p.n_tok), n = p.len[s];
            const unsigned long long mine = __ballot(s0 + lane < p.n_seq && first <= token && token < e);
            if (mine) {
                const int l = __builtin_ctzll(mine);
                seq = s0 + l;
                end = __builtin_amdgcn_readlane(e, l);
                len = __builtin_amdgcn_readlane(n, l);
            }
        }
        if (seq < 0) return false;
    } else {
        if (token >= p.n_seq) return false;
        seq = token;
        end = token + 1;
        len = p.len[seq];
    }
    at.pos = len - (end - token);
    at.page = -1;
    if (at.pos >= 0 && at.pos >> p.page_log < p.max_page)
        at.page = page_of(p, p.table + (size_t)seq * p.max_page, at.pos);
    return true;
}

__device__ __forceinline__ void turn(const PagedStoreArgs &a, int pos, int pair, float &c, float &s) {
    const double turns = (double)pos * a.freqs[pair] * 0.15915494309189533577;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    c *= a.mscale;
    s *= a.mscale;
}

// 16 positions of a sequence that lie together in a page, some of its new tokens among them.
constexpr int POS = 16;
struct Block {
    int before, first;  // position of the sequence's first new token, and its row
    int pos0, page;     // first position, and its page
    int lo, hi;         // the new tokens' places among the 16
};
// Block number `block` of the batch's. False: it is none, or has no page.
__device__ __forceinline__ bool block_of(const PagedArgs &p, int block, Block &at) {
    const int lane = threadIdx.x & 63;
    int seq = -1, end = 0, len = 0;
    for (int s0 = 0; s0 < p.n_seq; s0 += WAVE) {
        const int s = s0 + lane;
        int units = 0, f = s, e = s + 1, n = 0;
        if (s < p.n_seq) {
            n = p.len[s];
            if (p.start) {
                f = min(max(p.start[s], 0), p.n_tok);
                e = max(min(p.start[s + 1], p.n_tok), f);
            }
            // the table's positions [n - tokens, n)
            const long long top = min((long long)n, (long long)p.max_page << p.page_log);
            const long long from = max((long long)n - (e - f), 0LL);
            units = from < top ? (int)((top - 1) / POS - from / POS + 1) : 0;
        }
        const int sum = wave_incl_sum_i(units);
        const unsigned long long past = __ballot(sum > block);
        if (past) {
            const int l = __builtin_ctzll(past);
            block -= __builtin_amdgcn_readlane(sum - units, l);
            seq = s0 + l;
            at.first = __builtin_amdgcn_readlane(f, l);
            end = __builtin_amdgcn_readlane(e, l);
            len = __builtin_amdgcn_readlane(n, l);
            break;
        }
        block -= __builtin_amdgcn_readlane(sum, 63);
    }
    if (seq < 0) return false;
    at.before = len - (end - at.first);
    at.pos0 = (max(at.before, 0) / POS + block) * POS;
    at.page = page_of(p, p.table + (size_t)seq * p.max_page, at.pos0);
    at.lo = max(at.before - at.pos0, 0);
    at.hi = min(len - at.pos0, POS);
    return at.page >= 0;
}

// ---- queries and keys ---------------------------------------------------------------

// Sum over the LANES (8, 16 or 32) lanes of a head.
template <int LANES> __device__ __forceinline__ float head_sum(float x) {
    x += dpp<DPP_XOR1>(0.0f, x);
    x += dpp<DPP_XOR2>(0.0f, x);
    x += dpp<DPP_HALF_MIRROR>(0.0f, x);
    if constexpr (LANES >= 16) x += dpp<DPP_MIRROR>(0.0f, x);
    if constexpr (LANES == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

// A lane has two runs of four dimensions of a head: with n_rot / 8 lanes for the rotated part, dimensions 4 l and
// n_rot / 2 + 4 l (or, interleaved and behind n_rot, 8 l and 8 l + 4), which holds four whole pairs either way.
// n_rot % 8 == 0. WAVES: waves that share a token's heads.
template <class E, int HD, int WAVES>
__device__ __forceinline__ void store_token(const PagedStoreArgs &a, int token, int wave) {
    typedef typename E::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int LANES = HD / 8, HEADS = WAVE / LANES, AHEAD = 3;
    const PagedArgs &p = a.p;
    const int lane = threadIdx.x & 63, l = lane % LANES;
    const bool turned = l < a.n_rot / 8, halves = turned && !a.interleaved;
    const int d0 = halves ? 4 * l : 8 * l, d1 = halves ? a.n_rot / 2 + 4 * l : 8 * l + 4;
    const int nq = a.x[0] ? p.n_head : 0, n = nq + p.n_kv_head;
    const int first = wave * HEADS + lane / LANES;
    // the heads' values do not depend on where the token goes
    const auto value = [&](int h, int d) {
        const int which = h < nq ? 0 : 1;
        return *(const f4 *)(a.x[which] + (size_t)token * a.ld[which] + (size_t)(which ? h - nq : h) * HD + d);
    };
    f4 x[AHEAD][2];
    const auto load = [&](int i, int h) { x[i][0] = value(min(h, n - 1), d0), x[i][1] = value(min(h, n - 1), d1); };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(i, first + i * HEADS * WAVES);
    f4 w[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (a.norm[i]) w[i][0] = *(const f4 *)(a.norm[i] + d0), w[i][1] = *(const f4 *)(a.norm[i] + d1);
    Place at;
    if (!place_of(p, token, at)) return;
    float c[4], s[4];
    if (turned) {
#pragma unroll
        for (int j = 0; j < 4; ++j) turn(a, at.pos, 4 * l + j, c[j], s[j]);
    }
    const size_t k_row = (((size_t)max(at.page, 0) * p.n_kv_head) << p.page_log) + (at.pos & ((1 << p.page_log) - 1));
    const auto put = [&](f4 u, f4 v, int h) {
        const int which = h < nq ? 0 : 1;
        if (a.norm[which]) {
            const f4 q = u * u + v * v;
            const float r = 1.0f / __builtin_sqrtf(head_sum<LANES>((q[0] + q[1]) + (q[2] + q[3])) * (1.0f / HD) + a.eps);
            // (both weights are in registers: which one is a choice of values)
            u = u * (which ? w[1][0] : w[0][0]) * r;
            v = v * (which ? w[1][1] : w[0][1]) * r;
        }
        if (turned) {
            f4 y, z;
            if (a.interleaved) {
                y = f4{u[0] * c[0] - u[1] * s[0], u[0] * s[0] + u[1] * c[0], u[2] * c[1] - u[3] * s[1], u[2] * s[1] + u[3] * c[1]};
                z = f4{v[0] * c[2] - v[1] * s[2], v[0] * s[2] + v[1] * c[2], v[2] * c[3] - v[3] * s[3], v[2] * s[3] + v[3] * c[3]};
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = u[j] * c[j] - v[j] * s[j], z[j] = u[j] * s[j] + v[j] * c[j];
            }
            u = y;
            v = z;
        }
        if (h >= n || (which && at.page < 0)) return;
        T *to = which ? (T *)p.k + (k_row + ((size_t)(h - nq) << p.page_log)) * HD
                      : (T *)a.q_out + ((size_t)token * nq + h) * HD;
        T4 y, z;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = E::put(u[j]), z[j] = E::put(v[j]);
        *(T4 *)(to + d0) = y;
        *(T4 *)(to + d1) = z;
    };
    // (a wave's heads end together: the last ones compute on what they have and do not store)
    for (int h = first; h - lane / LANES < n; h += AHEAD * HEADS * WAVES) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int here = h + i * HEADS * WAVES;
            put(x[i][0], x[i][1], here);
            load(i, here + AHEAD * HEADS * WAVES);
        }
    }
}

// Any even n_rot: a lane has pairs of single dimensions.
template <class E, int HD>
__device__ __forceinline__ void store_token_pairs(const PagedStoreArgs &a, int token) {
    typedef typename E::T T;
    constexpr int LANES = HD / 2 < WAVE ? HD / 2 : WAVE, PAIRS = HD / 2 / LANES, STEP = 4 * (WAVE / LANES);
    const PagedArgs &p = a.p;
    const int lane = threadIdx.x & (LANES - 1);
    Place at;
    if (!place_of(p, token, at)) return;
    const int half = a.n_rot / 2, nq = a.x[0] ? p.n_head : 0;
    float c[PAIRS], s[PAIRS];
    int e0[PAIRS], e1[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        const int pair = lane + LANES * i;
        const bool apart = pair < half && !a.interleaved;
        e0[i] = apart ? pair : 2 * pair;
        e1[i] = apart ? pair + half : 2 * pair + 1;
        if (pair < half) turn(a, at.pos, pair, c[i], s[i]);
    }
    for (int h = threadIdx.x / LANES; h < nq + p.n_kv_head; h += STEP) {
        const int which = h < nq ? 0 : 1, hh = which ? h - nq : h;
        const float *x = a.x[which] + (size_t)token * a.ld[which] + (size_t)hh * HD;
        const float *w = a.norm[which];
        float u[PAIRS], v[PAIRS];
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) u[i] = x[e0[i]], v[i] = x[e1[i]];
        if (w) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) sum += u[i] * u[i] + v[i] * v[i];
#pragma unroll
            for (int m = 1; m < LANES; m *= 2) sum += __shfl_xor(sum, m, LANES);
            const float r = 1.0f / __builtin_sqrtf(sum * (1.0f / HD) + a.eps);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) u[i] = u[i] * w[e0[i]] * r, v[i] = v[i] * w[e1[i]] * r;
        }
        if (which && at.page < 0) continue;
        T *y = which ? (T *)p.k + ((((size_t)at.page * p.n_kv_head + hh) << p.page_log) +
                                   (at.pos & ((1 << p.page_log) - 1))) * HD
                     : (T *)a.q_out + ((size_t)token * nq + hh) * HD;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            const bool turned = lane + LANES * i < half;
            y[e0[i]] = E::put(turned ? u[i] * c[i] - v[i] * s[i] : u[i]);
            y[e1[i]] = E::put(turned ? u[i] * s[i] + v[i] * c[i] : v[i]);
        }
    }
}

}  // namespace
}  // namespace llamd

// paged_store.hip -- new tokens' queries, keys and values into the form that the paged attention reads: per-head RMS
// norm, rotary positions, one rounding to the cache's type; keys and values go to the sequence's pages.
//
//   y = x * 1 / sqrt(mean(x^2) + eps) * w                        (with a weight; f32 sums)
//   (a, b) -> (a c - b s, a s + b c),  c = m cos(pos f_i), s = m sin(pos f_i)
//
// for the pairs i < n_rot / 2, dimensions (i, i + n_rot / 2) or (2 i, 2 i + 1); the rest of a head passes. The angle is
// formed in 64 bits and reduced to a fraction of a turn there: at position 10^6 a 32-bit angle is off by 0.03 radians.
#include "paged_util.hpp"

namespace llamd {
namespace {

// One workgroup per token: a wave per head (two heads of 64), each lane one pair of a head (two of 256), so that a lane's
// sine and cosine serve every head it meets.
template <class E, int HD>
__global__ __launch_bounds__(256) void paged_store(PagedStoreArgs a) {
    typedef typename E::T T;
    constexpr int LANES = HD / 2 < WAVE ? HD / 2 : WAVE;  // lanes per head
    constexpr int PAIRS = HD / 2 / LANES;                 // pairs per lane
    constexpr int STEP = 4 * (WAVE / LANES);              // heads per workgroup step
    const PagedArgs &p = a.p;
    const int token = blockIdx.x, lane = threadIdx.x & (LANES - 1), first = threadIdx.x / LANES;
    int seq = token, pos;
    if (p.start) {
        // sequences have ascending tokens: the one whose span holds this token
        int unit = token - min(max(p.start[0], 0), p.n_tok);
        if (unit < 0) return;
        seq = find_sequence(p.n_seq, unit, [&](int s) {
            const TokenSpan t = token_span(p, s);
            return t.end - t.first;
        });
        if (seq < 0) return;
        const TokenSpan t = token_span(p, seq);
        pos = p.len[seq] - (t.end - t.first) + unit;
    } else {
        if (seq >= p.n_seq) return;
        pos = p.len[seq] - 1;
    }
    int page = -1;
    if (pos >= 0 && pos >> p.page_log < p.max_page)
        page = page_of(p, p.table + (size_t)seq * p.max_page, pos);
    const int slot = pos & ((1 << p.page_log) - 1);

    const int half = a.n_rot / 2;
    float c[PAIRS], s[PAIRS];
    int e0[PAIRS], e1[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
        const int pair = lane + LANES * i;
        c[i] = 1.0f;
        s[i] = 0.0f;
        if (pair < half) {
            const double turns = (double)pos * a.freqs[pair] * 0.15915494309189533577;
            sincospif((float)(2.0 * (turns - rint(turns))), &s[i], &c[i]);
            c[i] *= a.mscale;
            s[i] *= a.mscale;
            e0[i] = a.interleaved ? 2 * pair : pair;
            e1[i] = a.interleaved ? 2 * pair + 1 : pair + half;
        } else {
            e0[i] = 2 * pair;
            e1[i] = 2 * pair + 1;
        }
    }

    const int nq = a.x[0] ? p.n_head : 0, nk = p.n_kv_head;
    for (int h = first; h < nq + nk; h += STEP) {
        const int which = h < nq ? 0 : 1, hh = which ? h - nq : h;
        const float *x = a.x[which] + (size_t)token * a.ld[which] + hh * HD;
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
            for (int i = 0; i < PAIRS; ++i) u[i] *= r * w[e0[i]], v[i] *= r * w[e1[i]];
        }
        T *y = which ? (T *)p.k + ((((size_t)max(page, 0) * nk + hh) << p.page_log) + slot) * HD
                     : (T *)a.q_out + ((size_t)token * nq + hh) * HD;
        if (which && page < 0) continue;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
            y[e0[i]] = E::put(u[i] * c[i] - v[i] * s[i]);
            y[e1[i]] = E::put(u[i] * s[i] + v[i] * c[i]);
        }
    }
    if (page < 0) return;
    const float *x = a.x[2] + (size_t)token * a.ld[2];
    T *v = (T *)p.v + (((size_t)page * nk * HD) << p.page_log) + slot;
    for (int i = threadIdx.x; i < nk * HD; i += 256) v[(size_t)i << p.page_log] = E::put(x[i]);
}

template <class E>
int store_as(const PagedStoreArgs &a, hipStream_t st) {
    const dim3 grid(a.p.n_tok), block(256);
    if (a.p.hd == 64) hipLaunchKernelGGL((paged_store<E, 64>), grid, block, 0, st, a);
    else if (a.p.hd == 128) hipLaunchKernelGGL((paged_store<E, 128>), grid, block, 0, st, a);
    else if (a.p.hd == 256) hipLaunchKernelGGL((paged_store<E, 256>), grid, block, 0, st, a);
    else return -1;
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace

int launch_paged_store(const PagedStoreArgs &a, int type, hipStream_t st) {
    if (type == PT_F32) return store_as<ElemF32>(a, st);
    if (type == PT_F16) return store_as<ElemF16>(a, st);
    if (type == PT_BF16) return store_as<ElemBF16>(a, st);
    return -1;
}

}  // namespace llamd

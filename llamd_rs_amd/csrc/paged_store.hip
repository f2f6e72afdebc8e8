// paged_store.hip -- new tokens' queries, keys and values into the form that the paged attention reads: per-head RMS
// norm, rotary positions, one rounding to the cache's type; keys and values go to the sequence's pages.
//
//   y = x * 1 / sqrt(mean(x^2) + eps) * w                        (with a weight; f32 sums)
//   (a, b) -> (a c - b s, a s + b c),  c = m cos(pos f_i), s = m sin(pos f_i)
//
// for the pairs i < n_rot / 2, dimensions (i, i + n_rot / 2) or (2 i, 2 i + 1); the rest of a head passes. The angle is
// formed in 64 bits and reduced to a fraction of a turn there: at position 10^6 a 32-bit angle is off by 0.03 radians.
//
// Bound: memory, 4 (H + 2 Hkv) hd bytes read and 2 or 4 of them written per token, and for a few tokens the chain of loads
// from the sequence's length to its page. One launch does two things:
//   queries and keys: a wave has a token (four waves share one when tokens are few), HD / 8 lanes a head, so that a lane's
//     four sines and cosines serve every head it meets, and loads and stores are 16 bytes (8 of a 16-bit type);
//   values: V pages hold a dimension's positions together, so a workgroup takes 16 positions that lie together in a page
//     and turns them in LDS.
#include <algorithm>

#include "paged_store.hpp"

namespace llamd {
namespace {

// ---- values ------------------------------------------------------------------------

// Unit number `unit`: a block of 16 positions and a kv head.
template <class E, int HD>
__device__ __forceinline__ void store_values(const PagedStoreArgs &a, int unit) {
    typedef typename E::T T;
    constexpr int ROW = HD + 4;
    __shared__ __align__(16) float tile[POS * ROW];
    const PagedArgs &p = a.p;
    const int kvh = unit % p.n_kv_head;
    Block at;
    if (!block_of(p, unit / p.n_kv_head, at)) return;
    const int before = at.before, pos0 = at.pos0, page = at.page, first = at.first, lo = at.lo, hi = at.hi;
    const float *x = a.x[2] + (size_t)kvh * HD;
    for (int i = threadIdx.x; i < POS * HD / 4; i += 256) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        if (r >= lo && r < hi)
            *(f4 *)(tile + r * ROW + d) = *(const f4 *)(x + (size_t)(first + (pos0 + r - before)) * a.ld[2] + d);
    }
    __syncthreads();
    T *v = (T *)p.v + ((((size_t)page * p.n_kv_head + kvh) * HD) << p.page_log) + (pos0 & ((1 << p.page_log) - 1));
    constexpr int RUN = E::RUN;
    for (int i = threadIdx.x; i < HD * (POS / RUN); i += 256) {
        const int d = i / (POS / RUN), r = i % (POS / RUN) * RUN;
        T *to = v + ((size_t)d << p.page_log) + r;
        if (r >= lo && r + RUN <= hi) {
            typedef T V __attribute__((ext_vector_type(RUN)));
            V y;
#pragma unroll
            for (int j = 0; j < RUN; ++j) y[j] = E::put(tile[(r + j) * ROW + d]);
            *(V *)to = y;
        } else {
            for (int j = max(lo - r, 0); j < min(hi - r, RUN); ++j) to[j] = E::put(tile[(r + j) * ROW + d]);
        }
    }
}

// The first `tokens` workgroups: queries and keys, WAVES waves per token (0: pairs of single dimensions); then values.
template <class E, int HD, int WAVES>
__global__ __launch_bounds__(256) void paged_store(PagedStoreArgs a, int tokens) {
    if ((int)blockIdx.x >= tokens) {
        store_values<E, HD>(a, blockIdx.x - tokens);
    } else if constexpr (WAVES) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), token = (blockIdx.x * 4 + wave) / WAVES;
        if (token < a.p.n_tok) store_token<E, HD, WAVES>(a, token, wave % WAVES);
    } else {
        store_token_pairs<E, HD>(a, blockIdx.x);
    }
}

template <class E, int HD>
int store_as(const PagedStoreArgs &a, hipStream_t st) {
    const PagedArgs &p = a.p;
    // 16-position blocks of all sequences: a whole one per 16 tokens, and two that are not
    const long long blocks = std::min((long long)p.n_tok / 16 + 2LL * p.n_seq, (long long)p.n_tok);
    const bool runs = a.n_rot % 8 == 0;
    // four waves per token while that leaves CUs idle otherwise
    const int waves = !runs ? 0 : p.n_tok < 2048 ? 4 : 1, tokens = waves == 1 ? (p.n_tok + 3) / 4 : p.n_tok;
    const long long grid = tokens + blocks * p.n_kv_head;
    if (grid > 0x7FFFFFFF / 256) return -1;
    const dim3 g((unsigned)grid), b(256);
    if (waves == 1) hipLaunchKernelGGL((paged_store<E, HD, 1>), g, b, 0, st, a, tokens);
    else if (waves) hipLaunchKernelGGL((paged_store<E, HD, 4>), g, b, 0, st, a, tokens);
    else hipLaunchKernelGGL((paged_store<E, HD, 0>), g, b, 0, st, a, tokens);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <class E>
int store_type(const PagedStoreArgs &a, hipStream_t st) {
    if (a.p.hd == 64) return store_as<E, 64>(a, st);
    if (a.p.hd == 128) return store_as<E, 128>(a, st);
    if (a.p.hd == 256) return store_as<E, 256>(a, st);
    return -1;
}

}  // namespace

int launch_paged_store(const PagedStoreArgs &a, int type, hipStream_t st) {
    if (type == PT_F32) return store_type<ElemF32>(a, st);
    if (type == PT_F16) return store_type<ElemF16>(a, st);
    if (type == PT_BF16) return store_type<ElemBF16>(a, st);
    return -1;
}

}  // namespace llamd

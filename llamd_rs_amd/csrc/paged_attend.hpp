// paged_attend.hpp -- causal attention over a paged cache: prompts (any number of new tokens per sequence, after any
// cached context) and decode batches (one token per sequence, prefixes that sequences share read once).
//
//   o = sum_j softmax_j(scale q . k_j) v_j,   j = 0 .. the token's position
//
// Rows: the query heads of a kv head's group, for all tokens of a sequence, are numbered token by token, and a tile
// takes consecutive ones: with 8 query heads per kv head, a tile of 256 rows is 32 tokens, whose keys and values are
// read once for all 8.
//
// Two ways to form O. tile_rows: many rows; the waves of a workgroup have 32 rows of their own each and share K and V
// tiles in LDS. few_rows: up to 16 rows; the waves share the rows and have positions of their own, read straight into the
// matrix operands. Either may have a part of a row's positions only; then O (unnormalised), the maximum and the sum
// go to scratch and paged_join or paged_join_decode puts the parts together, in a fixed order.
//
// 8-bit pages (e4m3 numbers with a power of two for each 16 positions): q, weights and products are bf16's. tile_rows widens K and V
// once for all rows, on their way into LDS; few_rows widens them in registers, K without its scale, which goes to the scores: 16
// bytes of a row are two steps' operands, so that a step is 64 positions.
//
// Bound and measured (32 query heads on 4 kv heads of 128, one MI355X). Long prompts of 16 bits: products and the softmax's
// vector work, one after the other (8192 tokens of bf16: matrix cores busy 46% of the cycles, vector units 53%; 560 us, 980
// TFLOP/s of the causal half, where a library product of 8192^3 reaches 1349); f32 110 to 119 of 154. Pieces and packed
// prompts: the steps of a CU's tiles, 1.1 us each, and 8 us to every workgroup's first product (512 tokens after 7000 81 us,
// 9 prompts of 192 to 700 tokens 41). Decode: memory, then the chain length -> table -> keys and the second launch (1 x 4100
// 12.8 us, 13 x 1000 in f32 20.4, 48 behind 4100 shared 25.8). 8-bit pages: 8192 tokens 562 to 603 us (912 to 978 TFLOP/s), 512
// after 7000 83 to 88, 9 packed prompts 40.3; decode 1 x 4100 12.3, 61 x 500 to 2000 (79 MB) 28.3, of these 23 at 3.4 TB/s and
// the join 5.4, 48 behind 4100 shared 25.4.
#pragma once

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "launch.hpp"
#include "paged_plan.hpp"
#include "paged_wave.hpp"

namespace llamd {
namespace {

// Parts of rows: a slot has the statistics (maximum, sum) of its rows and their O, four dimensions at a time:
// o[slot][HD / 4][rows].
struct Parts {
    float4 *o;
    float2 *ml;
};

// How a call is split (host).
struct Split {
    Parts many, few;     // of paged_tiles (blocks of 32 rows) and of paged_few
    int few_rows;        // rows of a slot of the latter: 16, or in decode a sequence's and kv head's, if fewer
    int parts;           // most parts of a row tile (prompt, prefix)
    int fine;            // parts of a shared prefix of 8-bit pages that may be short (prefix_parts); parts at the most
    int tiles;           // decode: tiles of shared prefixes that there are slots for
    double per_item;     // decode: 1 / (positions of all sequences' parts wanted, in steps)
    double per_row;      // decode: 1 / (parts of a sequence, in steps, while they are short)
};

// ---- rows ------------------------------------------------------------------------

// What a tile of rows belongs to.
struct Tile {
    int seq;              // the sequence whose table is read
    int n_kv;             // its positions that can be read
    int top;              // positions that the tile's last row attends to
    int first, end, len;  // prompt: the sequence's tokens and length; prefix: the group's sequences
    int rows;             // rows in the tile
};
// A row of it.
struct Row {
    long long at;         // token * n_head + head, -1: no row
    int limit;            // positions that it attends to
};

// Positions of a sequence of length n that the table can hold.
__device__ __forceinline__ int readable_of(const PagedArgs &p, int n) {
    return (int)min((long long)max(n, 0), min((long long)p.max_page << p.page_log, 0x7FFFFFFFLL));
}

// Tile number `tile` (R rows) of a prompt batch; it becomes its number within its sequence. False past the last. Every
// sequence's numbers come with the first loads: the search costs one trip to memory per 64 sequences.
template <int R>
__device__ __forceinline__ bool prompt_tile(const PagedArgs &p, int &tile, Tile &t) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < p.n_seq; s0 += WAVE) {
        const int s = s0 + lane;
        int units = 0, first = s, end = s + 1, len = 0;
        if (s < p.n_seq) {
            len = p.len[s];
            if (p.start) {
                first = min(max(p.start[s], 0), p.n_tok);
                end = max(min(p.start[s + 1], p.n_tok), first);
            }
            units = (int)(((long long)(end - first) * p.group + R - 1) / R);
        }
        const int sum = wave_incl_sum_i(units);
        const unsigned long long past = __ballot(sum > tile);
        if (past) {
            const int l = __builtin_ctzll(past);
            tile -= __builtin_amdgcn_readlane(sum - units, l);
            t.seq = s0 + l;
            t.first = __builtin_amdgcn_readlane(first, l);
            t.end = __builtin_amdgcn_readlane(end, l);
            t.len = __builtin_amdgcn_readlane(len, l);
            t.rows = (int)min((long long)(t.end - t.first) * p.group - (long long)R * tile, (long long)R);
            t.n_kv = readable_of(p, t.len);
            const int last = t.first + (int)(((long long)R * tile + t.rows - 1) / p.group);
            t.top = max(min(t.len - (t.end - last) + 1, t.n_kv), 0);
            return true;
        }
        tile -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// The same for tile number `order` of the batch's tiles by their positions, most first (in units of 2^STEP_LOG): long tiles
// that start last would leave the GPU to themselves. `unit` becomes the tile's number among all, `tile` that within its
// sequence. For batches of up to 64 sequences; larger ones, and one sequence, go from the last tile to the first.
template <int R, int STEP_LOG>
__device__ __forceinline__ bool prompt_tile_by_size(const PagedArgs &p, int order, int n_units, int &unit, int &tile, Tile &t) {
    if (p.n_seq == 1 || p.n_seq > WAVE) {
        unit = tile = n_units - 1 - order;
        return prompt_tile<R>(p, tile, t);
    }
    const int lane = threadIdx.x & 63;
    int tiles = 0, first = lane, end = lane + 1, len = 0;
    if (lane < p.n_seq) {
        len = p.len[lane];
        if (p.start) {
            first = min(max(p.start[lane], 0), p.n_tok);
            end = max(min(p.start[lane + 1], p.n_tok), first);
        }
        tiles = (int)(((long long)(end - first) * p.group + R - 1) / R);
    }
    const int n_kv = readable_of(p, len), before = len - (end - first);  // positions before its first token
    // tiles of the lane's sequence that have more than x positions: those whose last token is at x or further
    const auto more = [&](long long x) {
        if (x >= n_kv) return 0;
        const long long y = max(x - before, 0LL);  // token number y on
        if (y >= end - first) return 0;
        return tiles - (int)(y * p.group / R);
    };
    const auto sum = [](int x) { return wave_reduce(x, 0, [](int u, int v) { return u + v; }); };
    if (order >= sum(tiles)) return false;
    int most = wave_reduce(n_kv, 0, [](int u, int v) { return max(u, v); });
    // the least number of steps such that no more than `order` tiles have more
    int lo = 0, hi = ((most - 1) >> STEP_LOG) + 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sum(more((long long)mid << STEP_LOG)) <= order) hi = mid;
        else lo = mid + 1;
    }
    // (0 steps: the tiles that see nothing)
    const int above = more((long long)lo << STEP_LOG), upto = lo ? more((long long)(lo - 1) << STEP_LOG) : tiles;
    int at = order - sum(above);
    const int here = upto - above, scan = wave_incl_sum_i(here);
    const unsigned long long past = __ballot(scan > at);
    const int l = __builtin_ctzll(past);
    at -= __builtin_amdgcn_readlane(scan - here, l);
    // of a sequence's tiles, the last `above` have more
    tile = __builtin_amdgcn_readlane(tiles - above, l) - 1 - at;
    unit = __builtin_amdgcn_readlane(wave_incl_sum_i(tiles) - tiles, l) + tile;
    if (unit >= n_units) return false;  // starts that descend: sequences over the same tokens, more tiles than there are slots
    t.seq = l;
    t.first = __builtin_amdgcn_readlane(first, l);
    t.end = __builtin_amdgcn_readlane(end, l);
    t.len = __builtin_amdgcn_readlane(len, l);
    t.rows = (int)min((long long)(t.end - t.first) * p.group - (long long)R * tile, (long long)R);
    t.n_kv = readable_of(p, t.len);
    const int last = t.first + (int)(((long long)R * tile + t.rows - 1) / p.group);
    t.top = max(min(t.len - (t.end - last) + 1, t.n_kv), 0);
    return true;
}

// Row i of it (the last one for rows that it has not).
template <int R>
__device__ __forceinline__ Row prompt_row(const PagedArgs &p, int tile, const Tile &t, int kvh, int i) {
    const uint32_t at = (uint32_t)R * tile + min(i, t.rows - 1);
    const uint32_t tok = at / (uint32_t)p.group, head = at - tok * p.group;
    Row r;
    r.limit = max(min(t.len - (t.end - t.first) + (int)tok + 1, t.n_kv), 0);
    r.at = i < t.rows ? (long long)(t.first + tok) * p.n_head + kvh * p.group + head : -1;
    return r;
}

// A group of sequences: its members [first, end) and the positions that they share (whole pages of a table); none shared
// where a group has no two members.
struct Group {
    int first, end, shared;
};
__device__ __forceinline__ Group group_at(const PagedAttendArgs &a, int g) {
    Group x;
    x.first = min(max(a.group_at[g], 0), a.p.n_seq);
    x.end = min(max(a.group_at[g + 1], x.first), a.p.n_seq);
    x.shared = x.end - x.first < 2 ? 0 : shared_positions(a.shared[g], a.p.page_log, a.p.max_page);
    return x;
}
// The group of a sequence, by itself if it is in none.
__device__ __forceinline__ Group group_of(const PagedAttendArgs &a, int s, int &number) {
    Group x = {s, s + 1, 0};
    if (a.n_groups <= 8) {
        for (int g = 0; g < a.n_groups; ++g) {
            const Group y = group_at(a, g);
            if (s >= y.first && s < y.end) x = y, number = g;
        }
        return x;
    }
    int lo = 0, hi = a.n_groups;  // the last group that begins at or before s
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.group_at[mid] <= s) lo = mid + 1;
        else hi = mid;
    }
    if (lo) {
        const Group y = group_at(a, lo - 1);
        if (s >= y.first && s < y.end) x = y, number = lo - 1;
    }
    return x;
}

// Tile number `tile` of the rows of all groups that share something.
template <int R> __device__ __forceinline__ int prefix_units(const PagedAttendArgs &a, const Group &x) {
    return x.shared ? (int)(((long long)(x.end - x.first) * a.p.group + R - 1) / R) : 0;
}
template <int R>
__device__ __forceinline__ bool prefix_tile(const PagedAttendArgs &a, int &tile, Tile &t) {
    const int n = find_sequence(a.n_groups, tile, [&](int i) { return prefix_units<R>(a, group_at(a, i)); });
    if (n < 0) return false;
    const Group g = group_at(a, n);
    t.seq = t.first = g.first;
    t.end = g.end;
    t.rows = (int)min((long long)(g.end - g.first) * a.p.group - (long long)R * tile, (long long)R);
    t.n_kv = t.top = readable_of(a.p, g.shared);
    return true;
}
template <int R>
__device__ __forceinline__ Row prefix_row(const PagedAttendArgs &a, int tile, const Tile &t, int kvh, int i) {
    const uint32_t at = (uint32_t)R * tile + min(i, t.rows - 1);
    const uint32_t seq = t.first + at / (uint32_t)a.p.group, head = at % (uint32_t)a.p.group;
    Row r;
    r.limit = min(readable_of(a.p, a.p.len[seq]), t.n_kv);
    r.at = i < t.rows ? (long long)seq * a.p.n_head + kvh * a.p.group + head : -1;
    return r;
}

// ---- parts -----------------------------------------------------------------------

// Parts of a tile's `steps` steps of positions, and the steps of part z.
__device__ __forceinline__ int parts_of(int steps, int most, int least) {
    return max(min(most, steps / least), 1);
}
__device__ __forceinline__ int2 part_steps(int steps, int parts, int z) {
    return make_int2((int)((long long)steps * z / parts), (int)((long long)steps * (z + 1) / parts));
}

// Where a kv head's pages are.
template <class E> struct Pages {
    const typename E::P *k, *v;
    const int32_t *table;
    size_t step;  // elements between pages
    int mask;     // positions per page - 1
    const uint8_t *k_scale, *v_scale;  // 8-bit pages: of this kv head, step >> SCALE_LOG / HD bytes between pages
};
template <class E, int HD>
__device__ __forceinline__ Pages<E> pages_of(const PagedArgs &p, int seq, int kvh) {
    const size_t head = (size_t)kvh * HD << p.page_log;
    Pages<E> x = {(const typename E::P *)p.k + head, (const typename E::P *)p.v + head, p.table + (size_t)seq * p.max_page,
                  (size_t)p.n_kv_head * HD << p.page_log, (1 << p.page_log) - 1};
    if constexpr (bytes_of<E>) {
        const size_t first = (size_t)kvh << (p.page_log - SCALE_LOG);
        x.k_scale = p.k_scale + first;
        x.v_scale = p.v_scale + first;
    }
    return x;
}
// Where the scale of a position of a page lies.
template <class E> __device__ __forceinline__ size_t scale_at(const PagedArgs &p, const Pages<E> &pg, int page, int pos) {
    return (((size_t)page * p.n_kv_head) << (p.page_log - SCALE_LOG)) + ((pos & pg.mask) >> SCALE_LOG);
}

__device__ __forceinline__ float over(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

template <class E> __device__ __forceinline__ void put_out(void *out, bool f32, size_t at, float4 x) {
    if (f32) put4<ElemF32>(out, at, x);
    else put4<E>(out, at, x);
}

// ---- up to 16 rows -----------------------------------------------------------------

// x, as something that the compiler cannot keep the results of between tiles: addresses are cheaper made again than held
// in registers.
__device__ __forceinline__ uint32_t fresh(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// A row's runs for the first product of 16 rows. 8-bit pages: 16 bytes of K are the runs of two steps.
template <class E, int HD>
__device__ __forceinline__ void load_few(run4 (&q)[HD / (4 * E::RUN)], const void *from, long long at) {
    const typename E::T *x = (const typename E::T *)from + (size_t)max(at, 0LL) * HD;
    const int g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int c = 0; c < HD / (4 * E::RUN); ++c)
        q[c] = *(const run4 *)(x + (bytes_of<E> ? 2 * (4 * (c / 2) + g) + c % 2 : 4 * c + g) * E::RUN);
}

// Positions of a step of 16 rows.
template <class E> constexpr int few_positions = bytes_of<E> ? 64 : 32;

// 16 rows against 8-bit pages (see attend_few_runs): steps of 64 positions, position 16 g + 8 j + 4 b + i of a step in register i of
// block b and half j of group g's lanes.
template <int HD, int STRIDE, bool AGAIN>
__device__ __forceinline__ void attend_few8(const PagedArgs &p, const Pages<ElemE4M3> &pg, int n_kv, int limit, int begin,
                                            int end, const run4 (&q)[HD / 32], float scale, FewState<ElemE4M3, HD> &st) {
    typedef ElemE4M3 E;
    typedef FewState<E, HD> S;
    const int all = wave_reduce(limit, 0x7FFFFFFF, [](int x, int y) { return min(x, y); });
    const auto step = [&](auto masked, int t0) {
        const int lane = (AGAIN ? fresh(threadIdx.x) : threadIdx.x) & 63, g = lane >> 4, m = lane & 15;
        // the lane's page as a row of K (16 positions on per 4 rows), and as a group of positions
        const int k0 = t0 + SCALE_BLOCK * (m >> 2), v0 = t0 + SCALE_BLOCK * g;
        const int idk = pg.table[min(k0, n_kv - 1) >> p.page_log], idv = pg.table[min(v0, n_kv - 1) >> p.page_log];
        const bool ok = (unsigned)idv < (unsigned)p.n_page;
        // bit i: position t0 + i can be read
        const unsigned long long valid = __ballot(ok && t0 + lane < n_kv);
        if (!masked && valid != ~0ull) return false;
        const int page = ok ? idv : 0, page_k = (unsigned)idk < (unsigned)p.n_page ? idk : 0;
        const size_t at = scale_at(p, pg, page, v0);
        const uint32_t ek = pg.k_scale[at], ev = pg.v_scale[at];
        run4 k[4][HD / 64], v[S::DB];
        const uint8_t *x = pg.k + (size_t)page_k * pg.step + (size_t)((k0 & pg.mask) + (m & 3)) * HD + g * 16;
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) k[b][c] = *(const run4 *)(x + 4 * b * HD + 64 * c);
        const uint8_t *y = pg.v + (size_t)page * pg.step + ((size_t)m << p.page_log) + (v0 & pg.mask);
        const auto v_run = [&](int d, uint32_t plus) { return *(const run4 *)(y + (((size_t)(16 * d) << p.page_log) + plus)); };
        if constexpr (!masked) {
#pragma unroll
            for (int d = 0; d < S::DB; ++d) v[d] = v_run(d, 0u);
        }
        v4f s[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) s[b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    s[b] = mul16<E>(widen(k[b][c][2 * h], k[b][c][2 * h + 1], 0x1p-8f), q[2 * c + h], s[b]);
        if constexpr (masked) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = SCALE_BLOCK * g + 4 * b + i;
                    s[b][i] = t0 + n < limit && (valid >> n & 1) ? s[b][i] : NEG_INF;
                }
        }
        // (what lies in place of a scale that is none may be anything)
        const bool some = valid >> (SCALE_BLOCK * g) & 1;
        // (K was taken 2^-8 of its numbers, 1.75 at most: as they are, up to 448, large q would pass f32's range before the unit
        // is in. Inside that range: 0 scores, and masked ones, stay what they are)
        st.softmax(s, fminf(fmaxf(scale * unit_of(some ? ek : 127u) * 0x1p8f, 0x1p-126f), 0x1.fffffep127f));
        const float unit = unit_of(some ? ev : 127u);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const run4 w = S::weights(s, j);
            if constexpr (masked) {
                st.add_masked(
                    [&](int d, uint32_t plus) {
                        const run4 r = v_run(d, plus);
                        return widen(r[2 * j], r[2 * j + 1], unit);
                    },
                    (uint32_t)(valid >> (SCALE_BLOCK * g + 8 * j)), w, t0 + 8 * j, limit);
            } else {
#pragma unroll
                for (int d = 0; d < S::DB; ++d) st.o[d] = mul16<E>(widen(v[d][2 * j], v[d][2 * j + 1], unit), w, st.o[d]);
            }
        }
        return true;
    };
    int t0 = begin;
    while (!AGAIN && t0 < end && t0 + 64 <= all && step(std::false_type{}, t0)) t0 += STRIDE;
    for (; t0 < end; t0 += STRIDE) step(std::true_type{}, t0);
}

// 16 rows against the positions t0 .. t0 + 31 for t0 = begin, begin + STRIDE, ... below end; begin and STRIDE are multiples of
// 32 (few_positions), uniform over the wave. K of a step (and V, where the registers allow) is loaded whole before the first
// product.
template <class E, int HD, int STRIDE, bool AGAIN>
__device__ __forceinline__ void attend_few_runs(const PagedArgs &p, const Pages<E> &pg, int n_kv, int limit, int begin, int end,
                                                const run4 (&q)[HD / (4 * E::RUN)], float scale, FewState<E, HD> &st) {
    typedef typename E::T T;
    typedef FewState<E, HD> S;
    constexpr int RUN = E::RUN;
    constexpr bool EARLY = HD * sizeof(T) <= 512;
    const int all = wave_reduce(limit, 0x7FFFFFFF, [](int x, int y) { return min(x, y); });
    // a step; false, with nothing done, if it is not `masked` and some position in it cannot be read
    const auto step = [&](auto masked, int t0) {
        // (AGAIN: few registers are left, so addresses are made again every step)
        const int lane = (AGAIN ? fresh(threadIdx.x) : threadIdx.x) & 63, g = lane >> 4, m = lane & 15;
        // the pages of the two halves of the step
        const int id0 = pg.table[min(t0, n_kv - 1) >> p.page_log], id1 = pg.table[min(t0 + 16, n_kv - 1) >> p.page_log];
        const bool ok0 = (unsigned)id0 < (unsigned)p.n_page, ok1 = (unsigned)id1 < (unsigned)p.n_page;
        const size_t at0 = (size_t)(ok0 ? id0 : 0) * pg.step, at1 = (size_t)(ok1 ? id1 : 0) * pg.step;
        // bit i: position t0 + i can be read
        uint32_t valid = (ok0 ? 0x0000FFFFu : 0u) | (ok1 ? 0xFFFF0000u : 0u);
        if (n_kv - t0 < 32) valid &= (1u << (n_kv - t0)) - 1u;
        if (!masked && valid != 0xFFFFFFFFu) return false;
        run4 k[2][S::QS], v[S::PS][S::DB];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int r = few_row<E>(b, m);
            const T *x = pg.k + (r & 16 ? at1 : at0) + (size_t)((t0 + r) & pg.mask) * HD;
#pragma unroll
            for (int c = 0; c < S::QS; ++c) k[b][c] = *(const run4 *)(x + (4 * c + g) * RUN);
        }
        const auto v_run = [&](int c, int d, uint32_t plus) {
            const int r = (4 * c + g) * RUN;
            const T *x = pg.v + (r & 16 ? at1 : at0) + ((size_t)m << p.page_log) + ((t0 + r) & pg.mask);
            return *(const run4 *)(x + (((size_t)(16 * d) << p.page_log) + plus));
        };
        const auto load_v = [&]() {
#pragma unroll
            for (int c = 0; c < S::PS; ++c)
#pragma unroll
                for (int d = 0; d < S::DB; ++d) v[c][d] = v_run(c, d, 0u);
        };
        if constexpr (EARLY && !masked) load_v();
        v4f s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) s[b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < S::QS; ++c)
#pragma unroll
            for (int b = 0; b < 2; ++b) s[b] = mul16<E>(k[b][c], q[c], s[b]);
        if constexpr (!EARLY && !masked) load_v();
        if constexpr (masked) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = few_reg<E>(b, i, g);
                    s[b][i] = t0 + at < limit && (valid >> at & 1) ? s[b][i] : NEG_INF;
                }
        }
        st.softmax(s, scale);
#pragma unroll
        for (int c = 0; c < S::PS; ++c) {
            const run4 w = S::weights(s, c);
            if constexpr (masked) {
                st.add_masked([&](int d, uint32_t plus) { return v_run(c, d, plus); }, valid >> ((4 * c + g) * RUN), w,
                              t0 + 4 * RUN * c, limit);
            } else {
#pragma unroll
                for (int d = 0; d < S::DB; ++d) st.o[d] = mul16<E>(v[c][d], w, st.o[d]);
            }
        }
        return true;
    };
    // steps that all rows see whole, then the others
    int t0 = begin;
    while (!AGAIN && t0 < end && t0 + 32 <= all && step(std::false_type{}, t0)) t0 += STRIDE;
    for (; t0 < end; t0 += STRIDE) step(std::true_type{}, t0);
}

template <class E, int HD, int STRIDE, bool AGAIN = false>
__device__ __forceinline__ void attend_few(const PagedArgs &p, const Pages<E> &pg, int n_kv, int limit, int begin, int end,
                                           const run4 (&q)[HD / (4 * E::RUN)], float scale, FewState<E, HD> &st) {
    if constexpr (bytes_of<E>) attend_few8<HD, STRIDE, AGAIN>(p, pg, n_kv, limit, begin, end, q, scale, st);
    else attend_few_runs<E, HD, STRIDE, AGAIN>(p, pg, n_kv, limit, begin, end, q, scale, st);
}

// Rows of a wave of paged_tiles (32, from `limit` and `at` of their lanes) once more, 16 at a time straight from the pages,
// every infinity or NaN in V added only where it belongs. Slow, since a workgroup does it alone: one such value in a tile that
// some row sees in part makes a prompt of 4096 tokens 1128 us instead of 160, 63 of them 1545; 512 tokens after 7000 410
// instead of 85, 9 packed prompts 175 instead of 44. (Inline: a call would give the kernel scratch memory, with which
// workgroups start at a third of the rate, 14 us for 512 of them instead of 5.)
template <class E, int HD>
__device__ __forceinline__ void attend_again(const PagedAttendArgs &a, const Parts &parts, bool part, int seq, int n_kv,
                                             int kvh, int begin, int end, size_t slot, int limit, long long at) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll 1
    for (int b = 0; b < 2; ++b) {
        const int from = 16 * b + (lane & 15), lim = __shfl(limit, from, WAVE);
        const long long row = __shfl(at, from, WAVE);
        run4 q[HD / (4 * E::RUN)];
        load_few<E, HD>(q, a.q, row);
        FewState<E, HD> st;
        st.clear();
        attend_few<E, HD, few_positions<E>, true>(a.p, pages_of<E, HD>(a.p, seq, kvh), n_kv, lim, begin, end, q, a.scale, st);
        const float l = add_groups(st.l), f = over(l);
        if (part) {
            if (g == 0) parts.ml[slot * 32 + from] = make_float2(st.m, l);
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
                parts.o[(slot * (HD / 4) + 4 * d + g) * 32 + from] = make_float4(st.o[d][0], st.o[d][1], st.o[d][2], st.o[d][3]);
        } else if (row >= 0) {
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
                put_out<E>(a.out, a.out_f32, (size_t)row * HD + 16 * d + 4 * g,
                           make_float4(st.o[d][0] * f, st.o[d][1] * f, st.o[d][2] * f, st.o[d][3] * f));
        }
    }
}

// Least positions of a part of paged_few: one step of each wave. A sequence has no more than FEW_PARTS parts (each costs the
// join) unless they would have more than LONG_PART steps (1 x 9000 positions: 17 us, in 71 parts 19.4; 1 x 60000: 35 us in
// 118 parts, in 64 43).
template <class E> constexpr int few_step = 4 * few_positions<E>;
constexpr int FEW_PARTS = 64, LONG_PART = 4;

// A sequence's own positions in a decode batch (behind those that its group shares), cut into parts.
struct Own {
    int n, shared;  // positions that can be read; of these the group's
    __device__ __forceinline__ int tail() const { return max(n - shared, 0); }
    // parts of `cut`; one at least where nothing is shared, so that an empty sequence's rows are written
    __device__ __forceinline__ int units(int cut) const {
        const int u = tail() ? (tail() - 1) / cut + 1 : 0;
        return shared && n ? u : max(u, 1);
    }
};
__device__ __forceinline__ Own own_of(const PagedAttendArgs &a, int s) {
    Own x = {0, 0};
    if (s >= a.p.n_seq) return x;
    int number;
    x.n = readable_of(a.p, a.p.len[s]);
    if (a.n_groups) x.shared = group_of(a, s, number).shared;
    return x;
}
// The batch's parts. Up to 64 sequences lie in the lanes of a wave (`mine`), read once.
struct DecodePlan {
    Own mine;  // of sequence `lane`
    int cut;   // positions per part, so that all parts together are about as many as the host wants
};
template <class E> __device__ __forceinline__ DecodePlan decode_plan(const PagedAttendArgs &a, const Split &sp) {
    const int lane = threadIdx.x & 63;
    DecodePlan d;
    d.mine = own_of(a, lane);
    int most = d.mine.tail();
    double sum = (double)most;  // exact
    for (int s = lane + WAVE; s < a.p.n_seq; s += WAVE) {
        const int n = own_of(a, s).tail();
        sum += (double)n;
        most = max(most, n);
    }
    most = wave_reduce(most, 0, [](int x, int y) { return max(x, y); });
    // (a step less than 2^31 at most: one part)
    const double row = min(most * sp.per_row, (double)LONG_PART);
    d.cut = (int)min(max(ceil(max(wave_sum_d(sum) * sp.per_item, row)), 1.0) * few_step<E>, 2147483648.0 - few_step<E>);
    return d;
}
// The sequence of part number `part` (its number within the sequence afterwards); -1: past the last.
__device__ __forceinline__ int part_sequence(const PagedAttendArgs &a, const DecodePlan &d, int &part, Own &own) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < a.p.n_seq; s0 += WAVE) {
        const Own x = s0 ? own_of(a, s0 + lane) : d.mine;
        const int units = s0 + lane < a.p.n_seq ? x.units(d.cut) : 0, sum = wave_incl_sum_i(units);
        const unsigned long long past = __ballot(sum > part);
        if (past) {
            const int l = __builtin_ctzll(past);
            part -= __builtin_amdgcn_readlane(sum - units, l);
            own.n = __builtin_amdgcn_readlane(x.n, l);
            own.shared = __builtin_amdgcn_readlane(x.shared, l);
            return s0 + l;
        }
        part -= __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}
// Parts of the sequences before sequence `seq`, and its own positions.
__device__ __forceinline__ int parts_before(const PagedAttendArgs &a, const DecodePlan &d, int seq, Own &own) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 <= seq; s0 += WAVE) {
        const Own x = s0 ? own_of(a, s0 + lane) : d.mine;
        if (s0 + lane < seq) before += x.units(d.cut);
        if (seq - s0 < WAVE) {
            own.n = __builtin_amdgcn_readlane(x.n, seq - s0);
            own.shared = __builtin_amdgcn_readlane(x.shared, seq - s0);
        }
    }
    return wave_reduce(before, 0, [](int x, int y) { return x + y; });
}

// A workgroup's place in a grid of nx x ny.
struct Place {
    int x, y, nx, ny;
};

// What a workgroup of four waves keeps in LDS for up to 16 rows.
template <int HD> struct FewShared {
    float part[4][HD / 4][64];
    float2 stats[4][16];
};

// DECODE: at.x a part of a sequence, at.y a kv head and block of 16 of its query heads. Otherwise at.x a tile of 16 rows of a
// prompt batch and a kv head, at.y a part of its positions.
template <class E, int HD, bool DECODE>
__device__ __forceinline__ void few_rows(const PagedAttendArgs &a, const Split &sp, Place at, FewShared<HD> &shared) {
    typedef FewState<E, HD> S;
    auto &stats = shared.stats;
    auto &part = shared.part;
    const PagedArgs &p = a.p;
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Tile t;
    Row r;
    int begin, end, parts, kvh;
    size_t slot;
    if constexpr (DECODE) {
        const DecodePlan plan = decode_plan<E>(a, sp);
        const int cut = plan.cut;
        int unit = at.x;
        Own own;
        t.seq = part_sequence(a, plan, unit, own);
        if (t.seq < 0) return;
        const int per = (p.group + 15) / 16, head = (at.y % per) * 16 + m;
        kvh = at.y / per;
        t.n_kv = r.limit = own.n;
        r.at = head < p.group ? (long long)t.seq * p.n_head + kvh * p.group + head : -1;
        begin = (int)min((long long)own.shared + (long long)unit * cut, 0x7FFFFFFFLL);
        end = (int)min((long long)begin + cut, (long long)t.n_kv);
        parts = own.shared && own.n ? 2 : own.units(cut);
        slot = (size_t)at.x * at.ny + at.y;
    } else {
        kvh = at.x % p.n_kv_head;
        const int unit = at.nx / p.n_kv_head - 1 - at.x / p.n_kv_head;
        int tile = unit;
        if (!prompt_tile<16>(p, tile, t)) return;
        r = prompt_row<16>(p, tile, t, kvh, m);
        const int steps = (t.top + few_step<E> - 1) / few_step<E>;
        parts = parts_of(steps, sp.parts, 1);
        if (at.y >= parts) return;
        const int2 range = part_steps(steps, parts, at.y);
        begin = range.x * few_step<E>;
        end = min(range.y * few_step<E>, t.top);
        slot = (size_t)(unit * p.n_kv_head + kvh) * sp.parts + at.y;
    }
    run4 q[S::QS];
    load_few<E, HD>(q, a.q, r.at);
    S st;
    st.clear();
    attend_few<E, HD, few_step<E>>(p, pages_of<E, HD>(p, t.seq, kvh), t.n_kv, r.limit, begin + few_positions<E> * wave, end, q,
                                   a.scale, st);

    // the four waves' positions together: every wave adds a quarter of the dimensions
    const float mine = add_groups(st.l);
    if (g == 0) stats[wave][m] = make_float2(st.m, mine);
#pragma unroll
    for (int d = 0; d < S::DB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[wave][d * 4 + i][lane] = st.o[d][i];
    __syncthreads();
    float top = NEG_INF, l = 0.0f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, stats[w][m].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = exp2_fast(stats[w][m].x - against(top));
        l = __builtin_fmaf(stats[w][m].y, f[w], l);
    }
    const float by = parts > 1 ? 1.0f : over(l);
    if (parts > 1 && wave == 0 && g == 0 && m < sp.few_rows) sp.few.ml[slot * sp.few_rows + m] = make_float2(top, l);
#pragma unroll
    for (int j = 0; j < S::DB / 4; ++j) {
        const int d = wave * (S::DB / 4) + j;
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) x[i] = __builtin_fmaf(part[w][d * 4 + i][lane], f[w], x[i]);
            x[i] *= by;
        }
        const float4 y = make_float4(x[0], x[1], x[2], x[3]);
        if (parts > 1) {
            if (m < sp.few_rows) sp.few.o[(slot * (HD / 4) + 4 * d + g) * sp.few_rows + m] = y;
        } else if (r.at >= 0) {
            put_out<E>(a.out, a.out_f32, (size_t)r.at * HD + 16 * d + 4 * g, y);
        }
    }
}

template <class E, int HD, bool DECODE>
__global__ __launch_bounds__(256, E::RUN == 4 && HD <= 128 ? 3 : 1) void paged_few(PagedAttendArgs a, Split sp) {
    __shared__ __align__(16) FewShared<HD> shared;
    const int at = blockIdx.x, nx = gridDim.x;
    if constexpr (DECODE) {
        // all columns of a part together: parts that there are not come last (1 x 20000 positions: 25 us, first 20)
        const int cols = a.p.n_kv_head * ((a.p.group + 15) / 16);
        few_rows<E, HD, DECODE>(a, sp, {at / cols, at % cols, nx / cols, cols}, shared);
    } else {
        few_rows<E, HD, DECODE>(a, sp, {at, (int)blockIdx.y, nx, (int)gridDim.y}, shared);
    }
}

// ---- many rows -------------------------------------------------------------------

// Asks the scheduler for N reads of a block's operands 6 ahead of their products (left alone it places each right before
// its product, which then waits for LDS every time).
template <class E, int N> __device__ __forceinline__ void order_reads() {
    constexpr int MFMA = E::RUN == 8 ? 1 : 4, AHEAD = N < 6 ? N : 6;
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, MFMA, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * MFMA, 0);
}

// Positions per tile (two buffers of K and V in at most 128 KB), and least tiles of a part.
template <class E, int HD> __host__ __device__ constexpr int tile_positions() {
    return HD * sizeof(typename E::T) <= 512 ? 64 : 32;
}
template <class E> __host__ __device__ constexpr int tile_least() { return E::RUN == 8 ? 4 : 1; }
// ... of a part of a shared prefix, whose rows are few (48 sequences behind 4100 positions: 28.6 us, with 4 steps 30.9), and
// the most tiles that a prompt's rows are not split for: the join costs as much (512 tokens 22 us, in two parts 27; 1024 33,
// in four 41).
template <class E> __host__ __device__ constexpr int prefix_least() { return E::RUN == 8 ? 8 : 1; }
// 8-bit pages: up to Split::fine parts of 4 steps at least (8 sequences behind 7800 positions 20.3 us, by 8 steps 24.2; 64
// behind 1300 21.6 and 28.0; 20 behind 8700, heads of 256, 32.0 and 42.3).
constexpr int SHORT_PREFIX = 4;
template <class E> __device__ __forceinline__ int prefix_parts(const Split &sp, int steps) {
    const int parts = parts_of(steps, sp.parts, prefix_least<E>());
    return bytes_of<E> ? max(parts, parts_of(steps, sp.fine, SHORT_PREFIX)) : parts;
}
template <class E> __host__ __device__ constexpr int whole_steps() { return E::RUN == 8 ? 16 : 1; }
template <class E> __device__ __forceinline__ int prompt_parts(int steps, int most) {
    return steps <= whole_steps<E>() ? 1 : parts_of(steps, most, tile_least<E>());
}

template <class E, int HD> struct TileShared {
    run4 lds[2][2][tile_positions<E, HD>() * HD / E::RUN];  // two buffers of K and V
    int least[8];
};

// The runs as they are, or of 8-bit pages the widened ones.
template <int N, int M> __device__ __forceinline__ run4 (&of_raw(run4 (&x)[N], run4 (&)[M]))[N] { return x; }
template <int N> __device__ __forceinline__ run4 (&of_raw(run2 (&)[N], run4 (&x)[N]))[N] { return x; }

// W waves of 32 rows each. at.x: a tile and kv head, at.y: a part of its positions.
template <class E, int HD, int W, bool PREFIX>
__device__ __forceinline__ void tile_rows(const PagedAttendArgs &a, const Split &sp, Place at, TileShared<E, HD> &shared) {
    typedef typename E::T T;
    typedef RowState<E, HD> S;
    constexpr int RUN = E::RUN, R = 32 * W, THREADS = 64 * W;
    constexpr int KT = tile_positions<E, HD>();
    constexpr int SUB = KT / 32;
    constexpr int KCH = HD / RUN, VCH = KT / RUN;                 // 16-byte runs per row of a tile
    constexpr int N = KT * KCH / THREADS;                             // loads of each thread per K (V) tile
    typedef std::conditional_t<bytes_of<E>, run2, run4> Raw;          // a run as it lies in a page
    typedef typename E::P P;
    auto &lds = shared.lds;
    auto &least = shared.least;
    const PagedArgs &p = a.p;
    const int lane = threadIdx.x & 63, m = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    const int kvh = at.x % p.n_kv_head;
    int unit = at.x / p.n_kv_head, tile = unit;
    Tile t;
    Row row;
    if constexpr (PREFIX) {
        if (!prefix_tile<R>(a, tile, t)) return;
        row = prefix_row<R>(a, tile, t, kvh, 32 * wave + m);
    } else {
        if (!prompt_tile_by_size<R, KT == 64 ? 6 : 5>(p, unit, at.nx / p.n_kv_head, unit, tile, t)) return;
        row = prompt_row<R>(p, tile, t, kvh, 32 * wave + m);
    }
    const int steps = (t.top + KT - 1) / KT, parts = PREFIX ? prefix_parts<E>(sp, steps) : prompt_parts<E>(steps, sp.parts);
    if (at.y >= parts) return;
    const int2 range = part_steps(steps, parts, at.y);
    const Pages<E> g = pages_of<E, HD>(p, t.seq, kvh);
    // the table's entry for position step * KT + lane, looked at a step later (a use at once would wait for it)
    const auto entry = [&](int step) { return g.table[min(step * KT + (lane & (KT - 1)), t.n_kv - 1) >> p.page_log]; };
    int next = range.x < range.y ? entry(range.x) : 0;  // the first one is what everything waits for
    // positions that all rows attend to, and that any of this wave's does
    const int mine = wave_reduce(row.limit, 0x7FFFFFFF, [](int x, int y) { return min(x, y); });
    if (lane == 0) least[wave] = mine;
    __syncthreads();
    int all = least[0];
#pragma unroll
    for (int w = 1; w < W; ++w) all = min(all, least[w]);
    all = __builtin_amdgcn_readfirstlane(all);
    const int any = wave_reduce(row.limit, 0, [](int x, int y) { return max(x, y); });

    run4 q[S::QS];
    {
        const T *x = (const T *)a.q + (size_t)max(row.at, 0LL) * HD;
#pragma unroll
        for (int c = 0; c < S::QS; ++c) q[c] = *(const run4 *)(x + (2 * c + (lane >> 5)) * RUN);
    }
    S st;
    st.clear();

    // runs of a tile's row are exchanged by the row's number, so that 16 lanes that read the same run of consecutive
    // rows meet all banks
    const auto k_swap = [](int r) { return KCH >= 16 ? r & 15 : (r >> 1) & 7; };
    const auto v_swap = [](int r) { return VCH >= 16 ? r & 15 : (r >> 1) & 7; };
    // This thread's runs of a K and V tile: number at = 256 i + thread, in row at / KCH (at / VCH). A tile inside one page
    // is a uniform address and a lane's offset; with smaller pages every run asks for its page. They pass through
    // registers: loads straight into LDS return a quarter as much per cycle.
    const bool one_page = 1 << p.page_log >= KT;
    // (step's page: the table's entry for its position of this lane)
    const auto page_or_0 = [&](int id) { return (unsigned)id < (unsigned)p.n_page ? id : 0; };
    // (8-bit pages: and the scales, of the lane's position for K, of its run for V)
    uint32_t k_unit = 0, v_unit = 0;
    const auto load_k = [&](Raw (&x)[N], int step, int id) {
        const int t0 = step * KT;
        const uint32_t tid = fresh(threadIdx.x);
        if constexpr (bytes_of<E>) k_unit = g.k_scale[scale_at(p, g, page_or_0(id), t0 + (tid & (KT - 1)))];
        if (one_page) {
            const int page = page_or_0(__builtin_amdgcn_readfirstlane(id));
            const char *k = (const char *)(g.k + (size_t)page * g.step + (size_t)(t0 & g.mask) * HD);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = *(const Raw *)(k + i * (THREADS * sizeof(Raw)) + tid * sizeof(Raw));
        } else {
            // (a wave's 64 runs are rows of one page: 64 / KCH rows from a multiple of that)
            static_assert(64 / KCH <= 16, "a wave's runs in one page");
            const int page = page_or_0(id);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = (THREADS * i + 64 * wave) / KCH;
                const char *k = (const char *)(g.k + (size_t)__builtin_amdgcn_readlane(page, r) * g.step +
                                               (size_t)((t0 + r) & g.mask) * HD);
                x[i] = *(const Raw *)(k + (tid & 63) * sizeof(Raw));
            }
        }
    };
    const auto load_v = [&](Raw (&x)[N], int step, int id) {
        const int t0 = step * KT;
        const uint32_t tid = fresh(threadIdx.x);
        if (one_page) {
            const int page = page_or_0(__builtin_amdgcn_readfirstlane(id));
            if constexpr (bytes_of<E>) v_unit = g.v_scale[scale_at(p, g, page, t0 + tid % VCH * RUN)];
            const char *v = (const char *)(g.v + (size_t)page * g.step + (t0 & g.mask));
            const uint32_t v_lane = (uint32_t)(((tid / VCH) << p.page_log) + (tid % VCH) * RUN) * (uint32_t)sizeof(P);
#pragma unroll
            for (int i = 0; i < N; ++i)
                x[i] = *(const Raw *)(v + (size_t)i * ((THREADS / VCH * sizeof(P)) << p.page_log) + v_lane);
        } else {
            const int page = page_or_0(id);
            const uint32_t c = tid % VCH;
            const int of_run = __shfl(page, c * RUN, WAVE);
            if constexpr (bytes_of<E>) v_unit = g.v_scale[scale_at(p, g, of_run, t0 + c * RUN)];
            const P *v = g.v + (size_t)of_run * g.step + ((t0 + c * RUN) & g.mask);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = *(const Raw *)(v + ((size_t)((THREADS * i + tid) / VCH) << p.page_log));
        }
    };
    // positions of a step that can be read
    const auto readable = [&](int step, int id) {
        return __ballot((unsigned)id < (unsigned)p.n_page && step * KT + (lane & (KT - 1)) < t.n_kv);
    };
    // the loaded runs into their buffer; V at positions that cannot be read may be anything: 0 in its place
    // (8-bit pages: as bf16, once for all rows; widened by each wave for its own, the tile's 128 conversions per wave
    // would cost as much as its products)
    const auto put_k = [&](const Raw (&x)[N], int step) {
        run4 *to = lds[step & 1][0];
        const uint32_t tid = fresh(threadIdx.x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t r = (THREADS * i + tid) / KCH;
            run4 y;
            if constexpr (bytes_of<E>)  // (the wave's rows have one scale)
                y = widen(x[i][0], x[i][1], unit_of(__builtin_amdgcn_readlane(k_unit, (THREADS * i + 64 * wave) / KCH)));
            else y = x[i];
            to[r * KCH + ((tid % KCH) ^ k_swap(r))] = y;
        }
    };
    // (a position that a row does not attend to weighs nothing, whatever lies there; but nothing times an infinity or NaN
    // is NaN: where some row does not see all of a tile that has one, the rows are done again, attend_again)
    uint32_t bad = 0;
    const auto put_v = [&](Raw (&raw)[N], int step, unsigned long long valid) {
        run4 *to = lds[step & 1][1];
        const uint32_t tid = fresh(threadIdx.x);
        run4 wide_runs[bytes_of<E> ? N : 1];
        if constexpr (bytes_of<E>) {
#pragma unroll
            for (int i = 0; i < N; ++i) wide_runs[i] = widen(raw[i][0], raw[i][1], unit_of(v_unit));
        }
        run4 (&x)[N] = of_raw(raw, wide_runs);
        if (valid != ~0ull) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = keep_elements<E>(x[i], (uint32_t)(valid >> (tid % VCH * RUN)));
        }
        if ((step + 1) * KT > all) {
#pragma unroll
            for (int i = 0; i < N; ++i) bad |= any_not_finite<E>(x[i]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t r = (THREADS * i + tid) / VCH;
            to[r * VCH + ((tid % VCH) ^ v_swap(r))] = x[i];
        }
    };

    if (range.x < range.y) {
        const int last = range.y - 1;
        Raw kr[N], vr[N];
        load_k(kr, range.x, next);
        load_v(vr, range.x, next);
        unsigned long long valid = readable(range.x, next);
        put_k(kr, range.x);
        put_v(vr, range.x, valid);
        next = entry(min(range.x + 1, last));
        const auto attend_step = [&](auto masked, int step) {
            __syncthreads();  // the step's tile is there, and the other buffer is read
            const int t0 = step * KT;
            if (step < last) {
                load_k(kr, step + 1, next);
                load_v(vr, step + 1, next);
            }
            const int after = entry(min(step + 2, last));
            if (!masked || t0 < any) {
                const run4 *kt = lds[step & 1][0], *vt = lds[step & 1][1];
                // this lane's first run of a K and V tile's block; the others by exchanging bits of its place
                const uint32_t x = fresh(threadIdx.x);
                const int h = x >> 5 & 1, m = x & 31;
                const int k_first = kv_row<E>(m) * KCH + (h ^ k_swap(kv_row<E>(m))), v_first = m * VCH + (h ^ v_swap(m));
                // (the wave that has products to issue goes first: the other one of its SIMD has exponentials, more often
                // than not, and both pipes are busy; 8192 tokens 575 -> 568 us)
                __builtin_amdgcn_s_setprio(1);
                v16f s[SUB];
#pragma unroll
                for (int b = 0; b < SUB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
                // every operand is read AHEAD products before its own (left alone, the compiler reads it right before, and
                // each product waits for LDS)
                constexpr int NK = SUB * S::QS, AHEAD = 6;
                run4 ring[AHEAD];
                const auto read = [&](int i) {
                    if (i < NK) ring[i % AHEAD] = kt[32 * (i % SUB) * KCH + (k_first ^ (2 * (i / SUB)))];
                };
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) read(i);
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    s[i % SUB] = Mma<E>::mul(ring[i % AHEAD], q[i / SUB], s[i % SUB]);
                    read(i + AHEAD);
                }
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(0);
                if constexpr (masked) {
                    // bit 32 b + kv_reg(i, 0): the row attends to that register's position
                    const int seen = row.limit - t0;
                    unsigned long long mask = seen >= 64 ? valid : seen > 0 ? valid & ((1ull << seen) - 1) : 0ull;
                    if (__any(mask != ~0ull)) {
                        mask >>= RUN * h;
#pragma unroll
                        for (int b = 0; b < SUB; ++b)
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                s[b][i] = (uint32_t)(mask >> (32 * b)) >> kv_reg<E>(i, 0) & 1u ? s[b][i] : NEG_INF;
                    }
                }
                st.template softmax<SUB>(s, a.scale);
#pragma unroll
                for (int c = 0; c < SUB * S::PS; ++c) {
                    const run4 w = S::weights(s[c / S::PS], c % S::PS);
#pragma unroll
                    for (int d = 0; d < S::DB; ++d)
                        st.o[d] = Mma<E>::mul(vt[32 * d * VCH + (v_first ^ (2 * c))], w, st.o[d]);
                }
                order_reads<E, SUB * S::PS * S::DB>();
            }
            if (step < last) {
                valid = readable(step + 1, next);
                put_k(kr, step + 1);
                put_v(vr, step + 1, valid);
                next = after;
            }
        };
        // steps that all rows see whole, then the others: in one loop, the two would meet with their scores in different
        // registers, and every step would move them
        int step = range.x;
        for (; step < min(all / KT, range.y) && valid == ~0ull; ++step) attend_step(std::false_type{}, step);
        for (; step < range.y; ++step) attend_step(std::true_type{}, step);
    }
    const size_t slot = ((size_t)(unit * p.n_kv_head + kvh) * sp.parts + at.y) * W + wave;
    const bool part = PREFIX || parts > 1;
    if (range.x < range.y && range.y * KT > all) {
        // (`least` was read before the first tile's barrier)
        const bool some = __any(bad != 0);
        if (lane == 0) least[wave] = some;
        __syncthreads();
        int again = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) again |= least[w];
        again = __builtin_amdgcn_readfirstlane(again);
        if (again) {
            attend_again<E, HD>(a, sp.many, part, t.seq, t.n_kv, kvh, range.x * KT, min(range.y * KT, any), slot, row.limit,
                                row.at);
            return;
        }
    }
    const float l = add_halves(st.l), f = part ? 1.0f : over(l);
    const int h = lane >> 5;
    if (part && h == 0) sp.many.ml[slot * 32 + m] = make_float2(st.m, l);
#pragma unroll
    for (int d = 0; d < S::DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int four = 8 * d + i / 2 + h;  // dimensions 4 four ..
            const float4 y = make_float4(st.o[d][i] * f, st.o[d][i + 1] * f, st.o[d][i + 2] * f, st.o[d][i + 3] * f);
            if (part) sp.many.o[(slot * (HD / 4) + four) * 32 + m] = y;
            else if (row.at >= 0) put_out<E>(a.out, a.out_f32, (size_t)row.at * HD + 4 * four, y);
        }
}

template <class E, int HD, int W>
__global__ __launch_bounds__(64 * W, W == 8 || HD * sizeof(typename E::T) <= 256 ? 2 : 1)
void paged_tiles(PagedAttendArgs a, Split sp) {
    __shared__ __align__(16) TileShared<E, HD> shared;
    tile_rows<E, HD, W, false>(a, sp, {(int)blockIdx.x, (int)blockIdx.y, (int)gridDim.x, (int)gridDim.y}, shared);
}

// A decode batch with groups: the first nx * ny workgroups have the tiles of the shared positions, the others the
// sequences' own, which run beside them (48 sequences, 4100 shared positions and up to 500 of their own: 22 us; as two
// launches 15.5 + 14.5).
template <class E, int HD>
__global__ __launch_bounds__(256, HD * sizeof(typename E::T) <= 256 ? 2 : 1) void paged_decode(PagedAttendArgs a, Split sp,
                                                                                           int nx, int ny, int cols) {
    __shared__ __align__(16) union {
        TileShared<E, HD> tile;
        FewShared<HD> few;
    } shared;
    int at = blockIdx.x;
    if (at < nx * ny) {
        tile_rows<E, HD, 4, true>(a, sp, {at % nx, at / nx, nx, ny}, shared.tile);
    } else {
        at -= nx * ny;
        few_rows<E, HD, true>(a, sp, {at / cols, at % cols, ((int)gridDim.x - nx * ny) / cols, cols}, shared.few);
    }
}

// ---- the parts together ------------------------------------------------------------

// Up to ROWS rows, 32 of their dimensions (share number blockIdx.z), out of `n` parts: part z's statistics of row r are
// ml(z, r), its O of four dimensions o(z, r, four). Groups of threads share the parts among them, and the first loads of O do
// not wait for the statistics: few loads wait for each other, which is what this would spend its time on (1 x 4100
// positions, 33 parts: 14 -> 7 us).
constexpr int JOIN_MOST = 256, TILE_PARTS = 64;  // parts of a row at the most, of a prompt's tile
template <class E, int HD, int ROWS, class Ml, class O, class At>
__device__ __forceinline__ void join(const PagedAttendArgs &a, int n, int rows, Ml ml, O o, At at) {
    constexpr int FOURS = 8, GROUPS = 256 / (ROWS * FOURS), K = 256 / ROWS, HELD = 4;
    __shared__ float2 stats[JOIN_MOST * ROWS];
    __shared__ float side[K][ROWS];
    __shared__ float4 sums[GROUPS][FOURS * ROWS];
    const int r = threadIdx.x % ROWS, k = threadIdx.x / ROWS, f = k % FOURS, group = k / FOURS;
    const int four = blockIdx.z * FOURS + f;
    const bool here = r < rows;
    for (int z = k; z < n; z += K) stats[z * ROWS + r] = here ? ml(z, r) : make_float2(NEG_INF, 0.0f);
    float4 held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int z = group + i * GROUPS;
        held[i] = here && z < n ? o(z, r, four) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float top = NEG_INF;
    for (int z = k; z < n; z += K) top = fmaxf(top, stats[z * ROWS + r].x);  // this thread's own writes
    side[k][r] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < K; ++i) top = fmaxf(top, side[i][r]);
    __syncthreads();
    float l = 0.0f;
    for (int z = k; z < n; z += K) {
        const float2 x = stats[z * ROWS + r];
        const float w = exp2_fast(x.x - against(top));
        stats[z * ROWS + r].x = w;
        l = __builtin_fmaf(x.y, w, l);
    }
    side[k][r] = l;
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < K; ++i) l += side[i][r];
    const float by = over(l);
    const long long row = here ? at(r) : -1;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto add = [&](float4 x, float w) {
        y.x = __builtin_fmaf(x.x, w, y.x);
        y.y = __builtin_fmaf(x.y, w, y.y);
        y.z = __builtin_fmaf(x.z, w, y.z);
        y.w = __builtin_fmaf(x.w, w, y.w);
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int z = group + i * GROUPS;
        if (z < n) add(held[i], stats[z * ROWS + r].x);
    }
    if (here) {
#pragma unroll 8
        for (int z = group + HELD * GROUPS; z < n; z += GROUPS) add(o(z, r, four), stats[z * ROWS + r].x);
    }
    sums[group][f * ROWS + r] = y;
    __syncthreads();
    if (row >= 0 && !group) {
#pragma unroll
        for (int i = 1; i < GROUPS; ++i) add(sums[i][f * ROWS + r], 1.0f);
        put_out<E>(a.out, a.out_f32, (size_t)row * HD + 4 * four, make_float4(y.x * by, y.y * by, y.z * by, y.w * by));
    }
}

// The same for 16 rows with few parts and all their dimensions: every thread adds the parts of its own runs of four, whose
// first loads do not wait for the statistics either. Bound: memory (512 tokens, 4 parts, 34 MB read: 8.3 us, by join 9.5).
template <class E, int HD, class Ml, class O, class At>
__device__ __forceinline__ void join_whole(const PagedAttendArgs &a, int n, int rows, Ml ml, O o, At at) {
    constexpr int ROWS = 16, K = 256 / ROWS, RUNS = HD / 4 / K, HELD = 4;
    __shared__ float2 stats[TILE_PARTS * ROWS];
    const int r = threadIdx.x % ROWS, k = threadIdx.x / ROWS;
    const bool here = r < rows;
    for (int z = k; z < n; z += K) stats[z * ROWS + r] = here ? ml(z, r) : make_float2(NEG_INF, 0.0f);
    float4 held[HELD][RUNS];
#pragma unroll
    for (int z = 0; z < HELD; ++z)
#pragma unroll
        for (int i = 0; i < RUNS; ++i) held[z][i] = here && z < n ? o(z, r, k + K * i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
    float top = NEG_INF, l = 0.0f;
    for (int z = 0; z < n; ++z) top = fmaxf(top, stats[z * ROWS + r].x);
    const float ref = against(top);
    float4 y[RUNS];
#pragma unroll
    for (int i = 0; i < RUNS; ++i) y[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto add = [&](int z, const float4 (&x)[RUNS]) {
        const float2 s = stats[z * ROWS + r];
        const float w = exp2_fast(s.x - ref);
        l = __builtin_fmaf(s.y, w, l);
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            y[i].x = __builtin_fmaf(x[i].x, w, y[i].x);
            y[i].y = __builtin_fmaf(x[i].y, w, y[i].y);
            y[i].z = __builtin_fmaf(x[i].z, w, y[i].z);
            y[i].w = __builtin_fmaf(x[i].w, w, y[i].w);
        }
    };
#pragma unroll
    for (int z = 0; z < HELD; ++z)
        if (z < n) add(z, held[z]);
#pragma unroll 2
    for (int z = HELD; z < n; ++z) {
        float4 x[RUNS];
#pragma unroll
        for (int i = 0; i < RUNS; ++i) x[i] = here ? o(z, r, k + K * i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        add(z, x);
    }
    const long long row = here ? at(r) : -1;
    if (row < 0) return;
    const float by = over(l);
#pragma unroll
    for (int i = 0; i < RUNS; ++i)
        put_out<E>(a.out, a.out_f32, (size_t)row * HD + 4 * (k + K * i),
                   make_float4(y[i].x * by, y[i].y * by, y[i].z * by, y[i].w * by));
}

// blockIdx.x: a tile of R rows and kv head of a prompt batch, blockIdx.y: 16 of its rows.
template <class E, int HD, int R>
__global__ __launch_bounds__(256) void paged_join(PagedAttendArgs a, Split sp) {
    const PagedArgs &p = a.p;
    const int unit = blockIdx.x / p.n_kv_head, kvh = blockIdx.x % p.n_kv_head;
    constexpr bool FEW = R == 16;
    constexpr int STEP = FEW ? few_step<E> : tile_positions<E, HD>();
    int tile = unit;
    Tile t;
    if (!prompt_tile<R>(p, tile, t)) return;
    const int steps = (t.top + STEP - 1) / STEP, parts = FEW ? parts_of(steps, sp.parts, 1) : prompt_parts<E>(steps, sp.parts);
    const int first = 16 * blockIdx.y;
    if (parts < 2 || first >= t.rows) return;
    const Parts x = FEW ? sp.few : sp.many;
    const size_t slot = (size_t)(unit * p.n_kv_head + kvh) * sp.parts;
    const int block = FEW ? 0 : first / 32, place = FEW ? 0 : first % 32;
    const auto at = [&](int z) { return FEW ? slot + z : (slot + z) * (R / 32) + block; };
    const auto ml = [&](int z, int r) { return x.ml[at(z) * (FEW ? 16 : 32) + place + r]; };
    const auto o = [&](int z, int r, int four) { return x.o[(at(z) * (HD / 4) + four) * (FEW ? 16 : 32) + place + r]; };
    const auto row = [&](int r) { return prompt_row<R>(p, tile, t, kvh, first + r).at; };
    if constexpr (FEW) join<E, HD, 16>(a, parts, min(t.rows - first, 16), ml, o, row);
    else join_whole<E, HD>(a, parts, min(t.rows - first, 16), ml, o, row);
}

// blockIdx.x: a sequence, blockIdx.y: a kv head and block of 16 of its query heads. R: rows of the prefix's tiles. ROWS: at
// least the rows of a slot.
template <class E, int HD, int R, int ROWS>
__global__ __launch_bounds__(256) void paged_join_decode(PagedAttendArgs a, Split sp) {
    const PagedArgs &p = a.p;
    const int lane = threadIdx.x & 63, seq = blockIdx.x, per = (p.group + 15) / 16;
    const int kvh = blockIdx.y / per, head = (blockIdx.y % per) * 16;
    const DecodePlan plan = decode_plan<E>(a, sp);
    Own own;
    const int before = parts_before(a, plan, seq, own), units = own.units(plan.cut);
    const bool prefix = own.shared && own.n;
    if (!prefix && units < 2) return;
    int parts = 0, base = 0;  // of the prefix, and the number of the group's first row among its 32-row blocks
    long long first = 0;
    if (prefix) {
        int number = 0, tiles = 0;
        const Group g = group_of(a, seq, number);
        for (int i = lane; i < number; i += WAVE) tiles = add_tiles(tiles, prefix_units<R>(a, group_at(a, i)), sp.tiles);
        base = wave_reduce(tiles, 0, [](int x, int y) { return x + y; });
        constexpr int KT = tile_positions<E, HD>();
        parts = prefix_parts<E>(sp, (readable_of(p, g.shared) + KT - 1) / KT);
        first = (long long)(seq - g.first) * p.group + head;
    }
    const auto many = [&](int z, int r) {  // the slot of a row's 32-row block
        const long long x = first + r;
        const size_t tile = (size_t)tile_of_row(base, x, R, sp.tiles);
        return (tile * p.n_kv_head + kvh) * sp.parts * (R / 32) + (size_t)z * (R / 32) + (size_t)(x % R) / 32;
    };
    const auto few = [&](int z) { return (size_t)(before + z - parts) * gridDim.y + blockIdx.y; };
    const int w = sp.few_rows;
    join<E, HD, ROWS>(
        a, parts + units, min(p.group - head, 16),
        [&](int z, int r) {
            return z < parts ? sp.many.ml[many(z, r) * 32 + (first + r) % 32] : sp.few.ml[few(z) * w + r];
        },
        [&](int z, int r, int four) {
            return z < parts ? sp.many.o[(many(z, r) * (HD / 4) + four) * 32 + (first + r) % 32]
                             : sp.few.o[(few(z) * (HD / 4) + four) * w + r];
        },
        [&](int r) { return (long long)seq * p.n_head + kvh * p.group + head + r; });
}

// ---- launches ------------------------------------------------------------------------

constexpr int CUS = 256;

// Scratch for slots of both kinds; false: none is to be had.
bool room(Split &sp, size_t many, size_t few, int few_rows, int hd) {
    const size_t o_many = many * hd * 32, o_few = few * hd * few_rows;  // floats
    char *p = (char *)lib_scratch((o_many + o_few) * 4 + (many * 32 + few * few_rows) * 8);
    if (!p) return false;
    sp.many.o = (float4 *)p;
    sp.few.o = (float4 *)(p + o_many * 4);
    sp.many.ml = (float2 *)(p + (o_many + o_few) * 4);
    sp.few.ml = sp.many.ml + many * 32;
    sp.few_rows = few_rows;
    return true;
}

int queued() { return hipGetLastError() == hipSuccess ? 0 : -1; }

template <class E, int HD, int W>
int prompt_tiles(const PagedAttendArgs &a, hipStream_t st) {
    const PagedArgs &p = a.p;
    constexpr int R = 32 * W, KT = tile_positions<E, HD>();
    const long long rows = (long long)p.n_tok * p.group, tiles = rows / R + std::min(p.n_seq, p.n_tok);
    const long long busy = (rows + R - 1) / R * p.n_kv_head, want = CUS * 8 / W;
    const long long top = (long long)p.max_page << p.page_log;
    const long long most = top <= KT * whole_steps<E>() ? 1 : top / (KT * tile_least<E>());
    Split sp{};
    // parts for two workgroups per CU (single calls, 512 tokens after 7000: 91 us, for four 98, in one part 163); f32's steps
    // are long, and a causal prompt's last tile has twice the steps of the mean: up to 4 parts where the workgroups then
    // need two turns (2048 tokens of 12 heads of 64 114 us, 142 in one turn, 4096 282, 389)
    const long long turns = E::RUN == 4 ? std::min(2 * want / busy, 4LL) : 0;
    sp.parts = at_least_one(std::max(want / busy, turns), most, TILE_PARTS);
    if (tiles * p.n_kv_head > 0x7FFFFFFF / 512) return -1;
    if (sp.parts > 1 && !room(sp, (size_t)tiles * p.n_kv_head * sp.parts * W, 0, 16, HD)) return -1;
    const dim3 grid((unsigned)(tiles * p.n_kv_head), sp.parts);
    hipLaunchKernelGGL((paged_tiles<E, HD, W>), grid, dim3(64 * W), 0, st, a, sp);
    if (sp.parts > 1) hipLaunchKernelGGL((paged_join<E, HD, R>), dim3(grid.x, R / 16), dim3(256), 0, st, a, sp);
    return queued();
}

// Workgroups of paged_few that are resident at once.
template <int HD> constexpr int few_resident() { return (HD <= 128 ? 3 : 2) * CUS; }

template <class E, int HD>
int prompt_few(const PagedAttendArgs &a, hipStream_t st) {
    const PagedArgs &p = a.p;
    // as many workgroups as are resident (16 tokens after 12000 positions: 33.5 us, for 2 per CU 42, for 4 40)
    const TilePlan plan = plan_tiles((long long)p.n_tok * p.group, std::min(p.n_seq, p.n_tok), 16, p.n_kv_head, few_resident<HD>(),
                                     ((long long)p.max_page << p.page_log) / few_step<E>, 128);
    const long long tiles = plan.tiles;
    Split sp{};
    sp.parts = plan.parts;
    if (tiles * p.n_kv_head > 0x7FFFFFFF / 512) return -1;
    if (sp.parts > 1 && !room(sp, 0, (size_t)tiles * p.n_kv_head * sp.parts, 16, HD)) return -1;
    const dim3 grid((unsigned)(tiles * p.n_kv_head), sp.parts);
    hipLaunchKernelGGL((paged_few<E, HD, false>), grid, dim3(256), 0, st, a, sp);
    if (sp.parts > 1) hipLaunchKernelGGL((paged_join<E, HD, 16>), dim3(grid.x, 1, HD / 32), dim3(256), 0, st, a, sp);
    return queued();
}

// Whether eight waves' rows fit the registers of four SIMDs.
template <class E, int HD> constexpr bool wide() { return HD * sizeof(typename E::T) <= 256; }

template <class E, int HD>
int prompt_as(const PagedAttendArgs &a, hipStream_t st) {
    const PagedArgs &p = a.p;
    const long long total = (long long)p.n_tok * p.group, rows = total / p.n_seq;  // and of a sequence, on average
    const long long top = (long long)p.max_page << p.page_log;
    // few rows per sequence or in all, or little work by what the table holds: 16-row tiles spread it further, but each reads
    // its keys again (32 query and 4 kv heads of bf16: 45 tokens 6.3 us, in larger tiles 9.6; 16 after 500 positions 14.3 and
    // 21.5, after 3000 20.8 and 22.7, after 12000 36 and 42; 64 after 500, 1.2 M rows x positions, 16.8 and 20.6; 32 after
    // 3000, 3.1 M, 27.9 and 20.9). The wrong way at its far end: 24 after 12000 46 and 36, 16 after 30000 66 and 56. One way
    // for the whole batch, by its mean: a long prompt among many short sequences, or in a list of mostly empty places, is
    // taken 16 rows at a time (4096 tokens in 1024 places 939 us, in 256 165, alone 154; 2000 tokens beside 400 single ones 311,
    // in two calls 60 and 87)
    if (rows <= 64 || total * p.n_kv_head <= 768 || total * p.n_kv_head * top <= 5 << 19) return prompt_few<E, HD>(a, st);
    // 8-bit pages, whose 16-row steps are 64 positions: also where tiles would not be split and the 16-row ones are resident
    // at once with some to spare (256 tokens after 500 positions 15.8 us, in larger tiles 25.0; 9 x 40 after 900 18.6 and 30.6;
    // 16 query and 8 kv heads: 512 tokens 11.4 and 18.6; heads of 256: 9 x 100 after 900 38.9 and 55.7). Beyond: 9 x 100 after
    // 900 of 16 and 8 heads, 584 tiles, 31.8 and 32.4; 400 tokens, 800 tiles, 19.2 and 17.1; 128 tokens after 1500 25.2 and 20.6.
    // Missed: sequences behind longer contexts (16 of up to 20 tokens after 2000, 38.8, in 16-row tiles 28.2), and any whose table
    // is wider than they need, since the lengths are on the device (the first three with tables of 17 to 2048 pages: 27.3, 32.7, 21.0)
    if (bytes_of<E> && top <= tile_positions<E, HD>() * whole_steps<E>() && total * p.n_kv_head <= 16 * few_resident<HD>() * 3 / 4)
        return prompt_few<E, HD>(a, st);
    // eight waves where all CUs still have work (32 query heads on 4: 4096 tokens 175 us, four waves 195; 3000 110 and 101)
    if constexpr (wide<E, HD>())
        if (rows >= 1024 && total * p.n_kv_head >= 512 * 256) return prompt_tiles<E, HD, 8>(a, st);
    return prompt_tiles<E, HD, 4>(a, st);
}

template <class E, int HD>
int decode_as(const PagedAttendArgs &a, hipStream_t st) {
    const PagedArgs &p = a.p;
    constexpr int R = 128, KT = tile_positions<E, HD>();
    const int per = (p.group + 15) / 16, cols = p.n_kv_head * per;
    const long long top = (long long)p.max_page << p.page_log;
    Split sp{};
    // parts of the sequences' own positions: 4 workgroups per CU, one part per sequence at least (64 x 500 to 2000 positions,
    // 164 MB: 37.5 us, 2 per CU 44, 1 per CU 51; all of 2000, 263 MB: 52.6, 51.6, 47.5); a row's should fill the GPU once
    // where there are few columns
    const int target = std::min(std::max(1, 4 * CUS / cols), JOIN_MOST - 66);
    sp.per_item = 1.0 / ((double)target * few_step<E>);
    sp.per_row = 1.0 / ((double)std::max(FEW_PARTS, CUS / cols) * few_step<E>);
    const long long items = std::min<long long>((long long)p.n_seq + target + 1,
                                                (long long)p.n_seq * ((top + few_step<E> - 1) / few_step<E>));
    long long tiles = 0, slots = 0;
    if (a.n_groups) {
        // (groups of one sequence share nothing)
        const TilePlan plan = plan_tiles((long long)p.n_seq * p.group, std::min(a.n_groups, p.n_seq / 2), R, p.n_kv_head, 2 * CUS,
                                         top / (KT * prefix_least<E>()), 64);
        tiles = plan.tiles;
        sp.parts = plan.parts;
        sp.tiles = (int)tiles;
        // short parts in two fifths of the places, two workgroups per CU, that the sequences' own positions leave: past that
        // two tiles share a CU (4 kv heads, 48 sequences behind 4100: 8 parts 26.5 us, 10 25.5, 12 24.4, 14 26.4, 16 28.6;
        // behind 3900 26.4, 23.9, 26.3, 27.5, 28.8; 32 behind 4100 25.7, 24.5, 23.0, 22.6, 23.0; where nothing is left,
        // 12 kv heads of 64 and 64 sequences behind 3600, 7 parts 25.8 us, 11 26.6)
        const long long filled = std::max(((long long)p.n_seq * p.group + R - 1) / R, (long long)std::min(a.n_groups, p.n_seq / 2));
        sp.fine = bytes_of<E> && tiles ? at_least_one((2LL * CUS - (long long)p.n_seq * cols) * 2 / (5 * filled * p.n_kv_head),
                                                      top / (KT * SHORT_PREFIX), 64) : 1;
        sp.parts = std::max(sp.parts, sp.fine);
        slots = tiles * p.n_kv_head * sp.parts * 4;
    }
    if (items * cols > 0x7FFFFFFF / 512 || cols > 65535 || tiles * p.n_kv_head > 0x7FFFFFFF / 512) return -1;
    const bool join = a.n_groups || top > few_step<E>;
    if (join && !room(sp, slots, (size_t)items * cols, std::min(p.group, 16), HD)) return -1;
    if (a.n_groups) {
        const long long nx = tiles * p.n_kv_head, grid = nx * sp.parts + items * cols;
        if (grid > 0x7FFFFFFF / 512) return -1;
        hipLaunchKernelGGL((paged_decode<E, HD>), dim3((unsigned)grid), dim3(256), 0, st, a, sp, (int)nx, sp.parts, cols);
    } else {
        hipLaunchKernelGGL((paged_few<E, HD, true>), dim3((unsigned)(items * cols)), dim3(256), 0, st, a, sp);
    }
    if (join) {
        const dim3 grid(p.n_seq, cols, HD / 32);
        if (p.group <= 8) hipLaunchKernelGGL((paged_join_decode<E, HD, R, 8>), grid, dim3(256), 0, st, a, sp);
        else hipLaunchKernelGGL((paged_join_decode<E, HD, R, 16>), grid, dim3(256), 0, st, a, sp);
    }
    return queued();
}

template <class E>
int paged_attend(const PagedAttendArgs &a, bool decode, hipStream_t st) {
    const std::lock_guard<std::mutex> lk(lib_scratch_mutex());
    if (a.p.hd == 64) return decode ? decode_as<E, 64>(a, st) : prompt_as<E, 64>(a, st);
    if (a.p.hd == 128) return decode ? decode_as<E, 128>(a, st) : prompt_as<E, 128>(a, st);
    if (a.p.hd == 256) return decode ? decode_as<E, 256>(a, st) : prompt_as<E, 256>(a, st);
    return -1;
}

}  // namespace
}  // namespace llamd

// paged_attend.hpp -- causal attention over a paged cache: prompts (any number of new tokens per sequence, after any
// cached context) and decode batches (one token per sequence, prefixes that sequences share read once).
//
//   o = sum_j softmax_j(scale q . k_j) v_j,   j = 0 .. the token's position
//
// Rows: the query heads of a kv head's group, for all tokens of a sequence, are numbered token by token, and a tile
// takes consecutive ones: with 8 query heads per kv head, a tile of 256 rows is 32 tokens, whose keys and values are
// read once for all 8.
//
// Two kernels form O. paged_tiles: many rows; the waves of a workgroup have rows of their own and share K and V tiles in
// LDS. paged_rows: up to 32 rows; the waves share the rows and have positions of their own, read straight into the
// matrix operands. Either may have a part of a row's positions only; then O (unnormalised), the maximum and the sum
// go to scratch and paged_join puts the parts together.
#pragma once

#include <algorithm>
#include <mutex>

#include "launch.hpp"
#include "paged_wave.hpp"

namespace llamd {
namespace {

// What prompt and decode calls of this batch are split into (host), and where parts lie.
struct Split {
    float4 *part_o;   // [slot][HD / 8][64] a 32-row block's O: 4 dimensions of a row per lane
    float2 *part_ml;  // [slot][32] maximum and sum
    int parts;        // most parts of a row tile (prompt, prefix)
    int prefix_slots; // decode: slots [0, prefix_slots) are the prefix's
    int target;       // decode: workgroups wanted per kv head and block of 32 heads
};

// ---- rows ------------------------------------------------------------------------

// A tile's rows, and this lane's of them.
struct Tile {
    int seq;              // the sequence whose table is read
    int n_kv;             // its positions that can be read
    int top;              // positions that the tile's last row attends to
};
struct Row {
    long long at;         // token * n_head + head, -1: no row
    int limit;            // positions that it attends to
};

// Tile number `tile` (R rows) of a prompt batch; false past the last. rows_end: rows in it.
template <int R>
__device__ __forceinline__ bool prompt_tile(const PagedArgs &p, int &tile, Tile &t, int &rows_end, TokenSpan &span) {
    t.seq = find_sequence(p.n_seq, tile, [&](int s) {
        const TokenSpan x = token_span(p, s);
        return (int)(((long long)(x.end - x.first) * p.group + R - 1) / R);
    });
    if (t.seq < 0) return false;
    span = token_span(p, t.seq);
    rows_end = (int)min((long long)(span.end - span.first) * p.group - (long long)R * tile, (long long)R);
    t.n_kv = held(p, t.seq);
    const int last = span.first + (int)(((long long)R * tile + rows_end - 1) / p.group);
    t.top = max(min(p.len[t.seq] - (span.end - last) + 1, t.n_kv), 0);
    return true;
}

// Row i of it (the last one for rows that it has not).
template <int R>
__device__ __forceinline__ Row prompt_row(const PagedArgs &p, int tile, const Tile &t, int rows_end, TokenSpan span, int kvh,
                                          int i) {
    const long long at = (long long)R * tile + min(i, rows_end - 1);
    const int tok = span.first + (int)(at / p.group), head = (int)(at % p.group);
    Row r;
    r.limit = max(min(p.len[t.seq] - (span.end - tok) + 1, t.n_kv), 0);
    r.at = i < rows_end ? (long long)tok * p.n_head + kvh * p.group + head : -1;
    return r;
}

// The group of a sequence: its members [first, end) and the positions that they share (whole pages); none shared where a
// group has no two members.
struct Group {
    int first, end, shared;
};
__device__ __forceinline__ Group group_at(const PagedAttendArgs &a, int g) {
    Group x;
    x.first = min(max(a.group_at[g], 0), a.p.n_seq);
    x.end = min(max(a.group_at[g + 1], x.first), a.p.n_seq);
    x.shared = x.end - x.first < 2 ? 0 : max(a.shared[g], 0) & ~((1 << a.p.page_log) - 1);
    return x;
}
__device__ __forceinline__ Group group_of(const PagedAttendArgs &a, int s, int *number = nullptr) {
    int lo = 0, hi = a.n_groups;  // the last group that begins at or before s
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.group_at[mid] <= s) lo = mid + 1;
        else hi = mid;
    }
    Group x = {s, s + 1, 0};
    if (lo) {
        const Group y = group_at(a, lo - 1);
        if (s >= y.first && s < y.end) {
            x = y;
            if (number) *number = lo - 1;
        }
    }
    return x;
}

// Tile number `tile` of the rows of all groups that share something.
template <int R>
__device__ __forceinline__ int prefix_units(const PagedAttendArgs &a, int g) {
    const Group x = group_at(a, g);
    return x.shared ? (int)(((long long)(x.end - x.first) * a.p.group + R - 1) / R) : 0;
}
template <int R>
__device__ __forceinline__ bool prefix_tile(const PagedAttendArgs &a, int &tile, Tile &t, int &rows_end, Group &g) {
    const int n = find_sequence(a.n_groups, tile, [&](int i) { return prefix_units<R>(a, i); });
    if (n < 0) return false;
    g = group_at(a, n);
    rows_end = (int)min((long long)(g.end - g.first) * a.p.group - (long long)R * tile, (long long)R);
    t.seq = g.first;
    t.n_kv = t.top = (int)min((long long)g.shared, (long long)a.p.max_page << a.p.page_log);
    return true;
}
template <int R>
__device__ __forceinline__ Row prefix_row(const PagedAttendArgs &a, int tile, const Tile &t, int rows_end, const Group &g,
                                          int kvh, int i) {
    const long long at = (long long)R * tile + min(i, rows_end - 1);
    const int seq = g.first + (int)(at / a.p.group), head = (int)(at % a.p.group);
    Row r;
    r.limit = min(held(a.p, seq), t.n_kv);
    r.at = i < rows_end ? (long long)seq * a.p.n_head + kvh * a.p.group + head : -1;
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

template <class E, int HD>
__device__ __forceinline__ void write_part(const Split &sp, size_t slot, const RowState<E, HD> &st, float l) {
    const int lane = threadIdx.x & 63;
    float4 *o = sp.part_o + slot * (HD / 8 * 64) + lane;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            o[(d * 4 + i / 4) * 64] = make_float4(st.o[d][i], st.o[d][i + 1], st.o[d][i + 2], st.o[d][i + 3]);
    if (lane < 32) sp.part_ml[slot * 32 + lane] = make_float2(st.m, l);
}

// ---- one wave, straight from the pages -----------------------------------------------

// Where a kv head's pages are.
template <class E> struct Pages {
    const typename E::T *k, *v;
    const int32_t *table;
    size_t step;  // elements between pages
    int mask;     // positions per page - 1
};
template <class E, int HD>
__device__ __forceinline__ Pages<E> pages_of(const PagedArgs &p, int seq, int kvh) {
    const size_t head = (size_t)kvh * HD << p.page_log;
    return {(const typename E::T *)p.k + head, (const typename E::T *)p.v + head, p.table + (size_t)seq * p.max_page,
            (size_t)p.n_kv_head * HD << p.page_log, (1 << p.page_log) - 1};
}

template <class E, int HD>
__device__ __forceinline__ void load_rows(run4 (&q)[HD / (2 * E::RUN)], const void *from, long long at) {
    const typename E::T *x = (const typename E::T *)from + (size_t)max(at, 0LL) * HD;
    const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int c = 0; c < HD / (2 * E::RUN); ++c) q[c] = *(const run4 *)(x + (2 * c + h) * E::RUN);
}

// 32 rows against the positions t0 .. t0 + 31 of every STRIDE from `begin` to `end` (a multiple of 32 from begin, or
// all that the rows attend to).
template <class E, int HD, int STRIDE>
__device__ __forceinline__ void attend_pages(const PagedArgs &p, const Pages<E> &g, const Tile &t, int limit, int begin,
                                             int end, const run4 (&q)[HD / (2 * E::RUN)], float scale,
                                             RowState<E, HD> &st) {
    typedef typename E::T T;
    typedef RowState<E, HD> S;
    constexpr int RUN = E::RUN;
    const int lane = threadIdx.x & 63, h = lane >> 5;
    for (int t0 = begin; t0 < end; t0 += STRIDE) {
        const int pos = t0 + kv_row<E>(lane & 31), posc = min(pos, t.n_kv - 1);
        const int page = page_of(p, g.table, posc);
        // bit m: the position of the first product's row m can be read
        const uint32_t valid = (uint32_t)__ballot(page >= 0 && pos < t.n_kv);
        const T *k = g.k + (size_t)max(page, 0) * g.step + (size_t)(posc & g.mask) * HD;
        v16f s[1];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[0][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < S::QS; ++c) s[0] = Mma<E>::mul(*(const run4 *)(k + (2 * c + h) * RUN), q[c], s[0]);
        const bool whole = __all(limit >= t0 + 32) && valid == 0xFFFFFFFFu;
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool seen = t0 + kv_reg<E>(i, h) < limit && (valid >> (8 * (i >> 2) + (i & 3) + 4 * h) & 1);
                s[0][i] = seen ? s[0][i] : NEG_INF;
            }
        }
        st.template softmax<1>(s, scale);
#pragma unroll
        for (int c = 0; c < S::PS; ++c) {
            const run4 w = S::weights(s[0], c);
            const int vp = t0 + RUN * (2 * c + h), vpc = min(vp, (t.n_kv - 1) & ~(RUN - 1));
            const int page = page_of(p, g.table, vpc);
            const T *v = g.v + (size_t)max(page, 0) * g.step + (vpc & g.mask);
            const auto v_run = [&](int d) { return *(const run4 *)(v + ((size_t)(32 * d + (lane & 31)) << p.page_log)); };
            if (whole) {
#pragma unroll
                for (int d = 0; d < S::DB; ++d) st.o[d] = Mma<E>::mul(v_run(d), w, st.o[d]);
            } else {
                // positions that no row attends to may hold anything
                const int n = page < 0 ? 0 : min(max(end - vp, 0), RUN);
                st.add_masked(v_run, (1u << n) - 1u, w, t0 + 2 * RUN * c, limit);
            }
        }
    }
}

// ---- many rows -------------------------------------------------------------------

typedef __attribute__((address_space(3))) void *lds_ptr;

// x, as something that the compiler cannot keep the results of between tiles: addresses are cheaper made again than held
// in registers.
__device__ __forceinline__ uint32_t fresh(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

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

// Least steps of a part.
constexpr int TILE_STEPS = 4;

// O over the sum, to this lane's row (at < 0: none).
template <class E, int HD>
__device__ __forceinline__ void write_rows(void *out, bool f32, long long at, RowState<E, HD> &st, float l) {
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[d][i] *= f;
    if (at >= 0) st.write(out, f32, (size_t)at);
}

// A wave's rows once more, straight from the pages, every infinity or NaN in V added only where it belongs. A function of
// its own: its registers would cost paged_tiles some of the reads that it keeps in flight.
struct Again {
    PagedArgs p;
    Split sp;
    Tile t;
    int kvh, begin, end;
    const void *q;
    void *out;  // null: a part, to `slot`
    bool out_f32;
    float scale;
    size_t slot;
};
template <class E, int HD>
__device__ __attribute__((noinline)) void attend_again(const Again &x, int limit, long long at) {
    run4 q[HD / (2 * E::RUN)];
    load_rows<E, HD>(q, x.q, at);
    RowState<E, HD> st;
    st.clear();
    attend_pages<E, HD, 32>(x.p, pages_of<E, HD>(x.p, x.t.seq, x.kvh), x.t, limit, x.begin, x.end, q, x.scale, st);
    const float l = add_halves(st.l);
    if (x.out) write_rows<E, HD>(x.out, x.out_f32, at, st, l);
    else write_part<E, HD>(x.sp, x.slot, st, l);
}

// W waves of 32 rows each.
template <class E, int HD, int W, bool PREFIX>
__global__ __launch_bounds__(64 * W, W == 8 || HD * sizeof(typename E::T) <= 256 ? 2 : 1) void paged_tiles(PagedAttendArgs a, Split sp) {
    typedef typename E::T T;
    typedef RowState<E, HD> S;
    constexpr int RUN = E::RUN, R = 32 * W, THREADS = 64 * W;
    constexpr int KT = HD * sizeof(T) * 256 <= 131072 ? 64 : 32;  // positions per tile: two buffers of K and V in 128 KB
    constexpr int SUB = KT / 32;
    constexpr int KCH = HD / RUN, VCH = KT / RUN;                 // 16-byte runs per row of a tile
    constexpr int N = KT * KCH / THREADS;                             // loads of each thread per K (V) tile
    __shared__ __align__(16) run4 lds[2][2][KT * KCH];
    const PagedArgs &p = a.p;
    const int lane = threadIdx.x & 63, m = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // the last tiles, which have the most positions, go first
    const int unit = gridDim.x / p.n_kv_head - 1 - blockIdx.x / p.n_kv_head, kvh = blockIdx.x % p.n_kv_head;
    int tile = unit, rows_end;
    Tile t;
    Row row;
    if constexpr (PREFIX) {
        Group g;
        if (!prefix_tile<R>(a, tile, t, rows_end, g)) return;
        row = prefix_row<R>(a, tile, t, rows_end, g, kvh, 32 * wave + m);
    } else {
        TokenSpan span;
        if (!prompt_tile<R>(p, tile, t, rows_end, span)) return;
        row = prompt_row<R>(p, tile, t, rows_end, span, kvh, 32 * wave + m);
    }
    const int steps = (t.top + KT - 1) / KT, parts = parts_of(steps, sp.parts, TILE_STEPS);
    if ((int)blockIdx.y >= parts) return;
    const int2 range = part_steps(steps, parts, blockIdx.y);
    // positions that all rows of this wave attend to, and that any does
    const int all = wave_reduce(row.limit, 0x7FFFFFFF, [](int x, int y) { return min(x, y); });
    const int any = wave_reduce(row.limit, 0, [](int x, int y) { return max(x, y); });

    run4 q[S::QS];
    load_rows<E, HD>(q, a.q, row.at);
    S st;
    st.clear();
    const Pages<E> g = pages_of<E, HD>(p, t.seq, kvh);

    // runs of a tile's row are exchanged by the row's number, so that 16 lanes that read the same run of consecutive
    // rows meet all banks
    const auto k_swap = [](int r) { return KCH >= 16 ? r & 15 : (r >> 1) & 7; };
    const auto v_swap = [](int r) { return VCH >= 16 ? r & 15 : (r >> 1) & 7; };
    // the table's entry for position step * KT + lane, looked at a step later (a use at once would wait for it)
    const auto entry = [&](int step) { return g.table[min(step * KT + (lane & (KT - 1)), t.n_kv - 1) >> p.page_log]; };
    // This thread's runs of a K and V tile: number at = 256 i + thread, in row at / KCH (at / VCH). A tile inside one page
    // is a uniform address and a lane's offset; with smaller pages every run asks for its page. They pass through
    // registers: loads straight into LDS return a quarter as much per cycle.
    const bool one_page = 1 << p.page_log >= KT;
    // (step's page: the table's entry for its position of this lane)
    const auto page_or_0 = [&](int id) { return (unsigned)id < (unsigned)p.n_page ? id : 0; };
    const auto load_k = [&](run4 (&x)[N], int step, int id) {
        const int t0 = step * KT;
        const uint32_t tid = fresh(threadIdx.x);
        if (one_page) {
            const int page = page_or_0(__builtin_amdgcn_readfirstlane(id));
            const char *k = (const char *)(g.k + (size_t)page * g.step + (size_t)(t0 & g.mask) * HD);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = *(const run4 *)(k + i * (THREADS * 16) + tid * 16);
        } else {
            const int page = page_or_0(id);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint32_t r = (THREADS * i + tid) / KCH, c = tid % KCH;
                x[i] = *(const run4 *)(g.k + (size_t)__shfl(page, r, WAVE) * g.step +
                                       (size_t)((t0 + r) & g.mask) * HD + c * RUN);
            }
        }
    };
    const auto load_v = [&](run4 (&x)[N], int step, int id) {
        const int t0 = step * KT;
        const uint32_t tid = fresh(threadIdx.x);
        if (one_page) {
            const int page = page_or_0(__builtin_amdgcn_readfirstlane(id));
            const char *v = (const char *)(g.v + (size_t)page * g.step + (t0 & g.mask));
            const uint32_t v_lane = (uint32_t)(((tid / VCH) << p.page_log) + (tid % VCH) * RUN) * (uint32_t)sizeof(T);
#pragma unroll
            for (int i = 0; i < N; ++i)
                x[i] = *(const run4 *)(v + (size_t)i * ((THREADS / VCH * sizeof(T)) << p.page_log) + v_lane);
        } else {
            const int page = page_or_0(id);
            const uint32_t c = tid % VCH;
            const T *v = g.v + (size_t)__shfl(page, c * RUN, WAVE) * g.step + ((t0 + c * RUN) & g.mask);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = *(const run4 *)(v + ((size_t)((THREADS * i + tid) / VCH) << p.page_log));
        }
    };
    // positions of a step that can be read
    const auto readable = [&](int step, int id) {
        return __ballot((unsigned)id < (unsigned)p.n_page && step * KT + (lane & (KT - 1)) < t.n_kv);
    };
    // the loaded runs into their buffer; V at positions that cannot be read may be anything: 0 in its place
    const auto put_k = [&](const run4 (&x)[N], int step) {
        run4 *to = lds[step & 1][0];
        const uint32_t tid = fresh(threadIdx.x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t r = (THREADS * i + tid) / KCH;
            to[r * KCH + ((tid % KCH) ^ k_swap(r))] = x[i];
        }
    };
    const auto put_v = [&](run4 (&x)[N], int step, unsigned long long valid) {
        run4 *to = lds[step & 1][1];
        const uint32_t tid = fresh(threadIdx.x);
        if (valid != ~0ull) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = keep_elements<E>(x[i], (uint32_t)(valid >> (tid % VCH * RUN)));
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t r = (THREADS * i + tid) / VCH;
            to[r * VCH + ((tid % VCH) ^ v_swap(r))] = x[i];
        }
    };

    bool again = false;
    if (range.x < range.y) {
        const int last = range.y - 1;
        run4 kr[N], vr[N];
        int next = entry(range.x);
        load_k(kr, range.x, next);
        load_v(vr, range.x, next);
        unsigned long long valid = readable(range.x, next);
        put_k(kr, range.x);
        put_v(vr, range.x, valid);
        next = entry(min(range.x + 1, last));
        for (int step = range.x; step < range.y; ++step) {
            __syncthreads();  // the step's tile is there, and the other buffer is read
            const int t0 = step * KT;
            if (step < last) {
                load_k(kr, step + 1, next);
                load_v(vr, step + 1, next);
            }
            const int after = entry(min(step + 2, last));
            if (t0 < any) {
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
#pragma unroll
                for (int c = 0; c < S::QS; ++c)
#pragma unroll
                    for (int b = 0; b < SUB; ++b) s[b] = Mma<E>::mul(kt[32 * b * KCH + (k_first ^ (2 * c))], q[c], s[b]);
                order_reads<E, SUB * S::QS>();
                __builtin_amdgcn_s_setprio(0);
                if (t0 + KT > all || valid != ~0ull) {
                    // a position that a row does not attend to weighs nothing, whatever lies there; but nothing times an
                    // infinity or NaN is NaN: where V has one, these rows are done again (attend_again)
#pragma unroll
                    for (int b = 0; b < SUB; ++b)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int at = 32 * b + kv_reg<E>(i, h);
                            s[b][i] = t0 + at < row.limit && (valid >> at & 1) ? s[b][i] : NEG_INF;
                        }
                    uint32_t bad = 0;
#pragma unroll 4
                    for (int i = 0; i < KT * KCH / 64; ++i) bad |= not_finite<E>(vt[i * 64 + (x & 63)]);
                    again |= __any(bad != 0);
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
        }
    }
    const size_t slot = ((size_t)(unit * p.n_kv_head + kvh) * sp.parts + blockIdx.y) * W + wave;
    if (again) {
        Again x;
        x.p = p;
        x.sp = sp;
        x.t = t;
        x.kvh = kvh;
        x.begin = range.x * KT;
        x.end = min(range.y * KT, any);
        x.q = a.q;
        x.out = PREFIX || parts > 1 ? nullptr : a.out;
        x.out_f32 = a.out_f32;
        x.scale = a.scale;
        x.slot = slot;
        attend_again<E, HD>(x, row.limit, row.at);
        return;
    }
    const float l = add_halves(st.l);
    if (PREFIX || parts > 1) write_part<E, HD>(sp, slot, st, l);
    else write_rows<E, HD>(a.out, a.out_f32, row.at, st, l);
}

// ---- up to 32 rows ---------------------------------------------------------------

// Least positions of a part: one step of each wave.
constexpr int ROWS_STEP = 128;

// A decode batch's own positions (behind the shared ones): tail(s) of sequence s, cut into parts of `cut`.
struct DecodePlan {
    int cut;
};
__device__ __forceinline__ int tail_of(const PagedAttendArgs &a, int s) {
    const int n = held(a.p, s);
    return a.n_groups ? max(n - group_of(a, s).shared, 0) : n;
}
__device__ __forceinline__ DecodePlan decode_plan(const PagedAttendArgs &a, const Split &sp) {
    const int lane = threadIdx.x & 63;
    double sum = 0.0;  // exact: lengths are integers
    for (int s = lane; s < a.p.n_seq; s += WAVE) sum += (double)tail_of(a, s);
    sum = wave_sum_d(sum);
    DecodePlan d;
    // (at most 2^31 - 1 positions per sequence: a part of a whole sequence at the most)
    d.cut = (int)min(max(ceil(sum / sp.target / ROWS_STEP), 1.0) * ROWS_STEP, 2147483520.0);
    return d;
}
// Parts of sequence s: one at least where nothing is shared, so that an empty sequence's rows are written.
__device__ __forceinline__ int decode_units(const PagedAttendArgs &a, const DecodePlan &d, int s) {
    const int n = held(a.p, s), shared = a.n_groups ? group_of(a, s).shared : 0;
    const int units = n > shared ? (n - shared - 1) / d.cut + 1 : 0;
    return shared && n ? units : max(units, 1);
}

// DECODE: blockIdx.x a part of a sequence, blockIdx.y a kv head and block of 32 of its query heads. Otherwise blockIdx.x
// a tile of 32 rows of a prompt batch and a kv head, blockIdx.y a part of its positions.
template <class E, int HD, bool DECODE>
__global__ __launch_bounds__(256) void paged_rows(PagedAttendArgs a, Split sp) {
    typedef RowState<E, HD> S;
    __shared__ float stats[2][4][32];
    __shared__ __align__(16) float part[2][S::DB * 16][64];
    const PagedArgs &p = a.p;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
    Tile t;
    Row r;
    int begin, end, parts, kvh;
    size_t slot;
    if constexpr (DECODE) {
        const DecodePlan plan = decode_plan(a, sp);
        int unit = blockIdx.x;
        t.seq = find_sequence(p.n_seq, unit, [&](int s) { return decode_units(a, plan, s); });
        if (t.seq < 0) return;
        const int per = (p.group + 31) / 32, head = (blockIdx.y % per) * 32 + (lane & 31);
        kvh = blockIdx.y / per;
        t.n_kv = r.limit = held(p, t.seq);
        const int shared = a.n_groups ? group_of(a, t.seq).shared : 0;
        r.at = head < p.group ? (long long)t.seq * p.n_head + kvh * p.group + head : -1;
        begin = (int)min((long long)shared + (long long)unit * plan.cut, 0x7FFFFFFFLL);
        end = (int)min((long long)begin + plan.cut, (long long)t.n_kv);
        parts = shared && t.n_kv ? 2 : decode_units(a, plan, t.seq);
        slot = sp.prefix_slots + (size_t)blockIdx.x * gridDim.y + blockIdx.y;
    } else {
        kvh = blockIdx.x % p.n_kv_head;
        const int unit = gridDim.x / p.n_kv_head - 1 - blockIdx.x / p.n_kv_head;
        int tile = unit, rows_end;
        TokenSpan span;
        if (!prompt_tile<32>(p, tile, t, rows_end, span)) return;
        r = prompt_row<32>(p, tile, t, rows_end, span, kvh, lane & 31);
        const int steps = (t.top + ROWS_STEP - 1) / ROWS_STEP;
        parts = parts_of(steps, sp.parts, 1);
        if ((int)blockIdx.y >= parts) return;
        const int2 range = part_steps(steps, parts, blockIdx.y);
        begin = range.x * ROWS_STEP;
        end = min(range.y * ROWS_STEP, t.top);
        slot = (size_t)(unit * p.n_kv_head + kvh) * sp.parts + blockIdx.y;
    }
    run4 q[S::QS];
    load_rows<E, HD>(q, a.q, r.at);
    S st;
    st.clear();
    attend_pages<E, HD, ROWS_STEP>(p, pages_of<E, HD>(p, t.seq, kvh), t, r.limit, begin + 32 * wave, end, q, a.scale, st);

    // the four waves' positions together
    st.l = add_halves(st.l);
    if (h == 0) {
        stats[0][wave][lane] = st.m;
        stats[1][wave][lane] = st.l;
    }
    __syncthreads();
    float m = NEG_INF, l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, stats[0][w][lane & 31]);
#pragma unroll
    for (int w = 0; w < 4; ++w)
        l = __builtin_fmaf(stats[1][w][lane & 31], exp2_fast(stats[0][w][lane & 31] - against(m)), l);
    const float f = exp2_fast(st.m - against(m)) * (parts > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l);
#pragma unroll
    for (int d = 0; d < S::DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[d][i] *= f;
#pragma unroll
    for (int half = 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int d = 0; d < S::DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) part[wave - half][d * 16 + i][lane] = st.o[d][i];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int d = 0; d < S::DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) st.o[d][i] += part[wave][d * 16 + i][lane];
        }
        __syncthreads();
    }
    if (wave) return;
    if (parts > 1) {
        st.m = m;
        write_part<E, HD>(sp, slot, st, l);
    } else if (r.at >= 0) {
        st.write(a.out, a.out_f32, (size_t)r.at);
    }
}

// ---- the parts together ------------------------------------------------------------

// Adds parts [0, n) of a 32-row block, slot(z) each, to the running maximum, sum and this wave's quarter of O; twice
// over the statistics, once over O.
template <int HD, class Slot>
__device__ __forceinline__ float join_top(const Split &sp, int n, float top, Slot slot) {
    for (int z = 0; z < n; ++z) top = fmaxf(top, sp.part_ml[slot(z) * 32 + (threadIdx.x & 31)].x);
    return top;
}
template <int HD, class Slot>
__device__ __forceinline__ void join_add(const Split &sp, int n, float top, float &l, float4 (&o)[HD / 32], Slot slot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int z = 0; z < n; ++z) {
        const float2 ml = sp.part_ml[slot(z) * 32 + (lane & 31)];
        const float f = exp2_fast(ml.x - against(top));
        l = __builtin_fmaf(ml.y, f, l);
        const float4 *x = sp.part_o + slot(z) * (HD / 8 * 64) + lane;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            const float4 y = x[(wave * (HD / 32) + i) * 64];
            o[i].x = __builtin_fmaf(y.x, f, o[i].x);
            o[i].y = __builtin_fmaf(y.y, f, o[i].y);
            o[i].z = __builtin_fmaf(y.z, f, o[i].z);
            o[i].w = __builtin_fmaf(y.w, f, o[i].w);
        }
    }
}
template <class E, int HD>
__device__ __forceinline__ void join_write(const PagedAttendArgs &a, float l, const float4 (&o)[HD / 32], long long at) {
    const int h = (threadIdx.x >> 5) & 1, wave = threadIdx.x >> 6;
    if (at < 0) return;
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
        const int q = wave * (HD / 32) + i;  // four dimensions 32 (q / 4) + 8 (q % 4) + 4 h
        const size_t to = (size_t)at * HD + 32 * (q / 4) + 8 * (q % 4) + 4 * h;
        const float4 x = make_float4(o[i].x * f, o[i].y * f, o[i].z * f, o[i].w * f);
        if (a.out_f32) put4<ElemF32>(a.out, to, x);
        else put4<E>(a.out, to, x);
    }
}

// blockIdx.x: a tile of R rows and kv head of a prompt batch, blockIdx.y: 32 of its rows.
template <class E, int HD, int R>
__global__ __launch_bounds__(256) void paged_join(PagedAttendArgs a, Split sp) {
    const PagedArgs &p = a.p;
    const int unit = blockIdx.x / p.n_kv_head, kvh = blockIdx.x % p.n_kv_head;
    constexpr int KT = R == 32 ? ROWS_STEP : HD * sizeof(typename E::T) * 256 <= 131072 ? 64 : 32;
    int tile = unit, rows_end;
    Tile t;
    TokenSpan span;
    if (!prompt_tile<R>(p, tile, t, rows_end, span)) return;
    const int parts = parts_of((t.top + KT - 1) / KT, sp.parts, R == 32 ? 1 : TILE_STEPS);
    if (parts < 2 || 32 * (int)blockIdx.y >= rows_end) return;
    const Row r = prompt_row<R>(p, tile, t, rows_end, span, kvh, 32 * blockIdx.y + (threadIdx.x & 31));
    const auto slot = [&](int z) {
        return ((size_t)(unit * p.n_kv_head + kvh) * sp.parts + z) * (R / 32) + blockIdx.y;
    };
    float l = 0.0f;
    float4 o[HD / 32] = {};
    join_add<HD>(sp, parts, join_top<HD>(sp, parts, NEG_INF, slot), l, o, slot);
    join_write<E, HD>(a, l, o, r.at);
}

// blockIdx.x: a sequence, blockIdx.y: a kv head and block of 32 of its query heads. R: rows of the prefix's tiles.
template <class E, int HD, int R>
__global__ __launch_bounds__(256) void paged_join_decode(PagedAttendArgs a, Split sp) {
    const PagedArgs &p = a.p;
    const int lane = threadIdx.x & 63, seq = blockIdx.x, per = (p.group + 31) / 32;
    const int kvh = blockIdx.y / per, head = (blockIdx.y % per) * 32 + (lane & 31);
    const DecodePlan plan = decode_plan(a, sp);
    const int units = decode_units(a, plan, seq);
    int number = 0;
    const Group g = a.n_groups ? group_of(a, seq, &number) : Group{seq, seq + 1, 0};
    const bool prefix = g.shared && held(p, seq);
    if (!prefix && units < 2) return;
    int before = 0;  // parts of the sequences before this one
    for (int s = lane; s < seq; s += WAVE) before += decode_units(a, plan, s);
    before = wave_reduce(before, 0, [](int x, int y) { return x + y; });
    const auto slot = [&](int z) { return sp.prefix_slots + (size_t)(before + z) * gridDim.y + blockIdx.y; };
    float top = join_top<HD>(sp, units, NEG_INF, slot), l = 0.0f;
    float4 o[HD / 32] = {};
    if (prefix) {
        // this lane's row among the group's: its 32-row block and its place there, in the prefix's parts
        int tiles = 0;
        for (int i = lane; i < number; i += WAVE) tiles += prefix_units<R>(a, i);
        tiles = wave_reduce(tiles, 0, [](int x, int y) { return x + y; });
        const int n_kv = (int)min((long long)g.shared, (long long)p.max_page << p.page_log);
        constexpr int KT = HD * sizeof(typename E::T) * 256 <= 131072 ? 64 : 32;
        const int parts = parts_of((n_kv + KT - 1) / KT, sp.parts, TILE_STEPS);
        const long long row = (long long)(seq - g.first) * p.group + min(head, p.group - 1);
        const size_t unit = tiles + (size_t)(row / R);
        const auto at = [&](int z) {
            return ((unit * p.n_kv_head + kvh) * sp.parts + z) * (R / 32) + (size_t)(row % R) / 32;
        };
        const int place = (int)(row & 31), wave = threadIdx.x >> 6;
        for (int z = 0; z < parts; ++z) top = fmaxf(top, sp.part_ml[at(z) * 32 + place].x);
        for (int z = 0; z < parts; ++z) {
            const float2 ml = sp.part_ml[at(z) * 32 + place];
            const float f = exp2_fast(ml.x - against(top));
            l = __builtin_fmaf(ml.y, f, l);
            const float4 *x = sp.part_o + at(z) * (HD / 8 * 64) + (lane & 32) + place;
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
                const float4 y = x[(wave * (HD / 32) + i) * 64];
                o[i].x = __builtin_fmaf(y.x, f, o[i].x);
                o[i].y = __builtin_fmaf(y.y, f, o[i].y);
                o[i].z = __builtin_fmaf(y.z, f, o[i].z);
                o[i].w = __builtin_fmaf(y.w, f, o[i].w);
            }
        }
    }
    join_add<HD>(sp, units, top, l, o, slot);
    join_write<E, HD>(a, l, o, head < p.group ? (long long)seq * p.n_head + kvh * p.group + head : -1);
}

// ---- launches ------------------------------------------------------------------------

constexpr int CUS = 256;

size_t slot_bytes(int hd) { return (size_t)hd * 128 + 256; }

// Scratch for `slots` parts (null: none is needed, or none is to be had).
bool room(Split &sp, size_t slots, int hd) {
    if (!slots) return true;
    char *p = (char *)lib_scratch(slots * slot_bytes(hd));
    if (!p) return false;
    sp.part_o = (float4 *)p;
    sp.part_ml = (float2 *)(p + slots * (size_t)hd * 128);
    return true;
}

int queued() { return hipGetLastError() == hipSuccess ? 0 : -1; }

template <class E, int HD, int W>
int prompt_tiles(const PagedAttendArgs &a, hipStream_t st) {
    const PagedArgs &p = a.p;
    constexpr int R = 32 * W, KT = HD * sizeof(typename E::T) * 256 <= 131072 ? 64 : 32;
    const long long rows = (long long)p.n_tok * p.group, tiles = rows / R + p.n_seq;
    const long long busy = (rows + R - 1) / R * p.n_kv_head, want = CUS * 8 / W;
    const long long most = ((long long)p.max_page << p.page_log) / (KT * TILE_STEPS);
    Split sp{};
    sp.parts = (int)std::max(1LL, std::min({(want + busy - 1) / busy, most, 64LL}));
    if (tiles * p.n_kv_head > 0x7FFFFFFF / 256) return -1;
    if (sp.parts > 1 && !room(sp, (size_t)tiles * p.n_kv_head * sp.parts * (R / 32), HD)) return -1;
    const dim3 grid((unsigned)(tiles * p.n_kv_head), sp.parts);
    hipLaunchKernelGGL((paged_tiles<E, HD, W, false>), grid, dim3(64 * W), 0, st, a, sp);
    if (sp.parts > 1)
        hipLaunchKernelGGL((paged_join<E, HD, R>), dim3(grid.x, R / 32), dim3(256), 0, st, a, sp);
    return queued();
}

template <class E, int HD>
int prompt_rows(const PagedAttendArgs &a, hipStream_t st) {
    const PagedArgs &p = a.p;
    const long long rows = (long long)p.n_tok * p.group, tiles = rows / 32 + p.n_seq;
    const long long busy = (rows + 31) / 32 * p.n_kv_head, want = 2 * CUS;
    const long long most = ((long long)p.max_page << p.page_log) / ROWS_STEP;
    Split sp{};
    sp.parts = (int)std::max(1LL, std::min({(want + busy - 1) / busy, most, 256LL}));
    if (tiles * p.n_kv_head > 0x7FFFFFFF / 256) return -1;
    if (sp.parts > 1 && !room(sp, (size_t)tiles * p.n_kv_head * sp.parts, HD)) return -1;
    const dim3 grid((unsigned)(tiles * p.n_kv_head), sp.parts);
    hipLaunchKernelGGL((paged_rows<E, HD, false>), grid, dim3(256), 0, st, a, sp);
    if (sp.parts > 1) hipLaunchKernelGGL((paged_join<E, HD, 32>), dim3(grid.x, 1), dim3(256), 0, st, a, sp);
    return queued();
}

template <class E, int HD>
int prompt_as(const PagedAttendArgs &a, hipStream_t st) {
    const long long rows = (long long)a.p.n_tok * a.p.group / a.p.n_seq;  // of a sequence, on average
    if (rows <= 96) return prompt_rows<E, HD>(a, st);
    return rows >= 1024 ? prompt_tiles<E, HD, 8>(a, st) : prompt_tiles<E, HD, 4>(a, st);
}

template <class E, int HD, int W>
int decode_with(const PagedAttendArgs &a, hipStream_t st) {
    const PagedArgs &p = a.p;
    constexpr int R = 32 * W, KT = HD * sizeof(typename E::T) * 256 <= 131072 ? 64 : 32;
    const int per = (p.group + 31) / 32, cols = p.n_kv_head * per;
    const long long top = (long long)p.max_page << p.page_log;
    Split sp{};
    // parts of the sequences' own positions: 4 workgroups per CU, one part per sequence at least
    sp.target = std::max(1, 4 * CUS / cols);
    const long long cut_min = ROWS_STEP, items =
        std::min<long long>((long long)p.n_seq + sp.target, (long long)p.n_seq * ((top + cut_min - 1) / cut_min));
    long long tiles = 0;
    if (a.n_groups) {
        const long long rows = (long long)p.n_seq * p.group;
        tiles = rows / R + a.n_groups;
        const long long busy = (rows + R - 1) / R * p.n_kv_head, want = CUS * 8 / W;
        sp.parts = (int)std::max(1LL, std::min({(want + busy - 1) / busy, top / (KT * TILE_STEPS), 64LL}));
        const long long slots = tiles * p.n_kv_head * sp.parts * (R / 32);
        if (slots > 0x7FFFFFFF / 256) return -1;
        sp.prefix_slots = (int)slots;
    }
    if (items > 0x7FFFFFFF / 256 || cols > 65535) return -1;
    const bool join = a.n_groups || top > ROWS_STEP;
    if (join && !room(sp, sp.prefix_slots + (size_t)items * cols, HD)) return -1;
    if (a.n_groups)
        hipLaunchKernelGGL((paged_tiles<E, HD, W, true>), dim3((unsigned)(tiles * p.n_kv_head), sp.parts), dim3(64 * W),
                           0, st, a, sp);
    hipLaunchKernelGGL((paged_rows<E, HD, true>), dim3((unsigned)items, cols), dim3(256), 0, st, a, sp);
    if (join) hipLaunchKernelGGL((paged_join_decode<E, HD, R>), dim3(p.n_seq, cols), dim3(256), 0, st, a, sp);
    return queued();
}

template <class E, int HD>
int decode_as(const PagedAttendArgs &a, hipStream_t st) {
    const long long rows = a.n_groups ? (long long)a.p.n_seq * a.p.group / a.n_groups : 0;  // of a group, on average
    return rows >= 1024 ? decode_with<E, HD, 8>(a, st) : decode_with<E, HD, 4>(a, st);
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

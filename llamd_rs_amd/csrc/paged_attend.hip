// paged_attend.hip -- causal attention over a paged cache: prompts (any number of new tokens per sequence, after any
// cached context) and decode batches (one token per sequence).
//
//   o = sum_j softmax_j(scale q . k_j) v_j,   j = 0 .. the token's position
//
// Rows: the query heads of a kv head's group, for all tokens of a sequence, are numbered token by token, and a tile
// takes consecutive ones: with 8 query heads per kv head, a tile of 32 rows is 4 tokens, whose keys and values are read
// once for all 8.
#include "launch.hpp"
#include "paged_wave.hpp"

namespace llamd {
namespace {

// Where a workgroup's rows are, and this lane's row.
struct Rows {
    int seq;
    int n_kv;             // positions of the sequence that can be read
    int top;              // positions that the tile's last row attends to
    int limit;            // positions that this lane's row attends to
    long long row;        // token * n_head + head, -1: no row
};

// Tile `tile` (32 rows) of the whole batch; false past the last.
__device__ __forceinline__ bool prompt_rows(const PagedArgs &p, int tile, int kvh, Rows &r) {
    const int seq = find_sequence(p.n_seq, tile, [&](int s) {
        const TokenSpan t = token_span(p, s);
        return (int)(((long long)(t.end - t.first) * p.group + 31) / 32);
    });
    if (seq < 0) return false;
    const TokenSpan t = token_span(p, seq);
    const int n_rows_end = (int)min((long long)(t.end - t.first) * p.group - 32LL * tile, 32LL);
    const int i = threadIdx.x & 31;
    const long long at = 32LL * tile + min(i, n_rows_end - 1);
    const int tok = t.first + (int)(at / p.group), head = (int)(at % p.group);
    const int last = t.first + (int)((32LL * tile + n_rows_end - 1) / p.group);
    r.seq = seq;
    r.n_kv = held(p, seq);
    r.limit = max(min(p.len[seq] - (t.end - tok) + 1, r.n_kv), 0);
    r.top = max(min(p.len[seq] - (t.end - last) + 1, r.n_kv), 0);
    r.row = i < n_rows_end ? (long long)tok * p.n_head + kvh * p.group + head : -1;
    return true;
}

template <class E, int HD, bool DECODE>
__global__ __launch_bounds__(256) void paged_rows(PagedAttendArgs a) {
    typedef typename E::T T;
    typedef RowState<E, HD> S;
    constexpr int RUN = E::RUN;
    __shared__ float stats[2][4][32];
    __shared__ __align__(16) float part[2][S::DB * 16][64];
    const PagedArgs &p = a.p;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6, kvh = blockIdx.y;
    const int slot_mask = (1 << p.page_log) - 1;
    Rows r;
    int shared = 0;
    const int32_t *own, *first;
    if constexpr (DECODE) {
        const int per = (p.group + 31) / 32, part_of = blockIdx.x % per;
        r.seq = blockIdx.x / per;
        r.n_kv = r.limit = r.top = held(p, r.seq);
        const int head = part_of * 32 + (lane & 31);
        r.row = head < p.group ? (long long)r.seq * p.n_head + kvh * p.group + head : -1;
        own = first = p.table + (size_t)r.seq * p.max_page;
        if (a.n_groups) {
            int unit = r.seq - max(a.group_at[0], 0);
            const int g = unit < 0 ? -1 : find_sequence(a.n_groups, unit, [&](int i) {
                return max(a.group_at[i + 1] - max(a.group_at[i], 0), 0);
            });
            if (g >= 0) {
                shared = max(a.shared[g], 0) & ~slot_mask;  // whole pages
                first = p.table + (size_t)min(max(a.group_at[g], 0), r.seq) * p.max_page;
            }
        }
    } else {
        if (!prompt_rows(p, blockIdx.x, kvh, r)) return;
        own = first = p.table + (size_t)r.seq * p.max_page;
    }
    const size_t kv_page = (size_t)p.n_kv_head * HD << p.page_log, kv_head = (size_t)kvh * HD << p.page_log;
    const T *kc = (const T *)p.k + kv_head, *vc = (const T *)p.v + kv_head;

    run4 q[S::QS];
    {
        const T *x = (const T *)a.q + max(r.row, 0LL) * HD;
#pragma unroll
        for (int c = 0; c < S::QS; ++c) q[c] = *(const run4 *)(x + (2 * c + h) * RUN);
    }
    S st;
    st.clear();
    const auto page_at = [&](int pos) { return page_of(p, pos < shared ? first : own, pos); };

    for (int t0 = 32 * wave; t0 < r.top; t0 += 128) {
        const int pos = t0 + kv_row<E>(lane & 31), posc = min(pos, r.n_kv - 1);
        const int page = page_at(posc);
        // bit m: the position of the first product's row m can be read
        const uint32_t valid = (uint32_t)__ballot(page >= 0 && pos < r.n_kv);
        const T *k = kc + (size_t)max(page, 0) * kv_page + (size_t)(posc & slot_mask) * HD;
        v16f s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < S::QS; ++c) s = Mma<E>::mul(*(const run4 *)(k + (2 * c + h) * RUN), q[c], s);
        const bool whole = __all(r.limit >= t0 + 32) && valid == 0xFFFFFFFFu;
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int m = 8 * (i >> 2) + (i & 3);
                const bool seen = t0 + kv_reg<E>(i, h) < r.limit && (valid >> (m + 4 * h) & 1);
                s[i] = seen ? s[i] : NEG_INF;
            }
        }
        st.softmax(s, a.scale);
#pragma unroll
        for (int c = 0; c < S::PS; ++c) {
            float x[RUN];
#pragma unroll
            for (int j = 0; j < RUN; ++j) x[j] = s[c * RUN + j];
            const run4 pr = to_run<E>(x);
            const int vp = t0 + 2 * RUN * c + RUN * h, vpc = min(vp, (r.n_kv - 1) & ~(RUN - 1));
            const int page = page_at(vpc);
            const T *v = vc + (size_t)max(page, 0) * kv_page + (vpc & slot_mask);
            if (whole) {
#pragma unroll
                for (int d = 0; d < S::DB; ++d)
                    st.o[d] = Mma<E>::mul(*(const run4 *)(v + ((size_t)(32 * d + (lane & 31)) << p.page_log)), pr, st.o[d]);
            } else {
                // positions that no row attends to may hold anything
                const int n = page < 0 ? 0 : min(max(r.top - vp, 0), RUN);
                st.add_masked([&](int d) { return *(const run4 *)(v + ((size_t)(32 * d + (lane & 31)) << p.page_log)); },
                              (1u << n) - 1u, pr, t0 + 2 * RUN * c, r.limit);
            }
        }
    }

    // the four waves' positions together
    st.l += other_half(st.l);
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
    const float f = l == 0.0f ? 0.0f : exp2_fast(st.m - against(m)) / l;
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
    if (wave || r.row < 0) return;
#pragma unroll
    for (int d = 0; d < S::DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const size_t at = (size_t)r.row * HD + 32 * d + 2 * i + 4 * h;
            if (a.out_f32) {
                *(float4 *)((float *)a.out + at) =
                    make_float4(st.o[d][i], st.o[d][i + 1], st.o[d][i + 2], st.o[d][i + 3]);
            } else {
                typedef T V __attribute__((ext_vector_type(4)));
                V v;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = E::put(st.o[d][i + j]);
                *(V *)((T *)a.out + at) = v;
            }
        }
}

template <class E, int HD>
int attend_as(const PagedAttendArgs &a, bool decode, hipStream_t st) {
    const PagedArgs &p = a.p;
    if (decode) {
        const dim3 grid(p.n_seq * ((p.group + 31) / 32), p.n_kv_head);
        hipLaunchKernelGGL((paged_rows<E, HD, true>), grid, dim3(256), 0, st, a);
    } else {
        const long long tiles = ((long long)p.n_tok * p.group) / 32 + p.n_seq;
        if (tiles > 0x7FFFFFFFLL / 256) return -1;
        hipLaunchKernelGGL((paged_rows<E, HD, false>), dim3((unsigned)tiles, p.n_kv_head), dim3(256), 0, st, a);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <class E>
int attend_type(const PagedAttendArgs &a, bool decode, hipStream_t st) {
    if (a.p.hd == 64) return attend_as<E, 64>(a, decode, st);
    if (a.p.hd == 128) return attend_as<E, 128>(a, decode, st);
    if (a.p.hd == 256) return attend_as<E, 256>(a, decode, st);
    return -1;
}

int attend(const PagedAttendArgs &a, int type, bool decode, hipStream_t st) {
    if (type == PT_F32) return attend_type<ElemF32>(a, decode, st);
    if (type == PT_F16) return attend_type<ElemF16>(a, decode, st);
    if (type == PT_BF16) return attend_type<ElemBF16>(a, decode, st);
    return -1;
}

}  // namespace

int launch_paged_prompt(const PagedAttendArgs &a, int type, hipStream_t st) { return attend(a, type, false, st); }
int launch_paged_decode(const PagedAttendArgs &a, int type, hipStream_t st) { return attend(a, type, true, st); }

}  // namespace llamd

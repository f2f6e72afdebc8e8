// paged.cpp -- the C entry points of the paged cache (include/llamd_hip.h): argument checks and descriptors for the
// kernels of paged_store.hip and paged_attend.hpp. Lengths, starts, tables and groups are device arrays that the host
// does not read, so that a captured call follows them; the kernels keep them inside the buffers given here.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/llamd_hip.h"
#include "errors.hpp"
#include "launch.hpp"
#include "paged.hpp"

using namespace llamd;

namespace {

bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

int type_bytes(int type) { return type == PT_F32 ? 4 : type == PT_F16 || type == PT_BF16 ? 2 : 0; }

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + nb && y < x + na;
}

size_t page_bytes(const llamd_hip_pages *c) {
    return (size_t)c->n_page * c->n_head_kv * c->page * c->hd * type_bytes(c->type);
}

// Whether [x, x + n) meets the K or V pages.
bool meets_pages(const llamd_hip_pages *c, const void *x, size_t n) {
    return overlap(x, n, c->k, page_bytes(c)) || overlap(x, n, c->v, page_bytes(c));
}

// The checks that every entry point shares; -1 with the reason.
int describe(const char *what, const llamd_hip_pages *c, const llamd_hip_batch *b, int n_head, PagedArgs *p) {
    if (!c || !b) return set_error("%s: null descriptor", what);
    if (!c->k || !c->v || !aligned(c->k) || !aligned(c->v))
        return set_error("%s: K and V pages must be 16-byte aligned device memory", what);
    if (!type_bytes(c->type)) return set_error("%s: type %d (0 f32, 1 f16, 30 bf16)", what, c->type);
    if (c->hd != 64 && c->hd != 128 && c->hd != 256) return set_error("%s: head_dim %d (64, 128 or 256)", what, c->hd);
    if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)))
        return set_error("%s: page of %d positions (a power of two, 16 to 256)", what, c->page);
    if (c->n_page <= 0) return set_error("%s: %d pages", what, c->n_page);
    if (c->n_head_kv <= 0 || n_head <= 0 || n_head % c->n_head_kv || n_head > 65535)
        return set_error("%s: n_head %d, n_head_kv %d", what, n_head, c->n_head_kv);
    if (b->n_seq < 0 || b->n_tok < 0 || b->max_page <= 0)
        return set_error("%s: n_seq %d, n_tok %d, max_page %d", what, b->n_seq, b->n_tok, b->max_page);
    if ((long long)b->max_page * c->page > 1 << 30)
        return set_error("%s: tables of %d pages of %d (2^30 positions at most)", what, b->max_page, c->page);
    if (overlap(c->k, page_bytes(c), c->v, page_bytes(c))) return set_error("%s: K overlaps V", what);
    if (b->n_seq && (!b->len || !b->table)) return set_error("%s: null lengths or table", what);
    if (((uintptr_t)b->start | (uintptr_t)b->len | (uintptr_t)b->table) & 3)
        return set_error("%s: starts, lengths and table must be 4-byte aligned", what);
    if (!b->start && b->n_tok < b->n_seq)
        return set_error("%s: %d tokens for %d sequences of one token", what, b->n_tok, b->n_seq);
    p->k = c->k;
    p->v = c->v;
    p->start = b->start;
    p->len = b->len;
    p->table = b->table;
    p->n_page = c->n_page;
    p->page_log = __builtin_ctz(c->page);
    p->n_kv_head = c->n_head_kv;
    p->hd = c->hd;
    p->n_seq = b->n_seq;
    p->n_tok = b->n_tok;
    p->max_page = b->max_page;
    p->n_head = n_head;
    p->group = n_head / c->n_head_kv;
    return 0;
}

int describe_attend(const char *what, const llamd_hip_pages *c, const llamd_hip_batch *b, const void *q, int n_head,
                    float scale, int out_type, void *out, PagedAttendArgs *a) {
    if (describe(what, c, b, n_head, &a->p)) return -1;
    if (!q || !out || !aligned(q) || !aligned(out)) return set_error("%s: q and out must be 16-byte aligned", what);
    const float by = (float)(scale * 1.4426950408889634074);  // (past the largest f32: 0 scores would be NaN)
    if (!(scale > 0.0f) || !isfinite(by)) return set_error("%s: scale %g", what, (double)scale);
    if (out_type != c->type && out_type != PT_F32)
        return set_error("%s: out_type %d (the cache's, %d, or f32)", what, out_type, c->type);
    const size_t values = (size_t)b->n_tok * n_head * c->hd;
    if (overlap(q, values * type_bytes(c->type), out, values * type_bytes(out_type)))
        return set_error("%s: out overlaps q", what);
    if (meets_pages(c, out, values * type_bytes(out_type))) return set_error("%s: out overlaps the pages", what);
    a->q = q;
    a->out = out;
    a->out_f32 = out_type == PT_F32;
    a->scale = by;
    return 0;
}

int attend(const char *what, const PagedAttendArgs &a, int type, bool decode) {
    const auto launch = type == PT_F32 ? launch_paged_attend_f32
                        : type == PT_F16 ? launch_paged_attend_f16 : launch_paged_attend_bf16;
    return launch(a, decode, lib_stream()) ? set_error("%s: launch", what) : 0;
}

}  // namespace

extern "C" {

int llamd_hip_rope_freqs(int n_rot, double base, double factor, int orig_ctx, double beta_fast, double beta_slow,
                         double *freqs, float *mscale) {
    if (!freqs || !mscale || n_rot <= 0 || n_rot % 2) return set_error("rope_freqs: n_rot %d", n_rot);
    if (!(base > 1.0) || !isfinite(base) || !(factor > 0.0) || !isfinite(factor) || orig_ctx < 0 ||
        (orig_ctx && (!(beta_slow > 0.0) || !(beta_fast >= beta_slow) || !isfinite(beta_fast))))
        return set_error("rope_freqs: base %g, factor %g, orig_ctx %d, beta %g, %g", base, factor, orig_ctx,
                         beta_fast, beta_slow);
    // the (fractional) pair that turns `beta` times over the trained context
    const auto pair_of = [&](double beta) {
        return n_rot * log(orig_ctx / (2.0 * M_PI * beta)) / (2.0 * log(base));
    };
    double low = 0.0, high = 0.0;
    if (orig_ctx) {
        low = std::max(floor(pair_of(beta_fast)), 0.0);
        high = std::min(ceil(pair_of(beta_slow)), (double)(n_rot - 1));
    }
    for (int i = 0; i < n_rot / 2; ++i) {
        const double f = pow(base, -2.0 * i / n_rot);
        const double ramp =
            orig_ctx ? std::min(std::max((i - low) / std::max(high - low, 1e-3), 0.0), 1.0) : 1.0;
        freqs[i] = f * (1.0 - ramp) + f / factor * ramp;
    }
    *mscale = orig_ctx ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    return 0;
}

int llamd_hip_paged_store(const llamd_hip_pages *c, const llamd_hip_batch *b, const float *q, int ld_q,
                          const float *k, int ld_k, const float *v, int ld_v, const float *q_norm,
                          const float *k_norm, float eps, const double *freqs, int n_rot, int interleaved,
                          float mscale, int n_head, void *q_out) {
    PagedStoreArgs a{};
    if (describe("paged_store", c, b, n_head, &a.p)) return -1;
    if (!k || !v || !q != !q_out) return set_error("paged_store: k, v, and q with q_out or neither");
    if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(q_out) || !aligned(q_norm) || !aligned(k_norm))
        return set_error("paged_store: q, k, v, q_out and the norm weights must be 16-byte aligned");
    const int kv = c->n_head_kv * c->hd;
    if ((q && (ld_q < n_head * c->hd || ld_q % 4)) || ld_k < kv || ld_k % 4 || ld_v < kv || ld_v % 4)
        return set_error("paged_store: row lengths %d, %d, %d (at least the heads', multiples of 4)", ld_q, ld_k, ld_v);
    if (n_rot < 0 || n_rot > c->hd || n_rot % 2 || (n_rot && !freqs) || ((uintptr_t)freqs & 7) || (interleaved & ~1))
        return set_error("paged_store: n_rot %d (even, at most %d, with 8-byte aligned frequencies), interleaved %d", n_rot, c->hd,
                         interleaved);
    if (!(eps >= 0.0f) || !isfinite(eps) || !isfinite(mscale))
        return set_error("paged_store: eps %g, mscale %g", (double)eps, (double)mscale);
    // (the rows up to the last one's end)
    const size_t rows = b->n_tok ? b->n_tok - 1 : 0, n_k = (rows * ld_k + kv) * 4, n_v = (rows * ld_v + kv) * 4;
    if (meets_pages(c, k, n_k) || meets_pages(c, v, n_v)) return set_error("paged_store: k or v overlaps the pages");
    if (q) {
        const size_t n_q = (rows * ld_q + (size_t)n_head * c->hd) * 4;
        const size_t n_out = (size_t)b->n_tok * n_head * c->hd * type_bytes(c->type);
        if (overlap(q, n_q, q_out, n_out) || overlap(k, n_k, q_out, n_out) || overlap(v, n_v, q_out, n_out))
            return set_error("paged_store: q_out overlaps q, k or v");
        if (meets_pages(c, q, n_q)) return set_error("paged_store: q overlaps the pages");
        if (meets_pages(c, q_out, n_out)) return set_error("paged_store: q_out overlaps the pages");
    }
    if (!b->n_seq || !b->n_tok) return 0;
    a.x[0] = q;
    a.x[1] = k;
    a.x[2] = v;
    a.ld[0] = ld_q;
    a.ld[1] = ld_k;
    a.ld[2] = ld_v;
    a.norm[0] = q_norm;
    a.norm[1] = k_norm;
    a.eps = eps;
    a.freqs = freqs;
    a.n_rot = n_rot;
    a.interleaved = interleaved;
    a.mscale = mscale;
    a.q_out = q_out;
    return launch_paged_store(a, c->type, lib_stream()) ? set_error("paged_store: launch") : 0;
}

int llamd_hip_paged_prompt(const llamd_hip_pages *c, const llamd_hip_batch *b, const void *q, int n_head, float scale,
                           int out_type, void *out) {
    PagedAttendArgs a{};
    if (describe_attend("paged_prompt", c, b, q, n_head, scale, out_type, out, &a)) return -1;
    if (!b->n_seq || !b->n_tok) return 0;
    return attend("paged_prompt", a, c->type, false);
}

int llamd_hip_paged_decode(const llamd_hip_pages *c, const llamd_hip_batch *b, const int32_t *group,
                           const int32_t *shared, int n_group, const void *q, int n_head, float scale, int out_type,
                           void *out) {
    PagedAttendArgs a{};
    if (describe_attend("paged_decode", c, b, q, n_head, scale, out_type, out, &a)) return -1;
    if (b->n_tok < b->n_seq)
        return set_error("paged_decode: %d tokens for %d sequences", b->n_tok, b->n_seq);
    if (n_group < 0 || n_group > b->n_seq || (n_group && (!group || !shared)))
        return set_error("paged_decode: %d groups of %d sequences", n_group, b->n_seq);
    if (((uintptr_t)group | (uintptr_t)shared) & 3)
        return set_error("paged_decode: groups must be 4-byte aligned");
    if (!b->n_seq) return 0;
    a.group_at = group;
    a.shared = shared;
    a.n_groups = n_group;
    return attend("paged_decode", a, c->type, true);
}

}  // extern "C"

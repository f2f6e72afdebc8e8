// paged.cpp -- the C entry points of the paged caches (include/llamd_hip.h): argument checks and descriptors for the
// kernels of paged_store.hip, paged8_store.hip and paged_attend.hpp. Lengths, starts, tables and groups are device arrays that the host
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

// A cache as the checks see it. `type` is that of q and of results by default; an 8-bit cache has scales.
struct Cache {
    void *k, *v;
    uint8_t *k_scale, *v_scale;
    int type, element, n_page, page, n_head_kv, hd;  // element: bytes

    size_t bytes() const { return (size_t)n_page * n_head_kv * page * hd * element; }
    size_t scale_bytes() const { return k_scale ? (size_t)n_page * n_head_kv * (page / SCALE_BLOCK) : 0; }
};

bool cache_of(const char *what, const llamd_hip_pages *c, Cache *x) {
    if (!c) return set_error("%s: null descriptor", what), false;
    *x = {c->k, c->v, nullptr, nullptr, c->type, type_bytes(c->type), c->n_page, c->page, c->n_head_kv, c->hd};
    if (!x->element) return set_error("%s: type %d (0 f32, 1 f16, 30 bf16)", what, c->type), false;
    return true;
}

bool cache_of(const char *what, const llamd_hip_pages8 *c, Cache *x) {
    if (!c) return set_error("%s: null descriptor", what), false;
    *x = {c->k, c->v, c->k_scale, c->v_scale, PT_BF16, 1, c->n_page, c->page, c->n_head_kv, c->hd};
    if (!c->k_scale || !c->v_scale || (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3))
        return set_error("%s: the scales must be 4-byte aligned device memory", what), false;
    return true;
}

// Whether [x, x + n) meets the K or V pages, or their scales.
bool meets_pages(const Cache &c, const void *x, size_t n) {
    return overlap(x, n, c.k, c.bytes()) || overlap(x, n, c.v, c.bytes()) ||
           overlap(x, n, c.k_scale, c.scale_bytes()) || overlap(x, n, c.v_scale, c.scale_bytes());
}

// The checks that every entry point shares; -1 with the reason.
int describe(const char *what, const Cache &cache, const llamd_hip_batch *b, int n_head, PagedArgs *p) {
    const Cache *c = &cache;
    if (!b) return set_error("%s: null descriptor", what);
    if (!c->k || !c->v || !aligned(c->k) || !aligned(c->v))
        return set_error("%s: K and V pages must be 16-byte aligned device memory", what);
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
    if (overlap(c->k, c->bytes(), c->v, c->bytes())) return set_error("%s: K overlaps V", what);
    if (c->k_scale) {
        const size_t n = c->scale_bytes();
        if (overlap(c->k_scale, n, c->v_scale, n) || overlap(c->k_scale, n, c->k, c->bytes()) ||
            overlap(c->k_scale, n, c->v, c->bytes()) || overlap(c->v_scale, n, c->k, c->bytes()) ||
            overlap(c->v_scale, n, c->v, c->bytes()))
            return set_error("%s: scales overlap each other or the pages", what);
    }
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
    p->k_scale = c->k_scale;
    p->v_scale = c->v_scale;
    return 0;
}

int describe_attend(const char *what, const Cache &cache, const llamd_hip_batch *b, const void *q, int n_head,
                    float scale, int out_type, void *out, PagedAttendArgs *a) {
    const Cache *c = &cache;
    if (describe(what, cache, b, n_head, &a->p)) return -1;
    if (!q || !out || !aligned(q) || !aligned(out)) return set_error("%s: q and out must be 16-byte aligned", what);
    const float by = (float)(scale * 1.4426950408889634074);  // (past the largest f32: 0 scores would be NaN)
    if (!(scale > 0.0f) || !isfinite(by)) return set_error("%s: scale %g", what, (double)scale);
    if (out_type != c->type && out_type != PT_F32)
        return set_error("%s: out_type %d (q's, %d, or f32)", what, out_type, c->type);
    const size_t values = (size_t)b->n_tok * n_head * c->hd;
    if (overlap(q, values * type_bytes(c->type), out, values * type_bytes(out_type)))
        return set_error("%s: out overlaps q", what);
    if (meets_pages(cache, out, values * type_bytes(out_type))) return set_error("%s: out overlaps the pages", what);
    a->q = q;
    a->out = out;
    a->out_f32 = out_type == PT_F32;
    a->scale = by;
    return 0;
}

int attend(const char *what, const PagedAttendArgs &a, const Cache &c, bool decode) {
    const auto launch = c.k_scale ? launch_paged_attend_e4m3
                        : c.type == PT_F32 ? launch_paged_attend_f32
                        : c.type == PT_F16 ? launch_paged_attend_f16 : launch_paged_attend_bf16;
    return launch(a, decode, lib_stream()) ? set_error("%s: launch", what) : 0;
}

// New tokens into the cache, of either kind.
template <class Pages>
int store(const char *what, const Pages *pages, const llamd_hip_batch *b, const float *q, int ld_q, const float *k, int ld_k,
          const float *v, int ld_v, const float *q_norm, const float *k_norm, float eps, const double *freqs, int n_rot,
          int interleaved, float mscale, int n_head, void *q_out) {
    PagedStoreArgs a{};
    Cache cache;
    if (!cache_of(what, pages, &cache) || describe(what, cache, b, n_head, &a.p)) return -1;
    const Cache *c = &cache;
    if (!k || !v || !q != !q_out) return set_error("%s: k, v, and q with q_out or neither", what);
    if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(q_out) || !aligned(q_norm) || !aligned(k_norm))
        return set_error("%s: q, k, v, q_out and the norm weights must be 16-byte aligned", what);
    const int kv = c->n_head_kv * c->hd;
    if ((q && (ld_q < n_head * c->hd || ld_q % 4)) || ld_k < kv || ld_k % 4 || ld_v < kv || ld_v % 4)
        return set_error("%s: row lengths %d, %d, %d (at least the heads', multiples of 4)", what, ld_q, ld_k, ld_v);
    if (n_rot < 0 || n_rot > c->hd || n_rot % 2 || (n_rot && !freqs) || ((uintptr_t)freqs & 7) || (interleaved & ~1))
        return set_error("%s: n_rot %d (even, at most %d, with 8-byte aligned frequencies), interleaved %d", what, n_rot, c->hd,
                         interleaved);
    if (!(eps >= 0.0f) || !isfinite(eps) || !isfinite(mscale))
        return set_error("%s: eps %g, mscale %g", what, (double)eps, (double)mscale);
    // (the rows up to the last one's end)
    const size_t rows = b->n_tok ? b->n_tok - 1 : 0, n_k = (rows * ld_k + kv) * 4, n_v = (rows * ld_v + kv) * 4;
    if (meets_pages(cache, k, n_k) || meets_pages(cache, v, n_v)) return set_error("%s: k or v overlaps the pages", what);
    if (q) {
        const size_t n_q = (rows * ld_q + (size_t)n_head * c->hd) * 4;
        const size_t n_out = (size_t)b->n_tok * n_head * c->hd * type_bytes(c->type);
        if (overlap(q, n_q, q_out, n_out) || overlap(k, n_k, q_out, n_out) || overlap(v, n_v, q_out, n_out))
            return set_error("%s: q_out overlaps q, k or v", what);
        if (meets_pages(cache, q, n_q)) return set_error("%s: q overlaps the pages", what);
        if (meets_pages(cache, q_out, n_out)) return set_error("%s: q_out overlaps the pages", what);
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
    const int rc = c->k_scale ? launch_paged8_store(a, lib_stream()) : launch_paged_store(a, c->type, lib_stream());
    return rc ? set_error("%s: launch", what) : 0;
}

template <class Pages>
int prompt(const char *what, const Pages *pages, const llamd_hip_batch *b, const void *q, int n_head, float scale, int out_type,
           void *out) {
    PagedAttendArgs a{};
    Cache c;
    if (!cache_of(what, pages, &c) || describe_attend(what, c, b, q, n_head, scale, out_type, out, &a)) return -1;
    if (!b->n_seq || !b->n_tok) return 0;
    return attend(what, a, c, false);
}

template <class Pages>
int decode(const char *what, const Pages *pages, const llamd_hip_batch *b, const int32_t *group, const int32_t *shared,
           int n_group, const void *q, int n_head, float scale, int out_type, void *out) {
    PagedAttendArgs a{};
    Cache c;
    if (!cache_of(what, pages, &c) || describe_attend(what, c, b, q, n_head, scale, out_type, out, &a)) return -1;
    if (b->n_tok < b->n_seq)
        return set_error("%s: %d tokens for %d sequences", what, b->n_tok, b->n_seq);
    if (n_group < 0 || n_group > b->n_seq || (n_group && (!group || !shared)))
        return set_error("%s: %d groups of %d sequences", what, n_group, b->n_seq);
    if (((uintptr_t)group | (uintptr_t)shared) & 3)
        return set_error("%s: groups must be 4-byte aligned", what);
    if (!b->n_seq) return 0;
    a.group_at = group;
    a.shared = shared;
    a.n_groups = n_group;
    return attend(what, a, c, true);
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
    return store("paged_store", c, b, q, ld_q, k, ld_k, v, ld_v, q_norm, k_norm, eps, freqs, n_rot, interleaved, mscale, n_head, q_out);
}

int llamd_hip_paged_prompt(const llamd_hip_pages *c, const llamd_hip_batch *b, const void *q, int n_head, float scale,
                           int out_type, void *out) {
    return prompt("paged_prompt", c, b, q, n_head, scale, out_type, out);
}

int llamd_hip_paged_decode(const llamd_hip_pages *c, const llamd_hip_batch *b, const int32_t *group,
                           const int32_t *shared, int n_group, const void *q, int n_head, float scale, int out_type,
                           void *out) {
    return decode("paged_decode", c, b, group, shared, n_group, q, n_head, scale, out_type, out);
}

int llamd_hip_paged8_store(const llamd_hip_pages8 *c, const llamd_hip_batch *b, const float *q, int ld_q,
                          const float *k, int ld_k, const float *v, int ld_v, const float *q_norm,
                          const float *k_norm, float eps, const double *freqs, int n_rot, int interleaved,
                          float mscale, int n_head, void *q_out) {
    return store("paged8_store", c, b, q, ld_q, k, ld_k, v, ld_v, q_norm, k_norm, eps, freqs, n_rot, interleaved, mscale, n_head, q_out);
}

int llamd_hip_paged8_prompt(const llamd_hip_pages8 *c, const llamd_hip_batch *b, const void *q, int n_head, float scale,
                           int out_type, void *out) {
    return prompt("paged8_prompt", c, b, q, n_head, scale, out_type, out);
}

int llamd_hip_paged8_decode(const llamd_hip_pages8 *c, const llamd_hip_batch *b, const int32_t *group,
                           const int32_t *shared, int n_group, const void *q, int n_head, float scale, int out_type,
                           void *out) {
    return decode("paged8_decode", c, b, group, shared, n_group, q, n_head, scale, out_type, out);
}

}  // extern "C"

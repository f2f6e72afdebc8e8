"""The paged cache's operators against 64-bit restatements (paged_reference), where they can go wrong: lengths of zero
and one, tiles and pages that end inside each other, page sizes, shared and missing pages, far positions, rows that
belong to no sequence, infinities and NaN in masked places, groups, captured calls. Bounds are paged_reference's."""
import ctypes as C

import numpy as np
import pytest

import paged_reference as R

pytestmark = pytest.mark.gpu
KINDS = ["bf16", "f16", "f32"]


def rounded(x, kind):
    from llamd_rs_amd import rocm
    if kind == "bf16":
        return rocm.from_bf16(rocm.to_bf16(x))
    return np.asarray(x, np.float16 if kind == "f16" else np.float32).astype(np.float32)


def tables(rng, lengths, page, spare=2):
    """Pages in a random order; unused entries are -1. (table, n_page)"""
    need = [-(-n // page) for n in lengths]
    order = rng.permutation(sum(need) + spare)
    t = np.full((len(lengths), max(max(need), 1)), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = order[at:at + n]
        at += n
    return t, len(order)


def dense(pages_k, pages_v, row, n):
    """K, V [n, kv heads, hd] of a table row's first n positions."""
    page = pages_k.shape[2]
    at = np.arange(n)
    ids = row[at // page]
    return pages_k[ids, :, at % page], pages_v[ids, :, :, at % page]


def filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths, garbage=np.nan):
    """A cache with values at the lengths' positions and `garbage` everywhere else."""
    c = gpu.PagedCache(kind, n_page, page, heads, kvh, hd)
    k = np.full(c.shape_k, garbage, np.float32)
    v = np.full(c.shape_v, garbage, np.float32)
    for row, n in zip(table, lengths):
        at = np.arange(n)
        k[row[at // page], :, at % page] = rounded(rng.standard_normal((n, kvh, hd)) * 1.5, kind)
        v[row[at // page], :, :, at % page] = rounded(rng.standard_normal((n, kvh, hd)), kind)
    c.write(k, v)
    return c, k, v


# ---- store ------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd,page,n_rot,interleaved,norm", [
    (32, 4, 128, 64, 128, False, True), (16, 8, 128, 16, 64, True, False), (12, 12, 64, 32, 64, False, True),
    (3, 1, 64, 16, 32, False, True), (8, 2, 256, 128, 256, True, True), (5, 5, 256, 256, 100, False, False),
    (2, 1, 128, 32, 0, False, True)])
def test_store(gpu, kind, heads, kvh, hd, page, n_rot, interleaved, norm):
    rng = np.random.default_rng(11)
    new, old = [1, 0, 37, 2, 70, 1], [0, 5, 3, 900, 61, 15]
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[2], 2 + np.cumsum(new)])
    tokens = start[-1] + 3   # two rows before the first sequence and three behind the last
    q, k, v = (rng.standard_normal((tokens, h * hd)).astype(np.float32) * 2 for h in (heads, kvh, kvh))
    qw, kw = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)) if norm else (None, None)
    freqs, m = (gpu.rope_freqs(n_rot, 1e6, 4.0, 512) if n_rot else (None, 1.0))
    c = gpu.PagedCache(kind, n_page, page, heads, kvh, hd)
    before_k = rounded(rng.standard_normal(c.shape_k), kind)
    before_v = rounded(rng.standard_normal(c.shape_v), kind)
    c.write(before_k, before_v)
    got = c.store(q, k, v, table, lengths, start, qw, kw, 1e-5, freqs, interleaved, m)
    got_k, got_v = c.read()
    want_k, bound_k = before_k.astype(np.float64), np.zeros(c.shape_k)
    want_v, bound_v = before_v.astype(np.float64), np.zeros(c.shape_v)
    want_q, bound_q = np.zeros((tokens, heads, hd)), np.zeros((tokens, heads, hd))
    for s in range(len(new)):
        rows = slice(start[s], start[s + 1])
        pos = np.arange(old[s], lengths[s])
        if not len(pos):
            continue
        want_q[rows], bound_q[rows] = R.store(q[rows].reshape(-1, heads, hd), qw, pos, freqs, n_rot, interleaved, m, 1e-5, kind)
        ids, slots = table[s][pos // page], pos % page
        want_k[ids, :, slots], bound_k[ids, :, slots] = R.store(k[rows].reshape(-1, kvh, hd), kw, pos, freqs, n_rot,
                                                                interleaved, m, 1e-5, kind)
        want_v[ids, :, :, slots] = rounded(v[rows].reshape(-1, kvh, hd), kind)
    R.check(got, want_q.reshape(tokens, -1), bound_q.reshape(tokens, -1), "q")
    R.check(got_k, want_k, bound_k, "k")
    assert np.array_equal(got_v, want_v.astype(np.float32))


@pytest.mark.parametrize("kind", KINDS)
def test_store_far_positions(gpu, kind):
    """Angles of a million radians, where 32 bits would be off by a few hundredths."""
    rng = np.random.default_rng(12)
    heads, kvh, hd, page = 4, 2, 128, 256
    lengths = [1_000_000, 262_145, 7]
    table = np.full((3, 3907), -1, np.int32)
    table[0, 999_999 // page], table[1, 262_144 // page], table[2, 0] = 1, 0, 2
    q, k, v = (rng.standard_normal((3, h * hd)).astype(np.float32) for h in (heads, kvh, kvh))
    freqs, m = gpu.rope_freqs(hd, 10000.0)
    c = gpu.PagedCache(kind, 3, page, heads, kvh, hd)
    got = c.store(q, k, v, table, lengths, None, None, None, 1e-6, freqs, False, m)
    want, bound = R.store(q.reshape(3, heads, hd), None, np.array(lengths) - 1, freqs, hd, False, m, 0, kind)
    R.check(got, want.reshape(3, -1), bound.reshape(3, -1))
    want, bound = R.store(k.reshape(3, kvh, hd), None, np.array(lengths) - 1, freqs, hd, False, m, 0, kind)
    got_k, _ = c.read()
    for s, n in enumerate(lengths):
        at = (n - 1)
        R.check(got_k[table[s, at // page], :, at % page], want[s], bound[s])


def test_store_without_a_place(gpu):
    """Missing pages, ids outside the cache, tokens before position 0 and past the table: q is turned, nothing is stored."""
    rng = np.random.default_rng(13)
    heads, kvh, hd, page = 4, 2, 64, 16
    c = gpu.PagedCache("f32", 4, page, heads, kvh, hd)
    table = np.array([[0, -1], [4, 1], [1 << 30, 2], [3, 3]], np.int32)
    lengths, start = [17, 3, 16, 34], [0, 2, 6, 8, 11]  # sequence 1: four tokens, the first at position -1
    q, k, v = (rng.standard_normal((11, h * hd)).astype(np.float32) for h in (heads, kvh, kvh))
    freqs, m = gpu.rope_freqs(hd, 10000.0)
    got = c.store(q, k, v, table, lengths, start, None, None, 1e-6, freqs)
    pos = np.array([15, 16, -1, 0, 1, 2, 14, 15, 31, 32, 33])
    want, bound = R.store(q.reshape(11, heads, hd), None, pos, freqs, hd, False, m, 0, "f32")
    R.check(got, want.reshape(11, -1), bound.reshape(11, -1))
    got_k, got_v = c.read()
    want_k, bound_k = np.zeros(c.shape_k), np.zeros(c.shape_k)
    want_v = np.zeros(c.shape_v)
    w, b = R.store(k.reshape(11, kvh, hd), None, pos, freqs, hd, False, m, 0, "f32")
    for t, (s, at) in enumerate(zip([0, 0, 1, 1, 1, 1, 2, 2, 3, 3, 3], pos)):
        if 0 <= at < 32 and 0 <= table[s, at // page] < 4:
            want_k[table[s, at // page], :, at % page], bound_k[table[s, at // page], :, at % page] = w[t], b[t]
            want_v[table[s, at // page], :, :, at % page] = v[t].reshape(kvh, hd)
    R.check(got_k, want_k, bound_k)
    assert np.array_equal(got_v, want_v.astype(np.float32))


def test_store_side_by_side_and_without_q(gpu):
    """Q, K and V as one matrix's columns; then K and V alone."""
    rng = np.random.default_rng(14)
    L, heads, kvh, hd, page, n = gpu.lib(), 4, 2, 64, 16, 21
    wide = (heads + 2 * kvh) * hd + 8
    x = rng.standard_normal((n, wide)).astype(np.float32)
    q, k, v = (np.ascontiguousarray(x[:, a * hd:b * hd]) for a, b in ((0, 4), (4, 6), (6, 8)))
    c, d = (gpu.PagedCache("f16", 4, page, heads, kvh, hd) for _ in range(2))
    table = np.array([[2, 0]], np.int32)
    freqs, _ = gpu.rope_freqs(hd, 10000.0)
    want = c.store(q, k, v, table, [n], [0, n], None, None, 1e-6, freqs)
    X, F = gpu.DeviceBuffer.from_array(x), gpu.DeviceBuffer.from_array(freqs)
    out = gpu.DeviceBuffer.from_array(np.zeros((n, heads * hd), np.float16))
    b, keep = d._batch(table, [n], [0, n], n)
    P, B = C.byref(d.pages), C.byref(b)
    at = [X.ptr + 4 * hd * i for i in (0, 4, 6)]
    assert L.llamd_hip_paged_store(P, B, at[0], wide, at[1], wide, at[2], wide, None, None, 1e-6, F.ptr, hd, 0, 1.0,
                                   heads, out.ptr) == 0
    assert np.array_equal(out.download(np.empty((n, heads * hd), np.float16)).astype(np.float32), want)
    assert all(np.array_equal(a, b) for a, b in zip(c.read(), d.read()))
    d.write(np.zeros(d.shape_k, np.float32), np.zeros(d.shape_v, np.float32))
    assert L.llamd_hip_paged_store(P, B, None, 0, at[1], wide, at[2], wide, None, None, 1e-6, F.ptr, hd, 0, 1.0,
                                   heads, None) == 0
    assert all(np.array_equal(a, b) for a, b in zip(c.read(), d.read()))


# ---- prompts ----------------------------------------------------------------------

def want_prompt(q, pages_k, pages_v, table, lengths, start, heads, kvh, hd, scale, kind, out_kind=None):
    page, n_page = pages_k.shape[2], len(pages_k)
    out = np.zeros((len(q), heads, hd))
    bound = np.zeros((len(q), heads, hd))
    for s, n in enumerate(lengths):
        a, b = start[s], start[s + 1]
        if a == b:
            continue
        n = min(n, table.shape[1] * page)
        at = np.arange(max(n, 0))
        ids = table[s][at // page]
        there = (ids >= 0) & (ids < n_page)
        ids = np.where(there, ids, 0)
        k, v = pages_k[ids, :, at % page], pages_v[ids, :, :, at % page]
        limits = lengths[s] - (b - np.arange(a, b)) + 1
        out[a:b], bound[a:b] = R.attend(q[a:b].reshape(-1, heads, hd), k, v, limits, scale, kind, out_kind, there)
    return out.reshape(len(q), -1), bound.reshape(len(q), -1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd,page,new,old", [
    (32, 4, 128, 64, [1, 0, 5, 33], [0, 7, 60, 31]),
    (16, 8, 128, 16, [64, 1, 17], [0, 15, 130]),
    (12, 12, 64, 32, [1, 31, 32, 33, 65], [0, 1, 0, 63, 200]),
    (16, 1, 64, 16, [3, 40], [0, 300]),
    (3, 1, 64, 128, [70, 2], [129, 0]),
    (40, 1, 128, 64, [9], [50]),
    (8, 2, 256, 32, [20, 7], [3, 100]),
    (4, 4, 128, 256, [130], [190])])
def test_prompt(gpu, kind, heads, kvh, hd, page, new, old):
    rng = np.random.default_rng(21)
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[0], np.cumsum(new)])
    tokens = start[-1] + 2
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((tokens, heads * hd)) * 1.5, kind)
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, hd ** -0.5, kind)
    R.check(c.prompt(q, table, lengths, start), want, bound)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd,new,old", [
    (4, 4, 64, [700], [0]), (8, 1, 128, [300, 1, 290], [500, 2000, 0]), (4, 4, 128, [200], [2500]), (2, 1, 256, [150], [900]),
    (12, 4, 64, [5, 260], [6000, 11])])
def test_prompt_long(gpu, kind, heads, kvh, hd, new, old):
    rng = np.random.default_rng(22)
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, 32)
    start = np.concatenate([[0], np.cumsum(new)])
    c, k, v = filled(gpu, rng, kind, table, n_page, 32, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((start[-1], heads * hd)) * 2, kind)
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, 0.1, kind)
    R.check(c.prompt(q, table, lengths, start, scale=0.1), want, bound)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_prompt_f32_result(gpu, kind):
    rng = np.random.default_rng(23)
    table, n_page = tables(rng, [90, 4], 16)
    c, k, v = filled(gpu, rng, kind, table, n_page, 16, 8, 2, 128, [90, 4])
    q = rounded(rng.standard_normal((34, 8 * 128)), kind)
    want, bound = want_prompt(q, k, v, table, [90, 4], [0, 30, 34], 8, 2, 128, 128 ** -0.5, kind, "f32")
    R.check(c.prompt(q, table, [90, 4], [0, 30, 34], f32_out=True), want, bound)


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_missing_pages_and_empty_rows(gpu, kind):
    """Ids outside the cache, tokens before position 0, a length past the table: such positions have no part, and rows
    that see nothing are 0."""
    rng = np.random.default_rng(24)
    heads, kvh, hd, page = 8, 2, 64, 16
    lengths, new = [70, 20, 3, 100, 40], [40, 20, 9, 50, 3]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    table = table[:, :5].copy()           # sequence 3's last 20 positions are past the table
    table[0, 1], table[0, 3] = -1, n_page
    table[1, :] = [1 << 30, -5, -1, -1, -1]  # sequence 1 has no pages at all
    start = np.concatenate([[0], np.cumsum(new)])
    q = rounded(rng.standard_normal((start[-1], heads * hd)), kind)
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, hd ** -0.5, kind)
    got = c.prompt(q, table, lengths, start)
    R.check(got, want, bound)
    assert not got[40:60].any() and not got[60:66].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_prompt_not_finite_values_stay_with_those_who_see_them(gpu, kind, bad):
    """A token with infinities or NaN in V (and, further on, in K) touches no row before it, in any sequence."""
    rng = np.random.default_rng(25)
    heads, kvh, hd, page = 4, 2, 64, 16
    table, n_page = tables(rng, [90, 50], page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, [90, 50])
    for pos in (47, 66):
        v[table[0, pos // page], 1, 5:40:7, pos % page] = bad
    k[table[0, 70 // page], 0, 70 % page, 3] = np.nan
    c.write(k, v)
    start = [0, 90, 140]
    q = rounded(rng.standard_normal((140, heads * hd)), kind)
    want, bound = want_prompt(q, k, v, table, [90, 50], start, heads, kvh, hd, hd ** -0.5, kind)
    assert np.isfinite(want[:47]).all() and np.isfinite(want[90:]).all() and not np.isfinite(want[47]).all()
    R.check(c.prompt(q, table, [90, 50], start), want, bound)


@pytest.mark.parametrize("kind", KINDS)
def test_scores_of_minus_infinity(gpu, kind):
    """Keys of minus infinity weigh nothing beside others; a row that sees nothing else gives 0."""
    rng = np.random.default_rng(40)
    heads, kvh, hd, page = 4, 2, 64, 16
    table, n_page = tables(rng, [80, 20], page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, [80, 20])
    q = rounded(np.abs(rng.standard_normal((100, heads * hd))) + 0.5, kind)
    k[table[0, 33 // page], :, 33 % page, 5] = -np.inf
    for pos in range(20):
        k[table[1, pos // page], 0, pos % page, 7] = -np.inf
    c.write(k, v)
    # position 33 of the first sequence weighs nothing: as if it were not visible; the second one's first kv head has no
    # finite score
    want, bound = np.zeros((100, heads, hd)), np.zeros((100, heads, hd))
    for s, (first, n) in enumerate(((0, 80), (80, 20))):
        at = np.arange(n)
        ids = table[s][at // page]
        rows = slice(first, first + n)
        want[rows], bound[rows] = R.attend(q[rows].reshape(-1, heads, hd), k[ids, :, at % page], v[ids, :, :, at % page],
                                           at + 1, hd ** -0.5, kind, None, at != 33 if s == 0 else None)
    assert np.isnan(want[80:, :2]).all() and np.isfinite(want[:80]).all() and np.isfinite(want[80:, 2:]).all()
    want[80:, :2] = bound[80:, :2] = 0
    lists = [80, 20], [0, 80, 100]
    R.check(c.prompt(q, table, *lists), want.reshape(100, -1), bound.reshape(100, -1))
    R.check(c.decode(q[[79, 99]], table, [80, 20]), want[[79, 99]].reshape(2, -1), bound[[79, 99]].reshape(2, -1))


def test_prompt_starts_that_make_no_sense(gpu):
    """Starts that descend or leave the buffer never reach past it; the sequences that do make sense are right."""
    rng = np.random.default_rng(26)
    heads, kvh, hd, page = 4, 2, 64, 16
    table, n_page = tables(rng, [30, 30, 30], page)
    c, k, v = filled(gpu, rng, "f16", table, n_page, page, heads, kvh, hd, [30, 30, 30])
    q = rounded(rng.standard_normal((40, heads * hd)), "f16")
    start = [0, 10, 1 << 30, 20]
    want, bound = want_prompt(q, k, v, table, [30], [0, 10], heads, kvh, hd, hd ** -0.5, "f16")
    got = c.prompt(q, table, [30, 30, 30], start)
    R.check(got[:10], want[:10], bound[:10])
    got = c.prompt(q, table, [30, -7, -(1 << 31)], [0, 10, 20, 40])
    R.check(got[:10], want[:10], bound[:10])
    assert not got[10:].any()


def test_prompt_many_sequences(gpu):
    """More sequences than a wave has lanes, some without tokens."""
    rng = np.random.default_rng(27)
    heads, kvh, hd, page = 4, 1, 64, 16
    new = [int(n) for n in rng.integers(0, 4, 150)]
    lengths = [n + int(x) for n, x in zip(new, rng.integers(0, 40, 150))]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, "bf16", table, n_page, page, heads, kvh, hd, lengths)
    start = np.concatenate([[0], np.cumsum(new)])
    q = rounded(rng.standard_normal((start[-1], heads * hd)), "bf16")
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, hd ** -0.5, "bf16")
    R.check(c.prompt(q, table, lengths, start), want, bound)


# ---- decode -----------------------------------------------------------------------

def want_decode(q, k, v, table, lengths, heads, kvh, hd, scale, kind, group=(), shared=()):
    out, bound = [], []
    page = k.shape[2]
    t = table.copy()
    rows = []
    for s in range(len(lengths)):
        g = [i for i in range(len(shared)) if group[i] <= s < group[i + 1]]
        n = min(max(lengths[s], 0), t.shape[1] * page)
        at = np.arange(n)
        ids = t[s][at // page]
        if g:
            ids = np.where(at < max(shared[g[0]], 0) // page * page, t[group[g[0]]][at // page], ids)
        there = (ids >= 0) & (ids < len(k))
        ids = np.where(there, ids, 0)
        rows.append(R.attend(q[s:s + 1].reshape(1, heads, hd), k[ids, :, at % page], v[ids, :, :, at % page], [n], scale,
                             kind, None, there))
    out, bound = (np.concatenate(x).reshape(len(lengths), -1) for x in zip(*rows))
    return out, bound


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd,page,lengths", [
    (32, 4, 128, 64, [1, 0, 63, 64, 65, 700]), (16, 8, 128, 16, [31, 32, 33, 129]), (12, 12, 64, 32, [5, 300, 1]),
    (16, 1, 64, 128, [2000, 3]), (40, 1, 64, 16, [77, 400]), (8, 2, 256, 256, [600, 1, 255]), (3, 1, 128, 16, [4100])])
def test_decode(gpu, kind, heads, kvh, hd, page, lengths):
    rng = np.random.default_rng(31)
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((len(lengths) + 1, heads * hd)) * 1.5, kind)
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, kind)
    got = c.decode(q, table, lengths)
    R.check(got[:-1], want, bound)
    assert not got[-1].any()   # the row behind the last sequence


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,page,lengths", [
    (8, 1, 256, [26_000]), (4, 4, 64, [11_000, 0, 3, 40_000]), (20, 1, 128, [9_000, 130]), (16, 8, 32, [8_321, 8_320, 8_193])])
def test_decode_long(gpu, kind, heads, kvh, page, lengths):
    """As many parts of a row as there may be, and parts of several steps."""
    rng = np.random.default_rng(38)
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, 64, lengths)
    q = rounded(rng.standard_normal((len(lengths), heads * 64)) * 1.5, kind)
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, 64, 0.125, kind)
    R.check(c.decode(q, table, lengths), want, bound)


def shared_tables(rng, group, shared, lengths, page):
    """Tables whose groups share the pages that their prefix fills; (table, n_page, pages that copies are made of)."""
    table, n_page = tables(rng, lengths, page)
    copies = []
    for g, n in enumerate(shared):
        for s in range(group[g] + 1, group[g + 1]):
            full = min(n, lengths[s]) // page
            table[s, :full] = table[group[g], :full]
            if n % page and lengths[s] > full * page:
                copies.append((table[s, full], table[group[g], full], n % page))
    return table, n_page, copies


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kvh,hd,page,group,shared,lengths", [
    (32, 4, 128, 64, [0, 6], [128], [129, 300, 128, 700, 1000, 131]),
    (16, 8, 128, 16, [0, 2, 3, 8], [40, 17, 100], [45, 41, 60, 100, 101, 300, 116, 117]),
    (12, 12, 64, 32, [1, 5], [333], [20, 334, 600, 333, 400, 7]),
    (16, 1, 64, 16, [0, 3, 3, 6], [2000, 5, 0], [2100, 2001, 2500, 30, 40, 50]),
    (8, 2, 256, 64, [0, 20], [70], [71 + i for i in range(20)]),
    (8, 1, 128, 32, [0, 40], [900], [901 + 3 * i for i in range(40)])])
def test_decode_shared_prefix(gpu, kind, heads, kvh, hd, page, group, shared, lengths):
    rng = np.random.default_rng(32)
    table, n_page, copies = shared_tables(rng, group, shared, lengths, page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    for to, of, n in copies:
        k[to, :, :n], v[to, :, :, :n] = k[of, :, :n], v[of, :, :, :n]
    c.write(k, v)
    q = rounded(rng.standard_normal((len(lengths), heads * hd)) * 1.5, kind)
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, kind, group, shared)
    R.check(c.decode(q, table, lengths, group, shared), want, bound)
    # the same batch without the groups
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, kind)
    R.check(c.decode(q, table, lengths), want, bound)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_prefix_is_read_through_the_first_sequence(gpu, kind):
    """Members need no table entries for the shared positions; members shorter than the prefix, an empty one, missing
    pages and a first sequence shorter than the prefix it lends."""
    rng = np.random.default_rng(33)
    heads, kvh, hd, page = 8, 2, 128, 16
    lengths, group, shared = [200, 130, 50, 0, 97, 40, 90], [0, 5, 7], [96, 64]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    table[1:5, :6] = -1
    table[0, 2] = n_page + 3
    table[6, 4] = -1
    q = rounded(rng.standard_normal((7, heads * hd)), kind)
    # sequence 5 holds 40 positions in 3 pages; position 48 on of its group has no page, what lies in page 2 from 8 on is
    # whatever the cache holds
    k[table[5, 2], :, 8:], v[table[5, 2], :, :, 8:] = 0.5, 0.25
    c.write(k, v)
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, kind, group, shared)
    got = c.decode(q, table, lengths, group, shared)
    R.check(got, want, bound)
    assert not got[3].any()


def test_decode_groups_that_make_no_sense(gpu):
    """Descending or outlying group starts and lengths: no access past the arrays, sequences in no group are right."""
    rng = np.random.default_rng(34)
    heads, kvh, hd, page, lengths = 4, 2, 64, 16, [30, 40, 50]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, "f16", table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((3, heads * hd)), "f16")
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "f16")
    for group, shared in (([2, 1 << 30], [-5]), ([1, 0, 0], [1 << 30, 7]), ([-9, -3, -(1 << 31)], [4, 4]), ([3, 9], [20])):
        R.check(c.decode(q, table, lengths, group, shared), want, bound)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_batch_of_many(gpu, kind):
    rng = np.random.default_rng(35)
    heads, kvh, hd, page = 8, 2, 64, 16
    lengths = [int(n) for n in rng.integers(0, 200, 130)]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((130, heads * hd)), kind)
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, kind)
    R.check(c.decode(q, table, lengths), want, bound)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_decode_not_finite_values_that_a_member_does_not_see(gpu, kind, bad):
    """Infinities and NaN at shared positions behind a short member's length (the prefix's tiles), and at positions behind
    a sequence's length in its last page."""
    rng = np.random.default_rng(36)
    heads, kvh, hd, page = 8, 2, 64, 32
    lengths, group, shared = [300, 70, 310, 256, 40], [0, 4], [256]
    table, n_page, _ = shared_tables(rng, group, shared, lengths, page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    for pos in (80, 255):
        v[table[0, pos // page], 0, 3:50:5, pos % page] = bad
    v[table[0, 280 // page], 1, 7, 280 % page] = bad
    c.write(k, v)
    q = rounded(rng.standard_normal((5, heads * hd)), kind)
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, kind, group, shared)
    assert np.isfinite(want[[1, 4]]).all() and not np.isfinite(want[0]).all() and not np.isfinite(want[3]).all()
    R.check(c.decode(q, table, lengths, group, shared), want, bound)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_many_groups_in_a_large_batch(gpu, kind):
    """More groups than are looked through one by one, more sequences than a wave has lanes; groups of one and of none,
    sequences before, between and behind the groups."""
    rng = np.random.default_rng(37)
    heads, kvh, hd, page, n = 4, 2, 64, 16, 150
    sizes = [2, 1, 0, 7, 3, 30, 1, 2, 2, 5, 17, 4, 33, 2, 6]
    group = [4] + [4 + x for x in np.cumsum(sizes).tolist()]
    shared = [int(x) for x in rng.integers(0, 120, len(sizes))]
    lengths = [int(x) for x in rng.integers(0, 60, n)]
    for g, m in enumerate(shared):
        for s in range(group[g], group[g + 1]):
            lengths[s] = m + int(rng.integers(0, 90)) if s % 5 else int(rng.integers(0, 90))
    for g, m in enumerate(shared):
        if group[g + 1] > group[g]:
            lengths[group[g]] = max(lengths[group[g]], m)
    table, n_page, copies = shared_tables(rng, group, shared, lengths, page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    for to, of, m in copies:
        k[to, :, :m], v[to, :, :, :m] = k[of, :, :m], v[of, :, :, :m]
    c.write(k, v)
    q = rounded(rng.standard_normal((n, heads * hd)) * 1.5, kind)
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, kind, group, shared)
    R.check(c.decode(q, table, lengths, group, shared), want, bound)


def test_starts_and_groups_over_the_same_rows(gpu):
    """Starts (of sequences, of groups) that go back to 0 again and again claim more tiles than the rows make: nothing past
    the rows or the scratch is touched, and the calls after that are right."""
    rng = np.random.default_rng(39)
    heads, kvh, hd, page, n = 16, 1, 64, 16, 20
    lengths = [1500] * n
    table, n_page = tables(rng, lengths[:1], page)
    c, k, v = filled(gpu, rng, "bf16", table, n_page, page, heads, kvh, hd, lengths[:1])
    q = rounded(rng.standard_normal((100, heads * hd)), "bf16")
    many = np.repeat(table, n, 0)
    got = c.prompt(q, many, lengths, [0, 90] * (n // 2) + [0])
    assert not got[90:].any()
    got = c.decode(q[:n], many, lengths, [0, n] * (n // 2) + [0], [1400] * n)
    got = c.decode(q[:n], many, lengths, [0, n] * 3, [1400] * 5)
    want, bound = want_prompt(q, k, v, table, [1500], [0, 90], heads, kvh, hd, hd ** -0.5, "bf16")
    R.check(c.prompt(q, table, [1500], [0, 90])[:90], want[:90], bound[:90])
    want, bound = want_decode(q[:n], k, v, many, lengths, heads, kvh, hd, hd ** -0.5, "bf16", [0, n], [1400])
    R.check(c.decode(q[:n], many, lengths, [0, n], [1400]), want, bound)


# ---- large calls --------------------------------------------------------------------

def some_prompt_rows(c, q, k, v, table, lengths, start, heads, kvh, hd, kind, picked):
    """Results of the picked tokens of a prompt batch against the restatement."""
    got = c.prompt(q, table, lengths, start)
    page = k.shape[2]
    for s, n in enumerate(lengths):
        rows = np.array([t for t in picked if start[s] <= t < start[s + 1]])
        if not len(rows):
            continue
        at = np.arange(n)
        ids = table[s][at // page]
        limits = n - (start[s + 1] - rows) + 1
        want, bound = R.attend(q[rows].reshape(-1, heads, hd), k[ids, :, at % page], v[ids, :, :, at % page], limits,
                               hd ** -0.5, kind)
        R.check(got[rows], want.reshape(len(rows), -1), bound.reshape(len(rows), -1), s)


@pytest.mark.parametrize("kind,heads,kvh,hd,page,new,old", [
    ("bf16", 32, 4, 128, 64, [5000], [0]), ("f16", 32, 8, 64, 16, [4200], [77]), ("f32", 40, 20, 64, 32, [3700], [5]),
    ("bf16", 64, 8, 128, 128, [1100, 1300], [900, 0]), ("f16", 16, 2, 256, 64, [2100], [0]),
    ("f32", 12, 12, 64, 64, [2050], [0]), ("f32", 8, 1, 256, 16, [900], [300])])
def test_prompt_of_thousands(gpu, kind, heads, kvh, hd, page, new, old):
    rng = np.random.default_rng(51)
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[0], np.cumsum(new)])
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((start[-1], heads * hd)) * 1.5, kind)
    edges = [0, 1, 31, 32, 63, 64, 127, start[-1] - 1, start[-1] - 2, start[-1] // 2] + [int(x) for x in start[1:-1]]
    picked = sorted(set(edges + rng.integers(0, start[-1], 8).tolist()))
    some_prompt_rows(c, q, k, v, table, lengths, start, heads, kvh, hd, kind, picked)


@pytest.mark.parametrize("kind,heads,kvh,hd,page,n,old", [
    ("bf16", 32, 4, 128, 64, 4200, 0), ("f16", 64, 8, 64, 16, 2100, 90), ("f32", 8, 2, 256, 16, 300, 40),
    ("f16", 16, 2, 256, 32, 500, 0), ("f32", 16, 4, 128, 128, 600, 1000), ("bf16", 32, 4, 128, 64, 200, 3000)])
def test_prompt_not_finite_values_in_large_tiles(gpu, kind, heads, kvh, hd, page, n, old):
    """The first rows that see an infinity or NaN in V, the last that do not, and rows of every wave about them; two
    in one tile of positions, in different heads."""
    rng = np.random.default_rng(56)
    length = n + old
    table, n_page = tables(rng, [length], page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, [length])
    q = rounded(rng.standard_normal((n, heads * hd)), kind)
    spots = [(old + n // 2, 3, np.nan, 0), (old + n // 2 + 5, hd - 1, np.inf, kvh - 1), (old + n - 40, 0, -np.inf, 0)]
    for pos, d, bad, h in spots:
        v[table[0, pos // page], h, d, pos % page] = bad
    c.write(k, v)
    near = [n // 2 + i for i in (-33, -9, -1, 0, 1, 4, 5, 6, 20, 33)] + [0, n - 41, n - 40, n - 1]
    some_prompt_rows(c, q, k, v, table, [length], np.array([0, n]), heads, kvh, hd, kind, near)


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_of_many_long_sequences(gpu, kind):
    """More sequences than a wave has lanes, with enough rows each for the tiles; one without tokens, one of one."""
    rng = np.random.default_rng(52)
    heads, kvh, hd, page = 16, 1, 64, 32
    new = [int(x) for x in rng.integers(5, 40, 70)]
    new[3], new[66] = 0, 1
    lengths = [a + int(b) for a, b in zip(new, rng.integers(0, 300, 70))]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[0], np.cumsum(new)])
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((start[-1], heads * hd)), kind)
    picked = sorted(set([int(x) for x in start[:-1] if x < start[-1]] + rng.integers(0, start[-1], 30).tolist()))
    some_prompt_rows(c, q, k, v, table, lengths, start, heads, kvh, hd, kind, picked)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n_rot,interleaved", [(64, False), (128, True), (20, True)])
def test_store_of_thousands(gpu, kind, n_rot, interleaved):
    """2300 tokens in 5 sequences: one wave per token, and values over many blocks of positions."""
    rng = np.random.default_rng(53)
    heads, kvh, hd, page = 4, 2, 128, 32
    new, old = [1200, 0, 1, 1000, 99], [3, 9, 31, 17, 0]
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[0], np.cumsum(new)])
    n = int(start[-1])
    q, k, v = (rng.standard_normal((n, h * hd)).astype(np.float32) for h in (heads, kvh, kvh))
    freqs, m = gpu.rope_freqs(n_rot, 10000.0)
    w = (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32)
    c = gpu.PagedCache(kind, n_page, page, heads, kvh, hd)
    got = c.store(q, k, v, table, lengths, start, w, w, 1e-6, freqs, interleaved, m)
    got_k, got_v = c.read()
    want_k, bound_k, want_v = np.zeros(c.shape_k), np.zeros(c.shape_k), np.zeros(c.shape_v)
    for s in range(5):
        rows, pos = slice(start[s], start[s + 1]), np.arange(old[s], lengths[s])
        if not len(pos):
            continue
        want, bound = R.store(q[rows].reshape(-1, heads, hd), w, pos, freqs, n_rot, interleaved, m, 1e-6, kind)
        R.check(got[rows], want.reshape(len(pos), -1), bound.reshape(len(pos), -1), s)
        ids, slots = table[s][pos // page], pos % page
        want_k[ids, :, slots], bound_k[ids, :, slots] = R.store(k[rows].reshape(-1, kvh, hd), w, pos, freqs, n_rot,
                                                                interleaved, m, 1e-6, kind)
        want_v[ids, :, :, slots] = rounded(v[rows].reshape(-1, kvh, hd), kind)
    R.check(got_k, want_k, bound_k, "k")
    assert np.array_equal(got_v, want_v.astype(np.float32))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_pages_past_32_bits(gpu, kind):
    """A cache of more than 2^32 elements: the same tokens at its far end and in a small cache give the same bits."""
    rng = np.random.default_rng(54)
    L, heads, kvh, hd, page = gpu.lib(), 8, 8, 256, 256
    size = 4 if kind == "f32" else 2
    n_page = 2 ** 32 // (kvh * hd * page) + 9
    total = n_page * kvh * hd * page * size
    far_k, far_v = gpu.DeviceBuffer(total), gpu.DeviceBuffer(total)
    near = gpu.PagedCache(kind, 9, page, heads, kvh, hd)
    far = gpu.Pages(far_k.ptr, far_v.ptr, near.pages.type, n_page, page, kvh, hd)
    lengths, start = [300, 700], [0, 300, 1000]
    table = np.array([[0, 1, -1], [7, 3, 5]], np.int32)
    freqs, _ = gpu.rope_freqs(hd, 1e6)
    x = [gpu.DeviceBuffer.from_array(rng.standard_normal((1000, h * hd)).astype(np.float32)) for h in (heads, kvh, kvh)]
    f = gpu.DeviceBuffer.from_array(freqs)
    got = []
    for pages, ids in ((near.pages, table), (far, np.where(table < 0, -1, table + n_page - 9).astype(np.int32))):
        t, o, d = (gpu.DeviceBuffer.from_array(np.zeros((1000, heads * hd), near.dtype)) for _ in range(3))
        b, keep = near._batch(ids, lengths, start, 1000)
        P, B = C.byref(pages), C.byref(b)
        assert L.llamd_hip_paged_store(P, B, x[0].ptr, heads * hd, x[1].ptr, kvh * hd, x[2].ptr, kvh * hd, None, None, 1e-6,
                                       f.ptr, hd, 0, 1.0, heads, t.ptr) == 0
        assert L.llamd_hip_paged_prompt(P, B, t.ptr, heads, hd ** -0.5, near.pages.type, o.ptr) == 0
        assert L.llamd_hip_paged_decode(P, B, None, None, 0, t.ptr, heads, hd ** -0.5, near.pages.type, d.ptr) == 0
        got.append([y.download(np.empty((1000, heads * hd), near.dtype)) for y in (t, o, d)])
    assert got[0][1].any() and got[0][2][:2].any()
    assert all(np.array_equal(a, b) for a, b in zip(*got))
    far_k.close(), far_v.close()


def test_calls_from_two_threads(gpu):
    """Calls of different sizes from two threads share the library's scratch: each gets what it gets alone."""
    import threading
    rng = np.random.default_rng(55)
    heads, kvh, hd, page = 8, 1, 64, 16
    jobs = []
    for lengths, new in (([900, 3000], 1), ([700], 90)):
        table, n_page = tables(rng, lengths, page)
        c, _, _ = filled(gpu, rng, "bf16", table, n_page, page, heads, kvh, hd, lengths)
        q = rounded(rng.standard_normal((new * len(lengths), heads * hd)), "bf16")
        jobs.append((lambda c=c, q=q, t=table, n=lengths: c.decode(q, t, n)) if new == 1 else
                    (lambda c=c, q=q, t=table, n=lengths, m=new: c.prompt(q, t, n, [0, m])))
    alone = [j() for j in jobs]
    seen = [[], []]

    def run(i):
        for _ in range(12):
            seen[i].append(jobs[i]())

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(seen[i]) == 12 and all(np.array_equal(x, alone[i]) for x in seen[i])


# ---- together ---------------------------------------------------------------------

def run_calls(gpu, c, b, dev, heads, hd, group=None):
    L, P, B = gpu.lib(), C.byref(c.pages), C.byref(b)
    kvh = c.pages.n_head_kv
    number = c.pages.type
    assert L.llamd_hip_paged_store(P, B, dev["q"].ptr, heads * hd, dev["k"].ptr, kvh * hd, dev["v"].ptr, kvh * hd,
                                   dev["w"].ptr, dev["w"].ptr, 1e-6, dev["f"].ptr, hd, 0, 1.0, heads, dev["t"].ptr) == 0
    if group is None:
        assert L.llamd_hip_paged_prompt(P, B, dev["t"].ptr, heads, hd ** -0.5, number, dev["o"].ptr) == 0
    else:
        assert L.llamd_hip_paged_decode(P, B, group[0].ptr, group[1].ptr, 1, dev["t"].ptr, heads, hd ** -0.5, number,
                                        dev["o"].ptr) == 0


@pytest.mark.parametrize("kind", KINDS)
def test_a_prompt_and_the_steps_after_it(gpu, kind):
    """A system prompt, users that fork from it, their own prompts, then decode steps: every result against 64-bit
    attention over the values that the cache holds."""
    rng = np.random.default_rng(41)
    heads, kvh, hd, page, base = 8, 2, 128, 16, 75
    freqs, m = gpu.rope_freqs(hd, 1e6)
    w = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    c = gpu.PagedCache(kind, 64, page, heads, kvh, hd)

    def step(new, lengths, table, group=None, shared=None):
        n = sum(new)
        q, k, v = (rng.standard_normal((n, h * hd)).astype(np.float32) for h in (heads, kvh, kvh))
        start = np.concatenate([[0], np.cumsum(new)])
        turned = c.store(q, k, v, table, lengths, start, w, w, 1e-6, freqs)
        pages_k, pages_v = c.read()
        if group is None:
            got = c.prompt(turned, table, lengths, start)
            want, bound = want_prompt(turned, pages_k, pages_v, table, lengths, start, heads, kvh, hd, hd ** -0.5, kind)
        else:
            got = c.decode(turned, table, lengths, group, shared)
            want, bound = want_decode(turned, pages_k, pages_v, table, lengths, heads, kvh, hd, hd ** -0.5, kind, group, shared)
        R.check(got, want, bound)

    table = np.full((3, 12), -1, np.int32)
    table[0, :6] = [9, 3, 50, 7, 22, 41]
    step([base], [base], table[:1])
    full = base // page
    k, v = c.read()
    for s in (1, 2):  # the page that the prompt ends in is copied
        table[s, :full], table[s, full] = table[0, :full], 10 + s
        k[10 + s], v[10 + s] = k[table[0, full]], v[table[0, full]]
    c.write(k, v)
    table[0, 6:9], table[1, 5:9], table[2, 5:9] = [30, 31, 32], [33, 34, 35, 36], [60, 61, 62, 63]
    lengths = [base + 20, base + 1, base + 33]
    step([20, 1, 33], lengths, table)
    for _ in range(4):
        lengths = [n + 1 for n in lengths]
        step([1, 1, 1], lengths, table, [0, 3], [base])


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_captured_calls_follow_the_device(gpu, kind):
    """Store, prompt and decode captured once, replayed with other lengths, tables and inputs, with eager calls (also
    larger ones) between the replays: every replay gives the eager call's bits."""
    L = gpu.lib()
    rng = np.random.default_rng(42)
    heads, kvh, hd, page, n_page = 8, 2, 64, 16, 300
    c = gpu.PagedCache(kind, n_page, page, heads, kvh, hd)
    freqs, _ = gpu.rope_freqs(hd, 1e6)

    def inputs(n):
        x = {k: rng.standard_normal((n, h * hd)).astype(np.float32) for k, h in (("q", heads), ("k", kvh), ("v", kvh))}
        x["w"], x["f"] = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32), freqs
        return x

    for mode in ("prompt", "decode"):
        n_tok, n_seq, max_page = (40, 3, 60) if mode == "prompt" else (4, 4, 60)
        dev = {k: gpu.DeviceBuffer.from_array(x) for k, x in inputs(n_tok).items()}
        for k in "to":
            dev[k] = gpu.DeviceBuffer.from_array(np.zeros((n_tok, heads * hd), c.dtype))
        b, keep = c._batch(np.zeros((n_seq, max_page), np.int32), np.zeros(n_seq), np.zeros(n_seq + 1), n_tok)
        group = None if mode == "prompt" else [gpu.DeviceBuffer.from_array(np.array(x, np.int32)) for x in ([0, 4], [0])]
        fill = lambda: c.write(*(np.zeros(s, np.float32) for s in (c.shape_k, c.shape_v)))  # noqa: E731
        assert L.llamd_fwd_begin_capture() == 0
        run_calls(gpu, c, b, dev, heads, hd, group)
        assert L.llamd_fwd_end_capture() == 0
        for turn, lengths in enumerate(([20, 30, 9, 40], [900, 700, 15, 12], [1, 1, 1, 1], [500, 40, 950, 60])):
            lengths = lengths[:n_seq]
            new = [1] * 4 if mode == "decode" else [min(n, 12) for n in lengths]
            order = rng.permutation(n_page)
            table = np.stack([order[i * max_page:(i + 1) * max_page] for i in range(n_seq)]).astype(np.int32)
            keep[0].upload(np.array(lengths, np.int32))
            keep[1].upload(table)
            keep[2].upload(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
            if group:
                group[1].upload(np.array([min(lengths) - 1], np.int32))
            for k, x in inputs(n_tok).items():
                dev[k].upload(x)
            got = []
            for graph in (False, True):
                fill()
                for k in "to":
                    dev[k].upload(np.zeros((n_tok, heads * hd), c.dtype))
                if graph:
                    assert L.llamd_fwd_graph_launch() == 0
                else:
                    run_calls(gpu, c, b, dev, heads, hd, group)
                assert L.llamd_fwd_sync() == 0
                got.append([dev[k].download(np.empty((n_tok, heads * hd), c.dtype)) for k in "to"] + list(c.read()))
                # a larger call between: its scratch may move the library's
                big_t, big_n = tables(rng, [1500 * (turn + 1)], page, 0)
                if not graph and big_n <= n_page:
                    big = gpu.PagedCache(kind, big_n, page, heads, kvh, hd)
                    big.prompt(rng.standard_normal((600, heads * hd)), big_t, [1500 * (turn + 1)], [0, 600])
                    big.close()
            assert got[0][1].any()
            for x, y in zip(*got):
                assert np.array_equal(x, y), (mode, turn)
        L.llamd_fwd_graph_destroy()
    assert L.llamd_fwd_last_error() == 0

"""The 8-bit cache's operators against 64-bit restatements, where they can go wrong: units that grow token by token, blocks and
pages that end inside each other, missing pages, rows that see nothing, NaN and scales of any byte in masked places, groups,
captured calls. Attention's bounds are paged_reference's for a bf16 cache of the values that the pages hold."""
import ctypes as C

import numpy as np
import pytest

import paged8_reference as R8
import paged_reference as R
from test_gpu_paged import rounded, shared_tables, tables, want_decode, want_prompt

pytestmark = pytest.mark.gpu


def filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths, spread=2.0):
    """(cache, K, V): values of different sizes at the lengths' positions, NaN everywhere else, and any byte for the scales
    of 16 positions that have none."""
    c = gpu.PagedCache8(n_page, page, heads, kvh, hd)
    k, v = np.full(c.shape_k, np.nan, np.float32), np.full(c.shape_v, np.nan, np.float32)
    for row, n in zip(table, lengths):
        at = np.arange(n)
        size = np.exp2(rng.uniform(-spread, spread, (2, -(-n // 16), kvh, 1))).repeat(16, 1)[:, :n]
        k[row[at // page], :, at % page] = rng.standard_normal((n, kvh, hd)) * size[0]
        v[row[at // page], :, :, at % page] = rng.standard_normal((n, kvh, hd)) * size[1]
    c.write(k, v)
    none = np.isnan(k).reshape(n_page, kvh, page // 16, -1).all(-1)
    b = [x.copy() for x in c.read_bytes()]
    for s in b[2:]:
        s[none] = rng.choice([0, 1, 127, 254, 255], none.sum())
    c.write_bytes(*b)
    with np.errstate(all="ignore"):
        return (c, *c.read())


# ---- store ------------------------------------------------------------------------

def store_and_check(gpu, rng, heads, kvh, hd, page, n_rot, interleaved, norm, new, old, lead=2, behind=3, table=None):
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[lead], lead + np.cumsum(new)])
    tokens = start[-1] + behind
    q, k, v = (rng.standard_normal((tokens, h * hd)).astype(np.float32) * 2 for h in (heads, kvh, kvh))
    k *= np.exp2(rng.uniform(-3, 3, (tokens, 1))).astype(np.float32)
    v *= np.exp2(rng.uniform(-3, 3, (tokens, 1))).astype(np.float32)
    qw, kw = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)) if norm else (None, None)
    freqs, m = (gpu.rope_freqs(n_rot, 1e6, 4.0, 512) if n_rot else (None, 1.0))
    c, before_k, before_v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    scales = c.read_bytes()[2:]
    want_k, want_v = R8.Pages(before_k, scales[0]), R8.Pages(before_v.swapaxes(2, 3), scales[1])
    got = c.store(q, k, v, table, lengths, start, qw, kw, 1e-5, freqs, interleaved, m)
    want_q, bound_q = np.zeros((tokens, heads, hd)), np.zeros((tokens, heads, hd))
    for s in range(len(new)):
        rows, pos = slice(start[s], start[s + 1]), np.arange(old[s], lengths[s])
        if not len(pos):
            continue
        want_q[rows], bound_q[rows] = R.store(q[rows].reshape(-1, heads, hd), qw, pos, freqs, n_rot, interleaved, m, 1e-5, "bf16")
        y, off = R8.keys(k[rows].reshape(-1, kvh, hd), kw, pos, freqs, n_rot, interleaved, m, 1e-5)
        want_k.append(y, off, table[s], old[s], page)
        y = v[rows].reshape(-1, kvh, hd).astype(np.float64)
        want_v.append(y, np.zeros(y.shape), table[s], old[s], page)
    R.check(got, want_q.reshape(tokens, -1), bound_q.reshape(tokens, -1), "q")
    with np.errstate(all="ignore"):
        got_k, got_v = c.read()
    _, _, ks, vs = c.read_bytes()
    want_k.check(got_k, ks, "k")
    want_v.check(got_v.swapaxes(2, 3), vs, "v")
    assert np.array_equal(want_v.low, want_v.high)


@pytest.mark.parametrize("heads,kvh,hd,page,n_rot,interleaved,norm", [
    (32, 4, 128, 64, 128, False, True), (16, 8, 128, 16, 64, True, False), (12, 12, 64, 32, 64, False, True),
    (3, 1, 64, 16, 32, False, True), (8, 2, 256, 128, 256, True, True), (5, 5, 256, 256, 100, False, False),
    (6, 3, 64, 16, 18, True, True), (2, 1, 128, 32, 0, False, True)])
def test_store(gpu, heads, kvh, hd, page, n_rot, interleaved, norm):
    store_and_check(gpu, np.random.default_rng(11), heads, kvh, hd, page, n_rot, interleaved, norm, [1, 0, 37, 2, 70, 1],
                    [0, 5, 3, 900, 61, 15])


@pytest.mark.parametrize("n_rot,interleaved", [(64, False), (128, True), (20, True)])
def test_store_of_thousands(gpu, n_rot, interleaved):
    """One wave per token for the queries, and many blocks."""
    store_and_check(gpu, np.random.default_rng(12), 4, 2, 128, 32, n_rot, interleaved, True, [1200, 0, 1, 1000, 99],
                    [3, 9, 31, 17, 0])


def test_store_of_many_sequences(gpu):
    rng = np.random.default_rng(13)
    new = [int(x) for x in rng.integers(0, 4, 150)]
    store_and_check(gpu, rng, 4, 1, 64, 16, 64, False, True, new, [int(x) for x in rng.integers(0, 40, 150)])


def test_values_that_grow_token_by_token(gpu):
    """Token after token into the same 16 positions, larger and larger, smaller again: the units are those of the tokens stored
    at once, numbers that were rounded again are off below the normal numbers only."""
    rng = np.random.default_rng(14)
    heads, kvh, hd, page, n = 2, 2, 64, 32, 40
    size = np.exp2(rng.permutation(np.concatenate([np.arange(-12, 20), [60, -60, 100, -100, 0, 0, 1, 3]])))[:, None]
    k, v = (rng.standard_normal((n, kvh * hd)).astype(np.float32) * size.astype(np.float32) for _ in range(2))
    k[5], v[5] = 0, 0
    q = np.zeros((n, heads * hd), np.float32)
    one, each = (gpu.PagedCache8(2, page, heads, kvh, hd) for _ in range(2))
    table = np.array([[1, 0]], np.int32)
    one.store(q, k, v, table, [n], [0, n])
    want = [R8.Pages(np.zeros(one.shape_k), np.ones(one.shape_scale)) for _ in range(2)]
    for t in range(n):
        each.store(q[t:t + 1], k[t:t + 1], v[t:t + 1], table, [t + 1])
        for w, x in zip(want, (k, v)):
            w.append(x[t].astype(np.float64).reshape(1, kvh, hd), np.zeros((1, kvh, hd)), table[0], t, page)
    a, b = one.read_bytes(), each.read_bytes()
    assert np.array_equal(a[2], b[2]) and np.array_equal(a[3], b[3])
    for got in (one, each):
        x = got.read()
        want[0].check(x[0], got.read_bytes()[2], "k")
        want[1].check(x[1].swapaxes(2, 3), got.read_bytes()[3], "v")
    # normal numbers of the last unit are the same bytes
    for i, turn in ((0, lambda x: x), (1, lambda x: x.swapaxes(2, 3))):
        normal = (turn(a[i]) & 127) >= 8
        assert np.array_equal(turn(a[i])[normal], turn(b[i])[normal]) and normal.any()


def test_positions_behind_the_new_ones_stay(gpu):
    """What lies behind the new tokens in their 16 positions, and in the rest of the cache, keeps its bytes."""
    rng = np.random.default_rng(15)
    heads, kvh, hd, page = 4, 2, 128, 32
    c, _, _ = filled(gpu, rng, np.array([[0, 1, 2]]), 4, page, heads, kvh, hd, [96])
    before = c.read_bytes()
    x = [rng.standard_normal((3, h * hd)).astype(np.float32) * 50 for h in (heads, kvh, kvh)]
    c.store(*x, np.array([[2, 1]], np.int32), [40], [0, 3])  # positions 37 .. 39: page 1, slots 5 .. 7
    after = c.read_bytes()
    for i, (a, b) in enumerate(zip(before, after)):
        same = a == b
        if i < 2:
            s = same if i == 0 else same.swapaxes(2, 3)
            assert s[[0, 2, 3]].all() and s[1, :, 8:].all() and not s[1, :, 5:8].all()
        else:
            assert same[[0, 2, 3]].all() and same[1, :, 1].all() and (b[1, :, 0] > a[1, :, 0]).all()


def test_a_sequence_that_is_cut_and_goes_on(gpu):
    """Inside 16 positions the unit of the tokens cut off stays and those before keep their bytes; from a multiple of 16 on the
    unit is the new tokens'."""
    rng = np.random.default_rng(28)
    heads, kvh, hd, page = 2, 2, 64, 32
    table = np.array([[1, 0]], np.int32)
    c = gpu.PagedCache8(2, page, heads, kvh, hd)
    x = [rng.standard_normal((40, h * hd)).astype(np.float32) for h in (heads, kvh, kvh)]
    for a in x:
        a[20:24] *= 2.0 ** 12
    c.store(*x, table, [40], [0, 40])
    before = c.read_bytes()
    new = [rng.standard_normal((22, h * hd)).astype(np.float32) for h in (heads, kvh, kvh)]
    c.store(*(a[:3] for a in new), table, [23], [0, 3])      # positions 20 .. 22 again
    for i, turn in ((0, lambda b: b), (1, lambda b: b.swapaxes(2, 3))):
        after = c.read_bytes()
        assert np.array_equal(before[2 + i], after[2 + i])
        was, now = turn(before[i]), turn(after[i])
        assert np.array_equal(was[1, :, :20], now[1, :, :20]) and np.array_equal(was[1, :, 23:], now[1, :, 23:])
        got = turn(c.read()[i])[1, :, 20:23].swapaxes(0, 1).reshape(3, -1)
        unit = 2.0 ** (after[2 + i][1, :, 1].astype(float) - 127).repeat(hd)
        assert (np.abs(got - new[1 + i][:3]) <= np.maximum(2.0 ** -4 * np.abs(new[1 + i][:3]), 2.0 ** -10 * unit)).all()
    c.store(*new, table, [38], [0, 22])                      # positions 16 .. 37
    after = c.read_bytes()
    assert (after[2][1, :, 1] < before[2][1, :, 1]).all() and (after[3][1, :, 1] < before[3][1, :, 1]).all()
    got = c.read()[0][1, :, 16:].swapaxes(0, 1).reshape(16, -1)
    assert (np.abs(got - new[1][:16]) <= np.maximum(2.0 ** -4 * np.abs(new[1][:16]), 2.0 ** -10 * 2.0 ** -6)).all()


def test_not_finite_values_are_nan_and_do_not_count(gpu):
    rng = np.random.default_rng(16)
    heads, kvh, hd, page, n = 2, 1, 64, 16, 20
    x = {h: rng.standard_normal((n, h * hd)).astype(np.float32) for h in (heads, kvh)}
    k, v = x[kvh].copy(), x[kvh][::-1].copy()
    plain = gpu.PagedCache8(2, page, heads, kvh, hd)
    plain.store(x[heads], k, v, [[0, 1]], [n], [0, n])
    spots = [(3, 5, np.inf), (7, 60, -np.inf), (7, 61, np.nan), (18, 0, np.nan)]
    for t, d, bad in spots:
        k[t, d] = v[t, d] = bad
    k[19], v[19] = np.nan, np.inf
    c = gpu.PagedCache8(2, page, heads, kvh, hd)
    c.store(x[heads], k, v, [[0, 1]], [n], [0, n])
    a, b = plain.read_bytes(), c.read_bytes()
    bad = ~np.isfinite(k)
    got_k = gpu.from_e4m3(b[0]).reshape(2 * page, hd)[:n]
    got_v = gpu.from_e4m3(b[1]).transpose(0, 1, 3, 2).reshape(2 * page, hd)[:n]
    assert np.isnan(got_k[bad]).all() and np.isfinite(got_k[~bad]).all()
    assert np.isnan(got_v[~np.isfinite(v)]).all() and np.isfinite(got_v[np.isfinite(v)]).all()
    assert np.array_equal(a[2][0], b[2][0]) and np.array_equal(a[3][0], b[3][0])
    # a block of nothing finite
    c.store(x[heads][:1], np.full((1, hd), np.nan, np.float32), np.full((1, hd), np.inf, np.float32), [[0, 1]], [1])
    assert c.read_bytes()[2][0, 0, 0] == 1 and (c.read_bytes()[0][0, 0, 0] & 127 == 127).all()


def test_store_without_a_place(gpu):
    """Missing pages, ids outside the cache, tokens before position 0 and past the table: q is turned, nothing is stored."""
    rng = np.random.default_rng(17)
    heads, kvh, hd, page = 4, 2, 64, 16
    c = gpu.PagedCache8(4, page, heads, kvh, hd)
    table = np.array([[0, -1], [4, 1], [1 << 30, 2], [3, 3]], np.int32)
    lengths, start = [17, 3, 16, 32], [0, 2, 6, 8, 9]  # sequence 1: four tokens, the first at position -1
    q, k, v = (rng.standard_normal((9, h * hd)).astype(np.float32) for h in (heads, kvh, kvh))
    freqs, m = gpu.rope_freqs(hd, 10000.0)
    got = c.store(q, k, v, table, lengths, start, None, None, 1e-6, freqs)
    pos = np.array([15, 16, -1, 0, 1, 2, 14, 15, 31])
    want, bound = R.store(q.reshape(9, heads, hd), None, pos, freqs, hd, False, m, 0, "bf16")
    R.check(got, want.reshape(9, -1), bound.reshape(9, -1))
    w, off = R8.keys(k.reshape(9, kvh, hd), None, pos, freqs, hd, False, m, 0)
    want_k, want_v = (R8.Pages(np.zeros(c.shape_k), np.ones(c.shape_scale)) for _ in range(2))
    for t, (s, at) in enumerate(zip([0, 0, 1, 1, 1, 1, 2, 2, 3], pos)):
        if at < 0:
            continue
        want_k.append(w[t:t + 1], off[t:t + 1], table[s], at, page)
        want_v.append(v[t].reshape(1, kvh, hd).astype(np.float64), np.zeros((1, kvh, hd)), table[s], at, page)
    x = c.read()
    want_k.check(x[0], c.read_bytes()[2], "k")
    want_v.check(x[1].swapaxes(2, 3), c.read_bytes()[3], "v")


def test_store_side_by_side_and_without_q(gpu):
    """Q, K and V as one matrix's columns; then K and V alone."""
    rng = np.random.default_rng(18)
    L, heads, kvh, hd, page, n = gpu.lib(), 4, 2, 64, 16, 21
    wide = (heads + 2 * kvh) * hd + 8
    x = rng.standard_normal((n, wide)).astype(np.float32)
    q, k, v = (np.ascontiguousarray(x[:, a * hd:b * hd]) for a, b in ((0, 4), (4, 6), (6, 8)))
    table = np.array([[2, 0]], np.int32)
    freqs, _ = gpu.rope_freqs(hd, 10000.0)
    c = gpu.PagedCache8(4, page, heads, kvh, hd)
    want = c.store(q, k, v, table, [n], [0, n], None, None, 1e-6, freqs)
    X, F = gpu.DeviceBuffer.from_array(x), gpu.DeviceBuffer.from_array(freqs)
    out = gpu.DeviceBuffer.from_array(np.zeros((n, heads * hd), np.uint16))
    for with_q in (True, False):
        d = gpu.PagedCache8(4, page, heads, kvh, hd)
        b, keep = d._batch(table, [n], [0, n], n)
        at = [X.ptr + 4 * hd * i for i in (0, 4, 6)]
        assert L.llamd_hip_paged8_store(C.byref(d.pages), C.byref(b), at[0] if with_q else None, wide, at[1], wide, at[2], wide,
                                        None, None, 1e-6, F.ptr, hd, 0, 1.0, heads, out.ptr if with_q else None) == 0
        assert all(np.array_equal(a, b) for a, b in zip(c.read_bytes(), d.read_bytes()))
        assert np.array_equal(gpu.from_bf16(out.download(np.empty((n, heads * hd), np.uint16))), want)


# ---- prompts ----------------------------------------------------------------------

@pytest.mark.parametrize("heads,kvh,hd,page,new,old", [
    (32, 4, 128, 64, [1, 0, 5, 33], [0, 7, 60, 31]),
    (16, 8, 128, 16, [64, 1, 17], [0, 15, 130]),
    (12, 12, 64, 32, [1, 31, 32, 33, 65], [0, 1, 0, 63, 200]),
    (16, 1, 64, 16, [3, 40], [0, 300]),
    (3, 1, 64, 128, [70, 2], [129, 0]),
    (40, 1, 128, 64, [9], [50]),
    (8, 2, 256, 32, [20, 7], [3, 100]),
    (4, 4, 128, 256, [130], [190])])
def test_prompt(gpu, heads, kvh, hd, page, new, old):
    rng = np.random.default_rng(21)
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[0], np.cumsum(new)])
    tokens = start[-1] + 2
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((tokens, heads * hd)) * 1.5, "bf16")
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, hd ** -0.5, "bf16")
    got = c.prompt(q, table, lengths, start)
    R.check(got, want, bound)
    assert not got[-2:].any()


@pytest.mark.parametrize("heads,kvh,hd,page,new,old", [
    (4, 4, 64, 32, [700], [0]), (8, 1, 128, 16, [300, 1, 290], [500, 2000, 0]), (4, 4, 128, 64, [200], [2500]),
    (2, 1, 256, 16, [150], [900]), (12, 4, 64, 128, [5, 260], [6000, 11])])
def test_prompt_long(gpu, heads, kvh, hd, page, new, old):
    rng = np.random.default_rng(22)
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[0], np.cumsum(new)])
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((start[-1], heads * hd)) * 2, "bf16")
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, 0.1, "bf16")
    R.check(c.prompt(q, table, lengths, start, scale=0.1), want, bound)


@pytest.mark.parametrize("heads,kvh,hd,page,new,old", [
    (32, 4, 128, 64, [256], [500]), (8, 2, 128, 16, [90, 300, 1, 77], [600, 0, 700, 333]), (8, 2, 256, 64, [100, 33, 90], [900, 871, 4]),
    (12, 12, 64, 32, [512], [0]), (2, 2, 64, 128, [1000], [24])])
def test_prompt_of_a_turn(gpu, heads, kvh, hd, page, new, old):
    """Many rows after contexts of up to 1024 positions, as many as run at once and a few more."""
    rng = np.random.default_rng(24)
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[0], np.cumsum(new)])
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((start[-1] + 3, heads * hd)) * 1.5, "bf16")
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, hd ** -0.5, "bf16")
    got = c.prompt(q, table, lengths, start)
    R.check(got, want, bound)
    assert not got[-3:].any()


def test_f32_results(gpu):
    rng = np.random.default_rng(23)
    table, n_page = tables(rng, [90, 4], 16)
    c, k, v = filled(gpu, rng, table, n_page, 16, 8, 2, 128, [90, 4])
    q = rounded(rng.standard_normal((34, 8 * 128)), "bf16")
    want, bound = want_prompt(q, k, v, table, [90, 4], [0, 30, 34], 8, 2, 128, 128 ** -0.5, "bf16", "f32")
    R.check(c.prompt(q, table, [90, 4], [0, 30, 34], f32_out=True), want, bound)
    got = c.decode(q[[29, 33]], table, [90, 4], f32_out=True)
    R.check(got, want[[29, 33]], bound[[29, 33]])


@pytest.mark.parametrize("heads,kvh,hd,new", [(8, 2, 64, [40, 20, 9, 50, 3]), (32, 2, 128, [400, 200, 90, 300, 3])])
def test_prompt_missing_pages_and_empty_rows(gpu, heads, kvh, hd, new):
    """Ids outside the cache, tokens before position 0, a length past the table: such positions have no part, and rows
    that see nothing are 0. Few rows and large tiles."""
    rng = np.random.default_rng(24)
    page = 16
    lengths = [n + x for n, x in zip(new, [30, 0, -6, 50, 37])]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    table = table[:, :lengths[0] // page + 1].copy()
    table[0, 1], table[0, 3] = -1, n_page
    table[1, :] = -1
    table[1, :2] = [1 << 30, -5]  # sequence 1 has no pages at all
    start = np.concatenate([[0], np.cumsum(new)])
    q = rounded(rng.standard_normal((start[-1], heads * hd)), "bf16")
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, hd ** -0.5, "bf16")
    got = c.prompt(q, table, lengths, start)
    R.check(got, want, bound)
    assert not got[start[1]:start[2]].any() and not got[start[2]:start[2] + 6].any()


@pytest.mark.parametrize("heads,kvh,hd,page,n,old,spots", [
    (4, 2, 64, 16, 90, 0, (47, 66)), (32, 4, 128, 64, 2200, 0, (1100, 1105, 2160)), (16, 2, 256, 32, 500, 0, (250, 460)),
    (16, 4, 128, 128, 600, 1000, (1300, 1560))])
def test_prompt_nan_stays_with_those_who_see_it(gpu, heads, kvh, hd, page, n, old, spots):
    """NaN in V touches no row before it, and the rows after it in its dimensions only."""
    rng = np.random.default_rng(25)
    length = n + old
    table, n_page = tables(rng, [length], page)
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, [length])
    b = [x.copy() for x in c.read_bytes()]
    for i, pos in enumerate(spots):
        b[1][table[0, pos // page], i % kvh, 3 + i, pos % page] = 127
        v[table[0, pos // page], i % kvh, 3 + i, pos % page] = np.nan
    c.write_bytes(*b)
    q = rounded(rng.standard_normal((n, heads * hd)), "bf16")
    got = c.prompt(q, table, [length], [0, n])
    near = sorted({t for pos in spots for t in range(pos - old - 33, pos - old + 20, 7) if 0 <= t < n} |
                  {x for pos in spots for x in (pos - old - 1, pos - old)} | {0, n - 1})
    at = np.arange(length)
    ids = table[0][at // page]
    want, bound = R.attend(q[near].reshape(-1, heads, hd), k[ids, :, at % page], v[ids, :, :, at % page], old + np.array(near) + 1,
                           hd ** -0.5, "bf16")
    R.check(got[near], want.reshape(len(near), -1), bound.reshape(len(near), -1))
    assert np.isnan(want).any() and np.isfinite(want[0]).all()


def test_prompt_starts_that_make_no_sense(gpu):
    """Starts that descend or leave the buffer never reach past it; the sequences that do make sense are right."""
    rng = np.random.default_rng(26)
    heads, kvh, hd, page = 4, 2, 64, 16
    table, n_page = tables(rng, [30, 30, 30], page)
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, [30, 30, 30])
    q = rounded(rng.standard_normal((40, heads * hd)), "bf16")
    want, bound = want_prompt(q, k, v, table, [30], [0, 10], heads, kvh, hd, hd ** -0.5, "bf16")
    R.check(c.prompt(q, table, [30, 30, 30], [0, 10, 1 << 30, 20])[:10], want[:10], bound[:10])
    got = c.prompt(q, table, [30, -7, -(1 << 31)], [0, 10, 20, 40])
    R.check(got[:10], want[:10], bound[:10])
    assert not got[10:].any()
    x = [rng.standard_normal((40, h * hd)).astype(np.float32) for h in (heads, kvh, kvh)]
    c.store(*x, table, [30, 30, 30], [0, 10, 1 << 30, 20])
    c.store(*x, table, [30, -7, -(1 << 31)], [0, 10, 20, 40])


@pytest.mark.parametrize("heads,kvh,hd,page,new,old", [
    (32, 4, 128, 64, [5000], [0]), (32, 8, 64, 16, [4200], [77]), (64, 8, 128, 128, [1100, 1300], [900, 0]),
    (16, 2, 256, 64, [2100], [0]), (16, 1, 64, 32, [20] * 70, [100] * 70)])
def test_prompt_of_thousands(gpu, heads, kvh, hd, page, new, old):
    rng = np.random.default_rng(51)
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[0], np.cumsum(new)])
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((start[-1], heads * hd)) * 1.5, "bf16")
    edges = [0, 1, 31, 32, 63, 64, 127, start[-1] - 1, start[-1] - 2, start[-1] // 2] + [int(x) for x in start[1:-1]]
    picked = np.array(sorted(set(edges + rng.integers(0, start[-1], 8).tolist())))
    got = c.prompt(q, table, lengths, start)
    for s, n in enumerate(lengths):
        rows = picked[(picked >= start[s]) & (picked < start[s + 1])]
        at = np.arange(n)
        ids = table[s][at // page]
        want, bound = R.attend(q[rows].reshape(-1, heads, hd), k[ids, :, at % page], v[ids, :, :, at % page],
                               n - (start[s + 1] - rows) + 1, hd ** -0.5, "bf16")
        R.check(got[rows], want.reshape(len(rows), -1), bound.reshape(len(rows), -1), s)


# ---- decode -----------------------------------------------------------------------

@pytest.mark.parametrize("heads,kvh,hd,page,lengths", [
    (32, 4, 128, 64, [1, 0, 63, 64, 65, 700]), (16, 8, 128, 16, [31, 32, 33, 129]), (12, 12, 64, 32, [5, 300, 1]),
    (16, 1, 64, 128, [2000, 3]), (40, 1, 64, 16, [77, 400]), (8, 2, 256, 256, [600, 1, 255]), (3, 1, 128, 16, [4100]),
    (8, 1, 64, 256, [26_000]), (4, 4, 64, 64, [11_000, 0, 3, 40_000]), (20, 1, 64, 128, [9_000, 130])])
def test_decode(gpu, heads, kvh, hd, page, lengths):
    rng = np.random.default_rng(31)
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((len(lengths) + 1, heads * hd)) * 1.5, "bf16")
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "bf16")
    got = c.decode(q, table, lengths)
    R.check(got[:-1], want, bound)
    assert not got[-1].any()   # the row behind the last sequence


@pytest.mark.parametrize("heads,kvh,hd,page,group,shared,lengths", [
    (32, 4, 128, 64, [0, 6], [128], [129, 300, 128, 700, 1000, 131]),
    (16, 8, 128, 16, [0, 2, 3, 8], [40, 17, 100], [45, 41, 60, 100, 101, 300, 116, 117]),
    (12, 12, 64, 32, [1, 5], [333], [20, 334, 600, 333, 400, 7]),
    (16, 1, 64, 16, [0, 3, 3, 6], [2000, 5, 0], [2100, 2001, 2500, 30, 40, 50]),
    (8, 2, 256, 64, [0, 20], [70], [71 + i for i in range(20)]),
    (8, 1, 128, 32, [0, 40], [900], [901 + 3 * i for i in range(40)])])
def test_decode_shared_prefix(gpu, heads, kvh, hd, page, group, shared, lengths):
    rng = np.random.default_rng(32)
    table, n_page, copies = shared_tables(rng, group, shared, lengths, page)
    c, _, _ = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    b = [x.copy() for x in c.read_bytes()]
    for to, of, _ in copies:
        for x in b:
            x[to] = x[of]
    # what a copied page has behind the prefix, NaN or not, is some sequence's own
    for x in (b[0], b[1]):
        x[x & 127 == 127] = 3
    for x in (b[2], b[3]):
        x[(x < 100) | (x > 150)] = 120
    c.write_bytes(*b)
    k, v = c.read()
    q = rounded(rng.standard_normal((len(lengths), heads * hd)) * 1.5, "bf16")
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "bf16", group, shared)
    R.check(c.decode(q, table, lengths, group, shared), want, bound)
    # the same batch without the groups
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "bf16")
    R.check(c.decode(q, table, lengths), want, bound)


@pytest.mark.parametrize("heads,kvh,hd,page,group,shared,lengths", [
    (32, 4, 128, 64, [0, 8], [4100], [4101 + 37 * i for i in range(8)]),
    (8, 2, 256, 64, [1, 4], [2600], [5, 2601, 2600, 2900]),
    (8, 1, 64, 16, [0, 3, 6], [1500, 600], [1500, 1501, 1700, 601, 900, 650])])
def test_decode_long_shared_prefix(gpu, heads, kvh, hd, page, group, shared, lengths):
    """Few tiles of long prefixes, cut into short parts; the same call again gives the same bits."""
    rng = np.random.default_rng(35)
    table, n_page, copies = shared_tables(rng, group, shared, lengths, page)
    c, _, _ = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    b = [x.copy() for x in c.read_bytes()]
    for to, of, _ in copies:
        for x in b:
            x[to] = x[of]
    for x in (b[0], b[1]):
        x[x & 127 == 127] = 3
    for x in (b[2], b[3]):
        x[(x < 100) | (x > 150)] = 120
    c.write_bytes(*b)
    k, v = c.read()
    q = rounded(rng.standard_normal((len(lengths), heads * hd)) * 1.5, "bf16")
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "bf16", group, shared)
    got = c.decode(q, table, lengths, group, shared)
    R.check(got, want, bound)
    assert np.array_equal(got, c.decode(q, table, lengths, group, shared))


def test_decode_missing_pages_and_nan_that_a_member_does_not_see(gpu):
    rng = np.random.default_rng(36)
    heads, kvh, hd, page = 8, 2, 64, 32
    lengths, group, shared = [300, 70, 310, 256, 40], [0, 4], [256]
    table, n_page, _ = shared_tables(rng, group, shared, lengths, page)
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    b = [x.copy() for x in c.read_bytes()]
    for h, d, pos in ((0, 3, 80), (0, 44, 255), (1, 7, 280)):
        b[1][table[0, pos // page], h, d, pos % page] = 255
    c.write_bytes(*b)
    with np.errstate(all="ignore"):
        k, v = c.read()
    table[4, 1], table[2, 8] = -1, n_page + 3
    q = rounded(rng.standard_normal((5, heads * hd)), "bf16")
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "bf16", group, shared)
    assert np.isfinite(want[[1, 4]]).all() and not np.isfinite(want[0]).all() and not np.isfinite(want[3]).all()
    R.check(c.decode(q, table, lengths, group, shared), want, bound)


def test_decode_groups_that_make_no_sense(gpu):
    """Descending or outlying group starts and lengths: no access past the arrays, sequences in no group are right."""
    rng = np.random.default_rng(34)
    heads, kvh, hd, page, lengths = 4, 2, 64, 16, [30, 40, 50]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((3, heads * hd)), "bf16")
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "bf16")
    for group, shared in (([2, 1 << 30], [-5]), ([1, 0, 0], [1 << 30, 7]), ([-9, -3, -(1 << 31)], [4, 4]), ([3, 9], [20])):
        R.check(c.decode(q, table, lengths, group, shared), want, bound)


def test_decode_batch_of_many(gpu):
    rng = np.random.default_rng(35)
    heads, kvh, hd, page = 8, 2, 64, 16
    lengths = [int(n) for n in rng.integers(0, 200, 130)]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((130, heads * hd)), "bf16")
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "bf16")
    R.check(c.decode(q, table, lengths), want, bound)


@pytest.mark.parametrize("n", [1, 20, 700])
@pytest.mark.parametrize("k_unit,v_unit", [(20, 30), (100, 240), (127, 20), (1, 1), (127, 240)])
def test_far_scales(gpu, n, k_unit, v_unit):
    """Scales near the ends of what a byte says: keys near nothing weigh alike, masked ones nothing; values stay in proportion
    (f32 results, since bf16's smallest are cut off)."""
    rng = np.random.default_rng(33)
    heads, kvh, hd, page = 8, 2, 64, 16
    table, n_page = tables(rng, [n], page)
    c = gpu.PagedCache8(n_page, page, heads, kvh, hd)
    k, v = (rng.integers(0, 0x70, s).astype(np.uint8) | (rng.integers(0, 2, s) << 7).astype(np.uint8) for s in (c.shape_k, c.shape_v))
    if v_unit == 1:
        v |= 0x60  # (numbers whose product with 2^-126 is normal in f32)
    c.write_bytes(k, v, np.full(c.shape_scale, k_unit), np.full(c.shape_scale, v_unit))
    pages_k, pages_v = c.read()
    q = rounded(rng.standard_normal((1, heads * hd)), "bf16")
    want, bound = want_decode(q, pages_k, pages_v, table, [n], heads, kvh, hd, hd ** -0.5, "bf16")
    # sums of numbers around the smallest normal one are cut off there
    floor = n * 2.0 ** -126
    R.check(c.decode(q, table, [n], f32_out=True), want, bound + floor)
    if n == 700:
        many = np.repeat(q, 130, 0)
        want, bound = want_prompt(many, pages_k, pages_v, table, [n], [0, 130], heads, kvh, hd, hd ** -0.5, "bf16")
        R.check(c.prompt(many, table, [n], [0, 130], f32_out=True), want, bound + floor)


# ---- large caches, threads, graphs ----------------------------------------------------

def test_pages_past_32_bits(gpu):
    """A cache of more than 2^32 elements: the same tokens at its far end and in a small cache give the same bits."""
    rng = np.random.default_rng(54)
    L, heads, kvh, hd, page = gpu.lib(), 8, 8, 256, 256
    n_page = 2 ** 32 // (kvh * hd * page) + 9
    total = n_page * kvh * hd * page
    far_mem = [gpu.DeviceBuffer(total), gpu.DeviceBuffer(total), gpu.DeviceBuffer(total // hd // 16), gpu.DeviceBuffer(total // hd // 16)]
    near = gpu.PagedCache8(9, page, heads, kvh, hd)
    far = gpu.Pages8(*(m.ptr for m in far_mem), n_page, page, kvh, hd)
    lengths, start = [300, 700], [0, 300, 1000]
    table = np.array([[0, 1, -1], [7, 3, 5]], np.int32)
    freqs, _ = gpu.rope_freqs(hd, 1e6)
    x = [gpu.DeviceBuffer.from_array(rng.standard_normal((1000, h * hd)).astype(np.float32)) for h in (heads, kvh, kvh)]
    f = gpu.DeviceBuffer.from_array(freqs)
    got = []
    for pages, ids in ((near.pages, table), (far, np.where(table < 0, -1, table + n_page - 9).astype(np.int32))):
        t, o, d = (gpu.DeviceBuffer.from_array(np.zeros((1000, heads * hd), np.uint16)) for _ in range(3))
        b, keep = near._batch(ids, lengths, start, 1000)
        P, B = C.byref(pages), C.byref(b)
        assert L.llamd_hip_paged8_store(P, B, x[0].ptr, heads * hd, x[1].ptr, kvh * hd, x[2].ptr, kvh * hd, None, None, 1e-6,
                                        f.ptr, hd, 0, 1.0, heads, t.ptr) == 0
        assert L.llamd_hip_paged8_prompt(P, B, t.ptr, heads, hd ** -0.5, 30, o.ptr) == 0
        assert L.llamd_hip_paged8_decode(P, B, None, None, 0, t.ptr, heads, hd ** -0.5, 30, d.ptr) == 0
        got.append([y.download(np.empty((1000, heads * hd), np.uint16)) for y in (t, o, d)])
    assert got[0][1].any() and got[0][2][:2].any()
    assert all(np.array_equal(a, b) for a, b in zip(*got))
    for m in far_mem:
        m.close()


def run_calls(gpu, c, b, dev, heads, hd, group=None):
    L, P, B = gpu.lib(), C.byref(c.pages), C.byref(b)
    kvh = c.pages.n_head_kv
    assert L.llamd_hip_paged8_store(P, B, dev["q"].ptr, heads * hd, dev["k"].ptr, kvh * hd, dev["v"].ptr, kvh * hd,
                                    dev["w"].ptr, dev["w"].ptr, 1e-6, dev["f"].ptr, hd, 0, 1.0, heads, dev["t"].ptr) == 0
    if group is None:
        assert L.llamd_hip_paged8_prompt(P, B, dev["t"].ptr, heads, hd ** -0.5, 30, dev["o"].ptr) == 0
    else:
        assert L.llamd_hip_paged8_decode(P, B, group[0].ptr, group[1].ptr, 1, dev["t"].ptr, heads, hd ** -0.5, 30,
                                         dev["o"].ptr) == 0


def test_captured_calls_follow_the_device(gpu):
    """Store, prompt and decode captured once, replayed with other lengths, tables and inputs, with eager calls (also
    larger ones) between the replays: every replay gives the eager call's bits."""
    L = gpu.lib()
    rng = np.random.default_rng(42)
    heads, kvh, hd, page, n_page = 8, 2, 64, 16, 300
    c = gpu.PagedCache8(n_page, page, heads, kvh, hd)
    freqs, _ = gpu.rope_freqs(hd, 1e6)

    def inputs(n):
        x = {k: rng.standard_normal((n, h * hd)).astype(np.float32) for k, h in (("q", heads), ("k", kvh), ("v", kvh))}
        x["w"], x["f"] = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32), freqs
        return x

    for mode in ("prompt", "decode"):
        n_tok, n_seq, max_page = (40, 3, 60) if mode == "prompt" else (4, 4, 60)
        dev = {k: gpu.DeviceBuffer.from_array(x) for k, x in inputs(n_tok).items()}
        for k in "to":
            dev[k] = gpu.DeviceBuffer.from_array(np.zeros((n_tok, heads * hd), np.uint16))
        b, keep = c._batch(np.zeros((n_seq, max_page), np.int32), np.zeros(n_seq), np.zeros(n_seq + 1), n_tok)
        group = None if mode == "prompt" else [gpu.DeviceBuffer.from_array(np.array(x, np.int32)) for x in ([0, 4], [0])]
        blank = [np.full(s, 5, np.uint8) for s in (c.shape_k, c.shape_v)] + [np.full(c.shape_scale, 121, np.uint8)] * 2
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
                c.write_bytes(*blank)
                for k in "to":
                    dev[k].upload(np.zeros((n_tok, heads * hd), np.uint16))
                if graph:
                    assert L.llamd_fwd_graph_launch() == 0
                else:
                    run_calls(gpu, c, b, dev, heads, hd, group)
                assert L.llamd_fwd_sync() == 0
                got.append([dev[k].download(np.empty((n_tok, heads * hd), np.uint16)) for k in "to"] + list(c.read_bytes()))
                # a larger call between: its scratch may move the library's
                big_t, big_n = tables(rng, [1500 * (turn + 1)], page, 0)
                if not graph and big_n <= n_page:
                    big = gpu.PagedCache8(big_n, page, heads, kvh, hd)
                    big.prompt(rng.standard_normal((600, heads * hd)), big_t, [1500 * (turn + 1)], [0, 600])
                    big.close()
            assert got[0][1].any()
            for x, y in zip(*got):
                assert np.array_equal(x, y), (mode, turn)
        L.llamd_fwd_graph_destroy()
    assert L.llamd_fwd_last_error() == 0


def test_calls_from_two_threads(gpu):
    """Calls of different sizes from two threads share the library's scratch: each gets what it gets alone."""
    import threading
    rng = np.random.default_rng(55)
    heads, kvh, hd, page = 8, 1, 64, 16
    jobs = []
    for lengths, new in (([900, 3000], 1), ([700], 90)):
        table, n_page = tables(rng, lengths, page)
        c, _, _ = filled(gpu, rng, table, n_page, page, heads, kvh, hd, lengths)
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

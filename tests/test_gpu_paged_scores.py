"""Scores so large that neighbours in f32 are far apart: the softmax of finite scores is finite, whatever they are. Some rows have
such scores, made of powers of two and short factors so that they are exact in f32; the others of the same call have ordinary ones.

Two different scores lie 2^-4 of the largest apart, 2^20 at least here, so that a far row's result is the mean of V over the positions
that it sees and whose score is the largest. Weights there are equal, powers of two up to one common factor: off by P's rounding, the
sum over n positions and the result's own rounding. Ordinary rows have paged_reference's bounds."""
import numpy as np
import pytest

import paged_reference as R
from test_gpu_paged import rounded, shared_tables, tables

pytestmark = pytest.mark.gpu
FAR = 8  # dimensions that make a far row's scores

# powers of two: of a far row's q and of k, each within its type
SIZES = [("bf16", 14, 14), ("bf16", 60, 60), ("bf16", 0, 110), ("bf16", 119, 1), ("f32", 14, 13), ("f32", 50, 70), ("f32", 119, 0),
         ("f16", 14, 13), ("f16", 13, 14), ("8", 26, 1), ("8", 31, 0), ("8", 60, 60), ("8", 0, 115), ("8", 120, 0), ("8", 95, -60),
         ("8", -60, 119)]


def filled(gpu, rng, kind, size, table, n_page, page, heads, kvh, hd, lengths):
    """(cache, K, V): K's first dimensions 2^size times 1 to 1.75 of either sign, the same for all of a position."""
    c = gpu.PagedCache8(n_page, page, heads, kvh, hd) if kind == "8" else gpu.PagedCache(kind, n_page, page, heads, kvh, hd)
    cast = "bf16" if kind == "8" else kind
    k, v = np.zeros(c.shape_k, np.float32), np.zeros(c.shape_v, np.float32)
    for row, n in zip(table, lengths):
        at = np.arange(n)
        x = rounded(rng.standard_normal((n, kvh, hd)) * min(2.0 ** size, 1), cast)
        x[..., :FAR] = (2.0 ** size * rng.choice([-1.25, -1.0, 1.0, 1.25, 1.5, 1.75], (n, kvh)))[..., None]
        k[row[at // page], :, at % page] = x
        v[row[at // page], :, :, at % page] = rounded(rng.standard_normal((n, kvh, hd)), cast)
    c.write(k, v)
    return (c, *c.read())


def queries(rng, kind, size, tokens, heads, hd):
    """q, and which rows (token, head) are far: in a pattern that mixes them in every tile."""
    cast = "bf16" if kind == "8" else kind
    q = rounded(rng.standard_normal((tokens, heads, hd)), cast)
    far = rng.random((tokens, heads)) < 0.4
    q[..., :FAR] = 0
    q[far] = 0
    q[far, :FAR] = (2.0 ** size * rng.choice([-1.0, 1.0], far.sum()))[:, None]
    return q, far


def want_rows(q, far, k, v, limit, scale, kind):
    """(out, bound) of one token's heads over k, v [positions, kv heads, hd]."""
    heads, hd = q.shape
    cast = "bf16" if kind == "8" else kind
    out, bound = R.attend(q[None], k, v, [limit], scale, cast)
    out, bound = out[0], bound[0]
    for h in np.nonzero(far)[0]:
        kv = h * k.shape[1] // heads
        s = k[:limit, kv, 0].astype(np.float64) * float(q[h, 0])
        best = v[:limit, kv][s == s.max()].astype(np.float64)
        out[h] = best.mean(0)
        bound[h] = ((2 * limit + 16) * R.U + 2 * R.STEP[cast]) * np.abs(best).mean(0) + R.STEP[cast] * np.abs(out[h])
        if kind == "f16":
            bound[h] += 2.0 ** -25
    return out, bound


def dense(k, v, row, n, page):
    at = np.arange(n)
    return k[row[at // page], :, at % page], v[row[at // page], :, :, at % page]


@pytest.mark.parametrize("kind,q_size,k_size", SIZES)
@pytest.mark.parametrize("heads,kvh,hd,page,new,old", [(4, 2, 64, 16, [1, 9, 20], [3, 0, 300]),    # 16-row tiles
                                                       (4, 1, 256, 32, [40], [600]),
                                                       (32, 4, 128, 64, [300], [2000])])            # larger ones, in parts
def test_prompt(gpu, kind, q_size, k_size, heads, kvh, hd, page, new, old):
    rng = np.random.default_rng(31)
    lengths = [a + b for a, b in zip(new, old)]
    table, n_page = tables(rng, lengths, page)
    start = np.concatenate([[0], np.cumsum(new)])
    c, k, v = filled(gpu, rng, kind, k_size, table, n_page, page, heads, kvh, hd, lengths)
    q, far = queries(rng, kind, q_size, start[-1], heads, hd)
    got = c.prompt(q.reshape(start[-1], -1), table, lengths, start).reshape(q.shape)
    assert np.isfinite(got).all()
    for s in range(len(new)):
        kk, vv = dense(k, v, table[s], lengths[s], page)
        for t in range(0, new[s], max(new[s] // 12, 1)):
            row = start[s] + t
            want, bound = want_rows(q[row], far[row], kk, vv, old[s] + t + 1, hd ** -0.5, kind)
            R.check(got[row], want, bound, (s, t))


@pytest.mark.parametrize("kind,q_size,k_size", SIZES)
@pytest.mark.parametrize("heads,kvh,hd,page,lengths", [(4, 2, 64, 16, [1, 60, 700]), (32, 4, 128, 64, [4100, 5]),
                                                       (6, 2, 256, 128, [900])])
def test_decode(gpu, kind, q_size, k_size, heads, kvh, hd, page, lengths):
    rng = np.random.default_rng(32)
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, kind, k_size, table, n_page, page, heads, kvh, hd, lengths)
    q, far = queries(rng, kind, q_size, len(lengths), heads, hd)
    got = c.decode(q.reshape(len(lengths), -1), table, lengths).reshape(q.shape)
    for s, n in enumerate(lengths):
        want, bound = want_rows(q[s], far[s], *dense(k, v, table[s], n, page), n, hd ** -0.5, kind)
        R.check(got[s], want, bound, s)


@pytest.mark.parametrize("kind,q_size,k_size", SIZES)
def test_decode_shared_prefix(gpu, kind, q_size, k_size):
    """Positions of a row in large tiles and in 16-row ones, put together."""
    rng = np.random.default_rng(33)
    heads, kvh, hd, page, group, shared = 8, 2, 128, 32, [0, 12], [1536]
    lengths = [int(n) for n in rng.integers(1537, 1900, 12)]
    table, n_page, _ = shared_tables(rng, group, shared, lengths, page)
    c, k, v = filled(gpu, rng, kind, k_size, table, n_page, page, heads, kvh, hd, lengths)
    q, far = queries(rng, kind, q_size, 12, heads, hd)
    got = c.decode(q.reshape(12, -1), table, lengths, group, shared).reshape(q.shape)
    for s, n in enumerate(lengths):
        want, bound = want_rows(q[s], far[s], *dense(k, v, table[s], n, page), n, hd ** -0.5, kind)
        R.check(got[s], want, bound, s)

"""Plain 64-bit restatements of the paged-cache operators, with bounds on what the kernels' arithmetic may be off by.

Bounds. u = 2^-24 is half an f32 step, t half a step of the cache's type (f32 2^-24, f16 2^-11, bf16 2^-8), both relative.

store   y = a c - b s: the norm's sum, square root, division and product add at most (hd / 64 + 8) u to a and b, sine and
        cosine of a reduced angle 4 u of 1, the two products and their sum 3 u: 24 u (|a| + |b|) m covers head sizes up to
        256. Then one rounding: t |y|, or half the smallest f16 step (2^-25) below its normal range.
attend  a score's f32 error is at most e = (hd + 4) u scale sum |q_i k_i| (hd products and sums, one scaling, one
        subtraction of the maximum); exp2 and the statistics add 8 u and (n + 8) u: a weight is off by e + (n + 16) u
        relative, in the sum l too, so twice that. P's rounding is t p per position (f16: plus 2^-25 of the largest weight).
        O's sum over n positions adds n u, the exchange of partial results a few u. All of them times sum p |v|; then
        the result's own rounding t |o|."""
import numpy as np

U = 2.0 ** -24
STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def store(x, norm, pos, freqs, n_rot, interleaved, mscale, eps, kind):
    """Rows x [n, heads, hd] at positions pos: (y, bound)."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    y, size = x.copy(), np.abs(x)
    half = n_rot // 2
    if half:
        a = pos.astype(np.float64)[:, None] * freqs
        c, s = (f(a)[:, None] * mscale for f in (np.cos, np.sin))
        one = slice(0, n_rot, 2) if interleaved else slice(0, half)
        two = slice(1, n_rot, 2) if interleaved else slice(half, n_rot)
        u, v = x[..., one], x[..., two]
        y[..., one], y[..., two] = u * c - v * s, u * s + v * c
        size[..., one] = size[..., two] = (np.abs(u) + np.abs(v)) * abs(mscale)
    return y, 24 * U * size + STEP[kind] * np.abs(y) + 2.0 ** -25 * (kind == "f16")


def attend(q, k, v, limits, scale, kind, out_kind=None, visible=None):
    """q [n, heads, hd] against one sequence's k, v [positions, kv heads, hd]; row i sees positions below limits[i] that
    `visible` [positions] has. (out, bound)."""
    n, heads, hd = q.shape
    kvh = k.shape[1]
    out, bound = np.zeros((n, heads, hd)), np.zeros((n, heads, hd))
    for h in range(heads):
        kk, vv = k[:, h * kvh // heads].astype(np.float64), v[:, h * kvh // heads].astype(np.float64)
        for i in range(n):
            at = np.arange(min(max(limits[i], 0), len(kk)))
            if visible is not None:
                at = at[visible[at]]
            if not len(at):
                continue
            qq = q[i, h].astype(np.float64)
            with np.errstate(all="ignore"):
                s = kk[at] @ qq * scale
                size = np.abs(kk[at]) @ np.abs(qq) * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                o, spread = p @ vv[at], p @ np.abs(vv[at])
                e = 2 * ((hd + 4) * U * size.max() + (len(at) + 16) * U) + (len(at) + 8) * U
                if kind != "f32":
                    e += STEP[kind]
                b = e * spread + STEP[out_kind or kind] * np.abs(o)
                if kind == "f16":
                    b = b + 2.0 ** -25 * (p.max() * np.abs(vv[at]).sum(0) + 1)
            out[i, h], bound[i, h] = o, b
    return out, bound


def check(got, want, bound, what=""):
    """Non-finite values where the reference has them, the others within the bound."""
    got, fine = np.asarray(got, np.float64).reshape(want.shape), np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine), (what, np.argwhere(np.isfinite(got) != fine)[:4])
    off = np.abs(got[fine] - want[fine])
    bad = off > bound[fine]
    assert not bad.any(), (what, int(bad.sum()), float(off.max()), float((off / np.maximum(bound[fine], 1e-300)).max()))

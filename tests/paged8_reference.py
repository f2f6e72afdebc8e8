"""A plain 64-bit restatement of the store into 8-bit pages, with bounds on what the kernel's arithmetic may be off by.

Bounds. A key before its rounding is off by paged_reference's 24 u (|a| + |b|) m; a value by nothing. e4m3's half step is 2^-4 of
a value, or 2^-10 of the unit below the normal numbers (2^-6); a number that is rounded again when its unit grows changes below
the normal numbers of the new unit only, by half a step of it each time: 2^-10 of the last unit and less for those before,
2^-9 together. The unit is the one that the largest value needs; within its error of a border, the one on its other side."""
import numpy as np

import paged_reference as R
from llamd_rs_amd import rocm


class Pages:
    """Pages as numbers in 64 bits, in [page, kv head, slot, hd]: `y` what each stands for, `bound`; `unit` scale bytes, `low` and
    `high` the least and largest that the arithmetic may have made of them."""

    def __init__(self, values, unit):
        self.y, self.bound = values.astype(np.float64), np.zeros(values.shape)
        self.low, self.high = unit.astype(int), unit.astype(int)

    def append(self, y, off, row, first, page):
        """y [n, kv heads, hd], each off by `off`, at positions first .. of the sequence with this table row."""
        last = first + len(y)
        for b in range(max(first, 0) // 16, -(-last // 16)):
            lo, hi = max(first, 16 * b, 0), min(last, 16 * b + 16)
            if hi <= lo or 16 * b // page >= len(row) or not 0 <= row[16 * b // page] < len(self.y):
                continue
            at, slot, old = row[16 * b // page], 16 * b % page, lo - 16 * b
            part, part_off = y[lo - first:hi - first].swapaxes(0, 1), off[lo - first:hi - first].swapaxes(0, 1)
            with np.errstate(invalid="ignore"):
                fine = np.isfinite(part)
                size, err = np.where(fine, np.abs(part), 0), np.where(fine, part_off, 0)
            for name, top in (("low", np.maximum(size - err, 0)), ("high", size + err)):
                unit = rocm.scale_byte(top.max((1, 2)).astype(np.float32)).astype(int)
                u = getattr(self, name)
                u[at, :, slot // 16] = np.maximum(unit, u[at, :, slot // 16]) if old else unit
            step = 2.0 ** (self.high[at, :, slot // 16] - 127.0)[:, None, None]
            self.bound[at, :, slot:slot + old] = np.maximum(self.bound[at, :, slot:slot + old], 0) + 2.0 ** -9 * step
            new = slice(slot + old, slot + hi - 16 * b)
            self.y[at, :, new] = np.where(fine, part, np.nan)
            self.bound[at, :, new] = err + 2.0 ** -4 * (size + err) + 2.0 ** -10 * step

    def check(self, got, unit, what=""):
        assert ((unit >= self.low) & (unit <= self.high)).all(), (what, np.argwhere((unit < self.low) | (unit > self.high))[:4])
        R.check(got, self.y, self.bound, what)


def keys(x, norm, pos, freqs, n_rot, interleaved, mscale, eps):
    """(keys, what their arithmetic may be off by)."""
    y, bound = R.store(x, norm, pos, freqs, n_rot, interleaved, mscale, eps, "f32")
    return y, bound

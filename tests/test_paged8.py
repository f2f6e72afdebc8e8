"""The 8-bit cache's entry points without a GPU: what they refuse, and the number format on the host."""
import ctypes as C
import math

import numpy as np
import pytest

from llamd_rs_amd import rocm
from llamd_rs_amd._lib import last_error, lib

GOOD_PAGES = dict(k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=(3 << 20) + 4096, n_page=8, page=64, n_head_kv=4, hd=128)
GOOD_BATCH = dict(start=4 << 20, len=5 << 20, table=6 << 20, n_seq=2, n_tok=10, max_page=4)
FAR = 1 << 30  # addresses that nothing is ever read from: every call here is refused on the host


def call(name, pages=None, batch=None, **kw):
    c = C.byref(rocm.Pages8(**{**GOOD_PAGES, **(pages or {})}))
    b = C.byref(rocm.Batch(**{**GOOD_BATCH, **(batch or {})}))
    L = lib()
    if name == "store":
        a = dict(q=FAR, ld_q=4096, k=2 * FAR, ld_k=512, v=3 * FAR, ld_v=512, qn=None, kn=None, eps=1e-6, freqs=4 * FAR,
                 n_rot=128, interleaved=0, mscale=1.0, n_head=32, out=5 * FAR)
        a.update(kw)
        return L.llamd_hip_paged8_store(c, b, *a.values())
    a = dict(q=FAR, n_head=32, scale=0.1, out_type=30, out=2 * FAR)
    if name == "prompt":
        a.update(kw)
        return L.llamd_hip_paged8_prompt(c, b, *a.values())
    a = dict(group=None, shared=None, n_group=0, **a)
    a.update(kw)
    return L.llamd_hip_paged8_decode(c, b, *a.values())


@pytest.mark.parametrize("name", ["store", "prompt", "decode"])
@pytest.mark.parametrize("pages,batch", [
    (dict(k=None), {}), (dict(v=None), {}), (dict(k=(1 << 20) + 8), {}), (dict(k_scale=None), {}), (dict(v_scale=None), {}),
    (dict(k_scale=(3 << 20) + 2), {}), (dict(v_scale=(3 << 20) + 4097), {}), (dict(hd=96), {}), (dict(hd=0), {}),
    (dict(page=8), {}), (dict(page=48), {}), (dict(page=512), {}), (dict(page=0), {}), (dict(n_page=0), {}),
    (dict(n_head_kv=0), {}), (dict(n_head_kv=5), {}), (dict(n_head_kv=64), {}), (dict(v=(1 << 20) + 1024), {}),
    (dict(v_scale=(3 << 20) + 124), {}), (dict(k_scale=(1 << 20) + 64), {}), (dict(v_scale=(2 << 20) - 4), {}),
    (dict(k_scale=2 << 20), {}), ({}, dict(n_seq=-1)), ({}, dict(n_tok=-1)), ({}, dict(max_page=0)),
    ({}, dict(max_page=(1 << 24) + 1)), ({}, dict(len=None)), ({}, dict(table=None)), ({}, dict(start=None, n_tok=1)),
    ({}, dict(table=(6 << 20) + 1))])
def test_refused_descriptors(name, pages, batch):
    assert call(name, pages, batch) == -1
    assert "paged8_" + name in last_error()


@pytest.mark.parametrize("kw", [
    dict(k=None), dict(v=None), dict(q=None), dict(out=None), dict(q=FAR + 4), dict(k=FAR + 4), dict(v=FAR + 8),
    dict(out=5 * FAR + 2), dict(qn=FAR + 4), dict(kn=FAR + 4), dict(ld_q=4092), dict(ld_q=4097), dict(ld_k=508),
    dict(ld_v=514), dict(n_rot=127), dict(n_rot=-2), dict(n_rot=130), dict(freqs=None), dict(interleaved=2),
    dict(eps=-1.0), dict(eps=math.nan), dict(mscale=math.inf), dict(n_head=30), dict(n_head=0), dict(out=FAR),
    dict(out=2 * FAR + 512), dict(out=3 * FAR), dict(out=(1 << 20) + 4096), dict(out=(3 << 20) + 64),
    dict(out=(3 << 20) + 4096 + 112), dict(k=(3 << 20) + 16), dict(v=(3 << 20) + 4096), dict(q=(2 << 20) - 16),
    dict(k=(1 << 20) + 4096), dict(freqs=4 * FAR + 4)])
def test_refused_store(kw):
    assert call("store", **kw) == -1
    assert "paged8_store" in last_error()


@pytest.mark.parametrize("name", ["prompt", "decode"])
@pytest.mark.parametrize("kw", [
    dict(q=None), dict(out=None), dict(q=FAR + 8), dict(out=FAR + 2), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=math.nan), dict(scale=math.inf), dict(scale=3e38), dict(out_type=1), dict(out_type=7), dict(out=FAR),
    dict(out=FAR + 4096), dict(n_head=33), dict(out=(1 << 20) + 4096), dict(out=(3 << 20) + 64), dict(out=(2 << 20) - 16)])
def test_refused_attention(name, kw):
    assert call(name, **kw) == -1
    assert "paged8_" + name in last_error()


@pytest.mark.parametrize("batch,kw", [
    (dict(n_tok=1), {}), ({}, dict(n_group=-1)), ({}, dict(n_group=3, group=FAR, shared=FAR)),
    ({}, dict(n_group=1, group=FAR)), ({}, dict(n_group=1, shared=FAR)),
    ({}, dict(group=FAR + 2, shared=2 * FAR, n_group=1, out=3 * FAR))])
def test_refused_decode(batch, kw):
    assert call("decode", batch=batch, **kw) == -1
    assert "paged8_decode" in last_error()


def test_null_descriptors_and_empty_batches():
    c, b = rocm.Pages8(**GOOD_PAGES), rocm.Batch(**GOOD_BATCH)
    L = lib()
    assert L.llamd_hip_paged8_prompt(None, C.byref(b), FAR, 32, 0.1, 30, 2 * FAR) == -1
    assert L.llamd_hip_paged8_prompt(C.byref(c), None, FAR, 32, 0.1, 30, 2 * FAR) == -1
    for name in ("store", "prompt", "decode"):  # nothing to do: no device work, no error
        assert call(name, batch=dict(n_seq=0, n_tok=0)) == 0
    assert call("prompt", batch=dict(n_tok=0)) == 0
    assert call("store", batch=dict(n_tok=0)) == 0


@pytest.mark.parametrize("args", [(0, 16, 2, 1, 64), (4, 24, 2, 1, 64), (4, 0, 2, 1, 64), (4, 16, 2, 0, 64)])
def test_python_wrapper_refuses_before_the_device(args):
    with pytest.raises(ValueError):
        rocm.PagedCache8(*args)


def test_e4m3_on_the_host():
    """Every code stands for itself; between two neighbours the nearer one, of two the even code."""
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    values = rocm.from_e4m3(codes)
    assert values.max() == 448 and values[1] == 2.0 ** -9 and np.isnan(rocm.from_e4m3([127, 255])).all()
    assert np.array_equal(rocm.to_e4m3(values), codes)
    a = values[:127].astype(np.float64)
    middle, low = (a[1:] + a[:-1]) / 2, np.arange(126)
    assert np.array_equal(rocm.to_e4m3(middle), low + (low & 1))
    assert np.array_equal(rocm.to_e4m3(middle * (1 - 1e-9)), low) and np.array_equal(rocm.to_e4m3(middle * (1 + 1e-9)), low + 1)
    assert (rocm.to_e4m3([np.nan, np.inf, 1e9, 470.0]) & 127 == 127).all()


def test_scale_bytes_on_the_host():
    """The least power of two with which 448 of it covers the largest value."""
    top = np.array([448, np.nextafter(np.float32(448), np.float32(1e3)), 3.5, 4, 1e-3, 3.4e38, 1e-38, 1e-45, 0], np.float32)
    e = rocm.scale_byte(top).astype(int)
    assert e[0] == 127 and e[1] == 128 and e[2] == 120 and e[3] == 121 and (e[-3:] == 1).all()
    t = top[:6].astype(np.float64)
    assert (t <= 448 * 2.0 ** (e[:6] - 127)).all() and (t > 448 * 2.0 ** (e[:6] - 128)).all()


def test_numbers_rounded_again_on_the_host():
    """A unit that grows by steps: numbers that stay normal (2^-14 of 448 units or more) are those of one rounding, the others are
    off by less than 2^-9 of the last unit; up to 2^-10 of it they are 0 in one rounding."""
    rng = np.random.default_rng(1)
    x = np.concatenate([np.exp2(rng.uniform(-24, 8.8, 20_000)), [448.0, 2.0 ** -10, 2.0 ** -9]]) * rng.choice([-1, 1], 20_003)
    for steps in ([1], [3], [1, 1, 1, 1], [2, 5, 1], [1] * 9):
        y, unit = rocm.from_e4m3(rocm.to_e4m3(x)).astype(np.float64), 1.0
        for step in steps:
            unit *= 2.0 ** step
            y = rocm.from_e4m3(rocm.to_e4m3(y / 2.0 ** step)).astype(np.float64)
        once = rocm.from_e4m3(rocm.to_e4m3(x / unit)).astype(np.float64)
        large = np.abs(x / unit) >= 448 * 2.0 ** -14
        assert np.array_equal(y[large], once[large])
        assert (np.abs(y - x / unit) <= np.maximum(2.0 ** -4 * np.abs(x / unit), 2.0 ** -9)).all()
        assert (once[np.abs(x / unit) <= 2.0 ** -10] == 0).all()

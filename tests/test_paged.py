"""The paged-cache entry points without a GPU: what they refuse, and the rotary frequencies."""
import ctypes as C
import math

import numpy as np
import pytest

from llamd_rs_amd import rocm
from llamd_rs_amd._lib import HipError, last_error, lib

GOOD_PAGES = dict(k=1 << 20, v=2 << 20, type=30, n_page=8, page=64, n_head_kv=4, hd=128)
GOOD_BATCH = dict(start=3 << 20, len=4 << 20, table=5 << 20, n_seq=2, n_tok=10, max_page=4)
FAR = 1 << 30  # addresses that nothing is ever read from: every call here is refused on the host


def call(name, pages=None, batch=None, **kw):
    c = C.byref(rocm.Pages(**{**GOOD_PAGES, **(pages or {})}))
    b = C.byref(rocm.Batch(**{**GOOD_BATCH, **(batch or {})}))
    L = lib()
    if name == "store":
        a = dict(q=FAR, ld_q=4096, k=2 * FAR, ld_k=512, v=3 * FAR, ld_v=512, qn=None, kn=None, eps=1e-6, freqs=4 * FAR,
                 n_rot=128, interleaved=0, mscale=1.0, n_head=32, out=5 * FAR)
        a.update(kw)
        return L.llamd_hip_paged_store(c, b, *a.values())
    a = dict(q=FAR, n_head=32, scale=0.1, out_type=30, out=2 * FAR)
    if name == "prompt":
        a.update(kw)
        return L.llamd_hip_paged_prompt(c, b, *a.values())
    a = dict(group=None, shared=None, n_group=0, **a)
    a.update(kw)
    return L.llamd_hip_paged_decode(c, b, *a.values())


@pytest.mark.parametrize("name", ["store", "prompt", "decode"])
@pytest.mark.parametrize("pages,batch", [
    (dict(k=None), {}), (dict(v=None), {}), (dict(k=(1 << 20) + 8), {}), (dict(type=2), {}), (dict(hd=96), {}),
    (dict(hd=0), {}), (dict(page=8), {}), (dict(page=48), {}), (dict(page=512), {}), (dict(page=0), {}),
    (dict(n_page=0), {}), (dict(n_head_kv=0), {}), (dict(n_head_kv=5), {}), (dict(n_head_kv=64), {}),
    ({}, dict(n_seq=-1)), ({}, dict(n_tok=-1)), ({}, dict(max_page=0)), ({}, dict(max_page=(1 << 24) + 1)), ({}, dict(len=None)), ({}, dict(table=None)),
    ({}, dict(start=None, n_tok=1))])
def test_refused_descriptors(name, pages, batch):
    assert call(name, pages, batch) == -1
    assert "paged_" + name in last_error()


@pytest.mark.parametrize("kw", [
    dict(k=None), dict(v=None), dict(q=None), dict(out=None), dict(q=FAR + 4), dict(k=FAR + 4), dict(v=FAR + 8),
    dict(out=5 * FAR + 2), dict(qn=FAR + 4), dict(kn=FAR + 4), dict(ld_q=4092), dict(ld_q=4097), dict(ld_k=508),
    dict(ld_v=514), dict(n_rot=127), dict(n_rot=-2), dict(n_rot=130), dict(freqs=None), dict(interleaved=2),
    dict(eps=-1.0), dict(eps=math.nan), dict(mscale=math.inf), dict(n_head=30), dict(n_head=0), dict(out=FAR),
    dict(out=2 * FAR + 512), dict(out=3 * FAR)])
def test_refused_store(kw):
    assert call("store", **kw) == -1
    assert "paged_store" in last_error()


@pytest.mark.parametrize("name", ["prompt", "decode"])
@pytest.mark.parametrize("kw", [
    dict(q=None), dict(out=None), dict(q=FAR + 8), dict(out=FAR + 2), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=math.nan), dict(scale=math.inf), dict(out_type=1), dict(out_type=7), dict(out=FAR), dict(out=FAR + 4096),
    dict(n_head=33)])
def test_refused_attention(name, kw):
    assert call(name, **kw) == -1
    assert "paged_" + name in last_error()


@pytest.mark.parametrize("batch,kw", [
    (dict(n_tok=1), {}), ({}, dict(n_group=-1)), ({}, dict(n_group=3, group=FAR, shared=FAR)),
    ({}, dict(n_group=1, group=FAR)), ({}, dict(n_group=1, shared=FAR))])
def test_refused_decode(batch, kw):
    assert call("decode", batch=batch, **kw) == -1
    assert "paged_decode" in last_error()


@pytest.mark.parametrize("name,pages,batch,kw", [
    ("store", {}, {}, dict(out=(1 << 20) + 4096)), ("store", {}, {}, dict(out=(2 << 20) - 64)),
    ("store", {}, {}, dict(freqs=4 * FAR + 4)), ("store", {}, dict(start=(3 << 20) + 2), {}),
    ("prompt", {}, {}, dict(out=(1 << 20) + 4096)), ("prompt", {}, dict(table=(5 << 20) + 1), {}),
    ("prompt", dict(v=(1 << 20) + 1024), {}, {}), ("decode", {}, {}, dict(out=(2 << 20) + (1 << 19) - 16)),
    ("decode", {}, dict(len=(4 << 20) + 2), {}), ("decode", {}, {}, dict(group=FAR + 2, shared=2 * FAR, n_group=1, out=3 * FAR)),
    ("decode", dict(k=2 << 20), {}, {})])
def test_refused_overlaps_and_alignments(name, pages, batch, kw):
    assert call(name, pages, batch, **kw) == -1
    assert "paged_" + name in last_error()


def test_null_descriptors_and_empty_batches():
    c, b = rocm.Pages(**GOOD_PAGES), rocm.Batch(**GOOD_BATCH)
    L = lib()
    assert L.llamd_hip_paged_prompt(None, C.byref(b), FAR, 32, 0.1, 30, 2 * FAR) == -1
    assert L.llamd_hip_paged_prompt(C.byref(c), None, FAR, 32, 0.1, 30, 2 * FAR) == -1
    for name in ("store", "prompt", "decode"):  # nothing to do: no device work, no error
        assert call(name, batch=dict(n_seq=0, n_tok=0)) == 0
    assert call("prompt", batch=dict(n_tok=0)) == 0
    assert call("store", batch=dict(n_tok=0)) == 0


def test_python_wrapper_refuses_before_the_device():
    with pytest.raises(ValueError):
        rocm.PagedCache("f64", 4, 16, 2, 1, 64)
    with pytest.raises(ValueError):
        rocm.PagedCache("f16", 0, 16, 2, 1, 64)


def test_bf16_rounding_on_the_host():
    x = np.array([1.0, 1.00390625, 1.01171875, -2.5, 3.4e38, np.inf, np.nan, 1e-40], np.float32)
    got = rocm.from_bf16(rocm.to_bf16(x))
    # halfway cases go to the even neighbour; the largest f32 values round to infinity
    assert got[0] == 1.0 and got[1] == 1.0 and got[2] == np.float32(1.015625) and got[3] == -2.5
    assert np.isinf(got[4]) and np.isinf(got[5]) and np.isnan(got[6]) and got[7] > 0


# ---- the rotary frequencies -------------------------------------------------------

@pytest.mark.parametrize("n_rot,base", [(2, 10000.0), (64, 10000.0), (128, 1e6), (256, 5e5)])
def test_plain_and_linear_frequencies(n_rot, base):
    f, m = rocm.rope_freqs(n_rot, base)
    want = np.array([base ** (-2 * i / n_rot) for i in range(n_rot // 2)])
    assert m == 1.0 and np.allclose(f, want, rtol=1e-14, atol=0)
    g, m = rocm.rope_freqs(n_rot, base, factor=4.0)
    assert m == 1.0 and np.allclose(g, want / 4, rtol=1e-14, atol=0)


@pytest.mark.parametrize("n_rot,base,factor,orig", [(128, 1e6, 4.0, 32768), (64, 10000.0, 16.0, 4096)])
def test_frequencies_by_parts(n_rot, base, factor, orig):
    f, m = rocm.rope_freqs(n_rot, base, factor, orig)
    plain, _ = rocm.rope_freqs(n_rot, base)
    turns = plain * orig / (2 * math.pi)
    share = (plain - f) / (plain - plain / factor)   # 0 as trained .. 1 stretched
    assert abs(m - (0.1 * math.log(factor) + 1)) < 1e-6
    # the ramp runs between the whole pairs just outside the two turn counts
    i = np.arange(n_rot // 2)
    fast = math.floor(n_rot * math.log(orig / (2 * math.pi * 32)) / (2 * math.log(base)))
    slow = math.ceil(n_rot * math.log(orig / (2 * math.pi)) / (2 * math.log(base)))
    assert np.allclose(share[i <= fast], 0, atol=1e-9) and np.allclose(share[i >= slow], 1, atol=1e-9)
    assert (turns[i <= fast] >= 32 - 1e-9).all() and (turns[i >= slow] <= 1 + 1e-9).all()
    mid = (i > fast) & (i < slow)
    assert mid.any() and np.allclose(share[mid], (i[mid] - fast) / (slow - fast), atol=1e-9)


@pytest.mark.parametrize("args", [
    (0, 1e4), (3, 1e4), (64, 1.0), (64, math.nan), (64, 1e4, 0.0), (64, 1e4, math.inf), (64, 1e4, 2.0, -1),
    (64, 1e4, 2.0, 4096, 1.0, 32.0), (64, 1e4, 2.0, 4096, 32.0, 0.0)])
def test_refused_frequencies(args):
    with pytest.raises(HipError):
        rocm.rope_freqs(*args)


@pytest.mark.parametrize("name", ["prompt", "decode"])
def test_refused_scales_whose_exponent_of_two_is_no_number(name):
    """Weights are powers of two of scale * log2(e) times a score: where that passes f32's range, scores of 0 would be NaN."""
    for scale in (3e38, 2.4e38, -math.inf):
        assert call(name, scale=scale) == -1
        assert last_error() == "paged_%s: scale %g" % (name, np.float32(scale))


@pytest.mark.parametrize("kw", [
    dict(q=(1 << 20) + 4096), dict(k=(1 << 20) + 4096), dict(v=(2 << 20) + 4096), dict(k=(2 << 20) - 16), dict(v=(1 << 20) - 2048)])
def test_refused_store_of_rows_that_lie_in_the_pages(kw):
    """Pages are written while other workgroups read q, k and v."""
    assert call("store", **kw) == -1
    assert "overlaps the pages" in last_error()

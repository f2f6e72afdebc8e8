"""Sampling without a GPU: what the entry point refuses, the wrapper's rules, and the restatement on small rows."""
import numpy as np
import pytest

import sample_reference as S
from llamd_rs_amd import rocm
from llamd_rs_amd._lib import last_error, lib

FAR = 1 << 30  # addresses that nothing is ever read from: every call here is refused on the host


def call(**kw):
    a = dict(logits=FAR, ld=1000, n=1000, n_seq=4, how=2 * FAR, u=3 * FAR, ids=4 * FAR, prob=5 * FAR)
    a.update(kw)
    return lib().llamd_hip_sample(*a.values())


@pytest.mark.parametrize("kw", [
    dict(logits=None), dict(how=None), dict(u=None), dict(ids=None), dict(n=0), dict(n=-1), dict(n=(1 << 20) + 1, ld=1 << 21),
    dict(ld=999), dict(n_seq=-1), dict(n_seq=65536), dict(logits=FAR + 2), dict(how=2 * FAR + 8), dict(u=3 * FAR + 4),
    dict(ids=4 * FAR + 1), dict(prob=5 * FAR + 2), dict(ids=FAR), dict(ids=FAR + 15996), dict(prob=FAR + 4), dict(ids=2 * FAR),
    dict(prob=2 * FAR + 60), dict(ids=3 * FAR + 28), dict(prob=3 * FAR), dict(prob=4 * FAR + 12)])
def test_refused(kw):
    assert call(**kw) == -1
    assert last_error().startswith("sample: ")


def test_nothing_to_do():
    assert call(n_seq=0) == 0
    assert call(n_seq=0, logits=None, how=None, u=None, ids=None) == 0


def test_rules():
    r = rocm.sampling_rules(3, 0.5, [1, 2, 3], top_p=0.9)
    assert r["top_k"].tolist() == [1, 2, 3] and (r["temperature"] == 0.5).all() and (r["min_p"] == 0).all()
    assert (r["top_p"] == np.float32(0.9)).all() and r.nbytes == 48
    for bad in (dict(top_k=[1, 2]), dict(min_p=np.zeros((3, 1)))):
        with pytest.raises(ValueError):
            rocm.sampling_rules(3, **bad)
    for x, u in ((np.zeros((2, 4)), [0.5]), (np.zeros((2, 0)), 0.5), (np.zeros((2, 4)), np.zeros((2, 1)))):
        with pytest.raises(ValueError):
            rocm.sample(x, u)


def test_logits_of_more_than_two_axes_are_refused():
    """(Rows of what they hold would be drawn from: [2, 3, 100] as two rows of three logits.)"""
    for x in (np.zeros((2, 3, 100)), np.zeros((1, 1, 1, 5))):
        with pytest.raises(ValueError):
            rocm.sample(x, 0.5)
    head = rocm.LmHead.__new__(rocm.LmHead)  # (the check comes before the device)
    head.rows, head.blocks, head.max_seq, head._h = 100, 1, 8, None
    for x in (np.zeros((2, 256, 2)), np.zeros((1, 256, 1))):
        with pytest.raises(ValueError):
            head.sample(x, 0.5)


@pytest.mark.parametrize("top_k", [2.5, np.nan, np.inf, 1 << 31, -(1 << 31) - 1, [1, 2, (1 << 32) + 5], np.array([1, 2, 1 << 40]),
                                   np.array([0.5, 1, 2]), 1 << 70])
def test_a_top_k_that_is_no_whole_number_of_32_bits(top_k):
    """(Wrapped or cut short it would be another rule: 2^32 + 5 the first five.)"""
    with pytest.raises(ValueError):
        rocm.sampling_rules(3, top_k=top_k)


def test_a_top_k_of_any_number_type():
    for top_k in (7, 7.0, np.float32(7), np.uint64(7), [7, 7.0, np.int8(7)]):
        assert rocm.sampling_rules(3, top_k=top_k)["top_k"].tolist() == [7, 7, 7]
    for top_k in ((1 << 31) - 1, -(1 << 31)):
        assert rocm.sampling_rules(3, top_k=top_k)["top_k"].tolist() == [top_k] * 3


def test_the_restatement():
    """By hand: weights 1, 1/2, 1/2, 1/4 at ids 2, 0, 3, 1."""
    x = np.log(np.array([0.5, 0.25, 1, 0.5]))
    x[:] = np.float32(x)
    plain = (1, 0, 1, 0)
    assert [next(iter(S.choices(x, plain, u))) for u in (0.0, 0.2, 0.3, 0.4, 0.7, 0.8, 1.0)] == [0, 0, 1, 2, 2, 3, 3]
    # top-k 2: the largest and, of two equal ones, the lower id
    assert set(S.choices(x, (1, 2, 1, 0), 0.1)) == {0} and set(S.choices(x, (1, 2, 1, 0), 0.5)) == {2}
    # top-p of 0.6 of 9/4: 1 and 1/2; min-p 0.6: the largest; a half of the total: the largest
    assert set(S.choices(x, (1, 0, 0.6, 0), 0.9)) == {2} and set(S.choices(x, (1, 0, 0.6, 0), 0.2)) == {0}
    assert set(S.choices(x, (1, 0, 1, 0.6), 0.0)) == {2} and set(S.choices(x, (1, 0, 0.4, 0), 0.0)) == {2}
    assert S.choices(np.array([-np.inf, np.nan]), plain, 0.5) == {-1: [0.0]}
    assert set(S.choices(np.array([1.0, np.inf, 2, np.inf]), plain, 0.4)) == {1}

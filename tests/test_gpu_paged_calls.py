"""The paged cache's calls at their edges: numbers on the device that make no sense, an eager call beside a replayed graph, what
the library's scratch grows to. Values against paged_reference."""
import numpy as np
import pytest

import paged_reference as R
from test_gpu_paged import filled, rounded, tables, want_decode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("shared", [(1 << 31) - 1, (1 << 31) - 64, 1 << 30, 4096])
def test_groups_that_share_more_than_the_table_holds(gpu, page, shared):
    """Every position is then the group's, read through its first sequence; empty members give 0."""
    rng = np.random.default_rng(60)
    heads, kvh, hd = 8, 2, 64
    lengths, group = [300, 0, 290, 1, 0, 40], [0, 5]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, "bf16", table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((6, heads * hd)), "bf16")
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "bf16", group, [shared])
    got = c.decode(q, table, lengths, group, [shared])
    R.check(got, want, bound)
    assert not got[[1, 4]].any() and got[5].any()

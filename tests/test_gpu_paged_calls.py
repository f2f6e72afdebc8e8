"""The paged cache's calls at their edges: numbers on the device that make no sense, an eager call beside a replayed graph, what
the library's scratch grows to. Values against paged_reference."""
import ctypes as C

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


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_a_replayed_graph_beside_another_threads_calls(gpu, kind):
    """A graph's calls and eager ones use the same scratch: a replay from one thread falls between calls of another, never
    between the launches of one."""
    import threading
    L = gpu.lib()
    rng = np.random.default_rng(63)
    heads, kvh, hd, page = 8, 1, 64, 16
    tables_of = {}
    for name, lengths in (("replay", [900, 3000]), ("eager", [2500, 700])):
        table, n_page = tables(rng, lengths, page)
        c, _, _ = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
        tables_of[name] = c, table, lengths, rounded(rng.standard_normal((2, heads * hd)), kind)
    c, table, lengths, q = tables_of["replay"]
    b, keep = c._batch(table, lengths, None, 2)
    dq, out = gpu.DeviceBuffer.from_array(c.encode(q)), gpu.DeviceBuffer.from_array(np.zeros(q.shape, c.dtype))
    want = c.decode(q, table, lengths)
    other = [tables_of["eager"][0].decode(tables_of["eager"][3], *tables_of["eager"][1:3])]
    assert L.llamd_fwd_begin_capture() == 0
    assert L.llamd_hip_paged_decode(C.byref(c.pages), C.byref(b), None, None, 0, dq.ptr, heads, hd ** -0.5, c.pages.type,
                                    out.ptr) == 0
    assert L.llamd_fwd_end_capture() == 0
    replayed, done = [], threading.Event()

    def eager():
        try:
            for _ in range(60):
                other.append(tables_of["eager"][0].decode(tables_of["eager"][3], *tables_of["eager"][1:3]))
        finally:
            done.set()

    t = threading.Thread(target=eager)
    t.start()
    while not done.is_set():
        assert L.llamd_fwd_graph_launch() == 0
        replayed.append(c.decode_values(out.download(np.empty(q.shape, c.dtype))))
    t.join()
    L.llamd_fwd_graph_destroy()
    assert len(other) == 61 and replayed
    assert all(np.array_equal(x, other[0]) for x in other) and all(np.array_equal(x, want) for x in replayed)

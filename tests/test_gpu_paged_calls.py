"""The paged cache's calls at their edges: numbers on the device that make no sense, an eager call beside a replayed graph, what
the library's scratch grows to. Values against paged_reference."""
import ctypes as C
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

import paged_reference as R
from test_gpu_paged import filled, rounded, shared_tables, tables, want_decode, want_prompt

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


@pytest.mark.parametrize("heads,kvh", [(8, 2), (40, 1)])
@pytest.mark.parametrize("lengths,group", [([700], [0, 1]), ([0], [0, 1]), ([300, 40], [0, 1, 2]), ([5, 900, 33], [0, 0, 1, 2]), ([5, 900, 33], [1, 1, 1, 1])])
def test_groups_of_one_share_nothing(gpu, heads, kvh, lengths, group):
    """Such groups have no tiles: every sequence reads its own table."""
    rng = np.random.default_rng(65)
    hd, page = 128, 16
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, "f16", table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((len(lengths), heads * hd)), "f16")
    want, bound = want_decode(q, k, v, table, lengths, heads, kvh, hd, hd ** -0.5, "f16")
    R.check(c.decode(q, table, lengths, group, [256] * (len(group) - 1)), want, bound)


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


# ---- the scratch ------------------------------------------------------------------
# It never shrinks, and what other calls left would hide a call's own need: each of these runs in a process of its own.

HERE = Path(__file__).resolve().parent
MB = 1 << 20


def alone(name, *args):
    """Runs a function of this file in a fresh process."""
    code = f"import test_gpu_paged_calls as t\nfrom llamd_rs_amd import rocm\nt.{name}(rocm, *{args!r})\nprint('done', flush=True)"
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([str(HERE), str(HERE.parent)]))
    done = subprocess.run([sys.executable, "-c", code], cwd=HERE.parent, env=env, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0 and done.stdout.split()[-1:] == ["done"], done.stdout[-2000:] + done.stderr[-4000:]


def grown(gpu, call):
    """What a call returns, and by how many bytes the library's scratch grew in it (its other memory is freed)."""
    before = gpu.lib().llamd_rocm_free_mem()
    got = call()
    return got, before - gpu.lib().llamd_rocm_free_mem()


def pairs(gpu, n_seq, heads, width):
    """Sequences in pairs that share two pages, in a wide table."""
    rng = np.random.default_rng(61)
    hd, page = 128, 32
    group = list(range(0, n_seq + 1, 2))
    lengths = [70 + s % 9 for s in range(n_seq)]
    table, n_page, _ = shared_tables(rng, group, [64] * (n_seq // 2), lengths, page)
    c, k, v = filled(gpu, rng, "bf16", table, n_page, page, heads, heads, hd, lengths)
    q = rounded(rng.standard_normal((n_seq, heads * hd)), "bf16")
    wide = np.full((n_seq, width // page), -1, np.int32)
    wide[:, :table.shape[1]] = table
    shared = [64] * (n_seq // 2)
    got, more = grown(gpu, lambda: c.decode(q, wide, lengths, group, shared))
    want, bound = want_decode(q, k, v, table, lengths, heads, heads, hd, hd ** -0.5, "bf16", group, shared)
    R.check(got, want, bound)
    # slots of 128 rows (f32 values, two statistics): 5 for each of 512 workgroups, or one per pair and head; then small things
    assert more <= max(5 * 512, (n_seq // 2 + 2) * heads) * 128 * (hd * 4 + 8) + 8 * MB, more // MB


@pytest.mark.parametrize("n_seq,heads,width", [(64, 32, 8192), (128, 16, 16384)])
def test_scratch_of_many_small_groups(gpu, n_seq, heads, width):
    """Every group has tiles of its own: parts are for the tiles that there can be, not for rows packed into full ones."""
    alone("pairs", n_seq, heads, width)


def few_tokens(gpu, n_seq, tokens, heads, kvh):
    """A prompt batch of few tokens and many sequences that have none, as a captured call with places left looks."""
    rng = np.random.default_rng(62)
    hd, page = 128, 64
    new = [0] * n_seq
    for i in range(tokens):
        new[(i * 37 + 5) % n_seq] += 1
    lengths = [200 + 3 * s % 50 if n else 0 for s, n in enumerate(new)]
    table, n_page = tables(rng, lengths, page)
    wide = np.full((n_seq, 16384 // page), -1, np.int32)
    wide[:, :table.shape[1]] = table
    c, k, v = filled(gpu, rng, "bf16", table, n_page, page, heads, kvh, hd, lengths)
    start = np.concatenate([[0], np.cumsum(new)])
    q = rounded(rng.standard_normal((tokens, heads * hd)), "bf16")
    got, more = grown(gpu, lambda: c.prompt(q, wide, lengths, start))
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, hd ** -0.5, "bf16")
    R.check(got, want, bound)
    # slots of 16 rows: 5 for each of 768 workgroups, or one per tile and head; then small things
    assert more <= max(5 * 768, 2 * tokens * kvh) * 16 * (hd * 4 + 8) + 8 * MB, more // MB


@pytest.mark.parametrize("n_seq,tokens,heads,kvh", [(64, 1, 32, 4), (256, 8, 32, 32), (1000, 3, 8, 8), (40, 40, 12, 12)])
def test_scratch_of_sequences_without_tokens(gpu, n_seq, tokens, heads, kvh):
    """Tiles are counted for the sequences that can have tokens."""
    alone("few_tokens", n_seq, tokens, heads, kvh)


def moved_scratch(gpu, kind):
    L = gpu.lib()
    rng = np.random.default_rng(64)
    heads, kvh, hd, page = 8, 1, 128, 16
    lengths, start = [900, 2000, 50], [0, 20, 29, 40]
    table, n_page = tables(rng, lengths, page)
    c, k, v = filled(gpu, rng, kind, table, n_page, page, heads, kvh, hd, lengths)
    q = rounded(rng.standard_normal((40, heads * hd)), kind)
    want, bound = want_prompt(q, k, v, table, lengths, start, heads, kvh, hd, hd ** -0.5, kind)
    b, keep = c._batch(table, lengths, start, 40)
    dq, out = gpu.DeviceBuffer.from_array(c.encode(q)), gpu.DeviceBuffer.from_array(np.zeros(q.shape, c.dtype))
    assert L.llamd_fwd_begin_capture() == 0
    assert L.llamd_hip_paged_prompt(C.byref(c.pages), C.byref(b), dq.ptr, heads, hd ** -0.5, c.pages.type, out.ptr) == 0
    assert L.llamd_fwd_end_capture() == 0
    first = None
    big_q = rng.standard_normal((700, heads * hd))
    for turn, width in enumerate((3000, 9000, 3000)):
        out.upload(np.zeros(q.shape, c.dtype))
        assert L.llamd_fwd_graph_launch() == 0
        got = c.decode_values(out.download(np.empty(q.shape, c.dtype)))
        R.check(got, want, bound, turn)
        assert first is None or np.array_equal(got, first), turn
        first = got
        # an eager call whose parts (44 tiles of 128 rows, 11 parts: 33 MB) need more than the captured call's (3 MB)
        big_t, big_n = tables(rng, [width], page, 0)
        big = gpu.PagedCache(kind, big_n, page, heads, kvh, hd)
        _, more = grown(gpu, lambda: big.prompt(big_q, big_t, [width], [0, 700]))
        big.close()
        assert turn or more >= 32 * MB, more  # the scratch is another one now
    L.llamd_fwd_graph_destroy()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_a_graph_keeps_the_scratch_that_it_captured(gpu, kind):
    """A larger eager call replaces the library's scratch; replays go on in the one that they were captured with."""
    alone("moved_scratch", kind)

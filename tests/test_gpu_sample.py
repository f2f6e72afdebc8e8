"""Sampling against its restatement in extended precision (sample_reference), where it can go wrong: one logit and 2^20, rows at
any alignment, equal logits, masked and non-finite ones, rules at their ends, borders inside ties, random numbers at and past
their ends, replayed graphs, the LM head and an 8-bit cache in front of it."""
import numpy as np
import pytest

import sample_reference as S

pytestmark = pytest.mark.gpu

RULES = [(1, 0, 1, 0), (0.7, 50, 1, 0), (1.3, 0, 0.9, 0), (0.8, 40, 0.95, 0), (1, 0, 1, 0.05), (1, 200, 0.7, 0.01), (0, 5, 0.5, 0),
         (1.5, 3, 0.999, 0.5)]
LOWEST = float(np.finfo(np.float32).min)


def logits(rng, rows, n, spread=2.5):
    x = (rng.standard_normal((rows, n)) * spread).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, n, 4)] = 9 + rng.standard_normal(4)
    return x


def run(gpu, x, rules, u):
    t, k, p, m = (np.array(c) for c in zip(*rules))
    return gpu.sample(x, u, t.astype(np.float32), k.astype(np.int32), p.astype(np.float32), m.astype(np.float32))


def check(gpu, x, rules, u, what=""):
    x, u = np.asarray(x, np.float32), np.asarray(u, np.float64)
    ids, prob = run(gpu, x, rules, u)
    S.check(ids, prob, x, rules, u, what)
    return ids, prob


@pytest.mark.parametrize("n", [1, 2, 63, 256, 1000, 4095, 4096, 4097, 8193, 32001, 151936])
def test_sizes(gpu, n):
    rng = np.random.default_rng(n)
    x = logits(rng, len(RULES), n)
    check(gpu, x, RULES, rng.random(len(RULES)))


def test_largest(gpu):
    rng = np.random.default_rng(1)
    check(gpu, logits(rng, 3, 1 << 20), [RULES[0], RULES[3], RULES[2]], rng.random(3))


def test_many_rows(gpu):
    rng = np.random.default_rng(2)
    x = logits(rng, 300, 600)
    rules = [RULES[i % len(RULES)] for i in range(300)]
    check(gpu, x, rules, rng.random(300))


def test_more_rows_than_go_at_a_time(gpu):
    rng = np.random.default_rng(22)
    x = logits(rng, 2049, 41)
    check(gpu, x, [RULES[i % len(RULES)] for i in range(2049)], rng.random(2049))


@pytest.mark.parametrize("ends", [[0.0, 1.0 - 2.0 ** -53, 1.0, 2.0, -1.0, np.nan, np.inf, -np.inf]])
def test_random_numbers_at_their_ends(gpu, ends):
    rng = np.random.default_rng(3)
    for rule in RULES:
        check(gpu, np.repeat(logits(rng, 1, 5000), len(ends), 0), [rule] * len(ends), ends, rule)


@pytest.mark.parametrize("temperature", [0.0, -1.0, np.nan, 1e-30, 1e-6, 0.01, 30.0, 1e6, 1e30, np.inf])
def test_temperatures(gpu, temperature):
    rng = np.random.default_rng(4)
    rules = [(temperature, *r[1:]) for r in RULES]
    x = logits(rng, len(rules), 9000)
    x[:, 5::7] = -np.inf
    check(gpu, x, rules, rng.random(len(rules)))


def test_rules_at_their_ends(gpu):
    rng = np.random.default_rng(5)
    n = 5000
    rules = [(1, k, 1, 0) for k in (-5, 1, 2, n - 1, n, n + 1, 1 << 30)]
    rules += [(1, 0, p, 0) for p in (0.0, -1.0, -np.inf, 1e-12, 1 - 2.0 ** -24, 1.0, 2.0, np.nan, np.inf)]
    rules += [(1, 0, 1, m) for m in (-1.0, np.nan, 1e-30, 1.0, 2.0, np.inf)]
    rules += [(1, 1, 0.0, 2.0), (1, n - 1, 1 - 2.0 ** -24, 1e-30), (1, 20, 0.0, 0), (1, 2, 0.6, 0)]
    check(gpu, logits(rng, len(rules), n), rules, rng.random(len(rules)))


@pytest.mark.parametrize("n", [10, 300, 2048, 2049, 20_000, 151_936])
def test_equal_logits(gpu, n):
    """All logits equal: borders by index alone, in the list and (more than 2048) from the row."""
    rules = [(1, 0, 1, 0), (1, 7, 1, 0), (1, n - 1, 1, 0), (1, 0, 0.5, 0), (1, max(n // 2, 1), 0.25, 0), (1, 0, 0.999, 1.0)]
    for value in (0.0, -3.5, 1e30):
        check(gpu, np.full((len(rules), n), value, np.float32), rules, [0.3, 0.99, 0.7, 0.5, 0.999, 0.01], value)


@pytest.mark.parametrize("least", [float(np.nextafter(np.float32(1), np.float32(2))), 1.5, 2.0, 3e38, np.inf])
@pytest.mark.parametrize("n", [10, 2048, 2049, 40_000, 151_936])
def test_a_min_p_that_no_weight_reaches(gpu, n, least):
    """The first alone is kept, of equal maxima the one of the lowest id, whatever else the rule says."""
    rng = np.random.default_rng(24)
    rules = [(1, 0, 1, least), (0.5, 5, 1, least), (1, 0, 0.9, least), (2, n // 2, 0.3, least), (np.inf, 0, 1, least),
             (1, 5, 1, least), (1, 0, 1, least)]
    x = logits(rng, len(rules), n)
    first = rng.integers(1, n // 2, len(rules))
    for r in range(len(rules)):
        x[r, first[r]] = x[r, [first[r] + 1, n - 1]] = x[r].max() + 1
    x[5], first[5] = 0.25, 0
    x[6, first[6]] = x[6, first[6] + 1] = np.inf
    for u in (0.0, 0.4, 0.9, 1.0):
        ids, prob = check(gpu, x, rules, np.full(len(rules), u), u)
        assert np.array_equal(ids, first) and (prob == 1).all()


@pytest.mark.parametrize("values", [(0.0, -0.0, 1.0), (2.0, 2.25, 1.75, -8.0), (5.0, -np.inf, 4.0), (7.0, LOWEST), (1.0, 1 + 2.0 ** -23)])
@pytest.mark.parametrize("n", [500, 30_000])
def test_few_values(gpu, values, n):
    """Ties at every border; zeros of either sign are equal."""
    rng = np.random.default_rng(6)
    rules = RULES + [(1, n // 3, 1, 0), (1, n // 2, 0.5, 0), (0.5, 0, 0.3, 0), (1, 0, 0.5, 0.9)]
    check(gpu, rng.choice(np.array(values, np.float32), (len(rules), n)), rules, rng.random(len(rules)))


def test_values_that_are_no_numbers(gpu):
    rng = np.random.default_rng(7)
    n, rules = 6000, RULES
    for what in ("nan", "inf", "some inf", "masked", "lowest", "one", "none", "all nan", "all lowest", "huge"):
        x = logits(rng, len(rules), n)
        if what == "nan":
            x[:, ::3] = np.nan
        if what == "inf":
            x[:, 4321] = np.inf
        if what == "some inf":
            x[:, [7, 90, 5999]] = np.inf
        if what == "masked":
            x[:, rng.random(n) < 0.999] = -np.inf
        if what == "lowest":
            x[:, rng.random(n) < 0.9] = LOWEST
        if what == "one":
            x[:], x[:, 4097] = -np.inf, -1e30
        if what == "none":
            x[:] = -np.inf
        if what == "all nan":
            x[:] = np.nan
        if what == "all lowest":
            x[:] = LOWEST
        if what == "huge":
            x *= 1e37
        ids, prob = check(gpu, x, rules, rng.random(len(rules)), what)
        if what in ("none", "all nan"):
            assert (ids == -1).all() and (prob == 0).all()


@pytest.mark.parametrize("spread,temperature", [(1e-4, 1.0), (2.5, 50.0), (30.0, 1.0), (2.5, 1e4)])
def test_flat_and_steep_rows(gpu, spread, temperature):
    rng = np.random.default_rng(8)
    rules = [(temperature, k, p, m) for k in (0, 30, 20_000) for p in (1, 0.9, 0.3) for m in (0, 0.1)]
    x = (rng.standard_normal((len(rules), 40_000)) * spread).astype(np.float32)
    check(gpu, x, rules, rng.random(len(rules)))


@pytest.mark.parametrize("n,k", [(80_383, 1000), (80_383, 1004), (70_000, 600), (30_000, 374), (151_936, 1024)])
def test_a_top_k_of_most_groups(gpu, n, k):
    """The maxima of 64 values bound the k-th largest from far below, or there are fewer than k of them that are finite."""
    rng = np.random.default_rng(23)
    x = logits(rng, 6, n)
    x[1, rng.random(n) < 0.3] = -np.inf
    x[2, rng.random(n) < 0.97] = -np.inf
    x[3, :n // 2], x[3, n // 2 + 5000:] = -np.inf, -np.inf   # 5000 in a row, 79 groups
    x[4, 700:] = -np.inf
    x[5] = np.round(x[5] * 4) / 4
    rules = [(1, k, 1, 0), (0.8, k, 0.95, 0), (1.2, k, 1, 0.01), (1, k, 0.9, 0), (1, k, 1, 0), (0.7, k, 0.99, 0)]
    for turn in range(3):
        check(gpu, x, rules, rng.random(6), turn)


def test_an_outlier_below(gpu):
    """One logit far below the others stretches the bins: most others fall into one."""
    rng = np.random.default_rng(9)
    rules = [(1000.0, 500, 1, 0), (1000.0, 0, 0.5, 0), (1000.0, 9000, 0.2, 0)]
    x = rng.standard_normal((3, 10_000)).astype(np.float32)
    x[:, 77] = -30_000
    check(gpu, x, rules, rng.random(3))


@pytest.mark.parametrize("offset,pad", [(0, 0), (0, 4), (0, 3), (1, 0), (2, 5), (3, 1)])
def test_rows_of_any_alignment(gpu, offset, pad):
    """Rows apart, and not on 16 bytes; what lies between them is not looked at. Ids and probabilities behind stay."""
    rng = np.random.default_rng(10)
    L, n, rows = gpu.lib(), 9001, len(RULES)
    ld = n + pad
    flat = np.full(offset + rows * ld + 4, np.inf, np.float32)
    x = logits(rng, rows, n)
    for r in range(rows):
        flat[offset + r * ld:offset + r * ld + n] = x[r]
    u = rng.random(rows)
    rules = np.array([tuple(r) for r in RULES], gpu.SAMPLING)
    dev = [gpu.DeviceBuffer.from_array(a) for a in (flat, rules, u)]
    ids, prob = (gpu.DeviceBuffer.from_array(np.full(rows + 2, 77, t)) for t in (np.int32, np.float32))
    assert L.llamd_hip_sample(dev[0].ptr + 4 * offset, ld, n, rows, dev[1].ptr, dev[2].ptr, ids.ptr, prob.ptr) == 0
    got, p = ids.download(np.empty(rows + 2, np.int32)), prob.download(np.empty(rows + 2, np.float32))
    S.check(got, p, x, RULES, u)
    assert (got[rows:] == 77).all() and (p[rows:] == 77).all()
    assert L.llamd_hip_sample(dev[0].ptr + 4 * offset, ld, n, rows, dev[1].ptr, dev[2].ptr, ids.ptr, None) == 0
    assert np.array_equal(ids.download(np.empty(rows + 2, np.int32)), got)


@pytest.mark.parametrize("rule", [(1, 0, 1, 0), (0.9, 12, 1, 0), (1, 0, 0.8, 0), (1, 0, 1, 0.02)])
def test_every_share_of_u(gpu, rule):
    """Numbers spread evenly over [0, 1) draw each token as often as its probability says, to one."""
    rng = np.random.default_rng(11)
    rows, n = 2000, 300
    x = logits(rng, 1, n)
    u = (np.arange(rows) + 0.5) / rows
    ids, prob = run(gpu, np.repeat(x, rows, 0), [rule] * rows, u)
    assert (np.diff(ids) >= 0).all()   # in order of the ids
    seen = dict(zip(*np.unique(ids, return_counts=True)))
    for i, p in zip(ids, prob):
        assert abs(seen[i] - p * rows) <= 1 + 1e-3
    order, w = S._kept(x[0].astype(np.float64), rule, 0, 0)
    assert set(seen) <= set(order.tolist())


def test_calls_repeat_bit_for_bit(gpu):
    rng = np.random.default_rng(12)
    rules = [RULES[i % len(RULES)] for i in range(24)]
    x, u = logits(rng, 24, 50_000), rng.random(24)
    first = run(gpu, x, rules, u)
    for _ in range(8):
        assert all(np.array_equal(a, b) for a, b in zip(first, run(gpu, x, rules, u)))


def test_a_captured_call_follows_the_device(gpu):
    """Captured once, replayed with other logits, rules and numbers, with eager calls (also larger ones) between."""
    L, rng = gpu.lib(), np.random.default_rng(13)
    rows, n = 6, 20_000
    dev = [gpu.DeviceBuffer(b) for b in (rows * n * 4, rows * 16, rows * 8, rows * 4, rows * 4)]
    args = (dev[0].ptr, n, n, rows, *(d.ptr for d in dev[1:]))
    assert L.llamd_fwd_begin_capture() == 0
    assert L.llamd_hip_sample(*args) == 0
    assert L.llamd_fwd_end_capture() == 0
    for turn in range(4):
        rules = [RULES[(i + turn) % len(RULES)] for i in range(rows)]
        x, u = logits(rng, rows, n, 1 + turn), rng.random(rows)
        if turn == 2:
            x[:] = 1.0
        for d, a in zip(dev, (x, np.array([tuple(r) for r in rules], gpu.SAMPLING), u)):
            d.upload(a)
        for eager in (False, True):
            dev[3].upload(np.full(rows, -9, np.int32))
            assert (L.llamd_hip_sample(*args) if eager else L.llamd_fwd_graph_launch()) == 0
            ids, prob = dev[3].download(np.empty(rows, np.int32)), dev[4].download(np.empty(rows, np.float32))
            S.check(ids, prob, x, rules, u, (turn, eager))
            big = logits(rng, 200 * (turn + 1), 500)
            run(gpu, big, [RULES[3]] * len(big), rng.random(len(big)))
    L.llamd_fwd_graph_destroy()


def test_calls_from_two_threads(gpu):
    import threading
    rng = np.random.default_rng(14)
    jobs = [(logits(rng, 3, 40_000), [RULES[i] for i in (1, 2, 3)], rng.random(3)),
            (logits(rng, 40, 700), [RULES[i % 8] for i in range(40)], rng.random(40))]
    alone = [run(gpu, *j) for j in jobs]
    seen = [[], []]

    def many(i):
        for _ in range(12):
            seen[i].append(run(gpu, *jobs[i]))

    threads = [threading.Thread(target=many, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(seen[i]) == 12
        assert all(np.array_equal(a, b) for got in seen[i] for a, b in zip(got, alone[i]))


# ---- behind the LM head, and a whole step ---------------------------------------------

def test_lm_head(gpu):
    """Drawn from the head's own logits, which stay on the device; temperature 0 is its arg-max."""
    from llamd_rs_amd import synth
    rng = np.random.default_rng(15)
    rows, k, nseq = 3000, 512, 5
    head = gpu.LmHead(gpu.DeviceWeights.upload(synth.q6k_matrix(9, 0.05, rows, k), rows, k // 256), max_seq=8)
    x = (rng.standard_normal((nseq, k)) * 2).astype(np.float32)
    want, best = head.forward(x)
    u = rng.random(nseq)
    for rule in RULES:
        ids, prob = head.sample(x, u, *rule)
        S.check(ids, prob, want, [rule] * nseq, u, rule)
    ids, prob = head.sample(x, u, temperature=0)
    assert np.array_equal(ids, best) and (prob == 1).all()
    ids, _ = head.sample(x[:1], 0.5, top_k=1)
    assert ids[0] == best[0]
    for bad in (dict(x=x[:, :256], u=0.5), dict(x=np.zeros((9, k)), u=0.5), dict(x=x, u=[0.1, 0.2]), dict(x=x[:0], u=0.5)):
        with pytest.raises(ValueError):
            head.sample(**bad)


def test_steps_of_a_small_model(gpu):
    """Two users' tokens through an 8-bit cache, one layer's attention, the LM head and the draw, as a serving loop calls
    them: a prompt, then tokens fed back. Every attention against 64 bits over what the cache holds, every draw against the
    restatement."""
    import paged_reference as R
    from llamd_rs_amd import synth
    from test_gpu_paged import want_decode, want_prompt
    rng = np.random.default_rng(16)
    heads, kvh, hd, page, vocab, dim = 4, 2, 64, 16, 1500, 256
    embed = rng.standard_normal((vocab, dim)).astype(np.float32)
    w = {h: (rng.standard_normal((dim, h * hd)) / 16).astype(np.float32) for h in (heads, kvh)}
    head = gpu.LmHead(gpu.DeviceWeights.upload(synth.q6k_matrix(3, 0.1, vocab, dim), vocab, 1), max_seq=2)
    norm = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    freqs, _ = gpu.rope_freqs(hd, 1e4)
    c = gpu.PagedCache8(16, page, heads, kvh, hd)
    table = np.array([[3, 7, 1, 0], [2, 5, 9, 11]], np.int32)
    tokens, new, lengths = rng.integers(0, vocab, 30), [19, 11], [19, 11]
    rules = [(0.9, 40, 0.95, 0.0), (1.1, 0, 1.0, 0.02)]
    t, k, p, m = (np.array(x) for x in zip(*rules))
    drawn = []
    for step in range(8):
        x = embed[tokens]
        start = np.concatenate([[0], np.cumsum(new)])
        q = c.store(x @ w[heads], x @ w[kvh], x @ w[kvh] * 0.5, table, lengths, start, norm, norm, 1e-6, freqs)
        pages = c.read()
        if step == 0:
            o = c.prompt(q, table, lengths, start)
            want, bound = want_prompt(q, *pages, table, lengths, start, heads, kvh, hd, hd ** -0.5, "bf16")
        else:
            o = c.decode(q, table, lengths)
            want, bound = want_decode(q, *pages, table, lengths, heads, kvh, hd, hd ** -0.5, "bf16")
        R.check(o, want, bound, step)
        last = x[start[1:] - 1] + o[start[1:] - 1] @ w[heads].T
        u = rng.random(2)
        ids, prob = head.sample(last, u, t, k, p, m)
        S.check(ids, prob, head.forward(last)[0], rules, u, step)
        drawn.append(ids)
        tokens, new, lengths = ids, [1, 1], [n + 1 for n in lengths]
    assert len({tuple(d) for d in drawn}) > 4

"""Serving with an 8-bit cache and with sampled tokens, as cases that can be timed and compared.

  store   QK norm, rotary positions and the append of new tokens' keys and values to 8-bit pages (llamd_hip_paged8_store)
  prompt  causal attention of packed sequences' new tokens over such pages (llamd_hip_paged8_prompt)
  decode  attention of one token per sequence, prefixes that sequences share read once (llamd_hip_paged8_decode)
  sample  a token per row of logits: temperature, top-k, top-p, min-p and a given random number (llamd_hip_sample)

An element of a page is an e4m3 number times 2^(E - 127), with one byte E for every 16 positions of a page and kv head. K pages
are [page][kv head][slot][dimension], V pages [page][kv head][dimension][slot]. Head layouts and the vocabulary of 151936 are those
of this repository's tests and timed cases (32 query and 4 kv heads of 128, 16 and 8, 12 and 12 of 64), and one of wide heads.
"""
import ctypes
import math

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6
ROPE_BASE = 1e6
BF16 = 30  # ggml's number
F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BLOCK = 16    # positions that share a scale
TOP = 448.0   # the largest e4m3 number


# ---- the cases -----------------------------------------------------------------

def listed():
    wide = {"heads": 32, "kv_heads": 4, "hd": 128}
    rope = {"rot": 128, "interleaved": False, "factor": 1.0, "orig": 0}
    return [
        # one user's decode step: the smallest call there is
        {"name": "store_1", "kind": "store", **wide, "page": 64, "nseq": 1, "new": 1, "ctx": 900, "pad": 0, "norm": True, "fused": False,
         **rope},
        # several prompts of a model that rotates half of each head, pairs side by side, after cached pieces of any length
        {"name": "store_prompts", "kind": "store", "heads": 16, "kv_heads": 8, "hd": 128, "page": 16, "nseq": 5, "new": 700, "ctx": 333,
         "pad": 3, "norm": False, "fused": False, "rot": 64, "interleaved": True, "factor": 1.0, "orig": 0},
        # a large piece of a long document, positions stretched four times past the trained context, Q, K and V in one matrix
        {"name": "store_long", "kind": "store", **wide, "page": 64, "nseq": 1, "new": 8000, "ctx": 30000, "pad": 0, "norm": True,
         "fused": True, "rot": 128, "interleaved": False, "factor": 4.0, "orig": 10000},
        # several users' prompts packed into one pass, the buffer longer than they are
        {"name": "prompt_packed", "kind": "prompt", **wide, "page": 16, "nseq": 9, "new": 700, "ctx": 0, "pad": 13},
        # the next piece of a long prompt
        {"name": "prompt_chunk", "kind": "prompt", **wide, "page": 64, "nseq": 1, "new": 512, "ctx": 7000, "pad": 0},
        # a whole long prompt at once: the largest call
        {"name": "prompt_8192", "kind": "prompt", **wide, "page": 128, "nseq": 1, "new": 8192, "ctx": 0, "pad": 0},
        # one user deep in a long conversation
        {"name": "decode_1_4100", "kind": "decode", **wide, "page": 64, "nseq": 1, "ctx": 4100, "prefix": 0, "groups": 0},
        # a full batch of users at different lengths, where the cache's bytes count
        {"name": "decode_61_2000", "kind": "decode", **wide, "page": 32, "nseq": 61, "ctx": 2000, "prefix": 0, "groups": 0},
        # a batch behind one long system prompt
        {"name": "decode_shared", "kind": "decode", **wide, "page": 64, "nseq": 48, "ctx": 4600, "prefix": 4100, "groups": 1},
        # one user's next token with the usual settings: temperature, the 50 likeliest, of these 0.9 of the probability
        {"name": "sample_1", "kind": "sample", "rows": 1, "n": 151936, "pad": 0, "rule": "kp", "ties": False, "masked": 0.0},
        # a batch whose users have settings of their own, logits of 16 bits (many equal ones), tokens ruled out by a grammar
        {"name": "sample_mixed", "kind": "sample", "rows": 13, "n": 32001, "pad": 7, "rule": "mixed", "ties": True, "masked": 0.3},
        # a full batch with all of the vocabulary to choose from but the last tenth of the probability
        {"name": "sample_64", "kind": "sample", "rows": 64, "n": 151936, "pad": 0, "rule": "p", "ties": False, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


MOST_PAIRS = 8192 * 8192 // 2  # query-key pairs of a head in the largest listed case


def draw(rng):
    kind = rng.choice(["store", "prompt", "decode", "sample"])
    if kind == "sample":
        return {"kind": kind, "rows": _log(rng, 1, 64), "n": _log(rng, 500, 151936), "pad": rng.choice([0, 0, 5]),
                "rule": rng.choice(["kp", "p", "k", "t", "min", "mixed", "mixed"]), "ties": rng.random() < 0.4,
                "masked": rng.choice([0.0, 0.0, 0.3, 0.9])}
    heads, kv_heads, hd = rng.choice([(32, 4, 128), (32, 4, 128), (16, 8, 128), (12, 12, 64), (16, 1, 64), (8, 2, 256)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "hd": hd, "page": rng.choice([16, 32, 64, 64, 128])}
    if kind == "store":
        n = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 8000 // n))
        return {**case, "nseq": n, "new": new, "ctx": _log(rng, 1, max(1, min(30000, 131072 // n - new))),
                "pad": rng.choice([0, 0, 5]), "norm": rng.random() < 0.7, "fused": rng.random() < 0.5,
                "rot": hd // rng.choice([1, 1, 2]), "interleaved": rng.random() < 0.4, **rng.choice(
                    [{"factor": 1.0, "orig": 0}, {"factor": 2.0, "orig": 0}, {"factor": 4.0, "orig": 10000}])}
    if kind == "prompt":
        n = _log(rng, 1, 16)
        most = MOST_PAIRS // n
        new = _log(rng, 1, min(8192, math.isqrt(2 * most)))
        ctx = 0 if rng.random() < 0.5 else _log(rng, 1, max(1, min(8192, most // new - new)))
        return {**case, "nseq": n, "new": new, "ctx": ctx, "pad": rng.choice([0, 0, 13])}
    n = _log(rng, 1, 64)
    ctx = _log(rng, 16, min(16384, 262144 // n))
    groups = rng.choice([0, 1, 1, 3])
    groups = groups if groups <= n else 0
    return {**case, "nseq": n, "ctx": ctx, "prefix": int(ctx * rng.choice([0.5, 0.9, 0.97])) if groups else 0, "groups": groups}


# ---- inputs ----------------------------------------------------------------------

def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed(seed * 64 + stream)


def _normal(seed, stream, *shape, type=torch.float32):
    return torch.randn(*shape, generator=_gen(seed, stream), device=DEV, dtype=type)


def _uniform(seed, stream, *shape, type=torch.float32):
    return torch.rand(*shape, generator=_gen(seed, stream), device=DEV, dtype=type)


def _ragged(n, top, salt):
    """n lengths, the first of them `top`, the others from a quarter of it."""
    return [max(1, top - (s * salt % 97) * 3 * top // 384) for s in range(n)]


def _lengths(case):
    """(new tokens, positions in the cache with them) of each sequence."""
    n = case["nseq"]
    if case["kind"] == "decode":
        return [1] * n, [case["prefix"] + t for t in _ragged(n, case["ctx"] - case["prefix"], 41)]
    new = _ragged(n, case["new"], 41)
    old = _ragged(n, case["ctx"], 29) if case["ctx"] else [0] * n
    return new, [a + b for a, b in zip(new, old)]


def _group_starts(case):
    return [g * case["nseq"] // case["groups"] for g in range(case["groups"] + 1)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _frequencies(case):
    """(radians per position of each pair, magnitude). A factor stretches the positions; with the trained context length
    it does so by parts: pairs that turn less than once over it are stretched, those that turn over 32 times are not."""
    n, factor, orig = case["rot"], case["factor"], case["orig"]
    f = ROPE_BASE ** (-2.0 * torch.arange(n // 2, dtype=torch.float64) / n)
    if not orig:
        return f / factor, 1.0
    low = n * math.log(orig / (2 * math.pi * 32)) / (2 * math.log(ROPE_BASE))
    high = n * math.log(orig / (2 * math.pi)) / (2 * math.log(ROPE_BASE))
    low, high = max(math.floor(low), 0), min(math.ceil(high), n - 1)
    ramp = ((torch.arange(n // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1


def _filled(seed, stream, pages, kvh, page, hd):
    """(e4m3 bytes [pages, kvh, page, hd], scale bytes [pages, kvh, page / 16]) of normal values, blocks of different sizes."""
    x = _normal(seed, stream, pages, kvh, page // BLOCK, BLOCK, hd)
    x *= torch.exp2(2 * _uniform(seed, stream + 1, pages, kvh, page // BLOCK, 1, 1) - 1)
    e = torch.ceil(torch.log2(x.abs().amax((3, 4), keepdim=True) / TOP))
    x = (x * torch.exp2(-e)).to(F8).view(torch.uint8).reshape(pages, kvh, page, hd)
    return x, (e + 127).to(torch.uint8).reshape(pages, kvh, page // BLOCK)


def _prepare_sample(case, seed):
    rows, n = case["rows"], case["n"]
    x = torch.empty(rows, n + case["pad"], device=DEV)
    x[:, :n] = 2.5 * _normal(seed, 1, rows, n)
    # a few tokens that the model means
    likely = (_uniform(seed, 2, rows, 12) * n).long()
    x[:, :n].scatter_(1, likely, 9 + 2.5 * _normal(seed, 3, rows, 12))
    if case["ties"]:
        x = x.bfloat16().float()
    if case["masked"]:
        x[:, :n][_uniform(seed, 4, rows, n) < case["masked"]] = -math.inf
    x[:, n:] = 99.0
    host = np.random.default_rng(seed)
    how = np.zeros((rows, 4), np.float32)
    number = how.view(np.int32)[:, 1]
    how[:, 0] = host.uniform(0.6, 1.4, rows)
    how[:, 2] = 1
    which = host.integers(0, 6, rows) if case["rule"] == "mixed" else np.full(rows, ["kp", "p", "k", "t", "min"].index(case["rule"]))
    for r, w in enumerate(which.tolist()):
        if w in (0, 2):
            number[r] = host.choice([20, 50, 50, 200, 1000])
        if w in (0, 1):
            how[r, 2] = host.choice([0.5, 0.9, 0.9, 0.95])
        if w == 4:
            how[r, 3] = host.choice([0.01, 0.05, 0.1])
        if w == 5:
            how[r, 0] = 0
    return {"case": case, "x": x, "how": torch.from_numpy(how).to(DEV), "u": torch.from_numpy(host.random(rows)).to(DEV),
            "ids": torch.zeros(rows, dtype=torch.int32, device=DEV), "prob": torch.zeros(rows, device=DEV)}


def prepare(case, seed):
    kind = case["kind"]
    if kind == "sample":
        s = _prepare_sample(case, seed)
        torch.cuda.synchronize()
        return s
    heads, kvh, hd, page, n = case["heads"], case["kv_heads"], case["hd"], case["page"], case["nseq"]
    new, length = _lengths(case)
    # the table: sequences own pages from all over the cache; those of a group share the pages that its prefix fills
    need = [-(-x // page) for x in length]
    top = max(need)
    order = torch.randperm(sum(need) + 3, generator=_gen(seed, 1), device=DEV).tolist()
    table, at = [], 0
    for i in range(n):
        table.append([order[at + j] if j < need[i] else -1 for j in range(top)])
        at += need[i]
    pages = len(order)
    s = {"case": case}
    s["kc"], s["ks"] = _filled(seed, 2, pages, kvh, page, hd)
    v, s["vs"] = _filled(seed, 6, pages, kvh, page, hd)
    s["vc"] = v.transpose(2, 3).contiguous()
    if kind == "decode" and case["groups"]:
        starts, full, rest = _group_starts(case), case["prefix"] // page, case["prefix"] % page
        for a, b in zip(starts, starts[1:]):
            for i in range(a + 1, b):
                table[i][:full] = table[a][:full]
                if rest:  # the page that the prefix ends in is each sequence's own copy
                    for name in ("kc", "vc", "ks", "vs"):
                        s[name][table[i][full]] = s[name][table[a][full]]
    start = [sum(new[:i]) for i in range(n + 1)]
    tokens = start[-1] + case.get("pad", 0)
    s.update(start=_ints(start), length=_ints(length), table=_ints(table), tokens=tokens)
    if kind == "decode" and case["groups"]:
        s.update(group=_ints(starts), shared=_ints([case["prefix"]] * case["groups"]))
    if kind == "store":
        x = _normal(seed, 4, tokens, (heads + 2 * kvh) * hd)
        parts = x.split([heads * hd, kvh * hd, kvh * hd], 1)
        s["qkv"] = parts if case["fused"] else tuple(p.contiguous() for p in parts)
        s["norms"] = tuple(1 + 0.1 * _normal(seed, i, hd) for i in (8, 9)) if case["norm"] else None
        if case["norm"]:  # keys have a few channels that are larger than the others
            s["norms"][1][5::37] *= 4
        f, s["magnitude"] = _frequencies(case)
        s["freqs"] = f.to(DEV)
    else:
        s["q"] = _normal(seed, 4, tokens, heads * hd, type=torch.bfloat16)
    s["out"] = torch.zeros(tokens, heads * hd, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------------

def _positions(s):
    """The sequence of each token and its position."""
    start, length = s["start"].long(), s["length"].long()
    token = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(start[1:].contiguous(), token, right=True)
    seq = seq[seq < len(length)]
    return seq, length[seq] - (start[seq + 1] - token[:len(seq)])


def _turned(x, weight, s, pos):
    """x [tokens, heads, hd] normed by head and rotated, in 32 bits; the angles in 64."""
    case = s["case"]
    if weight is not None:
        x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight
    angle = pos[:, None].double() * s["freqs"]
    c, sn = ((f(angle) * s["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    n = case["rot"]
    x, rest = x[..., :n], x[..., n:]
    a, b = (x[..., 0::2], x[..., 1::2]) if case["interleaved"] else (x[..., :n // 2], x[..., n // 2:])
    a, b = a * c - b * sn, a * sn + b * c
    x = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([x, rest], -1)


def _unit(x):
    """The scale byte of values whose largest is x: the least E with x <= 448 * 2^(E - 127), 1 at least."""
    bits = x.view(torch.int32)
    return ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)).clamp_min(1)


def _append(x, cache, scales, values_last, s, seq, pos):
    """x [tokens, kvh, hd] into 8-bit pages; `values_last`: a page holds a dimension's positions together."""
    page = s["case"]["page"]
    flat = cache.transpose(2, 3) if values_last else cache  # [page][kv head][slot][dimension]
    at, slot = s["table"].long()[seq, pos // page], pos % page
    block = at * (page // BLOCK) + slot // BLOCK
    top = torch.zeros(scales.shape[0] * (page // BLOCK), x.shape[1], device=DEV)
    top = top.index_reduce(0, block, x.abs().amax(-1), "amax")
    touched = torch.zeros(len(top), dtype=torch.bool, device=DEV)
    touched[block] = True
    # the blocks with positions before the new ones: those of the sequences' first tokens
    begin = s["start"].long()[:-1]
    first_block, first_slot = block[begin], slot[begin] % BLOCK
    before = torch.zeros(len(top), dtype=torch.long, device=DEV)
    before[first_block] = first_slot
    old = scales.transpose(1, 2).reshape(len(top), -1).int()
    unit = torch.maximum(_unit(top), torch.where(before[:, None] > 0, old, 1))
    unit = torch.where(touched[:, None], unit, old)
    # those re-expressed
    i = torch.arange(BLOCK, device=DEV)
    b, j = torch.nonzero(i < before[first_block][:, None], as_tuple=True)
    b = first_block[b]
    where = (b // (page // BLOCK), slice(None), b % (page // BLOCK) * BLOCK + j)
    was = flat[where].contiguous().view(F8).float() * torch.exp2((old - unit)[b].float())[..., None]
    flat[where] = was.to(F8).view(torch.uint8)
    flat[at, :, slot] = (x * torch.exp2(127.0 - unit[block])[..., None]).to(F8).view(torch.uint8)
    scales.copy_(unit.to(torch.uint8).reshape(scales.shape[0], -1, scales.shape[1]).transpose(1, 2))


def _stored(s):
    return {"q": s["out"], "k": s["kc"].view(F8), "v": s["vc"].view(F8), "k_scale": s["ks"].view(E8), "v_scale": s["vs"].view(E8)}


def _store(s):
    case = s["case"]
    seq, pos = _positions(s)
    n = len(seq)
    q, k, v = (x[:n].reshape(n, -1, case["hd"]) for x in s["qkv"])
    wq, wk = s["norms"] or (None, None)
    s["out"][:n] = _turned(q, wq, s, pos).bfloat16().reshape(n, -1)
    _append(_turned(k, wk, s, pos), s["kc"], s["ks"], False, s, seq, pos)
    _append(v, s["vc"], s["vs"], True, s, seq, pos)
    return _stored(s)


def _attend(s):
    """Every sequence's tokens against all slots of its pages, what lies behind a token masked."""
    case = s["case"]
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    seq, pos = _positions(s)
    n, group = case["nseq"], heads // kvh
    row = torch.arange(len(seq), device=DEV) - s["start"].long()[seq]
    most = int(max(_lengths(case)[0]))
    q = torch.zeros(n, most, heads, hd, device=DEV)
    q[seq, row] = s["q"][:len(seq)].reshape(-1, heads, hd).float()
    at = torch.full((n, most), -1, dtype=torch.long, device=DEV)
    at[seq, row] = pos
    table = s["table"].long().clamp_min(0)
    slots = table.shape[1] * page
    unit = [torch.exp2(x[table].float() - 127).permute(0, 2, 1, 3).reshape(n, kvh, -1).repeat_interleave(BLOCK, 2)[..., None]
            for x in (s["ks"], s["vs"])]
    k = s["kc"][table].view(F8).permute(0, 2, 1, 3, 4).reshape(n, kvh, slots, hd).float() * unit[0]
    v = s["vc"][table].view(F8).permute(0, 2, 1, 4, 3).reshape(n, kvh, slots, hd).float() * unit[1]
    q = q.reshape(n, most, kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(n, kvh, most * group, hd)
    p = (q * (hd ** -0.5)) @ k.transpose(2, 3).contiguous()
    seen = (torch.arange(slots, device=DEV) <= at[:, :, None]).repeat_interleave(group, 1)[:, None]
    p = p.masked_fill_(~seen, -math.inf)
    p = (p - p.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.reshape(n, kvh, most, group, hd).permute(0, 2, 1, 3, 4).reshape(n, most, heads * hd)
    s["out"][:len(seq)] = o[seq, row].bfloat16()
    return s["out"]


def _sample(s):
    """In 64 bits: a token is chosen where a running sum passes a border."""
    n = s["case"]["n"]
    x = s["x"][:, :n].double()
    t, p, least = (s["how"][:, i:i + 1].double() for i in (0, 2, 3))
    k = s["how"].view(torch.int32)[:, 1:2]
    greedy = t <= 0
    w = ((x - x.amax(1, keepdim=True)) / torch.where(greedy, 1.0, t)).exp()
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(n, device=DEV)
    among = (rank < k) | (k <= 0)
    ws = torch.where(among, ws, 0.0)
    total = ws.cumsum(1)
    keep = among & ((total - ws < p * total[:, -1:]) | (p >= 1)) & (ws >= least)
    keep = torch.where(greedy, False, keep) | (rank == 0)
    w = torch.where(torch.zeros_like(keep).scatter_(1, order, keep), w, 0.0)
    total = w.cumsum(1)
    at = (total <= s["u"][:, None] * total[:, -1:]).sum(1, keepdim=True).clamp_max(n - 1)
    s["ids"].copy_(at[:, 0])
    s["prob"].copy_(w.gather(1, at)[:, 0] / total[:, -1])
    return {"ids": s["ids"], "prob": s["prob"]}


def _own_sample(s, L):
    case, x = s["case"], s["x"]
    if L.llamd_hip_sample(x.data_ptr(), x.stride(0), case["n"], case["rows"], s["how"].data_ptr(), s["u"].data_ptr(),
                          s["ids"].data_ptr(), s["prob"].data_ptr()):
        raise RuntimeError("sample: %s" % L.llamd_hip_last_error())
    return {"ids": s["ids"], "prob": s["prob"]}


def _own(s):
    """The library's call; the descriptors of the cache and the batch are made once, as a program does."""
    from llamd_rs_amd import rocm
    from llamd_rs_amd._lib import lib
    case, L = s["case"], lib()
    if case["kind"] == "sample":
        return _own_sample(s, L)
    if "pages" not in s:
        s["pages"] = rocm.Pages8(s["kc"].data_ptr(), s["vc"].data_ptr(), s["ks"].data_ptr(), s["vs"].data_ptr(), s["kc"].shape[0],
                                 case["page"], case["kv_heads"], case["hd"])
        s["batch"] = rocm.Batch(s["start"].data_ptr(), s["length"].data_ptr(), s["table"].data_ptr(), case["nseq"],
                                s["tokens"], s["table"].shape[1])
    pages, batch, out = ctypes.byref(s["pages"]), ctypes.byref(s["batch"]), s["out"].data_ptr()
    if case["kind"] == "store":
        (q, k, v), (wq, wk) = s["qkv"], s["norms"] or (None, None)
        rc = L.llamd_hip_paged8_store(
            pages, batch, q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
            wq.data_ptr() if case["norm"] else None, wk.data_ptr() if case["norm"] else None, EPS, s["freqs"].data_ptr(),
            case["rot"], int(case["interleaved"]), s["magnitude"], case["heads"], out)
        result = _stored(s)
    else:
        scale, result = case["hd"] ** -0.5, s["out"]
        if case["kind"] == "prompt":
            rc = L.llamd_hip_paged8_prompt(pages, batch, s["q"].data_ptr(), case["heads"], scale, BF16, out)
        else:
            group, shared = (s["group"].data_ptr(), s["shared"].data_ptr()) if case["groups"] else (None, None)
            rc = L.llamd_hip_paged8_decode(pages, batch, group, shared, case["groups"], s["q"].data_ptr(), case["heads"], scale,
                                           BF16, out)
    if rc:
        raise RuntimeError("%s: %s" % (case["kind"], L.llamd_hip_last_error()))
    return result


def run(state):
    if own:
        return _own(state)
    return {"store": _store, "sample": _sample}.get(state["case"]["kind"], _attend)(state)


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    if case["kind"] == "sample":
        # an exponential as 8 operations, a sum and two comparisons for each logit
        return {"bytes": case["rows"] * (4 * case["n"] + 32), "flops": 11 * case["rows"] * case["n"]}
    heads, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
    new, length = _lengths(case)
    if case["kind"] == "store":
        return {"bytes": sum(new) * hd * (heads * 6 + kvh * 10), "flops": sum(new) * (heads + kvh) * hd * (7 if case["norm"] else 3)}
    pairs = sum(n * x - n * (n - 1) // 2 for n, x in zip(new, length))
    read = sum(length)
    if case["kind"] == "decode" and case["groups"]:
        read -= (case["nseq"] - case["groups"]) * case["prefix"]
    return {"bytes": 2 * read * kvh * (hd + 1 / BLOCK) + 4 * sum(new) * heads * hd, "flops": 4 * pairs * heads * hd}


# ---- the same in 64 bits ------------------------------------------------------------------

def _exact_sample(case, seed):
    s = prepare(case, seed)
    ids, prob = np.zeros(case["rows"], np.int64), np.zeros(case["rows"])
    how, u = s["how"].cpu().numpy(), s["u"].cpu().numpy()
    for r, x in enumerate(s["x"][:, :case["n"]].cpu().numpy().astype(np.float64)):
        t, k, p, least = float(how[r, 0]), int(how[r:r + 1].view(np.int32)[0, 1]), float(how[r, 2]), float(how[r, 3])
        best = int(np.argmax(x))
        if t <= 0:
            ids[r], prob[r] = best, 1
            continue
        order = np.lexsort((np.arange(len(x)), -x))
        order = order[:k] if k > 0 else order
        w = np.exp((x[order] - x[best]) / t).astype(np.longdouble)
        if p < 1:
            before = np.concatenate([[0], np.cumsum(w)[:-1]])
            order = order[before < p * w.sum()]
        order = np.sort(order[np.exp((x[order] - x[best]) / t) >= min(least, 1)])
        w = np.exp((x[order] - x[best]) / t).astype(np.longdouble)
        at = min(int(np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right")), len(w) - 1)
        ids[r], prob[r] = order[at], w[at] / w.sum()
    return {"ids": torch.from_numpy(ids).int(), "prob": torch.from_numpy(prob)}


def _exact_append(y, cache, scales, row, first, page):
    """y [tokens, kvh, hd] at positions first .. of one sequence: cache [page][kv head][slot][hd] and scales hold numbers."""
    last = first + len(y)
    for b in range(first // BLOCK, (last - 1) // BLOCK + 1):
        lo, hi = max(first, b * BLOCK), min(last, b * BLOCK + BLOCK)
        at, slot, kept = int(row[b * BLOCK // page]), b * BLOCK % page, lo - b * BLOCK
        part = y[lo - first:hi - first].transpose(0, 1)
        need = torch.exp2(torch.ceil(torch.log2(part.abs().amax((1, 2)) / TOP)))
        old = scales[at, :, slot // BLOCK].clone()
        unit = torch.maximum(need, old) if kept else need
        if kept:
            cache[at, :, slot:slot + kept] *= (old / unit)[:, None, None]
        cache[at, :, slot + kept:slot + hi - b * BLOCK] = part / unit[:, None, None]
        scales[at, :, slot // BLOCK] = unit


def exact(case, seed):
    if case["kind"] == "sample":
        return _exact_sample(case, seed)
    s = prepare(case, seed)
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    new, length = _lengths(case)
    out = s["out"].double()
    kc, vc = s["kc"].view(F8).double(), s["vc"].view(F8).double().transpose(2, 3).contiguous()
    ks, vs = (torch.exp2(x.double() - 127) for x in (s["ks"], s["vs"]))
    first = 0
    if case["kind"] != "store":
        kc = kc * ks.repeat_interleave(BLOCK, 2)[..., None]
        vc = vc * vs.repeat_interleave(BLOCK, 2)[..., None]
    for i, (m, x) in enumerate(zip(new, length)):
        rows = slice(first, first + m)
        first += m
        owned = s["table"][i, :-(-x // page)].long()
        at = torch.arange(x - m, x, device=DEV)
        if case["kind"] == "store":
            f, magnitude = _frequencies(case)
            turn = torch.polar(torch.full((m, case["rot"] // 2), magnitude, dtype=torch.float64, device=DEV),
                               at[:, None].double() * f.to(DEV))
            done = []
            for which, h in ((0, heads), (1, kvh)):
                y = s["qkv"][which][rows].double().reshape(m, h, hd).clone()
                if case["norm"]:
                    y /= (y.square().sum(-1, keepdim=True) / hd + EPS).sqrt()
                    y *= s["norms"][which].double()
                half = case["rot"] // 2
                one = slice(0, case["rot"], 2) if case["interleaved"] else slice(0, half)
                two = slice(1, case["rot"], 2) if case["interleaved"] else slice(half, case["rot"])
                z = torch.complex(y[..., one].contiguous(), y[..., two].contiguous()) * turn[:, None]
                y[..., one], y[..., two] = z.real, z.imag
                done.append(y)
            out[rows] = done[0].reshape(m, -1)
            owned = owned.tolist()
            _exact_append(done[1], kc, ks, owned, x - m, page)
            _exact_append(s["qkv"][2][rows].double().reshape(m, kvh, hd), vc, vs, owned, x - m, page)
            continue
        q = s["q"][rows].double().reshape(m, kvh, heads // kvh, hd)
        behind = torch.arange(x, device=DEV)[None, :] > at[:, None]
        for h in range(kvh):
            k = kc[owned, h].reshape(-1, hd)[:x]
            v = vc[owned, h].reshape(-1, hd)[:x]
            for g in range(heads // kvh):
                a = (q[:, h, g] @ k.T) / math.sqrt(hd)
                a = torch.softmax(a.masked_fill_(behind, -math.inf), -1)
                head = h * (heads // kvh) + g
                out[rows, head * hd:(head + 1) * hd] = a @ v
    if case["kind"] != "store":
        return out
    return {"q": out, "k": kc, "v": vc.transpose(2, 3).contiguous(), "k_scale": ks, "v_scale": vs}

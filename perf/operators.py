"""The attention side of serving over a paged KV cache, as cases that can be timed and compared.

  store   QK norm, rotary positions and the append of new tokens' keys and values to the pages (llamd_hip_paged_store)
  prompt  causal attention of packed sequences' new tokens over their pages (llamd_hip_paged_prompt)
  decode  attention of one token per sequence, prefixes that sequences share read once (llamd_hip_paged_decode)

Head layouts are those of this repository's tests and timed cases (32 query and 4 kv heads of 128, 16 and 8, 12 and 12
of 64), and one of wide heads. K pages are [page][kv head][slot][dimension], V pages [page][kv head][dimension][slot].
"""
import ctypes
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-6
ROPE_BASE = 1e6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NUMBERS = {"f32": 0, "f16": 1, "bf16": 30}  # ggml's


# ---- the cases -----------------------------------------------------------------

def listed():
    wide = {"heads": 32, "kv_heads": 4, "hd": 128}
    plain_rope = {"rot": 128, "interleaved": False, "factor": 1.0, "orig": 0}
    return [
        # one user's decode step: the smallest call there is
        {"name": "store_1", "kind": "store", "type": "bf16", **wide, "page": 64, "nseq": 1, "new": 1, "ctx": 900, "pad": 0,
         "norm": True, "fused": False, **plain_rope},
        # a decode batch at different lengths, Q, K and V side by side in one matrix
        {"name": "store_16", "kind": "store", "type": "f16", **wide, "page": 16, "nseq": 16, "new": 1, "ctx": 1000, "pad": 3,
         "norm": True, "fused": True, **plain_rope},
        # a few prompts of a model that rotates half of each head, pairs side by side, without QK norm
        {"name": "store_prompts", "kind": "store", "type": "f32", "heads": 16, "kv_heads": 8, "hd": 128, "page": 32, "nseq": 5,
         "new": 700, "ctx": 0, "pad": 0, "norm": False, "fused": False, "rot": 64, "interleaved": True, "factor": 1.0, "orig": 0},
        # a large piece of a long document, positions stretched four times past the trained context
        {"name": "store_long", "kind": "store", "type": "bf16", **wide, "page": 64, "nseq": 1, "new": 8000, "ctx": 30000, "pad": 0,
         "norm": True, "fused": True, "rot": 128, "interleaved": False, "factor": 4.0, "orig": 10000},
        # a short prompt
        {"name": "prompt_45", "kind": "prompt", "type": "bf16", **wide, "page": 64, "nseq": 1, "new": 45, "ctx": 0, "pad": 0},
        # several users' prompts packed into one pass, the buffer longer than they are
        {"name": "prompt_packed", "kind": "prompt", "type": "f16", **wide, "page": 16, "nseq": 9, "new": 700, "ctx": 0, "pad": 13},
        # the next piece of a long prompt
        {"name": "prompt_chunk", "kind": "prompt", "type": "bf16", **wide, "page": 64, "nseq": 1, "new": 512, "ctx": 7000, "pad": 0},
        # a whole long prompt at once: the largest call
        {"name": "prompt_8192", "kind": "prompt", "type": "bf16", **wide, "page": 128, "nseq": 1, "new": 8192, "ctx": 0, "pad": 0},
        # prompts of a caller that keeps its cache in f32, as the rest of the library does
        {"name": "prompt_f32", "kind": "prompt", "type": "f32", "heads": 12, "kv_heads": 12, "hd": 64, "page": 32, "nseq": 2,
         "new": 700, "ctx": 300, "pad": 0},
        # one user deep in a long conversation
        {"name": "decode_1_4100", "kind": "decode", "type": "bf16", **wide, "page": 64, "nseq": 1, "ctx": 4100, "prefix": 0, "groups": 0},
        # a batch of users at different lengths, in f32
        {"name": "decode_13_1000", "kind": "decode", "type": "f32", **wide, "page": 32, "nseq": 13, "ctx": 1000, "prefix": 0,
         "groups": 0},
        # a batch behind one long system prompt
        {"name": "decode_shared", "kind": "decode", "type": "bf16", **wide, "page": 64, "nseq": 48, "ctx": 4600, "prefix": 4100,
         "groups": 1},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


MOST_PAIRS = 8192 * 8192 // 2  # query-key pairs of a head in the largest listed case


def draw(rng):
    heads, kv_heads, hd = rng.choice([(32, 4, 128), (32, 4, 128), (16, 8, 128), (12, 12, 64), (16, 1, 64), (8, 2, 256)])
    case = {"kind": rng.choice(["store", "prompt", "prompt", "decode", "decode"]), "type": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "heads": heads, "kv_heads": kv_heads, "hd": hd, "page": rng.choice([16, 32, 64, 64, 128])}
    if case["kind"] == "store":
        n = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 8000 // n))
        return {**case, "nseq": n, "new": new, "ctx": _log(rng, 1, max(1, min(30000, 131072 // n - new))),
                "pad": rng.choice([0, 0, 5]), "norm": rng.random() < 0.7, "fused": rng.random() < 0.5,
                "rot": hd // rng.choice([1, 1, 2]), "interleaved": rng.random() < 0.4, **rng.choice(
                    [{"factor": 1.0, "orig": 0}, {"factor": 2.0, "orig": 0}, {"factor": 4.0, "orig": 10000}])}
    if case["kind"] == "prompt":
        n = _log(rng, 1, 16)
        # f32 products run at a sixteenth of the 16-bit rate
        most = MOST_PAIRS // (16 if case["type"] == "f32" else 1) // n
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


def prepare(case, seed):
    kind, t, n = case["kind"], TYPES[case["type"]], case["nseq"]
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    new, length = _lengths(case)
    # the table: sequences own pages from all over the cache; those of a group share the pages that its prefix fills
    need = [-(-x // page) for x in length]
    top = max(need)
    order = torch.randperm(sum(need) + 3, generator=_gen(seed, 1), device=DEV).tolist()
    table, at = [], 0
    for s in range(n):
        table.append([order[at + i] if i < need[s] else -1 for i in range(top)])
        at += need[s]
    pages = len(order)
    s = {"case": case, "kc": _normal(seed, 2, pages, kvh, page, hd, type=t), "vc": _normal(seed, 3, pages, kvh, hd, page, type=t)}
    if kind == "decode" and case["groups"]:
        starts, full, rest = _group_starts(case), case["prefix"] // page, case["prefix"] % page
        for a, b in zip(starts, starts[1:]):
            for i in range(a + 1, b):
                table[i][:full] = table[a][:full]
                if rest:  # the page that the prefix ends in is each sequence's own copy
                    s["kc"][table[i][full], :, :rest] = s["kc"][table[a][full], :, :rest]
                    s["vc"][table[i][full], :, :, :rest] = s["vc"][table[a][full], :, :, :rest]
        s.update(group=_ints(starts), shared=_ints([case["prefix"]] * case["groups"]))
    start = [sum(new[:i]) for i in range(n + 1)]
    tokens = start[-1] + case.get("pad", 0)
    s.update(start=_ints(start), length=_ints(length), table=_ints(table), tokens=tokens)
    if kind == "store":
        x = _normal(seed, 4, tokens, (heads + 2 * kvh) * hd)
        parts = x.split([heads * hd, kvh * hd, kvh * hd], 1)
        s["qkv"] = parts if case["fused"] else tuple(p.contiguous() for p in parts)
        s["norms"] = tuple(1 + 0.1 * _normal(seed, i, hd) for i in (5, 6)) if case["norm"] else None
        f, s["magnitude"] = _frequencies(case)
        s["freqs"] = f.to(DEV)
    else:
        s["q"] = _normal(seed, 4, tokens, heads * hd, type=t)
    s["out"] = torch.zeros(tokens, heads * hd, dtype=t, device=DEV)
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


def _store(s):
    case, t = s["case"], TYPES[s["case"]["type"]]
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    seq, pos = _positions(s)
    n = len(seq)
    q, k, v = (x[:n].reshape(n, -1, hd) for x in s["qkv"])
    wq, wk = s["norms"] or (None, None)
    s["out"][:n] = _turned(q, wq, s, pos).to(t).reshape(n, heads * hd)
    at, slot = s["table"].long()[seq, pos // page], pos % page
    s["kc"][at, :, slot] = _turned(k, wk, s, pos).to(t)
    s["vc"][at, :, :, slot] = v.to(t)
    return {"q": s["out"], "k": s["kc"], "v": s["vc"]}


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
    k = s["kc"][table].permute(0, 2, 1, 3, 4).reshape(n, kvh, slots, hd).float()
    v = s["vc"][table].permute(0, 2, 1, 4, 3).reshape(n, kvh, slots, hd).float()
    q = q.reshape(n, most, kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(n, kvh, most * group, hd)
    p = (q * (hd ** -0.5)) @ k.transpose(2, 3).contiguous()
    seen = (torch.arange(slots, device=DEV) <= at[:, :, None]).repeat_interleave(group, 1)[:, None]
    p = p.masked_fill_(~seen, -math.inf)
    p = (p - p.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.reshape(n, kvh, most, group, hd).permute(0, 2, 1, 3, 4).reshape(n, most, heads * hd)
    s["out"][:len(seq)] = o[seq, row].to(s["out"].dtype)
    return s["out"]


def _own(s):
    """The library's call; the descriptors of the cache and the batch are made once, as a program does."""
    from llamd_rs_amd import rocm
    from llamd_rs_amd._lib import lib
    case, L = s["case"], lib()
    if "pages" not in s:
        s["pages"] = rocm.Pages(s["kc"].data_ptr(), s["vc"].data_ptr(), NUMBERS[case["type"]], s["kc"].shape[0], case["page"],
                                case["kv_heads"], case["hd"])
        s["batch"] = rocm.Batch(s["start"].data_ptr(), s["length"].data_ptr(), s["table"].data_ptr(), case["nseq"],
                                s["tokens"], s["table"].shape[1])
    pages, batch, out = ctypes.byref(s["pages"]), ctypes.byref(s["batch"]), s["out"].data_ptr()
    if case["kind"] == "store":
        (q, k, v), (wq, wk) = s["qkv"], s["norms"] or (None, None)
        rc = L.llamd_hip_paged_store(
            pages, batch, q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
            wq.data_ptr() if case["norm"] else None, wk.data_ptr() if case["norm"] else None, EPS, s["freqs"].data_ptr(),
            case["rot"], int(case["interleaved"]), s["magnitude"], case["heads"], out)
        result = {"q": s["out"], "k": s["kc"], "v": s["vc"]}
    else:
        scale, number, result = case["hd"] ** -0.5, NUMBERS[case["type"]], s["out"]
        if case["kind"] == "prompt":
            rc = L.llamd_hip_paged_prompt(pages, batch, s["q"].data_ptr(), case["heads"], scale, number, out)
        else:
            group, shared = (s["group"].data_ptr(), s["shared"].data_ptr()) if case["groups"] else (None, None)
            rc = L.llamd_hip_paged_decode(pages, batch, group, shared, case["groups"], s["q"].data_ptr(), case["heads"], scale,
                                          number, out)
    if rc:
        raise RuntimeError("%s: %s" % (case["kind"], L.llamd_hip_last_error()))
    return result


def run(state):
    if own:
        return _own(state)
    return _store(state) if state["case"]["kind"] == "store" else _attend(state)


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    heads, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
    size = 4 if case["type"] == "f32" else 2
    new, length = _lengths(case)
    if case["kind"] == "store":
        values = sum(new) * (heads + 2 * kvh) * hd
        return {"bytes": values * (4 + size), "flops": sum(new) * (heads + kvh) * hd * (7 if case["norm"] else 3)}
    pairs = sum(n * x - n * (n - 1) // 2 for n, x in zip(new, length))
    read = sum(length)
    if case["kind"] == "decode" and case["groups"]:
        read -= (case["nseq"] - case["groups"]) * case["prefix"]
    return {"bytes": size * (2 * read * kvh * hd + 2 * sum(new) * heads * hd), "flops": 4 * pairs * heads * hd}


# ---- the same in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["hd"], case["page"]
    new, length = _lengths(case)
    out = s["out"].double()
    kc, vc = s["kc"].double(), s["vc"].double()
    first = 0
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
            kc[owned[at // page], :, at % page] = done[1]
            vc[owned[at // page], :, :, at % page] = s["qkv"][2][rows].double().reshape(m, kvh, hd)
            continue
        q = s["q"][rows].double().reshape(m, kvh, heads // kvh, hd)
        behind = torch.arange(x, device=DEV)[None, :] > at[:, None]
        for h in range(kvh):
            k = kc[owned, h].reshape(-1, hd)[:x]
            v = vc[owned, h].transpose(1, 2).reshape(-1, hd)[:x]
            for g in range(heads // kvh):
                a = (q[:, h, g] @ k.T) / math.sqrt(hd)
                a = torch.softmax(a.masked_fill_(behind, -math.inf), -1)
                head = h * (heads // kvh) + g
                out[rows, head * hd:(head + 1) * hd] = a @ v
    return {"q": out, "k": kc, "v": vc} if case["kind"] == "store" else out

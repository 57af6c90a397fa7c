"""The operators of a decode step over quantised pages, as timed cases: rotary
positions, a page pool written and read back at slots, and attention of one new
token of each sequence over that pool.

A case is a dict of plain values. ``prepare`` makes what a program holds before
the call, ``run`` is one pass: the framework's calls where ``own`` is true, the
same in plain torch operations otherwise. ``work`` is what a pass cannot do
without, ``exact`` the result in 64 bits.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GROUP = 16  # int4 group of the cache


def _framework():
    path = os.path.join(os.getcwd(), "shadow-infer_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import shadowinfer_amd

    return shadowinfer_amd


def listed():
    return [
        # one new token of one sequence: the smallest call of a layer
        {"name": "rope_one_token", "kind": "rope", "T": 1, "Hq": 32, "Hk": 32, "D": 128, "R": 128,
         "layout": "half", "scaling": "none", "factor": 1.0, "base": 10000.0, "first": 4095,
         "dtype": "bf16", "transpose": False},
        # a long prompt's queries and grouped keys, far into a stretched context
        {"name": "rope_prompt_8192", "kind": "rope", "T": 8192, "Hq": 32, "Hk": 8, "D": 128,
         "R": 128, "layout": "interleaved", "scaling": "yarn", "factor": 16.0, "base": 10000.0,
         "first": 100000, "dtype": "bf16", "transpose": False},
        # part of an 80-wide head, ragged, rotated back (a gradient's direction)
        {"name": "rope_part_1003", "kind": "rope", "T": 1003, "Hq": 12, "Hk": 12, "D": 80, "R": 32,
         "layout": "half", "scaling": "bands", "factor": 8.0, "base": 500000.0, "first": 0,
         "dtype": "f16", "transpose": True},
        # one new token of each of 64 sequences into its page, int8 rows
        {"name": "cache_decode_64", "kind": "cache", "T": 64, "H": 8, "D": 128, "P": 32,
         "dtype": "bf16", "prec": "int8", "out": "bf16", "pad": 0.0, "rope": False},
        # a padded batch of an 80-wide model, fp32 rows kept as int8
        {"name": "cache_ragged_1003", "kind": "cache", "T": 1003, "H": 12, "D": 80, "P": 24,
         "dtype": "f32", "prec": "int8", "out": "f32", "pad": 0.1, "rope": False},
        # a prompt's keys rotated on their way into 16-bit pages
        {"name": "cache_rotated_2048", "kind": "cache", "T": 2048, "H": 8, "D": 128, "P": 16,
         "dtype": "bf16", "prec": "fp32", "out": "bf16", "pad": 0.0, "rope": True},
        # a long prompt of one layer of a 7B-shaped model, grouped int4
        {"name": "cache_prompt_8192", "kind": "cache", "T": 8192, "H": 32, "D": 128, "P": 32,
         "dtype": "bf16", "prec": "int4", "out": "bf16", "pad": 0.0, "rope": False},
        # the first answer of one short chat: 16-bit pages, a few of them
        {"name": "attend_one_100", "kind": "attend", "B": 1, "Hq": 32, "Hk": 32, "D": 128, "P": 32,
         "L": 100, "spread": 0.0, "window": 0, "q": "bf16", "dtype": "bf16", "prec": "fp32",
         "lse": False},
        # one sequence over a very long cache, grouped heads
        {"name": "attend_one_131072", "kind": "attend", "B": 1, "Hq": 32, "Hk": 8, "D": 128,
         "P": 32, "L": 131072, "spread": 0.0, "window": 0, "q": "bf16", "dtype": "bf16",
         "prec": "int8", "lse": False},
        # a serving batch of uneven lengths, one slot of it empty, int4 pages
        {"name": "attend_batch_64", "kind": "attend", "B": 64, "Hq": 32, "Hk": 8, "D": 128,
         "P": 16, "L": 4096, "spread": 1.0, "window": 0, "q": "bf16", "dtype": "bf16",
         "prec": "int4", "lse": True},
        # a small model in fp32 with odd pages, the last 1024 positions only
        {"name": "attend_window_80", "kind": "attend", "B": 7, "Hq": 12, "Hk": 4, "D": 80, "P": 24,
         "L": 2000, "spread": 0.7, "window": 1024, "q": "f32", "dtype": "f32", "prec": "int8",
         "lse": True},
        # a full batch of a 7B-shaped layer, every head its own keys
        {"name": "attend_full_8192", "kind": "attend", "B": 16, "Hq": 32, "Hk": 32, "D": 128,
         "P": 32, "L": 8192, "spread": 0.1, "window": 0, "q": "bf16", "dtype": "bf16",
         "prec": "int8", "lse": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "cache", "cache", "attend", "attend", "attend"])
    if kind == "rope":
        Hq, Hk = rng.choice([(32, 32), (32, 8), (16, 2), (12, 4), (8, 1)])
        D = rng.choice([64, 80, 128])
        scaling = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
        return {"kind": kind, "T": _log_int(rng, 1, 8192), "Hq": Hq, "Hk": Hk, "D": D,
                "R": rng.choice([D, D, D // 2, 32]), "layout": rng.choice(["half", "interleaved"]),
                "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 8.0, 32.0]),
                "base": rng.choice([10000.0, 500000.0]), "first": rng.choice([0, 1000, 100000]),
                "dtype": rng.choice(["bf16", "f16", "f32"]) if Hq < 32 else "bf16",
                "transpose": rng.random() < 0.25}
    if kind == "cache":
        H, D, dtype = rng.choice([4, 8, 12, 32]), rng.choice([64, 80, 128]), rng.choice(["bf16", "f16", "f32"])
        prec = rng.choice(["fp32", "fp16", "int8", "int4"])
        return {"kind": kind, "T": _log_int(rng, 1, 8192 if H < 32 else 4096), "H": H, "D": D,
                "P": rng.choice([1, 16, 24, 32, 64]), "dtype": dtype, "prec": prec,
                "out": rng.choice(["f32", dtype]), "pad": rng.choice([0.0, 0.0, 0.2]),
                "rope": prec == "fp32" and dtype != "f32" and rng.random() < 0.5}
    D = rng.choice([64, 80, 128, 128, 128])
    Hq, Hk = rng.choice([(32, 32), (32, 8), (32, 4), (16, 1), (12, 4), (12, 12)])
    L, dtype = _log_int(rng, 1, 65536), rng.choice(["bf16", "bf16", "f16", "f32"])
    case = {"kind": kind, "B": 1, "Hq": Hq, "Hk": Hk, "D": D, "P": rng.choice([8, 16, 24, 32, 64]),
            "L": L, "spread": 0.0, "window": rng.choice([0, 0, 0, 512]), "q": dtype, "dtype": dtype,
            "prec": rng.choice(["fp32", "fp16", "int8", "int8", "int4"]), "lse": rng.random() < 0.5}
    # tokens in all: the cache and the products of the largest listed case
    most = min(10 ** 9 // (2 * Hk * _row_bytes(case, D)), 2 * 10 ** 9 // (4 * Hq * D))
    case["L"] = min(L, most)
    case["B"] = min(_log_int(rng, 1, 64), most // case["L"])
    if case["B"] > 1:
        case["spread"] = rng.choice([0.0, 0.5, 1.0])
    return case


# ------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(g, T, H, D, dtype):
    """K and V of a projection, ``[T, H, D]`` views of one ``[T, 2 * H * D]``, 1%
    of the channels (at least one) eight times as large."""
    x = _normal(g, T, 2, H, D)
    for j in range(2):
        big = torch.randperm(D, generator=g, device="cuda")[:max(1, D // 100)]
        x[:, j, :, big] *= 8.0
    x = x.to(DTYPES[dtype])
    return x[:, 0], x[:, 1]


def _lengths(case):
    """Tokens of each sequence, from the longest down to (1 - spread) of it."""
    B, L = case["B"], case["L"]
    return [int(round(L * (1.0 - case["spread"] * i / max(1, B - 1)))) for i in range(B)]


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g, kind = _gen(seed), case["kind"]
    if kind == "rope":
        T, Hq, Hk, D = case["T"], case["Hq"], case["Hk"], case["D"]
        # queries and keys are columns of one projection q|k|v
        x = _normal(g, T, (Hq + 2 * Hk) * D).to(DTYPES[case["dtype"]])
        return {"q": x[:, :Hq * D].unflatten(1, (Hq, D)),
                "k": x[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D)),
                "positions": case["first"] + torch.randperm(T, generator=g, device="cuda")}
    if kind == "cache":
        T, P = case["T"], case["P"]
        k, v = _rows(g, T, case["H"], case["D"], case["dtype"])
        pages = (T + P - 1) // P + 8
        if T <= 64:  # single tokens of as many sequences: a page each
            pages = max(pages, T)
            slots = torch.randperm(pages, generator=g, device="cuda")[:T] * P
            slots += torch.randint(0, P, (T,), generator=g, device="cuda")
        else:        # a run of tokens over pages in no order
            order = torch.randperm(pages, generator=g, device="cuda")
            at = torch.arange(T, device="cuda")
            slots = order[at // P] * P + at % P
        if case["pad"]:
            slots = torch.where(torch.rand(T, generator=g, device="cuda") < case["pad"], -1, slots)
        return {"k": k, "v": v, "slots": slots, "page_count": pages, "positions": torch.arange(T, device="cuda")}
    B, P = case["B"], case["P"]
    order = torch.randperm(B, generator=g, device="cuda").tolist()
    lens = [_lengths(case)[i] for i in order]
    width = max(1, (max(lens) + P - 1) // P)
    need = [(n + P - 1) // P for n in lens]
    pages = sum(need) + 4
    free = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32, device="cuda")
    at, slots = 0, []
    for b in range(B):
        mine = free[at:at + need[b]]
        table[b, :need[b]] = mine
        at += need[b]
        t = torch.arange(lens[b], device="cuda")
        slots.append(mine.long()[t // P] * P + t % P)
    slots = torch.cat(slots)
    k, v = _rows(g, slots.numel(), case["Hk"], case["D"], case["dtype"])
    q = (_normal(g, B, case["Hq"], case["D"]) * 1.5).to(DTYPES[case["q"]])
    return {"q": q, "k": k, "v": v, "slots": slots, "page_count": pages, "table": table,
            "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda"), "lens": lens}


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "kind": case["kind"], **t}
    if case["kind"] == "rope" or case.get("rope"):
        state["freq"], state["gain"] = _frequencies(case)
        state["freq"] = torch.tensor(state["freq"], dtype=torch.float64, device="cuda")
        if own:
            state["rotary"] = _rotary(case)
    if case["kind"] in ("cache", "attend"):
        heads = case["H"] if case["kind"] == "cache" else case["Hk"]
        if own:
            state["pool"] = _framework().KVPagePool(
                t["page_count"], heads, case["D"], page_size=case["P"], precision=case["prec"],
                dtype=DTYPES[case["dtype"]], device="cuda", int4_group_size=GROUP)
        else:
            state["pages"] = _pages(case, t["page_count"], heads)
    if case["kind"] == "attend":  # the cache is there before the step
        if own:
            state["pool"].write(t["k"], t["v"], t["slots"])
        else:
            _write(state, t["k"], t["v"], t["slots"])
        del state["k"], state["v"], state["slots"]
    return state


def _rotary(case):
    f = _framework()
    D = case["D"]
    scaling = None
    if case.get("scaling", "none") != "none":
        scaling = f.RotaryScaling(case["scaling"], case["factor"], original_positions=4096)
    return f.RotaryEmbedding(D, rotary_dim=case.get("R", D), base=case.get("base", 10000.0),
                             layout=case.get("layout", "half"), scaling=scaling, device="cuda")


def run(state):
    case, kind = state["case"], state["kind"]
    if kind == "rope":
        if own:
            q, k = state["rotary"](state["positions"], state["q"], state["k"],
                                   transpose=case["transpose"])
        else:
            q, k = _rotate(state, state["q"]), _rotate(state, state["k"])
        return {"q": q, "k": k}
    if kind == "cache":
        out = DTYPES[case["out"]]
        if own:
            if case["rope"]:
                state["pool"].write(state["k"], state["v"], state["slots"],
                                    rotary=state["rotary"], positions=state["positions"])
            else:
                state["pool"].write(state["k"], state["v"], state["slots"])
            k, v = state["pool"].read(state["slots"], dtype=out)
        else:
            _write(state, _rotate(state, state["k"]) if case["rope"] else state["k"], state["v"],
                   state["slots"])
            k, v = _read(state, state["slots"], out)
        return {"k": k, "v": v}
    if own:
        got = _framework().paged_attention(state["q"], state["pool"], state["table"], state["lengths"],
                                           window=case["window"] or None, return_lse=case["lse"])
    else:
        got = _attend(state)
    return {"out": got[0], "lse": got[1]} if case["lse"] else {"out": got}


# --------------------------------------------------------- the plain form
def _frequencies(case):
    """Angle per position of each pair, and the factor on the rotated values."""
    R, base = case.get("R", case["D"]), case.get("base", 10000.0)
    kind, s, known = case.get("scaling", "none"), case.get("factor", 1.0), 4096
    if kind == "ntk":
        base *= s ** (R / (R - 2))
    f = [base ** (-2.0 * i / R) for i in range(R // 2)]
    if kind == "linear":
        f = [x / s for x in f]
    if kind == "bands":
        kept = []
        for x in f:
            turns = known * x / (2.0 * math.pi)  # turns over the known context: 1 and 4 are the edges
            share = min(1.0, max(0.0, (turns - 1.0) / 3.0))
            kept.append(x * share + x / s * (1.0 - share))
        f = kept
    if kind == "yarn":
        at = [R * math.log(known / (n * 2.0 * math.pi)) / (2.0 * math.log(base)) for n in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), R - 1)
        hi = hi + 0.001 if hi == lo else hi
        mix = [min(1.0, max(0.0, (i - lo) / (hi - lo))) for i in range(R // 2)]
        f = [x / s * m + x * (1.0 - m) for x, m in zip(f, mix)]
    return f, (0.1 * math.log(s) + 1.0 if kind == "yarn" else 1.0)


def _rotate(state, x):
    case, R = state["case"], 2 * state["freq"].numel()
    angle = state["positions"].double()[:, None, None] * state["freq"]
    cos, sin = (angle.cos() * state["gain"]).float(), (angle.sin() * state["gain"]).float()
    if case.get("transpose"):
        sin = -sin
    y = x.float()
    if case.get("layout", "half") == "half":
        a, b = y[..., :R // 2], y[..., R // 2:R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, y[..., R:]), -1).to(x.dtype)


def _pages(case, pages, heads):
    """Page tensors ``[pages + 1, heads, P, ...]``; rows of no slot go to the last page."""
    P, D, T = case["P"], case["D"], DTYPES[case["dtype"]]
    row, kept = {"fp32": (D, T), "fp16": (D, torch.float16), "int8": (D, torch.int8),
                 "int4": (D // 2, torch.uint8)}[case["prec"]]
    scales = {"int8": 1, "int4": D // GROUP}.get(case["prec"])
    got = {}
    for name in ("k", "v"):
        got[name] = torch.zeros(pages + 1, heads, P, row, dtype=kept, device="cuda")
        got["s" + name] = (None if scales is None else
                           torch.zeros(pages + 1, heads, P, scales, dtype=T, device="cuda"))
    return got


def _encode(x, prec):
    """Rows as the cache stores them, and their scales in x's type."""
    if prec in ("fp32", "fp16"):
        return (x if prec == "fp32" else x.half()), None
    steps, lo = (127.0, -128) if prec == "int8" else (7.0, -8)
    y = x if prec == "int8" else x.unflatten(-1, (-1, GROUP))
    top = y.abs().amax(-1, keepdim=True)
    s = top / torch.full_like(top, steps)
    s = torch.where(s == 0, torch.ones_like(s), s)
    q = (y / s).round().clamp(lo, steps)
    if prec == "int8":
        return q.to(torch.int8), s
    q = (q + 8).to(torch.uint8).flatten(-2)
    return q[..., 0::2] * 16 + q[..., 1::2], s.squeeze(-1)


def _decode(x, s, prec):
    """Stored rows as fp32 values."""
    if prec in ("fp32", "fp16"):
        return x.float()
    if prec == "int8":
        return x.float() * s.float()
    q = torch.stack((x // 16, x % 16), -1).flatten(-2).float() - 8.0
    return (q.unflatten(-1, (-1, GROUP)) * s.float()[..., None]).flatten(-2)


def _place(state, slots):
    P, pages = state["case"]["P"], state["pages"]["k"].shape[0]
    at = torch.where(slots < 0, (pages - 1) * P, slots)
    return at // P, at % P


def _write(state, k, v, slots):
    page, row = _place(state, slots)
    for name, x in (("k", k), ("v", v)):
        q, s = _encode(x, state["case"]["prec"])
        state["pages"][name][page, :, row] = q
        if s is not None:
            state["pages"]["s" + name][page, :, row] = s


def _read(state, slots, dtype):
    page, row = _place(state, slots)
    there = (slots >= 0)[:, None, None]
    got = []
    for name in ("k", "v"):
        s = state["pages"]["s" + name]
        x = _decode(state["pages"][name][page, :, row], None if s is None else s[page, :, row],
                    state["case"]["prec"])
        got.append(torch.where(there, x, torch.zeros_like(x)).to(dtype))
    return got


def _attend(state):
    case, pages, table = state["case"], state["pages"], state["table"].long()
    B, Hq, Hk, D = case["B"], case["Hq"], case["Hk"], case["D"]
    rows = []
    for name in ("k", "v"):  # [B, heads, positions, D]
        s = pages["s" + name]
        x = _decode(pages[name][table], None if s is None else s[table], case["prec"])
        rows.append(x.transpose(1, 2).reshape(B, Hk, -1, D))
    k, v = rows
    q = state["q"].float().reshape(B, Hk, Hq // Hk, D)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(D)
    at = torch.arange(k.shape[2], device="cuda")
    n = state["lengths"].long()[:, None]
    seen = at < n
    if case["window"]:
        seen = seen & (at >= n - case["window"])
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), torch.zeros_like(top), top)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen[:, None, :, None], v, torch.zeros_like(v))
    out = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.reshape(B, Hq, D).to(state["q"].dtype)
    if not case["lse"]:
        return out
    return out, (top + total.log()).reshape(B, Hq)


# --------------------------------------------------------------------- work
def _row_bytes(case, D):
    es = SIZE[case["dtype"]]
    return {"fp32": D * es, "fp16": 2 * D, "int8": D + es,
            "int4": D // 2 + D // GROUP * es}[case["prec"]]


def work(case):
    kind, D = case["kind"], case["D"]
    if kind == "rope":
        rows = case["T"] * (case["Hq"] + case["Hk"])
        return {"bytes": 2 * rows * D * SIZE[case["dtype"]] + 8 * case["T"],
                "flops": 3 * rows * case["R"]}
    if kind == "cache":
        rows = 2 * case["T"] * case["H"]
        stored = (1.0 - case["pad"]) * rows * _row_bytes(case, D)
        return {"bytes": (1.0 - case["pad"]) * rows * D * SIZE[case["dtype"]] + 2 * stored
                + rows * D * SIZE[case["out"]] + 16 * case["T"], "flops": 0}
    lens = [min(n, case["window"] or n) for n in _lengths(case)]
    q = case["B"] * case["Hq"] * D * SIZE[case["q"]]
    return {"bytes": 2 * sum(lens) * case["Hk"] * _row_bytes(case, D) + 2 * q
            + 4 * sum(-(-n // case["P"]) for n in lens),
            "flops": 4 * case["Hq"] * D * sum(lens)}


# ------------------------------------------------------- the same in 64 bits
def _exact_angles(case):
    """(angle per position of each pair, factor) by the same published rules, over tensors."""
    R, base, s = case.get("R", case["D"]), case.get("base", 10000.0), case.get("factor", 1.0)
    kind, i = case.get("scaling", "none"), torch.arange(R // 2, dtype=torch.float64)
    if kind == "ntk":
        base = base * math.pow(s, R / (R - 2.0))
    f = torch.exp(i * (-2.0 / R) * math.log(base))
    if kind == "linear":
        return f / s, 1.0
    if kind == "bands":
        wave = 2.0 * math.pi / f
        middle = (4096.0 / wave - 1.0) / (4.0 - 1.0)
        f = torch.where(wave > 4096.0, f / s, torch.where(wave < 1024.0, f, (1 - middle) * f / s + middle * f))
        return f, 1.0
    if kind == "yarn":
        def pair(turns):
            return R * math.log(4096.0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        first, last = max(float(math.floor(pair(32.0))), 0.0), min(float(math.ceil(pair(1.0))), R - 1.0)
        if first == last:
            last += 0.001
        slow = ((i - first) / (last - first)).clamp(0.0, 1.0)
        return slow * (f / s) + (1.0 - slow) * f, 0.1 * math.log(s) + 1.0
    return f, 1.0


def _exact_rotate(case, x, positions):
    f, gain = _exact_angles(case)
    angle = torch.outer(positions.double(), f.to(x.device))[:, None, :]
    turn = torch.polar(torch.full_like(angle, gain), -angle if case.get("transpose") else angle)
    R, y = case.get("R", case["D"]), x.double().clone()
    if case.get("layout", "half") == "half":
        z = torch.complex(y[..., :R // 2].contiguous(), y[..., R // 2:R].contiguous()) * turn
        y[..., :R // 2], y[..., R // 2:R] = z.real, z.imag
    else:
        z = torch.complex(y[..., 0:R:2].contiguous(), y[..., 1:R:2].contiguous()) * turn
        y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
    return y


def _exact_held(x, prec):
    """The values a cache of ``prec`` holds for the rows x, in 64 bits. Scales and
    quotients are rounded to x's type, as the format defines them."""
    T = x.dtype
    if prec == "fp32":
        return x.double()
    if prec == "fp16":
        return x.half().double()
    steps = 127.0 if prec == "int8" else 7.0
    y = x.double() if prec == "int8" else x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    # (float32 between 64 bits and a 16-bit type: the format's own roundings)
    s = (y.abs().max(-1, keepdim=True).values / steps).float().to(T).double()
    s = s.masked_fill(s == 0.0, 1.0)
    q = torch.round((y / s).float().to(T).double()).clamp(-steps - 1.0, steps)
    return (q * s).reshape(x.shape)


def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "rope":
        return {"q": _exact_rotate(case, t["q"], t["positions"]),
                "k": _exact_rotate(case, t["k"], t["positions"])}
    if kind == "cache":
        k = _exact_rotate(case, t["k"], t["positions"]) if case["rope"] else t["k"]
        there = (t["slots"] >= 0)[:, None, None]
        got = []
        for x in (k, t["v"]):
            x = x if x.dtype == torch.float64 else _exact_held(x, case["prec"])
            got.append(torch.where(there, x, torch.zeros((), dtype=torch.float64, device="cuda")))
        return {"k": got[0], "v": got[1]}
    Hq, Hk, D = case["Hq"], case["Hk"], case["D"]
    out = torch.zeros(case["B"], Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((case["B"], Hq), float("-inf"), dtype=torch.float64, device="cuda")
    at = 0
    for b, n in enumerate(t["lens"]):
        lo, hi = at + max(0, n - (case["window"] or n)), at + n
        at += n
        if lo == hi:
            continue
        k, v = _exact_held(t["k"][lo:hi], case["prec"]), _exact_held(t["v"][lo:hi], case["prec"])
        for h in range(Hk):
            rows = slice(h * (Hq // Hk), (h + 1) * (Hq // Hk))
            s = t["q"][b, rows].double() @ k[:, h].t().contiguous() / math.sqrt(D)
            lse[b, rows] = torch.logsumexp(s, -1)
            out[b, rows] = torch.softmax(s, -1) @ v[:, h].contiguous()
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}

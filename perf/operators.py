"""The operators of serving many sequences over one paged key/value cache, timed: rotary tables and rotation, the cache
written (quantized) and read back, and the attention of one new token a sequence.

With ``own`` false ``run`` computes them from elementary torch operations; with ``own`` true it calls the framework's
operators (``edgelm_amd.elmh.Context``, device pointers).

Kinds of case:
  table    cos and sin of the rotary angles, scaled for long contexts    rope_table_dev
  rope     heads rotated at given positions (half or interleaved pairs)  rope_dev
  store    new tokens' keys (rotated) and values written into the pages of their sequences, quantized where the cache is,
           and read back as the values that the cache then holds         paged_append_dev, paged_read_dev
  read     whole sequences read back from their pages                    paged_read_dev
  attend   one new token a sequence over its pages                       paged_attention_dev

The cache: keys and values in pools [page][kv head][slot][head_dim] of f32, f16, bf16, int8 (``q8``: one f32 scale per row,
[page][kv head][slot]) or 4-bit levels (``q4``: one f32 scale per 32 values, [page][kv head][group][slot]); a sequence's
position p is slot p % page_size of page table[sequence][p // page_size].
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
THETA = 10000.0


def listed():
    return [
        # the smallest decode step: one short chat on the 135M shape, the f32 cache that the framework has elsewhere
        dict(name="attend_chat_f32", kind="attend", dtype="f32", B=1, heads=9, kv=3, hd=64, page=16, top=137, lens="top", rope="half"),
        # one very long document: few (sequence, head) pairs, so the cache's length has to be split
        dict(name="attend_long_bf16", kind="attend", dtype="bf16", B=1, heads=32, kv=8, hd=128, page=64, top=100003, lens="top", rope="half"),
        # an ordinary serving batch of the 8B shape, sequences of every length, padding rows of length zero among them
        dict(name="attend_batch_q8", kind="attend", dtype="q8", B=32, heads=32, kv=8, hd=128, page=16, top=4096, lens="ragged", rope="half"),
        # a full batch with long contexts on a 4-bit cache: the largest
        dict(name="attend_large_q4", kind="attend", dtype="q4", B=64, heads=32, kv=8, hd=128, page=32, top=16384, lens="long", rope="none"),
        # a decode step's keys and values for a batch, some rows padding
        dict(name="store_step_q8", kind="store", dtype="q8", B=48, kv=8, hd=128, page=16, past=1500, new=1, rope="half", rot=128),
        # ragged prompts of a batch written at once, keys rotated over part of the head in interleaved pairs
        dict(name="store_prompt_q4", kind="store", dtype="q4", B=5, kv=8, hd=128, page=16, past=0, new=2111, rope="inter", rot=64),
        # a short f16 sequence read back into a contiguous cache
        dict(name="read_short_f16", kind="read", dtype="f16", B=1, kv=3, hd=64, page=16, top=131, lens="top", heads_first=True),
        # swapping a batch out: whole int8 sequences
        dict(name="read_batch_q8", kind="read", dtype="q8", B=12, kv=8, hd=128, page=32, top=6000, lens="ragged", heads_first=False),
        # a decode step's queries of a batch, each at its own position
        dict(name="rope_step", kind="rope", T=24, heads=32, hd=128, rot=128, rope="half", ctx=4096),
        # a long prompt's queries, a quarter of each head rotated in interleaved pairs
        dict(name="rope_prompt", kind="rope", T=7777, heads=32, hd=96, rot=24, rope="inter", ctx=8192),
        # tables of an ordinary context
        dict(name="table_linear", kind="table", n=4096, pos0=0, rot=64, scaling="linear", factor=2.0, orig=2048),
        # tables of a context stretched to a million positions
        dict(name="table_yarn", kind="table", n=1 << 20, pos0=0, rot=128, scaling="yarn", factor=32.0, orig=32768),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the ranges above: every cache type, head sizes 32 to 256, 1 to 8 kv heads of 1 to 8 queries, pages of 16 to
    128, 1 to 64 sequences of one to 131072 positions."""
    dearest = max(work(c)["bytes"] for c in listed())
    while True:
        kind = rng.choice(["attend", "attend", "attend", "store", "store", "read", "rope", "table"])
        dtype = rng.choice(["f32", "f16", "bf16", "q8", "q4"])
        hd = rng.choice([32, 64, 64, 96, 128, 128, 192, 256])
        kv = rng.choice([1, 2, 3, 4, 5, 8])
        page = rng.choice([16, 32, 64, 128])
        B = _log_int(rng, 1, 64)
        c = dict(kind=kind, dtype=dtype, B=B, kv=kv, hd=hd, page=page)
        if kind == "attend":
            c.update(heads=kv * rng.choice([1, 2, 3, 4, 7, 8]), top=_log_int(rng, 1, 131072), lens=rng.choice(["top", "ragged", "ragged", "long"]),
                     rope=rng.choice(["none", "half", "inter"]))
            if B * c["top"] * kv * hd > 64 * 16384 * 8 * 128:  # what the plain form lays out
                continue
        elif kind == "store":
            step = rng.random() < 0.5
            c.update(past=_log_int(rng, 1, 20000) if step else 0, new=1 if step else _log_int(rng, 2, 4096), rope=rng.choice(["none", "half", "inter"]),
                     rot=2 * rng.randint(4, hd // 2))
        elif kind == "read":
            c.update(top=_log_int(rng, 1, 16384), lens=rng.choice(["top", "ragged"]), heads_first=rng.random() < 0.5)
            if B * c["top"] > 300000:
                continue
        elif kind == "rope":
            c = dict(kind=kind, T=_log_int(rng, 1, 16384), heads=rng.choice([1, 3, 8, 9, 32]), hd=hd, rot=2 * rng.randint(1, hd // 2),
                     rope=rng.choice(["half", "inter"]), ctx=_log_int(rng, 1000, 131072))
        else:
            c = dict(kind=kind, n=_log_int(rng, 1, 1 << 19), pos0=rng.choice([0, _log_int(rng, 1, 1 << 19)]), rot=2 * rng.randint(4, 64),
                     scaling=rng.choice(["none", "linear", "bands", "yarn"]), factor=rng.uniform(1.5, 40.0), orig=_log_int(rng, 1024, 32768))
        if work(c)["bytes"] <= min(dearest, 2.2e8 if kind == "store" else 2e9):
            return c


# ------------------------------------------------------------------ a case's lengths, positions and sizes

def _lens(c):
    """Lengths of the case's sequences: `top` all alike; `ragged` spread from zero to top, the first at it; `long` in its upper
    half."""
    rng = random.Random(c["B"] * 1000003 + c["top"])
    lens = [c["top"]]
    for i in range(1, c["B"]):
        low = {"top": c["top"], "ragged": 0, "long": c["top"] // 2}[c["lens"]]
        n = rng.randint(low, c["top"])
        lens.append(0 if c["lens"] == "ragged" and i % 11 == 5 else n)
    return lens


def _tokens(c):
    """(sequence, position) of each token of a store or read case; a negative position is a padding row."""
    if c["kind"] == "read":
        return [(b, p) for b, n in enumerate(_lens(c)) for p in range(n)]
    rng = random.Random(c["B"] * 1000003 + c["new"] + c["past"])
    if c["new"] == 1:
        at = [rng.randint(c["past"] // 2, c["past"]) for _ in range(c["B"])]
        return [(b, -1 if b % 13 == 7 else p) for b, p in enumerate(at)]
    return [(b, p) for b in range(c["B"]) for p in range(c["new"] if b == 0 else rng.randint(c["new"] // 3, c["new"]))]


def _row_bytes(c):
    """Bytes of one cached row of head_dim values with its scales."""
    return {"f32": 4 * c["hd"], "f16": 2 * c["hd"], "bf16": 2 * c["hd"], "q8": c["hd"] + 4, "q4": c["hd"] // 2 + c["hd"] // 8}[c["dtype"]]


def work(case):
    c = case
    if c["kind"] == "table":
        return {"bytes": 4.0 * c["n"] * c["rot"], "flops": 20.0 * c["n"] * c["rot"]}
    if c["kind"] == "rope":  # x in, y out, the positions and the rows of the tables that they name
        return {"bytes": 4.0 * c["T"] * (2 * c["heads"] * c["hd"] + c["rot"] + 1), "flops": 3.0 * c["T"] * c["heads"] * c["rot"]}
    if c["kind"] in ("store", "read"):
        n = sum(p >= 0 for _, p in _tokens(c))
        f32, held = 8.0 * n * c["kv"] * c["hd"], 2.0 * n * c["kv"] * _row_bytes(c)
        if c["kind"] == "read":
            return {"bytes": held + f32, "flops": n * c["kv"] * c["hd"] * 2.0}
        turned = c["rot"] if c["rope"] != "none" else 0
        return {"bytes": 2 * (f32 + held) + 4.0 * n * turned, "flops": n * c["kv"] * (c["hd"] * 12.0 + 3.0 * turned)}
    seen = sum(_lens(c))
    return {"bytes": 2.0 * seen * c["kv"] * _row_bytes(c) + 8.0 * c["B"] * c["heads"] * c["hd"], "flops": 4.0 * seen * c["heads"] * c["hd"]}


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) % (1 << 62))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cache(c, g, lens, filled):
    """Pools, scales and a table of shuffled pages for sequences of these lengths. With `filled` every position holds a row
    and the slots behind the last one hold what memory may hold, NaN; else the pools are as a program clears them."""
    pages = [-(-n // c["page"]) for n in lens]
    most, total = max(1, max(pages)), max(1, sum(pages)) + 1
    order = torch.randperm(total, generator=g, device=DEV)[:sum(pages)].to(torch.int32)
    table = torch.full((len(lens), most), -1, dtype=torch.int32, device=DEV)
    owner = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(pages, device=DEV))
    first = torch.cumsum(torch.tensor([0] + pages[:-1], device=DEV), 0)
    nth = torch.arange(sum(pages), device=DEV) - first[owner]
    table[owner, nth] = order
    shape = (total, c["kv"], c["page"], c["hd"])
    t = {"table": table}
    behind = torch.zeros(total, c["page"], dtype=torch.bool, device=DEV)
    if filled:
        where = nth[:, None] * c["page"] + torch.arange(c["page"], device=DEV)
        behind[order.long()] = where >= torch.tensor(lens, device=DEV)[owner][:, None]
    if c["dtype"] in ("q8", "q4"):
        groups = 1 if c["dtype"] == "q8" else c["hd"] // 32
        for n in ("k", "v"):
            if c["dtype"] == "q8":
                t[n] = torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8) if filled else torch.zeros(shape, dtype=torch.int8, device=DEV)
                spread = 0.035
            else:
                half = shape[:3] + (c["hd"] // 2,)
                t[n] = torch.randint(0, 256, half, generator=g, device=DEV, dtype=torch.uint8) if filled else torch.zeros(half, dtype=torch.uint8, device=DEV)
                spread = 0.4
            s = torch.zeros(total, c["kv"], groups, c["page"], device=DEV)
            if filled:
                s = (torch.rand(s.shape, generator=g, device=DEV) + 0.5) * (spread / 2)
                if c["dtype"] == "q4":  # a group's scale has the sign of its largest value
                    s = s * (torch.randint(0, 2, s.shape, generator=g, device=DEV) * 2 - 1)
                s.masked_fill_(behind[:, None, None, :], math.nan)
            t[n + "s"] = s
    else:
        to = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[c["dtype"]]
        for n in ("k", "v"):
            t[n] = torch.zeros(shape, dtype=to, device=DEV)
            if filled:
                t[n].normal_(generator=g)
                t[n].masked_fill_(behind[:, None, :, None], math.nan)
    return t


def _tables(n, rot):
    inv = torch.tensor(THETA, dtype=torch.float64, device=DEV) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cos(a).float(), torch.sin(a).float()


def _inputs(c, seed):
    g = _generator(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    if c["kind"] == "table":  # the base differs from seed to seed: a program computes tables once a model
        return {"theta": 10000.0 * (1 + int(seed) % 997)}
    if c["kind"] == "rope":
        t = {"x": normal(c["T"], c["heads"] * c["hd"]), "pos": torch.randint(0, c["ctx"], (c["T"],), generator=g, device=DEV, dtype=torch.int32)}
        t["cos"], t["sin"] = _tables(c["ctx"], c["rot"])
        return t
    if c["kind"] == "attend":
        lens = _lens(c)
        t = _cache(c, g, lens, True)
        t["lens"], t["q"] = _ints(lens), normal(c["B"], c["heads"] * c["hd"])
        if c["rope"] != "none":
            t["cos"], t["sin"] = _tables(c["top"], c["hd"])
        return t
    tok = _tokens(c)
    lens = [0] * c["B"]
    for b, p in tok:
        lens[b] = max(lens[b], p + 1)
    t = _cache(c, g, lens, c["kind"] == "read")
    t["seq"], t["pos"] = _ints([b for b, _ in tok]), _ints([p for _, p in tok])
    if c["kind"] == "store":
        t["nk"], t["nv"] = normal(len(tok), c["kv"], c["hd"]), normal(len(tok), c["kv"], c["hd"])
        if c["rope"] != "none":
            t["cos"], t["sin"] = _tables(max(lens), c["rot"])
    return t


_context = None


def _elmh():
    """The framework's module and the process's context: a program makes one and keeps it."""
    global _context
    from edgelm_amd import elmh as E
    if _context is None:
        _context = E.Context(0)
    return E, _context


def _ptr(t, n):
    return t[n].data_ptr() if n in t else None


def prepare(case, seed):
    c = case
    t = _inputs(c, seed)
    s = {"c": c, "t": t}
    if c["kind"] == "table":
        s["cos"], s["sin"] = (torch.zeros(c["n"], c["rot"] // 2, device=DEV) for _ in range(2))
    elif c["kind"] == "rope":
        s["y"] = torch.zeros_like(t["x"])
    elif c["kind"] == "attend":
        s["out"] = torch.zeros_like(t["q"])
    else:
        n = t["pos"].numel()
        shape = (c["kv"], n, c["hd"]) if c.get("heads_first") else (n, c["kv"], c["hd"])
        s["k"], s["v"] = torch.zeros(shape, device=DEV), torch.zeros(shape, device=DEV)
    if own:  # the descriptors that a program keeps: where the pools and the rotary tables are
        E, ctx = _elmh()
        s["ctx"] = ctx
        if "table" in t:
            s["pages"] = E.KVPages(E.KV_DTYPES[c["dtype"]], c["kv"], c["hd"], c["page"], t["k"].shape[0], t["k"].data_ptr(), t["v"].data_ptr(),
                                   _ptr(t, "ks"), _ptr(t, "vs"))
        if "cos" in t:
            s["rope"] = E.Rope(t["cos"].data_ptr(), t["sin"].data_ptr(), t["cos"].shape[0], 2 * t["cos"].shape[1], c["rope"] == "inter")
        if c["kind"] == "table" and c["scaling"] != "none":
            kind = {"linear": E.ROPE_LINEAR, "bands": E.ROPE_BANDS, "yarn": E.ROPE_YARN}[c["scaling"]]
            s["scaling"] = E.RopeScaling(kind, c["factor"], c["orig"], *_betas(c), _magnitude(c))
    return s


def _betas(c):
    """(low, high): turns over the original context at which a pair counts as slow, and as fast."""
    return (1.0, 4.0) if c["scaling"] == "bands" else (1.0, 32.0)


def _magnitude(c):
    return 0.1 * math.log(c["factor"]) + 1.0 if c["scaling"] == "yarn" else 1.0


# ------------------------------------------------------------------ the framework's operators

def _run_own(s):
    c, t, ctx = s["c"], s["t"], s["ctx"]
    rope = s.get("rope")
    if c["kind"] == "table":
        ctx.rope_table_dev(s["cos"].data_ptr(), s["sin"].data_ptr(), c["pos0"], c["n"], c["rot"], t["theta"], s.get("scaling"))
        return [s["cos"], s["sin"]]
    if c["kind"] == "rope":
        ctx.rope_dev(t["x"].data_ptr(), s["y"].data_ptr(), c["T"], c["heads"], c["hd"], rope, t["pos"].data_ptr())
        return s["y"]
    most = t["table"].shape[1]
    if c["kind"] == "attend":
        ctx.paged_attention_dev(t["q"].data_ptr(), s["out"].data_ptr(), c["heads"], s["pages"], t["table"].data_ptr(), c["B"], most,
                                t["lens"].data_ptr(), c["top"], rope)
        return s["out"]
    n = t["pos"].numel()
    if c["kind"] == "store":
        ctx.paged_append_dev(t["nk"].data_ptr(), t["nv"].data_ptr(), n, s["pages"], t["table"].data_ptr(), c["B"], most, t["pos"].data_ptr(),
                             t["seq"].data_ptr(), rope)
    row, head = (c["hd"], n * c["hd"]) if c.get("heads_first") else (c["kv"] * c["hd"], c["hd"])
    ctx.paged_read_dev(s["k"].data_ptr(), s["v"].data_ptr(), n, s["pages"], t["table"].data_ptr(), c["B"], most, t["pos"].data_ptr(),
                       t["seq"].data_ptr(), row, head)
    return [s["k"], s["v"]]


# ------------------------------------------------------------------ the same in elementary operations

def _rotate(x, cos, sin, inter):
    """x [..., hd] rotated over its first 2 * cos.shape[-1] values: pairs (i, i + half), or (2i, 2i + 1)."""
    rot = 2 * cos.shape[-1]
    turned = x[..., :rot]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if inter else (turned[..., :rot // 2], turned[..., rot // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _levels(bytes4, keys):
    """The levels -8 .. 7 of packed 4-bit rows, in the order of their values. A byte holds two neighbouring values, the first
    in its low nibble; its place in the row: of a key, [c][j][b] for values 32 j + 8 c + 2 b; of a value row, [i][j] for
    values 32 j + 2 i."""
    lead, half = bytes4.shape[:-1], bytes4.shape[-1]
    groups = half // 16
    if keys:
        b = bytes4.view(*lead, 4, groups, 4).transpose(-3, -2)
    else:
        b = bytes4.view(*lead, 16, groups).transpose(-2, -1)
    b = b.reshape(*lead, half)
    return torch.stack([b & 15, b >> 4], -1).reshape(*lead, 2 * half).to(torch.float32) - 8


def _values(c, data, scales, keys):
    """Rows of the cache in 32 bits: data [..., hd or hd / 2], scales [..., groups]."""
    if c["dtype"] == "q8":
        return data.float() * scales
    if c["dtype"] == "q4":
        v = _levels(data, keys)
        return (v.view(*v.shape[:-1], -1, 32) * scales[..., None]).view(v.shape)
    return data.float()


def _pack(levels, keys):
    """_levels' inverse."""
    lead, hd = levels.shape[:-1], levels.shape[-1]
    u = (levels + 8).to(torch.uint8).view(*lead, hd // 2, 2)
    b = u[..., 0] | (u[..., 1] << 4)
    if keys:
        return b.view(*lead, hd // 32, 4, 4).transpose(-3, -2).reshape(*lead, hd // 2)
    return b.view(*lead, hd // 32, 16).transpose(-2, -1).reshape(*lead, hd // 2)


def _quantized(c, x):
    """(levels, scales) of rows x [..., hd]: q8 the largest magnitude / 127 a row; q4 the first value of largest magnitude
    / -8 per 32; levels to the nearest, halves away from zero."""
    if c["dtype"] == "q8":
        groups, lo, hi = x[..., None, :], -127.0, 127.0
        s = groups.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=x.device)
    else:
        groups, lo, hi = x.view(*x.shape[:-1], -1, 32), -8.0, 7.0
        s = groups.gather(-1, groups.abs().argmax(-1, keepdim=True)) / -8.0
    r = groups / torch.where(s == 0, torch.ones_like(s), s)
    q = (torch.sign(r) * torch.floor(r.abs() + 0.5)).clamp(lo, hi)
    return q.reshape(x.shape), s[..., 0]


def _slots(c, t):
    """(rows that are no padding, their pages, their slots)."""
    live = t["pos"] >= 0
    pos = t["pos"].clamp_min(0).long()
    return live, t["table"][t["seq"].long(), pos // c["page"]].clamp_min(0).long(), pos % c["page"]


def _plain_read(c, t, k_out, v_out):
    live, page, slot = _slots(c, t)
    for out, n in ((k_out, "k"), (v_out, "v")):
        scales = t[n + "s"][page, :, :, slot] if n + "s" in t else None
        rows = _values(c, t[n][page, :, slot], scales, n == "k")
        rows = torch.where(live[:, None, None], rows, torch.zeros_like(rows))
        out.copy_(rows.transpose(0, 1) if c.get("heads_first") else rows)
    return [k_out, v_out]


def _plain_store(c, t):
    live, page, slot = _slots(c, t)
    page, slot = page[live], slot[live]
    k = t["nk"][live]
    if "cos" in t:
        at = t["pos"][live].long()
        k = _rotate(k, t["cos"][at][:, None], t["sin"][at][:, None], c["rope"] == "inter")
    for x, n in ((k, "k"), (t["nv"][live], "v")):
        if n + "s" in t:
            q, sc = _quantized(c, x)
            t[n + "s"][page, :, :, slot] = sc
            x = _pack(q, n == "k") if c["dtype"] == "q4" else q
        t[n][page, :, slot] = x.to(t[n].dtype)


def _plain_attend(c, t, out):
    B, kv, hd, L = c["B"], c["kv"], c["hd"], t["table"].shape[1] * c["page"]
    at = t["table"].clamp_min(0).long()
    live = torch.arange(L, device=DEV) < t["lens"][:, None]
    q = t["q"].view(B, c["heads"], hd)
    if "cos" in t:
        p = (t["lens"] - 1).clamp_min(0).long()
        q = _rotate(q, t["cos"][p][:, None], t["sin"][p][:, None], c["rope"] == "inter")

    def rows(n):
        scales = t[n + "s"][at].transpose(-2, -1) if n + "s" in t else None
        r = _values(c, t[n][at], scales, n == "k").transpose(1, 2).reshape(B, kv, L, hd)
        return r.masked_fill_(~live[:, None, :, None], 0.0)

    score = torch.matmul(q.reshape(B, kv, -1, hd), rows("k").transpose(-2, -1)) / math.sqrt(hd)
    score.masked_fill_(~live[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p, rows("v")) / torch.where(total == 0, torch.ones_like(total), total)
    return out.copy_(y.reshape(B, -1))


def _frequencies(c, theta, dtype=torch.float64):
    """Angle per position of each pair, scaled for a longer context than the original one."""
    rot = c["rot"]
    i = torch.arange(rot // 2, dtype=dtype, device=DEV)
    f = torch.full_like(i, theta) ** (-2.0 * i / rot)
    low, high = _betas(c)
    if c["scaling"] == "linear":
        return f / c["factor"]
    if c["scaling"] == "bands":  # by the turns that a pair makes over the original context
        turns = c["orig"] * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return f * (keep + (1 - keep) / c["factor"])
    if c["scaling"] == "yarn":  # by the pair's index, between those that make `high` and `low` turns
        def pair(turns):
            return rot * math.log(c["orig"] / (2 * math.pi * turns)) / (2 * math.log(theta))
        lo, hi = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f * ((1 - ramp) + ramp / c["factor"])
    return f


def _plain_table(c, t, cos, sin):
    # angles in 64 bits: at position 10^6 an angle in 32 bits is off by 0.03
    a = torch.arange(c["pos0"], c["pos0"] + c["n"], dtype=torch.float64, device=DEV)[:, None] * _frequencies(c, t["theta"])
    cos.copy_(torch.cos(a) * _magnitude(c))
    sin.copy_(torch.sin(a) * _magnitude(c))
    return [cos, sin]


def run(state):
    s = state
    c, t = s["c"], s["t"]
    if own:
        return _run_own(s)
    if c["kind"] == "table":
        return _plain_table(c, t, s["cos"], s["sin"])
    if c["kind"] == "rope":
        p = t["pos"].long()
        y = _rotate(t["x"].view(c["T"], c["heads"], c["hd"]), t["cos"][p][:, None], t["sin"][p][:, None], c["rope"] == "inter")
        return s["y"].copy_(y.view(c["T"], -1))
    if c["kind"] == "attend":
        return _plain_attend(c, t, s["out"])
    if c["kind"] == "store":
        _plain_store(c, t)
    return _plain_read(c, t, s["k"], s["v"])


# ------------------------------------------------------------------ the same in 64 bits

def _turn64(x, cos, sin, inter):
    """x [n, heads, hd] as complex numbers times cos + i sin."""
    x, half = x.double(), cos.shape[-1]
    w = torch.complex(cos.double(), sin.double())[:, None]
    y = x.clone()
    if inter:
        z = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:-1], half, 2).contiguous()) * w
        y[..., :2 * half] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * w
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def _nibbles(hd, keys):
    """For each value of a row: the byte that holds it."""
    d = np.arange(hd)
    j, r = d // 32, d % 32
    at = (r // 8) * (hd // 8) + j * 4 + (r % 8) // 2 if keys else (r // 2) * (hd // 32) + j
    return torch.from_numpy(at).to(DEV)


def _rows64(c, t, n, page, slot):
    """Rows [tokens, kv, hd] of the cache at these pages and slots."""
    data = t[n][page, :, slot]
    if c["dtype"] in ("f32", "f16", "bf16"):
        return data.double()
    scale = t[n + "s"][page, :, :, slot].double()
    if c["dtype"] == "q8":
        return data.double() * scale
    at = _nibbles(c["hd"], n == "k")
    odd = torch.arange(c["hd"], device=DEV) % 2 == 1
    byte = data[..., at].int()
    return (torch.where(odd, byte >> 4, byte & 15).double() - 8) * scale.repeat_interleave(32, -1)


def _round32(x):
    """A 64-bit result rounded to 32 bits: a single-precision product, difference or quotient of 32-bit numbers."""
    return x.float().double()


def _held64(c, x):
    """The values that the cache holds of rows x (32-bit numbers in 64 bits). The scale and the quotients are single-precision
    ones: their rounding is part of the format."""
    if c["dtype"] in ("f32", "f16", "bf16"):
        return x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[c["dtype"]]).double()
    n, kv, hd = x.shape
    width = hd if c["dtype"] == "q8" else 32
    g = x.reshape(-1, width)
    mag = g.abs()
    if c["dtype"] == "q8":
        s, lo, hi = _round32(mag.max(1, keepdim=True).values / 127), -127, 127
    else:
        first = torch.where(mag == mag.max(1, keepdim=True).values, torch.arange(width, device=DEV), width).min(1, keepdim=True).values
        s, lo, hi = _round32(g.gather(1, first) / -8), -8, 7
    r = _round32(g / torch.where(s == 0, 1.0, s))
    level = torch.where(r < 0, -torch.floor(_round32(-r + 0.5)), torch.floor(_round32(r + 0.5))).clamp(lo, hi)
    return (level * s).reshape(n, kv, hd)


def _exact_store(c, t):
    k = t["nk"].double()
    live = t["pos"] >= 0
    if "cos" in t:  # the key is held in 32 bits before it is quantized: each product and difference is a single-precision one
        p = t["pos"].clamp_min(0).long()
        co, si = t["cos"].double()[p][:, None], t["sin"].double()[p][:, None]
        half = co.shape[-1]
        first = torch.arange(half, device=DEV) * (2 if c["rope"] == "inter" else 1)
        second = first + (1 if c["rope"] == "inter" else half)
        a, b = k[..., first].clone(), k[..., second].clone()
        k[..., first] = _round32(_round32(a * co) - _round32(b * si))
        k[..., second] = _round32(_round32(b * co) + _round32(a * si))
    return [torch.where(live[:, None, None], _held64(c, x), 0.0) for x in (k, t["nv"].double())]


def exact(case, seed):
    c = case
    t = _inputs(c, seed)
    if c["kind"] == "table":
        rot, th = c["rot"], t["theta"]
        f = []
        for i in range(rot // 2):
            w = math.exp(-2.0 * i / rot * math.log(th))
            if c["scaling"] == "linear":
                w /= c["factor"]
            elif c["scaling"] == "bands":
                wavelength = 2 * math.pi / w
                if wavelength > c["orig"] / 1.0:
                    w /= c["factor"]
                elif wavelength >= c["orig"] / 4.0:
                    smooth = (c["orig"] / wavelength - 1.0) / (4.0 - 1.0)
                    w = (1 - smooth) * w / c["factor"] + smooth * w
            elif c["scaling"] == "yarn":
                lo, hi = (rot / 2 * math.log(c["orig"] / (b * 2 * math.pi)) / math.log(th) for b in (32.0, 1.0))
                lo, hi = max(0, math.floor(lo)), min(rot - 1, math.ceil(hi))
                r = min(1.0, max(0.0, (i - lo) / (hi - lo if hi > lo else 0.001)))
                w = w / c["factor"] * r + w * (1 - r)
            f.append(w)
        m = 0.1 * math.log(c["factor"]) + 1.0 if c["scaling"] == "yarn" else 1.0
        a = torch.outer(torch.arange(c["pos0"], c["pos0"] + c["n"], device=DEV, dtype=torch.float64), torch.tensor(f, device=DEV, dtype=torch.float64))
        z = torch.polar(torch.full_like(a, m), a)
        return [z.real.contiguous(), z.imag.contiguous()]
    if c["kind"] == "rope":
        p = t["pos"].long()
        return _turn64(t["x"].view(c["T"], c["heads"], c["hd"]), t["cos"][p], t["sin"][p], c["rope"] == "inter").view(c["T"], -1)
    if c["kind"] == "store":
        return _exact_store(c, t)
    if c["kind"] == "read":
        p = t["pos"].long()
        page = t["table"][t["seq"].long(), p // c["page"]].long()
        rows = [_rows64(c, t, n, page, p % c["page"]) for n in ("k", "v")]
        return [r.transpose(0, 1).contiguous() if c["heads_first"] else r for r in rows]
    q = t["q"].view(c["B"], c["heads"], c["hd"]).double()
    out = torch.zeros_like(q)
    grp = c["heads"] // c["kv"]
    for b, n in enumerate(_lens(c)):
        if not n:
            continue
        qb = q[b:b + 1]
        if "cos" in t:
            qb = _turn64(qb, t["cos"][n - 1:n], t["sin"][n - 1:n], c["rope"] == "inter")
        p = torch.arange(n, device=DEV)
        page = t["table"][b].long()[p // c["page"]]
        k, v = (_rows64(c, t, m, page, p % c["page"]) for m in ("k", "v"))
        for h in range(c["kv"]):
            w = torch.softmax(qb[0, h * grp:(h + 1) * grp] @ k[:, h].T / math.sqrt(c["hd"]), 1)
            out[b, h * grp:(h + 1) * grp] = w @ v[:, h]
    return out.view(c["B"], -1)

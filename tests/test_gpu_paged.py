"""The paged key/value cache, its attention and the rotary operators (include/elmh.h) against plain numpy in 64 bits."""
import math

import numpy as np
import pytest

from edgelm_amd import elmh as E

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16", "q8", "q4"]
HDS = [32, 64, 96, 128, 192, 256]
EPS = 2.0 ** -24  # half a step of f32


def _up(ctx, *arrays):
    """Device copies, kept alive by the caller."""
    return [ctx.buffer(max(16, a.nbytes)).upload(a) for a in arrays]


def _free(*bufs):
    for b in bufs:
        b.free()


def _bf16(x):
    """f32 -> the bits of the nearest bf16, ties to even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def _level(r, lo, hi):
    return np.clip(np.sign(r) * np.floor(np.abs(r) + np.float32(0.5)), lo, hi).astype(np.float32)


def _nib_bytes(hd, keys):
    d = np.arange(hd)
    return (d % 32 // 8) * (hd // 8) + d // 32 * 4 + d % 8 // 2 if keys else d % 32 // 2 * (hd // 32) + d // 32


class Cache:
    """A paged cache on the device and its pools on the host. Rows are stored by this file's own statement of the format."""

    def __init__(self, ctx, dtype, n_kv, hd, page, n_pages, fill=None):
        self.ctx, self.dtype, self.n_kv, self.hd, self.page, self.n_pages = ctx, dtype, n_kv, hd, page, n_pages
        shape = (n_pages, n_kv, page)
        self.groups = {"q8": 1, "q4": hd // 32}.get(dtype, 0)
        kind = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "q8": np.int8, "q4": np.uint8}[dtype]
        width = hd // 2 if dtype == "q4" else hd
        # what was never written: NaN, or any levels under a NaN scale
        blank = {"f32": np.nan, "f16": np.nan, "bf16": 0x7FC1, "q8": -128, "q4": 0xA7}[dtype] if fill is None else fill
        self.pool = {n: np.full(shape + (width,), blank, kind) for n in "kv"}
        self.scale = {n: np.full((n_pages, n_kv, self.groups, page), np.nan, np.float32) for n in "kv"} if self.groups else {}

    def put(self, n, page, head, slot, x):
        """One row of f32 values."""
        x = np.asarray(x, np.float32)
        if self.dtype == "f32":
            self.pool[n][page, head, slot] = x
        elif self.dtype == "f16":
            self.pool[n][page, head, slot] = x.astype(np.float16)
        elif self.dtype == "bf16":
            self.pool[n][page, head, slot] = _bf16(x)
        elif self.dtype == "q8":
            s = np.float32(np.abs(x).max() / np.float32(127))
            self.pool[n][page, head, slot] = _level(x / (s if s else np.float32(1)), -127, 127)
            self.scale[n][page, head, 0, slot] = s
        else:
            g = x.reshape(-1, 32)
            s = g[np.arange(len(g)), np.abs(g).argmax(1)] / np.float32(-8)
            q = (_level(g / np.where(s == 0, np.float32(1), s)[:, None], -8, 7) + 8).astype(np.uint8).ravel()
            at = _nib_bytes(self.hd, n == "k")
            row = np.zeros(self.hd // 2, np.uint8)
            row[at[0::2]] = q[0::2] | q[1::2] << 4
            self.pool[n][page, head, slot] = row
            self.scale[n][page, head, :, slot] = s

    def get(self, n, page, head, slot):
        """The row's values in f64."""
        r = self.pool[n][page, head, slot]
        if self.dtype == "bf16":
            return (r.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        if self.dtype == "q8":
            return r.astype(np.float64) * np.float64(self.scale[n][page, head, 0, slot])
        if self.dtype == "q4":
            b = r[_nib_bytes(self.hd, n == "k")].astype(np.int32)
            q = np.where(np.arange(self.hd) % 2, b >> 4, b & 15) - 8
            return q * np.repeat(self.scale[n][page, head, :, slot].astype(np.float64), 32)
        return r.astype(np.float64)

    def send(self):
        arrays = [self.pool["k"], self.pool["v"]] + ([self.scale["k"], self.scale["v"]] if self.groups else [])
        self.bufs = _up(self.ctx, *arrays)
        ptrs = [b.ptr for b in self.bufs] + [None, None]
        self.pages = E.KVPages(E.KV_DTYPES[self.dtype], self.n_kv, self.hd, self.page, self.n_pages, *ptrs[:4])
        return self

    def fetch(self):
        """(pools, scales) now on the device."""
        pool = {n: b.download(self.pool[n].shape, self.pool[n].dtype) for n, b in zip("kv", self.bufs)}
        scale = {n: b.download(self.scale[n].shape, np.float32) for n, b in zip("kv", self.bufs[2:])}
        return pool, scale

    def free(self):
        _free(*self.bufs)


def _tables(n, rot, theta=10000.0):
    a = np.arange(n)[:, None] * theta ** (-np.arange(0, rot, 2) / rot)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


class RopeTables:
    def __init__(self, ctx, n, rot, inter):
        self.cos, self.sin = _tables(n, rot)
        self.rot, self.inter = rot, inter
        self.bufs = _up(ctx, self.cos, self.sin)
        self.rope = E.Rope(self.bufs[0].ptr, self.bufs[1].ptr, n, rot, int(inter))

    def turn(self, x, p):
        """x [..., hd] in its own precision, each product and sum rounded to it."""
        half, y = self.rot // 2, x.copy()
        a, b = (slice(0, self.rot, 2), slice(1, self.rot, 2)) if self.inter else (slice(0, half), slice(half, self.rot))
        c, s = self.cos[p].astype(x.dtype), self.sin[p].astype(x.dtype)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        return y

    def free(self):
        _free(*self.bufs)


def _table_of(rng, lens, page, n_pages, spare=1):
    """A page table of shuffled pages, entries behind a sequence's end naming no page."""
    need = [-(-n // page) for n in lens]
    most = max(1, max(need)) + spare
    order = iter(rng.permutation(n_pages)[:sum(need)])
    t = rng.choice(np.array([-1, n_pages, 2**31 - 1, -2**31], np.int64), (len(lens), most)).astype(np.int32)
    for s, k in enumerate(need):
        for i in range(k):
            t[s, i] = next(order)
    return t


def _fill(c, rng, table, lens, k_amp=1.0, v_amp=1.0):
    for s, n in enumerate(lens):
        for p in range(n):
            pg = table[s, p // c.page]
            if 0 <= pg < c.n_pages:
                for h in range(c.n_kv):
                    c.put("k", pg, h, p % c.page, rng.normal(0, k_amp, c.hd))
                    c.put("v", pg, h, p % c.page, rng.normal(0, v_amp, c.hd))


def _attention64(c, q, table, lens, rope=None):
    """(out [B, heads, hd], per-row tolerance of the 2-norm). A score is hd products of about its own size each rounded to f32
    once as it is added: some sqrt(hd) half steps of the score's size off, and a weight by as much of itself; eight times that
    covers every row of a test. The value sums add sqrt(len) half steps."""
    B, heads, hd = q.shape
    out, tol = np.zeros_like(q, np.float64), np.zeros((B, heads))
    for b, n in enumerate(lens):
        pos = [p for p in range(n) if 0 <= table[b, p // c.page] < c.n_pages]
        if not pos:
            continue
        qb = rope.turn(q[b].astype(np.float64), n - 1) if rope else q[b].astype(np.float64)
        for h in range(c.n_kv):
            k = np.stack([c.get("k", table[b, p // c.page], h, p % c.page) for p in pos])
            v = np.stack([c.get("v", table[b, p // c.page], h, p % c.page) for p in pos])
            for i in range(heads // c.n_kv * h, heads // c.n_kv * (h + 1)):
                s = k @ qb[i] / math.sqrt(hd)
                w = np.exp(s - s.max())
                o = (w / w.sum()) @ v
                out[b, i] = o
                amp = np.sqrt((k * qb[i]) ** 2 @ np.ones(hd) / hd).max() * math.sqrt(hd) / math.sqrt(hd) + np.abs(s).max()
                spread = np.sqrt((w / w.sum()) @ ((v - o) ** 2).sum(1))  # how far an output moves with a weight
                tol[b, i] = EPS * (8 * (math.sqrt(hd) * max(1.0, amp)) * (spread + np.linalg.norm(o)) + math.sqrt(n) * np.linalg.norm(o) + 8 * np.linalg.norm(o))
    return out, tol


def _attend(ctx, c, q, table, lens, max_len=None, rope=None, q_row=0):
    B, heads, hd = q.shape
    rows = q.reshape(B, heads * hd)
    if q_row:
        rows = np.concatenate([rows, np.full((B, q_row - heads * hd), np.nan, np.float32)], 1)
    qb, tb, lb, ob = _up(ctx, np.ascontiguousarray(rows), table, np.asarray(lens, np.int32), np.full((B, heads, hd), 7e7, np.float32))
    cap = table.shape[1] * c.page
    ctx.paged_attention_dev(qb.ptr, ob.ptr, heads, c.pages, tb.ptr, B, table.shape[1], lb.ptr,
                            max_len or max(1, min(cap, max(lens))), rope.rope if rope else None, q_row)
    out = ob.download((B, heads, hd), np.float32)
    _free(qb, tb, lb, ob)
    return out


def _check(got, want, tol):
    off = np.linalg.norm(got - want, axis=-1)
    assert np.isfinite(got).all()
    assert (off <= tol + 1e-37).all(), (off / np.maximum(tol, 1e-300)).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", HDS)
def test_attention_lengths(ctx, dtype, hd):
    """Sequences from none and one position to several parts, ends inside a page and inside a tile, pages in any order, slots
    behind the end holding NaN, table entries behind it naming no page; 1 to 8 queries a kv head."""
    print(f"attention {dtype} hd {hd}", flush=True)
    rng = np.random.default_rng([hd, DTYPES.index(dtype)])
    for page, n_kv, grp, lens in ((16, 2, 3, [1, 0, 15, 16, 17, 31, 33]), (48, 1, 8, [49, 130, 0, 257]), (128, 3, 1, [300, 64, 5])):
        n_pages = sum(-(-n // page) for n in lens) + 3
        table = _table_of(rng, lens, page, n_pages)
        c = Cache(ctx, dtype, n_kv, hd, page, n_pages)
        _fill(c, rng, table, lens)
        c.send()
        q = rng.normal(0, 1.5, (len(lens), n_kv * grp, hd)).astype(np.float32)
        want, tol = _attention64(c, q, table, lens)
        _check(_attend(ctx, c, q, table, lens), want, tol)
        # the same from a larger bound on the lengths: other parts
        _check(_attend(ctx, c, q, table, lens, max_len=table.shape[1] * page), want, tol)
        c.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grp", [2, 5, 15, 16, 17, 40])
def test_attention_groups(ctx, dtype, grp):
    """Query heads a kv head: a tile's sixteen columns partly used, full, and more than one tile; queries inside wider rows."""
    print(f"attention group {dtype} {grp}", flush=True)
    rng = np.random.default_rng(grp)
    lens, page, n_kv, hd = [70, 0, 9], 16, 2, 64
    table = _table_of(rng, lens, page, 9)
    c = Cache(ctx, dtype, n_kv, hd, page, 9)
    _fill(c, rng, table, lens)
    c.send()
    q = rng.normal(0, 1, (3, n_kv * grp, hd)).astype(np.float32)
    want, tol = _attention64(c, q, table, lens)
    _check(_attend(ctx, c, q, table, lens, q_row=n_kv * grp * hd + 37), want, tol)
    c.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,grp", [(256, 16), (256, 33), (192, 16), (128, 32)])
def test_attention_of_wide_tiles(ctx, dtype, hd, grp):
    """All sixteen columns at the large head sizes (66 KB of LDS at 256), split and in one part."""
    rng = np.random.default_rng([hd, grp])
    lens, page, n_kv = [600, 0, 40], 64, 1
    table = _table_of(rng, lens, page, 12)
    c = Cache(ctx, dtype, n_kv, hd, page, 12)
    _fill(c, rng, table, lens)
    c.send()
    q = rng.normal(0, 1, (3, grp, hd)).astype(np.float32)
    want, tol = _attention64(c, q, table, lens)
    _check(_attend(ctx, c, q, table, lens), want, tol)
    want, tol = _attention64(c, q, table, [512, 0, 40])
    _check(_attend(ctx, c, q, table, lens, max_len=512), want, tol)
    c.free()


@pytest.mark.parametrize("hd", HDS)
@pytest.mark.parametrize("grp", [1, 2, 3, 4, 5, 8, 9])
def test_attention_of_q4_columns(ctx, hd, grp):
    """Heads and groups of 32 values that share a tile's columns: as many as fit, fewer, one more; a row of the table without
    pages, sequences in one part and in several."""
    print(f"q4 columns hd {hd} group {grp}", flush=True)
    rng = np.random.default_rng([hd, grp])
    lens, page, n_kv = [700, 0, 37, 1, 60], 32, 2
    table = _table_of(rng, lens, page, 30)
    table[4, 0] = -1
    c = Cache(ctx, "q4", n_kv, hd, page, 30)
    _fill(c, rng, table, lens)
    c.send()
    q = rng.normal(0, 1, (5, n_kv * grp, hd)).astype(np.float32)
    want, tol = _attention64(c, q, table, lens)
    _check(_attend(ctx, c, q, table, lens), want, tol)
    want, tol = _attention64(c, q, table, [500, 0, 37, 1, 60])
    _check(_attend(ctx, c, q, table, [500, 0, 37, 1, 60], max_len=500), want, tol)
    c.free()


@pytest.mark.parametrize("dtype", ["f32", "q8"])
@pytest.mark.parametrize("rot,inter", [(128, False), (128, True), (64, False), (20, True), (22, False), (2, False)])
def test_attention_rotates_queries(ctx, dtype, rot, inter):
    rng = np.random.default_rng(rot)
    lens, page, n_kv, hd = [200, 1, 0, 33], 32, 2, 128
    table = _table_of(rng, lens, page, 20)
    c = Cache(ctx, dtype, n_kv, hd, page, 20)
    _fill(c, rng, table, lens)
    c.send()
    rope = RopeTables(ctx, 200, rot, inter)
    q = rng.normal(0, 1, (4, 6, hd)).astype(np.float32)
    want, tol = _attention64(c, q, table, lens, rope)
    _check(_attend(ctx, c, q, table, lens, max_len=200, rope=rope), want, 2 * tol)  # the rotation's own three roundings
    c.free()
    rope.free()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_missing_pages(ctx, dtype):
    """Entries that name no page, before the end too: their positions are left out; a sequence of none gives zeros. Lengths past
    the bound, and negative ones, are bounded."""
    rng = np.random.default_rng(3)
    lens, page, n_kv, hd = [100, 50, 64, 90], 16, 2, 96
    table = _table_of(rng, lens, page, 40)
    table[0, 2], table[0, 0], table[1, :], table[3, 5] = -1, 40, -7, 2**30
    c = Cache(ctx, dtype, n_kv, hd, page, 40)
    _fill(c, rng, table, lens)
    c.send()
    q = rng.normal(0, 1, (4, 4, hd)).astype(np.float32)
    want, tol = _attention64(c, q, table, lens)
    got = _attend(ctx, c, q, table, lens)
    _check(got, want, tol)
    assert not got[1].any()
    want, tol = _attention64(c, q, table, [64, 50, 64, 64])
    _check(_attend(ctx, c, q, table, [2**31 - 1, 50, 64, 90], max_len=64), want, tol)
    got = _attend(ctx, c, q, table, [-1, -2**31, 0, -5], max_len=64)
    assert not got.any()
    c.free()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_long_sequences(ctx, dtype):
    """Thousands of positions, split over workgroups and joined: a few pages repeated many times, as a table allows, so that the
    expected result needs only those pages' rows. The same bits every time."""
    print(f"attention long {dtype}", flush=True)
    rng = np.random.default_rng(11)
    page, n_kv, hd, n_pages = 16, 2, 64, 24
    lens = [40001, 0, 6000, 129, 20480]
    table = rng.integers(0, n_pages, (5, 2600)).astype(np.int32)
    c = Cache(ctx, dtype, n_kv, hd, page, n_pages)
    for p in range(n_pages):
        for h in range(n_kv):
            for s in range(page):
                c.put("k", p, h, s, rng.normal(0, 1, hd))
                c.put("v", p, h, s, rng.normal(0, 1, hd))
    c.send()
    q = rng.normal(0, 1, (5, 8, hd)).astype(np.float32)
    rows = {(n, p, h): np.stack([c.get(n, p, h, s) for s in range(page)]) for n in "kv" for p in range(n_pages) for h in range(n_kv)}
    want, tol = np.zeros(q.shape), np.zeros(q.shape[:2])
    for b, n in enumerate(lens):
        if not n:
            continue
        for i in range(8):
            h = i // 4
            k, v = (np.concatenate([rows[m, p, h] for p in table[b, :-(-n // page)]])[:n] for m in "kv")
            s = k @ q[b, i].astype(np.float64) / 8
            w = np.exp(s - s.max())
            want[b, i] = w / w.sum() @ v
            # as _attention64's, with scores of up to some 4 and value rows of norm 8 about their mean
            tol[b, i] = EPS * (8 * 8 * np.abs(s).max() * 8 / math.sqrt(n / 50) + math.sqrt(n) * np.linalg.norm(want[b, i]) + 8 * 8 / math.sqrt(n))
    got = _attend(ctx, c, q, table, lens)
    off = np.linalg.norm(got - want, axis=-1)
    assert (off <= tol + 1e-37).all(), (off / np.maximum(tol, 1e-300)).max()
    for _ in range(5):
        assert np.array_equal(got, _attend(ctx, c, q, table, lens))
    # a sequence's own result does not depend on its neighbours where the split is the same
    assert np.array_equal(got, _attend(ctx, c, q, table, lens, max_len=40001))
    c.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k_amp,v_amp,q_amp", [(1, 1, 40.0), (1e-6, 1, 1e6), (30.0, 200.0, 1e-3), (1, 1e-4, 0.0)])
def test_attention_magnitudes(ctx, dtype, k_amp, v_amp, q_amp):
    """One-hot softmaxes, tiny keys under huge queries, large values, queries of zeros."""
    rng = np.random.default_rng(5)
    if dtype == "f16" and k_amp < 1e-3:
        k_amp = 1e-3  # f16 holds 1e-6 only as a subnormal of three bits: that is the cache's rounding, not the attention's
    lens, page, n_kv, hd = [150, 77], 16, 1, 128
    table = _table_of(rng, lens, page, 20)
    c = Cache(ctx, dtype, n_kv, hd, page, 20)
    _fill(c, rng, table, lens, k_amp, v_amp)
    c.send()
    q = rng.normal(0, q_amp, (2, 4, hd)).astype(np.float32)
    want, tol = _attention64(c, q, table, lens)
    _check(_attend(ctx, c, q, table, lens), want, tol)
    c.free()


@pytest.mark.parametrize("dtype", ["q8", "q4"])
def test_attention_of_uneven_scales(ctx, dtype):
    """Rows of very different magnitude (the largest late, early and of tiny ones only), zero rows among them."""
    rng = np.random.default_rng(6)
    page, n_kv, hd, lens = 16, 1, 64, [320, 320, 320, 64]
    table = _table_of(rng, lens, page, 80)
    c = Cache(ctx, dtype, n_kv, hd, page, 80)
    amps = [lambda p: 10.0 ** (p / 16 - 10), lambda p: 10.0 ** (10 - p / 16), lambda p: 1e-30, lambda p: 0.0 if p % 3 else 1e-3]
    for b, n in enumerate(lens):
        for p in range(n):
            c.put("k", table[b, p // page], 0, p % page, rng.normal(0, 1, hd))
            c.put("v", table[b, p // page], 0, p % page, rng.normal(0, 1, hd) * amps[b](p))
    c.send()
    q = rng.normal(0, 1, (4, 4, hd)).astype(np.float32)
    want, tol = _attention64(c, q, table, lens)
    _check(_attend(ctx, c, q, table, lens), want, tol)
    c.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grp", [4, 8])
def test_attention_is_as_exact_as_f32(ctx, dtype, grp):
    """Queries, weights and sums keep their 24 bits. Scores of unit variance over 128 products: the partial sums of an f32
    accumulation grow to the score's size, each rounded by up to half a step, a third of that on average of squares:
    sqrt(128 / 3) = 6.5 half steps of error, which the weights carry into the output; rounding the queries, the scores, the weights and
    the output adds some two. 16 half steps leave a factor of two; pieces of one 16-bit type less would be a hundred off."""
    rng = np.random.default_rng(23)
    page, n_kv, hd, n_pages, lens = 16, 2, 128, 64, [1024, 1000]
    table = np.stack([rng.permutation(n_pages) for _ in lens]).astype(np.int32)
    c = Cache(ctx, dtype, n_kv, hd, page, n_pages)
    for p in range(n_pages):
        for h in range(n_kv):
            for s in range(page):
                c.put("k", p, h, s, rng.normal(0, 1, hd))
                c.put("v", p, h, s, rng.normal(0, 1, hd))
    c.send()
    q = rng.normal(0, 1, (2, n_kv * grp, hd)).astype(np.float32)
    want, _ = _attention64(c, q, table, lens)
    got = _attend(ctx, c, q, table, lens)
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= 16 * EPS, rel / EPS
    c.free()


@pytest.mark.parametrize("dtype", ["q8", "q4", "f32", "bf16"])
@pytest.mark.parametrize("k_amp,v_amp,q_amp", [(1e-30, 1e34, 1e30), (1e30, 1e-34, 1e-30)])
def test_attention_at_the_ends_of_the_range(ctx, dtype, k_amp, v_amp, q_amp):
    """Values and queries near the largest and smallest f32 holds, under keys that bring the scores back."""
    rng = np.random.default_rng(15)
    lens, page, n_kv, hd = [100, 33], 16, 2, 64
    table = _table_of(rng, lens, page, 12)
    c = Cache(ctx, dtype, n_kv, hd, page, 12)
    _fill(c, rng, table, lens, k_amp, v_amp)
    c.send()
    q = rng.normal(0, q_amp, (2, 4, hd)).astype(np.float32)
    want, tol = _attention64(c, q, table, lens)
    _check(_attend(ctx, c, q, table, lens) * 1.0, want, tol)
    c.free()


@pytest.mark.parametrize("dtype,hd", [("q8", 64), ("q4", 64), ("bf16", 128)])
def test_attention_of_many_sequences(ctx, dtype, hd):
    """More sequences than a wave has lanes, most of them short or empty, a few long ones that are split, at either end and
    between; and batches of 64 and 65. Pages shared by many sequences."""
    rng = np.random.default_rng(17)
    page, n_kv, n_pages = 16, 1, 12
    c = Cache(ctx, dtype, n_kv, hd, page, n_pages)
    for p in range(n_pages):
        for s in range(page):
            c.put("k", p, 0, s, rng.normal(0, 1, hd))
            c.put("v", p, 0, s, rng.normal(0, 1, hd))
    c.send()
    rows = {(n, p): np.stack([c.get(n, p, 0, s) for s in range(page)]) for n in "kv" for p in range(n_pages)}
    for n in (64, 65, 300) + ((4096,) if dtype == "q8" else ()):
        lens = rng.integers(0, 60, n)
        lens[rng.random(n) < 0.3] = 0
        lens[[0, n // 2, n - 1]] = [3000, 1700, 2500]
        table = rng.integers(0, n_pages, (n, 190)).astype(np.int32)
        q = rng.normal(0, 1, (n, 2, hd)).astype(np.float32)
        got = _attend(ctx, c, q, table, lens)
        for b in range(n):
            if not lens[b]:
                assert not got[b].any()
                continue
            k, v = (np.concatenate([rows[m, p] for p in table[b, :-(-lens[b] // page)]])[:lens[b]] for m in "kv")
            for i in range(2):
                s = k @ q[b, i].astype(np.float64) / math.sqrt(hd)
                w = np.exp(s - s.max())
                w /= w.sum()
                o = w @ v
                # as _attention64's
                amp = np.sqrt(((k * q[b, i]) ** 2).sum(1) / hd).max() + np.abs(s).max()
                spread = np.sqrt(w @ ((v - o) ** 2).sum(1))
                tol = EPS * (8 * math.sqrt(hd) * max(1.0, amp) * (spread + np.linalg.norm(o)) + (math.sqrt(lens[b]) + 8) * np.linalg.norm(o))
                assert np.linalg.norm(got[b, i] - o) <= tol, (n, b, i)
    c.free()


def test_attention_past_4_gb(ctx):
    """Pages far into pools of more than 4 GB (2^32 bytes, and 2^31 values in f16): addresses are 64-bit."""
    page, n_kv, hd, n_pages, lens = 128, 8, 256, 8400, [200, 129]
    rng = np.random.default_rng(8)
    assert n_pages * n_kv * page * hd > 2**31
    c = Cache(ctx, "f16", n_kv, hd, page, 4)
    small = _table_of(rng, lens, page, 4, spare=0)
    _fill(c, rng, small, lens)
    per = n_kv * page * hd * 2
    kb, vb = ctx.buffer(n_pages * per), ctx.buffer(n_pages * per)
    at = n_pages - 4
    for b, n in ((kb, "k"), (vb, "v")):
        h = np.ascontiguousarray(c.pool[n])
        ctx.memset_dev(b.ptr, 0xFF, per)  # page 0: NaN
        tmp = _up(ctx, h)[0]
        ctx.memcpy_d2d(b.ptr + at * per, tmp.ptr, h.nbytes)
        ctx.synchronize()
        tmp.free()
    c.pages = E.KVPages(E.F16, n_kv, hd, page, n_pages, kb.ptr, vb.ptr, None, None)
    q = rng.normal(0, 1, (2, 16, hd)).astype(np.float32)
    want, tol = _attention64(c, q, small, lens)
    far = (small + at).astype(np.int32)
    _check(_attend(ctx, c, q, far, lens), want, tol)
    # read back, and append there
    pos, seq = np.arange(120, 129, dtype=np.int32), np.ones(9, np.int32)
    pb, sb, tb = _up(ctx, pos, seq, far)
    ko, vo = ctx.buffer(9 * n_kv * hd * 4), ctx.buffer(9 * n_kv * hd * 4)
    ctx.paged_read_dev(ko.ptr, vo.ptr, 9, c.pages, tb.ptr, 2, far.shape[1], pb.ptr, sb.ptr)
    k = ko.download((9, n_kv, hd), np.float32)
    assert all(np.array_equal(k[i, h], c.get("k", small[1, p // page], h, p % page)) for i, p in enumerate(pos) for h in range(n_kv))
    ctx.paged_append_dev(vo.ptr, ko.ptr, 9, c.pages, tb.ptr, 2, far.shape[1], pb.ptr, sb.ptr)
    ctx.paged_read_dev(ko.ptr, vo.ptr, 9, c.pages, tb.ptr, 2, far.shape[1], pb.ptr, sb.ptr)
    assert np.array_equal(vo.download((9, n_kv, hd), np.float32), k)
    _free(pb, sb, tb, ko, vo, kb, vb)


# ------------------------------------------------------------------ rows written and read

def _special(rng, n, n_kv, hd):
    """Rows with ties, zeros, halves between levels, and magnitudes far apart."""
    x = rng.normal(0, 1, (n, n_kv, hd)).astype(np.float32)
    x *= np.float32(10.0) ** rng.integers(-12, 12, (n, n_kv, 1)).astype(np.float32)
    flat = x.reshape(-1, hd)
    flat[0] = 0
    if len(flat) > 4:
        flat[1] = np.where(np.arange(hd) % 2, -3, 3)                     # ties: the first of largest magnitude is positive
        flat[2] = np.where(np.arange(hd) % 5 == 0, -3, 2)                # and negative
        flat[3] = (np.arange(hd) % 16 - 8 + 0.5) * 0.25                  # halves
        flat[4] = np.arange(hd) % 32 == 31                               # one value, the group's last
    return np.clip(x, -6e4, 6e4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", HDS)
@pytest.mark.parametrize("rot,inter", [(0, False), (-1, False), (-1, True), (16, False), (14, False), (30, True)])
def test_append_and_read(ctx, dtype, hd, rot, inter):
    """Bit for bit: what is written (keys rotated over all of the head, 16, 14 or 30 values of it), what is left alone, what is
    read back; rows of padding, of no sequence, past the table, the pages or the rotary tables."""
    print(f"append {dtype} hd {hd} rot {rot} inter {inter}", flush=True)
    rng = np.random.default_rng([hd, rot + 5, inter])
    page, n_kv, n_pages = 16, 3, 12
    n_seqs, max_pages, max_pos = 4, 3, 45
    table = rng.permutation(n_pages).astype(np.int32).reshape(n_seqs, max_pages)
    table[3, 1], table[2, 2] = -1, n_pages
    rope = RopeTables(ctx, max_pos, hd if rot < 0 else rot, inter) if rot else None
    c = Cache(ctx, dtype, n_kv, hd, page, n_pages, fill=0x5A).send()
    pairs = [(0, 0), (0, 15), (0, 16), (1, 44), (1, 7), (2, 31), (3, 3), (2, 0), (0, 9), (1, 40)]
    skipped = [(0, -1), (0, 48), (1, 2**31 - 1), (1, -2**31), (4, 3), (-1, 3), (2**31 - 1, 0), (3, 16), (2, 32)] + ([(0, 45), (1, 47)] if rot else [])
    rows = [(s, p, True) for s, p in pairs] + [(s, p, False) for s, p in skipped]
    order = rng.permutation(len(rows))
    rows = [rows[i] for i in order]
    n = len(rows)
    k, v = _special(rng, n, n_kv, hd), _special(rng, n, n_kv, hd)
    for i, (s, p, live) in enumerate(rows):
        if live:
            for h in range(n_kv):
                c.put("k", table[s, p // page], h, p % page, rope.turn(k[i, h], p) if rope else k[i, h])
                c.put("v", table[s, p // page], h, p % page, v[i, h])
    seq, pos = np.array([r[0] for r in rows], np.int32), np.array([r[1] for r in rows], np.int32)
    kb, vb, tb, sb, pb = _up(ctx, k, v, table, seq, pos)
    ctx.paged_append_dev(kb.ptr, vb.ptr, n, c.pages, tb.ptr, n_seqs, max_pages, pb.ptr, sb.ptr, rope.rope if rope else None)
    pool, scale = c.fetch()
    for m in "kv":
        if dtype in ("f32", "f16"):  # zeros of both signs are one value
            assert np.array_equal(pool[m], c.pool[m])
        else:
            assert np.array_equal(pool[m], c.pool[m]), np.argwhere(pool[m] != c.pool[m])[:5]
        if scale:
            assert np.array_equal(scale[m], c.scale[m], equal_nan=True)
    # and back, into rows that hold something
    kb.upload(np.full_like(k, 123.0))
    vb.upload(np.full_like(v, 321.0))
    ctx.paged_read_dev(kb.ptr, vb.ptr, n, c.pages, tb.ptr, n_seqs, max_pages, pb.ptr, sb.ptr)
    for b, m, was in ((kb, "k", 123.0), (vb, "v", 321.0)):
        got = b.download(k.shape, np.float32)
        for i, (s, p, live) in enumerate(rows):
            in_table = live or (rot and (s, p) in ((0, 45), (1, 47)))  # the rotary tables do not bound a read
            for h in range(n_kv):
                if live:
                    assert np.array_equal(got[i, h], c.get(m, table[s, p // page], h, p % page).astype(np.float32)), (i, h)
                elif not in_table:
                    assert (got[i, h] == was).all()
    _free(kb, vb, tb, sb, pb)
    c.free()
    if rope:
        rope.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["fused", "heads_first", "odd", "unaligned"])
def test_append_and_read_strides(ctx, dtype, order):
    """Rows inside wider ones (a fused projection's), heads first (a contiguous cache), rows at odd distances, rows that start
    off 16 bytes. What lies between the rows read into stays."""
    rng = np.random.default_rng(2)
    n, n_kv, hd, page = 21, 2, 64, 16
    row, head, shift = {"fused": (5 * n_kv * hd, hd, 0), "heads_first": (hd, n * hd, 0), "odd": (n_kv * hd + 33, hd + 5, 0),
                        "unaligned": (n_kv * hd, hd, 3)}[order]
    size = shift + (n - 1) * row + (n_kv - 1) * head + hd
    src = rng.normal(0, 1, (2, size)).astype(np.float32)
    at = shift + np.arange(n)[:, None, None] * row + np.arange(n_kv)[None, :, None] * head + np.arange(hd)
    table = np.array([[1, 0]], np.int32)
    c = Cache(ctx, dtype, n_kv, hd, page, 2, fill=0).send()
    rope = RopeTables(ctx, 40, hd, False)
    for p in range(n):
        for h in range(n_kv):
            c.put("k", table[0, p // page], h, p % page, rope.turn(src[0][at[p, h]], p))
            c.put("v", table[0, p // page], h, p % page, src[1][at[p, h]])
    kb, vb, tb, sb, pb = _up(ctx, src[0], src[1], table, np.zeros(n, np.int32), np.arange(n, dtype=np.int32))
    ctx.paged_append_dev(kb.ptr + 4 * shift, vb.ptr + 4 * shift, n, c.pages, tb.ptr, 1, 2, pb.ptr, sb.ptr, rope.rope, row, head)
    pool, scale = c.fetch()
    for m in "kv":
        assert np.array_equal(pool[m], c.pool[m])
        if scale:
            assert np.array_equal(scale[m], c.scale[m], equal_nan=True)
    ctx.paged_read_dev(kb.ptr + 4 * shift, vb.ptr + 4 * shift, n, c.pages, tb.ptr, 1, 2, pb.ptr, sb.ptr, row, head)
    for b, m, x in ((kb, "k", src[0]), (vb, "v", src[1])):
        want = x.copy()
        for p in range(n):
            for h in range(n_kv):
                want[at[p, h]] = c.get(m, table[0, p // page], h, p % page)
        assert np.array_equal(b.download(want.shape, np.float32), want)
    _free(kb, vb, tb, sb, pb)
    c.free()
    rope.free()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_kv,hd,page", [(1, 96, 4096), (5, 32, 16), (8, 128, 48), (12, 64, 80), (64, 32, 16)])
@pytest.mark.parametrize("off", [0, 1])
def test_append_and_read_heads(ctx, dtype, n_kv, hd, page, off):
    """Kv heads that go to one workgroup in powers of two and not, page sizes that are no power of two and the largest, row i of
    sequence i, rotary tables on and off 16 bytes."""
    rng = np.random.default_rng([n_kv, hd])
    n, max_pos = 37, 9000
    cos, sin = _tables(max_pos, hd)
    cb, sb = _up(ctx, *[np.concatenate([np.full(off, 9, np.float32), t.ravel()]) for t in (cos, sin)])
    rope = E.Rope(cb.ptr + 4 * off, sb.ptr + 4 * off, max_pos, hd, 0)
    r = RopeTables.__new__(RopeTables)
    r.cos, r.sin, r.rot, r.inter = cos, sin, hd, False
    pos = rng.integers(0, min(max_pos, 2 * page), n).astype(np.int32)
    table = rng.permutation(2 * n).reshape(n, 2).astype(np.int32)
    c = Cache(ctx, dtype, n_kv, hd, page, 2 * n, fill=0).send()
    k, v = (rng.normal(0, 1, (n, n_kv, hd)).astype(np.float32) for _ in range(2))
    for i in range(n):
        for h in range(n_kv):
            c.put("k", table[i, pos[i] // page], h, pos[i] % page, r.turn(k[i, h], pos[i]))
            c.put("v", table[i, pos[i] // page], h, pos[i] % page, v[i, h])
    kb, vb, tb, pb = _up(ctx, k, v, table, pos)
    ctx.paged_append_dev(kb.ptr, vb.ptr, n, c.pages, tb.ptr, n, 2, pb.ptr, None, rope)
    pool, scale = c.fetch()
    for m in "kv":
        assert np.array_equal(pool[m], c.pool[m])
        if scale:
            assert np.array_equal(scale[m], c.scale[m], equal_nan=True)
    ctx.paged_read_dev(kb.ptr, vb.ptr, n, c.pages, tb.ptr, n, 2, pb.ptr)
    for b, m in ((kb, "k"), (vb, "v")):
        got = b.download(k.shape, np.float32)
        assert all(np.array_equal(got[i, h], c.get(m, table[i, pos[i] // page], h, pos[i] % page).astype(np.float32)) for i in range(n) for h in range(n_kv))
    _free(kb, vb, tb, pb, cb, sb)
    c.free()


def test_append_to_shared_pages(ctx):
    """One page in two sequences' rows of the table."""
    n_kv, hd, page = 2, 32, 16
    c = Cache(ctx, "q8", n_kv, hd, page, 2, fill=0).send()
    x = np.random.default_rng(1).normal(0, 1, (n_kv, hd)).astype(np.float32)
    table = np.array([[0], [1], [0]], np.int32)  # sequences 0 and 2 share page 0
    pos = np.array([3, 3, 9], np.int32)
    for s, p in enumerate(pos):
        for h in range(n_kv):
            for m in "kv":
                c.put(m, table[s, 0], h, p, x[h])
    xb, tb, pb = _up(ctx, np.stack([x] * 3), table, pos)
    ctx.paged_append_dev(xb.ptr, xb.ptr, 3, c.pages, tb.ptr, 3, 1, pb.ptr)
    pool, scale = c.fetch()
    assert all(np.array_equal(pool[m], c.pool[m]) and np.array_equal(scale[m], c.scale[m], equal_nan=True) for m in "kv")
    _free(xb, tb, pb)
    c.free()


# ------------------------------------------------------------------ rotary tables and rotation

@pytest.mark.parametrize("hd,rot,inter", [(64, 64, False), (64, 64, True), (128, 32, False), (80, 20, True), (96, 50, False), (2, 2, True), (256, 254, False)])
@pytest.mark.parametrize("T,heads", [(1, 1), (7, 3), (130, 9)])
def test_rope(ctx, hd, rot, inter, T, heads):
    """Bit for bit: at given positions and at consecutive ones, in place, in strided rows; rows at no position stay."""
    rng = np.random.default_rng([hd, rot, T])
    r = RopeTables(ctx, 500, rot, inter)
    x = rng.normal(0, 1, (T, heads, hd)).astype(np.float32)
    pos = rng.integers(0, 500, T).astype(np.int32)
    if T > 4:
        pos[1], pos[3] = -1, 500
    want = np.stack([r.turn(x[t], p) if 0 <= p < 500 else np.full_like(x[t], 9) for t, p in enumerate(pos)])
    xb, pb, yb = _up(ctx, x, pos, np.full_like(x, 9))
    ctx.rope_dev(xb.ptr, yb.ptr, T, heads, hd, r.rope, pb.ptr)
    assert np.array_equal(yb.download(x.shape, np.float32), want)
    ctx.rope_dev(xb.ptr, xb.ptr, T, heads, hd, r.rope, pos0=500 - T)
    want = np.stack([r.turn(x[t], 500 - T + t) for t in range(T)])
    assert np.array_equal(xb.download(x.shape, np.float32), want)
    wide = rng.normal(0, 1, (T, heads * hd + 7)).astype(np.float32)
    wb, zb = _up(ctx, wide, np.full((T, heads * hd + 3), 5, np.float32))
    ctx.rope_dev(wb.ptr, zb.ptr, T, heads, hd, r.rope, pos0=2, x_row=heads * hd + 7, y_row=heads * hd + 3)
    got = zb.download((T, heads * hd + 3), np.float32)
    want = np.stack([r.turn(wide[t, :heads * hd].reshape(heads, hd), 2 + t).ravel() for t in range(T)])
    assert np.array_equal(got[:, :heads * hd], want)
    assert (got[:-1, heads * hd:] == 5).all()
    _free(xb, pb, yb, wb, zb)
    r.free()


@pytest.mark.parametrize("rot", [64, 62])
def test_rope_of_many_rows(ctx, rot):
    """More rows than one launch has threads for at once."""
    T, heads, hd = 17003, 32, 64
    rng = np.random.default_rng(rot)
    r = RopeTables(ctx, 700, rot, False)
    x = rng.normal(0, 1, (T, heads, hd)).astype(np.float32)
    pos = rng.integers(0, 700, T).astype(np.int32)
    xb, pb = _up(ctx, x, pos)
    ctx.rope_dev(xb.ptr, xb.ptr, T, heads, hd, r.rope, pb.ptr)
    want, half = x.copy(), rot // 2
    c, s = r.cos[pos][:, None], r.sin[pos][:, None]
    want[..., :half], want[..., half:rot] = x[..., :half] * c - x[..., half:rot] * s, x[..., half:rot] * c + x[..., :half] * s
    assert np.array_equal(xb.download(x.shape, np.float32), want)
    _free(xb, pb)
    r.free()


@pytest.mark.parametrize("scaling", [None, E.RopeScaling(E.ROPE_LINEAR, 3.0), E.RopeScaling(E.ROPE_BANDS, 8.0, 8192, 1.0, 4.0),
                                     E.RopeScaling(E.ROPE_YARN, 16.0, 4096, 1.0, 32.0, 1.2772588722239781)])
@pytest.mark.parametrize("pos0,n,rot,theta", [(0, 1, 64, 10000.0), (0, 1000, 128, 500000.0), (1000003, 77, 96, 10000.0), (2**31 - 50, 40, 2, 1e6),
                                              (5, 33, 30, 100000.0)])
def test_rope_table(ctx, scaling, pos0, n, rot, theta):
    """A value is off by its rounding, half a step, and by what the angle's own rounding in f64 moves it: some 2^-50 of the angle
    (the frequency's power, the product, the reduction), which at 2^31 is 2e-6."""
    half = rot // 2
    cb, sb = _up(ctx, *[np.full(n * half + 3, 4.0, np.float32)] * 2)
    ctx.rope_table_dev(cb.ptr, sb.ptr, pos0, n, rot, theta, scaling)
    i = np.arange(half, dtype=np.longdouble)
    f = np.longdouble(theta) ** (-2 * i / rot)
    m = 1.0
    if scaling is not None:
        two_pi, fac, m = 2 * np.longdouble(math.pi), scaling.factor, scaling.magnitude
        if scaling.kind == E.ROPE_LINEAR:
            keep = np.zeros(half)
        elif scaling.kind == E.ROPE_BANDS:
            keep = np.clip((scaling.orig_ctx * f / two_pi - scaling.low) / (scaling.high - scaling.low), 0, 1)
        else:
            a, b = (rot * math.log(scaling.orig_ctx / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (scaling.high, scaling.low))
            a, b = max(math.floor(a), 0), min(math.ceil(b), rot - 1)
            keep = 1 - np.clip((i - a) / max(b - a, 0.001), 0, 1)
        f = f * (keep + (1 - keep) / fac)
    a = (pos0 + np.arange(n, dtype=np.longdouble))[:, None] * f
    for b, fn in ((cb, np.cos), (sb, np.sin)):
        got, want = b.download(n * half + 3, np.float32), (fn(a) * m).astype(np.float64).ravel()
        assert (got[n * half:] == 4.0).all()
        tol = np.abs(want) * EPS * 1.001 + m * np.abs(a.astype(np.float64)).ravel() * 2.0 ** -50 + 2.0 ** -60
        assert (np.abs(got[:n * half] - want) <= tol).all(), (np.abs(got[:n * half] - want) / tol).max()
    _free(cb, sb)


# ------------------------------------------------------------------ together, as they are used

@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_then_decode_steps(ctx, dtype):
    """Prompts through the contiguous attention, their caches moved into pages (keys as they are: rotated), then decode steps of
    the batch, each a step of elmh_attention_step_dev on the contiguous caches too. f32 pages give its results to f32's
    rounding, the others to their own: a row's rounding is half a step, 2^-12 (f16), 2^-9 (bf16), amax / 254 (q8), an eighth
    of the group's largest over two (q4), which moves an output by no more than some of that of a value's size."""
    rng = np.random.default_rng(21)
    n_kv, heads, hd, page, ctx_len = 2, 6, 64, 16, 96
    prompts, steps = [37, 5, 64], 6
    B = len(prompts)
    r = RopeTables(ctx, ctx_len, hd, False)
    c = Cache(ctx, dtype, n_kv, hd, page, 20, fill=0).send()
    table = rng.permutation(20)[:B * 6].reshape(B, 6).astype(np.int32)
    tb = _up(ctx, table)[0]
    kc = [[ctx.buffer(n_kv * ctx_len * hd * 4) for _ in range(2)] for _ in range(B)]
    for s, T in enumerate(prompts):
        q, k, v = (rng.normal(0, 1, (T, h, hd)).astype(np.float32) for h in (heads, n_kv, n_kv))
        qb, kb, vb, ob = _up(ctx, q, k, v, q)
        ctx.attention_dev(qb.ptr, kb.ptr, vb.ptr, ob.ptr, T, 0, heads, n_kv, hd, kc[s][0].ptr, kc[s][1].ptr, ctx_len, r.bufs[0].ptr, r.bufs[1].ptr)
        sb, pb = _up(ctx, np.full(T, s, np.int32), np.arange(T, dtype=np.int32))
        ctx.paged_append_dev(kc[s][0].ptr, kc[s][1].ptr, T, c.pages, tb.ptr, B, 6, pb.ptr, sb.ptr, None, hd, ctx_len * hd)
        ctx.synchronize()
        _free(qb, kb, vb, ob, sb, pb)
    rel = {"f32": 40 * EPS, "f16": 2.0 ** -11 * 2, "bf16": 2.0 ** -8 * 2, "q8": 0.04, "q4": 0.6}[dtype]
    for t in range(steps):
        q, k, v = (rng.normal(0, 1, (B, h, hd)).astype(np.float32) for h in (heads, n_kv, n_kv))
        pos = np.array([p + t for p in prompts], np.int32)
        qb, kb, vb, ob, pb, lb = _up(ctx, q, k, v, q, pos, pos + 1)
        ctx.paged_append_dev(kb.ptr, vb.ptr, B, c.pages, tb.ptr, B, 6, pb.ptr, None, r.rope)
        ctx.paged_attention_dev(qb.ptr, ob.ptr, heads, c.pages, tb.ptr, B, 6, lb.ptr, ctx_len, r.rope)
        got = ob.download(q.shape, np.float32)
        row = 4 * heads * hd
        for s in range(B):
            ctx.attention_step_dev(qb.ptr + s * row, kb.ptr + s * 4 * n_kv * hd, vb.ptr + s * 4 * n_kv * hd, ob.ptr + s * row, pb.ptr + 4 * s, heads,
                                   n_kv, hd, kc[s][0].ptr, kc[s][1].ptr, ctx_len, r.bufs[0].ptr, r.bufs[1].ptr)
        want = ob.download(q.shape, np.float32)
        assert np.linalg.norm(got - want) <= rel * np.linalg.norm(want), t
        _free(qb, kb, vb, ob, pb, lb)
    if dtype == "f32":  # the pages read back are the contiguous caches
        for s, T in enumerate(prompts):
            n = T + steps
            sb, pb, ko, vo = _up(ctx, np.full(n, s, np.int32), np.arange(n, dtype=np.int32), *[np.zeros((n_kv, ctx_len, hd), np.float32)] * 2)
            ctx.paged_read_dev(ko.ptr, vo.ptr, n, c.pages, tb.ptr, B, 6, pb.ptr, sb.ptr, hd, ctx_len * hd)
            for have, was in ((ko, kc[s][0]), (vo, kc[s][1])):
                assert np.array_equal(have.download((n_kv, ctx_len, hd), np.float32)[:, :n], was.download((n_kv, ctx_len, hd), np.float32)[:, :n])
            _free(sb, pb, ko, vo)
    for pair in kc:
        _free(*pair)
    tb.free()
    c.free()
    r.free()


def test_decode_step_in_graphs(ctx):
    """A captured step (append, then attention) replayed at growing lengths, two graphs of different batches sharing the
    context's scratch, eager calls between the replays: every replay gives the eager call's bits."""
    rng = np.random.default_rng(31)
    n_kv, heads, hd, page, B = 2, 8, 64, 16, 3
    c = Cache(ctx, "q8", n_kv, hd, page, 400, fill=0).send()
    table = rng.permutation(400)[:B * 130].reshape(B, 130).astype(np.int32)
    r = RopeTables(ctx, 2080, hd, False)
    lens0 = [2000, 300, 17]
    total = sum(lens0)
    k, v = (rng.normal(0, 1, (total, n_kv, hd)).astype(np.float32) for _ in range(2))
    tb, kb, vb, sb, pb = _up(ctx, table, k, v, np.repeat(np.arange(B), lens0).astype(np.int32), np.concatenate([np.arange(n) for n in lens0]).astype(np.int32))
    ctx.paged_append_dev(kb.ptr, vb.ptr, total, c.pages, tb.ptr, B, 130, pb.ptr, sb.ptr, r.rope)
    q1, k1, v1 = (rng.normal(0, 1, (B, h, hd)).astype(np.float32) for h in (heads, n_kv, n_kv))
    q, kn, vn, pos, lens, o = _up(ctx, q1, k1, v1, np.array(lens0, np.int32), np.array(lens0, np.int32) + 1, q1)
    o2 = ctx.buffer(q1.nbytes)

    def step(out, n):
        ctx.paged_append_dev(kn.ptr, vn.ptr, n, c.pages, tb.ptr, n, 130, pos.ptr, None, r.rope)
        ctx.paged_attention_dev(q.ptr, out.ptr, heads, c.pages, tb.ptr, n, 130, lens.ptr, 2080, r.rope)

    step(o, B)  # allocates the scratch
    step(o2, 1)
    graphs = []
    for out, n in ((o, B), (o2, 1)):
        ctx.graph_begin()
        step(out, n)
        graphs.append(ctx.graph_end())
    for t in range(5):
        q1, k1, v1 = (rng.normal(0, 1, (B, h, hd)).astype(np.float32) for h in (heads, n_kv, n_kv))
        for b, x in ((q, q1), (kn, k1), (vn, v1), (pos, np.array(lens0, np.int32) + t), (lens, np.array(lens0, np.int32) + t + 1)):
            b.upload(x)
        step(o, B)
        want = o.download((B, heads, hd), np.float32)
        o.upload(np.zeros_like(want))
        o2.upload(np.zeros_like(want))
        for g in graphs + graphs[::-1]:
            ctx.graph_launch(g)
        ctx.synchronize()
        got, got2 = o.download((B, heads, hd), np.float32), o2.download((1, heads, hd), np.float32)
        assert np.array_equal(got, want)
        step(o2, 1)
        assert np.array_equal(got2, o2.download((1, heads, hd), np.float32))
    for g in graphs:
        ctx.graph_destroy(g)
    _free(tb, kb, vb, sb, pb, q, kn, vn, pos, lens, o, o2)
    c.free()
    r.free()


def test_two_contexts_at_once(ctx):
    """Calls on two contexts' streams in flight together, each with split sequences and its own scratch."""
    rng = np.random.default_rng(41)
    other = E.Context(0)
    sides = []
    for c in (ctx, other):
        cache = Cache(c, "bf16", 2, 64, 16, 30)
        lens = [3000, 17, 2100]
        table = rng.integers(0, 30, (3, 190)).astype(np.int32)
        for p in range(30):
            for h in range(2):
                for s in range(16):
                    cache.put("k", p, h, s, rng.normal(0, 1, 64))
                    cache.put("v", p, h, s, rng.normal(0, 1, 64))
        cache.send()
        q = rng.normal(0, 1, (3, 8, 64)).astype(np.float32)
        sides.append((c, cache, q, _up(c, q, table, np.array(lens, np.int32), q), _attend(c, cache, q, table, lens)))
    for _ in range(20):
        for c, cache, q, (qb, tb, lb, ob), _ in sides:
            for _ in range(5):
                c.paged_attention_dev(qb.ptr, ob.ptr, 8, cache.pages, tb.ptr, 3, 190, lb.ptr, 3000)
    for c, cache, q, bufs, want in sides:
        assert np.array_equal(bufs[3].download(q.shape, np.float32), want)
        _free(*bufs)
        cache.free()
    other.close()


def test_scratch_does_not_grow_in_a_capture():
    """A capture that would need more scratch than the context has is refused, and the context goes on."""
    own = E.Context(0)
    rng = np.random.default_rng(1)
    c = Cache(own, "f16", 1, 64, 16, 4)
    table = np.tile(np.arange(4, dtype=np.int32), (1, 200))
    _fill(c, rng, table[:, :4], [64])
    c.send()
    q = rng.normal(0, 1, (1, 2, 64)).astype(np.float32)
    qb, ob, tb, lb = _up(own, q, q, table, np.array([12000], np.int32))
    own.graph_begin()
    with pytest.raises(E.ElmhError, match="during graph capture"):
        own.paged_attention_dev(qb.ptr, ob.ptr, 2, c.pages, tb.ptr, 1, 800, lb.ptr, 12000)
    own.graph_destroy(own.graph_end())
    own.paged_attention_dev(qb.ptr, ob.ptr, 2, c.pages, tb.ptr, 1, 800, lb.ptr, 12000)
    first = ob.download(q.shape, np.float32)
    own.graph_begin()
    own.paged_attention_dev(qb.ptr, ob.ptr, 2, c.pages, tb.ptr, 1, 800, lb.ptr, 12000)
    g = own.graph_end()
    ob.upload(np.zeros_like(q))
    own.graph_launch(g)
    own.synchronize()
    assert np.isfinite(first).all() and np.array_equal(ob.download(q.shape, np.float32), first)
    own.graph_destroy(g)
    _free(qb, ob, tb, lb)
    c.free()
    own.close()


def test_refusals_leave_the_context_usable(ctx):
    c = Cache(ctx, "f32", 1, 32, 16, 1, fill=0).send()
    b = ctx.buffer(4096)
    bad = E.KVPages(E.F32, 1, 40, 16, 1, b.ptr, b.ptr, None, None)
    with pytest.raises(E.ElmhError, match="head_dim"):
        ctx.paged_attention_dev(b.ptr, b.ptr + 64, 1, bad, b.ptr, 1, 1, b.ptr, 16)
    with pytest.raises(E.ElmhError, match="max_len"):
        ctx.paged_attention_dev(b.ptr, b.ptr + 64, 1, c.pages, b.ptr, 1, 1, b.ptr, 17)
    with pytest.raises(E.ElmhError, match="null"):
        ctx.paged_append_dev(None, b.ptr, 1, c.pages, b.ptr, 1, 1, b.ptr)
    with pytest.raises(E.ElmhError, match="overlap"):
        ctx.paged_read_dev(b.ptr, b.ptr, 2, c.pages, b.ptr, 1, 1, b.ptr, b.ptr, 16, 0)
    with pytest.raises(E.ElmhError, match="rot_dim"):
        ctx.rope_dev(b.ptr, b.ptr, 1, 1, 32, E.Rope(b.ptr, b.ptr, 4, 34, 0))
    with pytest.raises(E.ElmhError, match="theta"):
        ctx.rope_table_dev(b.ptr, b.ptr, 0, 4, 32, 0.5)
    ctx.rope_table_dev(b.ptr, b.ptr + 1024, 0, 4, 32, 10000.0)
    assert b.download((4, 16), np.float32)[0].tolist() == [1.0] * 16
    b.free()
    c.free()

"""elm_paged.h compiled by the host compiler and asked without a GPU: what the paged operators refuse, which page a position is
in (bad pages among them), how a sequence is split, the 4-bit rows' layout and the scaled rotary frequencies."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

from edgelm_amd import elmh as E

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = r"""
#include "elm_paged.h"
using namespace elmh;
static thread_local const char* last = "";
static int code(PagedFault f) { last = f.what ? f.what : ""; return f.code; }
extern "C" {
const char* what() { return last; }
int pages(const elmh_kv_pages* p) { return code(check_kv_pages(p)); }
int rows(const float* k, const float* v, int64_t n, int64_t row, int64_t head, const elmh_kv_pages* p, const int32_t* t, int ns,
         int mp, const int32_t* pos, const int32_t* seq, const elmh_rope* r, int written) {
  return code(check_paged_rows(k, v, n, row, head, p, t, ns, mp, pos, seq, r, written != 0));
}
int attn(const float* q, const float* o, int64_t qr, int nh, const elmh_kv_pages* p, const int32_t* t, int ns, int mp,
         const int32_t* lens, int ml, const elmh_rope* r) {
  return code(check_paged_attention(q, o, qr, nh, p, t, ns, mp, lens, ml, r));
}
int rope(const float* x, const float* y, int64_t T, int nh, int hd, int64_t xr, int64_t yr, const elmh_rope* r, const int32_t* p,
         int64_t p0) { return code(check_rope_rows(x, y, T, nh, hd, xr, yr, r, p, p0)); }
int table(const float* c, const float* s, int64_t p0, int64_t n, int rot, double th, const elmh_rope_scaling* sc) {
  return code(check_rope_table(c, s, p0, n, rot, th, sc));
}
int alone(int dt, int hd, int workgroups) { return part_alone(dt, hd, workgroups); }
int64_t page_of(const int32_t* row, int mp, int64_t np, int pos, int ps) { return kv_page_of(row, mp, np, pos, page_magic(ps)); }
int page_index_of(int pos, int ps) { return page_index(pos, page_magic(ps)); }
int extra(int dt, int hd, int rows, int n, int max_len) { return part_extra(part_workgroups(dt, hd), rows, n, max_len); }
int size(int dt, int hd, int rows, int n, int max_len, int extra, int total) {
  return part_size(total, part_rule(part_workgroups(dt, hd), rows, n, max_len, extra));
}
int count(int units, int per) { return part_count(units, part_inverse(per)); }
int begin(int units, int part, int parts) { return part_begin(units, part, parts); }
int ceil_div_of(int n, int d) { return ceil_of(n, ceil_div(d)); }
int kbyte(int d, int hd) { return q4_key_byte(d, hd); }
int vbyte(int d, int hd) { return q4_value_byte(d, hd); }
double freq(int rot, double th, const elmh_rope_scaling* sc, int i) {
  return rope_scaled(rope_band(rot, th, sc), std::pow(th, -2.0 * i / rot), i);
}
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "edgelm_amd", "csrc"),
                    "-I", os.path.join(ROOT, "include"), str(d / "shim.cpp"), "-o", str(d / "paged.so")], check=True)
    lib = C.CDLL(str(d / "paged.so"))
    v, i, l, f = C.c_void_p, C.c_int, C.c_int64, C.c_double
    p, r, s = C.POINTER(E.KVPages), C.POINTER(E.Rope), C.POINTER(E.RopeScaling)
    lib.what.restype = C.c_char_p
    lib.pages.argtypes = [p]
    lib.rows.argtypes = [v, v, l, l, l, p, v, i, i, v, v, r, i]
    lib.attn.argtypes = [v, v, l, i, p, v, i, i, v, i, r]
    lib.rope.argtypes = [v, v, l, i, i, l, l, r, v, l]
    lib.table.argtypes = [v, v, l, l, i, f, s]
    lib.page_of.argtypes, lib.page_of.restype = [v, i, l, i, i], l
    lib.freq.argtypes, lib.freq.restype = [i, f, s, i], f
    return lib


A = 0x1000  # an address: the checks read nothing through it


def _pages(**kw):
    d = dict(dtype=E.Q8, n_kv=8, head_dim=128, page_size=16, n_pages=100, k=A, v=A, k_scale=A, v_scale=A)
    d.update(kw)
    return E.KVPages(**d)


def _rope(**kw):
    d = dict(cos=A, sin=A, max_pos=4096, rot_dim=128, interleaved=0)
    d.update(kw)
    return E.Rope(**d)


@pytest.mark.parametrize("code,kw", [
    (0, {}), (0, dict(dtype=E.F32, k_scale=None, v_scale=None)), (0, dict(dtype=E.BF16)), (0, dict(page_size=4096)), (0, dict(page_size=48)),
    (0, dict(n_pages=2**31 - 1, n_kv=1)), (0, dict(n_pages=2**29 - 1)), (1, dict(n_pages=2**29)), (1, dict(n_pages=2**25, page_size=256)),
    (4, dict(dtype=3)), (4, dict(dtype=-1)), (4, dict(head_dim=80)), (4, dict(head_dim=160)), (4, dict(head_dim=0)), (4, dict(head_dim=512)),
    (1, dict(page_size=8)), (1, dict(page_size=24)), (1, dict(page_size=0)), (1, dict(page_size=8192)), (1, dict(n_kv=0)), (1, dict(n_kv=1025)),
    (1, dict(n_pages=0)), (1, dict(n_pages=2**31)), (1, dict(k=None)), (1, dict(v=None)), (1, dict(k=A + 8)), (1, dict(v=A + 4)),
    (1, dict(k_scale=None)), (1, dict(v_scale=None)), (1, dict(k_scale=A + 4)), (1, dict(dtype=E.Q4, v_scale=None)),
])
def test_pages(host, code, kw):
    assert host.pages(_pages(**kw)) == code, host.what()


def test_null_pages(host):
    assert host.pages(None) == 1


ROWS = dict(k=A, v=2 * A, n=5, row=0, head=0, pages=_pages(), table=A, n_seqs=5, max_pages=10, pos=A, seq=None, rope=None, written=0)


@pytest.mark.parametrize("code,kw", [
    (0, {}), (0, dict(rope=_rope())), (0, dict(rope=_rope(rot_dim=2, interleaved=1))), (0, dict(n=1000, seq=A)),
    (0, dict(row=128, head=5 * 128, written=1)), (0, dict(row=4096, head=128, written=1)), (0, dict(row=1, head=1)),
    (0, dict(k=2 * A)), (1, dict(k=2 * A, written=1)),
    (1, dict(k=None)), (1, dict(v=None)), (1, dict(pos=None)), (1, dict(table=None)), (1, dict(n=0)), (1, dict(n=-3)), (1, dict(n=6)),
    (0, dict(n=2**23, seq=A)), (1, dict(n=2**23 + 1, seq=A)), (1, dict(n_seqs=0)), (1, dict(max_pages=0)), (1, dict(max_pages=2**27)), (1, dict(row=-1)), (1, dict(head=-1)),
    (1, dict(row=2**41)), (1, dict(rope=_rope(rot_dim=130))), (1, dict(rope=_rope(rot_dim=3))), (1, dict(rope=_rope(rot_dim=0))),
    (1, dict(rope=_rope(cos=None))), (1, dict(rope=_rope(sin=None))), (1, dict(rope=_rope(max_pos=0))), (1, dict(rope=_rope(interleaved=2))),
    # rows written over each other
    (1, dict(row=128, head=128, written=1)), (1, dict(row=64, head=5 * 128, written=1)), (1, dict(row=1024, head=100, written=1)),
    (1, dict(row=128, head=4 * 128, written=1)),
    (4, dict(pages=_pages(head_dim=100))), (1, dict(pages=None)),
])
def test_rows(host, code, kw):
    assert host.rows(*{**ROWS, **kw}.values()) == code, host.what()


ATTN = dict(q=A, out=2 * A, q_row=0, n_heads=32, pages=_pages(), table=A, n_seqs=5, max_pages=10, lens=A, max_len=160, rope=None)


@pytest.mark.parametrize("code,kw", [
    (0, {}), (0, dict(n_heads=8)), (0, dict(n_heads=8 * 256)), (0, dict(max_len=1)), (0, dict(rope=_rope(max_pos=160))), (0, dict(q_row=5000)),
    (0, dict(n_seqs=4096)), (1, dict(n_seqs=4096, max_pages=2**24, max_len=2**24)),
    (1, dict(q=None)), (1, dict(out=None)), (1, dict(out=A)), (1, dict(lens=None)), (1, dict(table=None)), (1, dict(n_heads=0)), (1, dict(n_heads=33)),
    (1, dict(n_heads=4)), (1, dict(n_heads=8 * 257)), (1, dict(max_len=0)), (1, dict(max_len=161)), (1, dict(n_seqs=0)), (1, dict(n_seqs=4097)),
    (1, dict(q_row=-1)), (1, dict(rope=_rope(max_pos=159))), (1, dict(pages=_pages(k=None))), (4, dict(pages=_pages(dtype=7))),
])
def test_attention(host, code, kw):
    assert host.attn(*{**ATTN, **kw}.values()) == code, host.what()


ROPE = dict(x=A, y=2 * A, T=7, n_heads=3, hd=64, x_row=0, y_row=0, rope=_rope(rot_dim=64), pos=None, pos0=0)


@pytest.mark.parametrize("code,kw", [
    (0, {}), (0, dict(y=A)), (0, dict(y=A, x_row=200, y_row=200)), (0, dict(pos=A, pos0=-5)), (0, dict(pos0=4089)), (0, dict(hd=80)), (0, dict(x_row=1)),
    (1, dict(x=None)), (1, dict(y=None)), (1, dict(rope=None)), (1, dict(T=0)), (1, dict(T=2**24 + 1)), (1, dict(n_heads=0)), (1, dict(n_heads=4097)),
    (1, dict(hd=63)), (1, dict(hd=62)), (1, dict(hd=1026)), (1, dict(y_row=191)), (1, dict(y=A, x_row=200)), (1, dict(pos0=4090)), (1, dict(pos0=-1)),
    (1, dict(x_row=-1)), (1, dict(rope=_rope(rot_dim=66))),
])
def test_rope(host, code, kw):
    assert host.rope(*{**ROPE, **kw}.values()) == code, host.what()


TABLE = dict(c=A, s=A, pos0=0, n=100, rot=64, theta=10000.0, scaling=None)
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("code,kw", [
    (0, {}), (0, dict(scaling=E.RopeScaling(E.ROPE_LINEAR, 4.0))), (0, dict(scaling=E.RopeScaling(E.ROPE_YARN, 4.0, 4096))),
    (0, dict(scaling=E.RopeScaling(E.ROPE_BANDS, 8.0, 8192, 1.0, 4.0))), (0, dict(pos0=2**31 - 101)),
    (1, dict(c=None)), (1, dict(s=None)), (1, dict(pos0=-1)), (1, dict(n=0)), (1, dict(pos0=2**31 - 100)), (1, dict(rot=0)), (1, dict(rot=5)),
    (1, dict(rot=1026)), (1, dict(theta=1.0)), (1, dict(theta=NAN)), (1, dict(theta=INF)),
    (4, dict(scaling=E.RopeScaling(0, 4.0))), (4, dict(scaling=E.RopeScaling(4, 4.0))), (1, dict(scaling=E.RopeScaling(E.ROPE_LINEAR, 0.5))),
    (1, dict(scaling=E.RopeScaling(E.ROPE_LINEAR, NAN))), (1, dict(scaling=E.RopeScaling(E.ROPE_LINEAR, 2.0, magnitude=0.0))),
    (1, dict(scaling=E.RopeScaling(E.ROPE_YARN, 4.0, 0.0))), (1, dict(scaling=E.RopeScaling(E.ROPE_YARN, 4.0, 4096, 32.0, 1.0))),
    (1, dict(scaling=E.RopeScaling(E.ROPE_BANDS, 4.0, 4096, 0.0, 1.0))), (1, dict(scaling=E.RopeScaling(E.ROPE_BANDS, 4.0, INF, 1.0, 4.0))),
])
def test_rope_table(host, code, kw):
    assert host.table(*{**TABLE, **kw}.values()) == code, host.what()


def test_page_of_a_position(host):
    """Positions past the row, negative ones, and entries that name no page of the pool have none."""
    row = np.array([3, -1, 99, 100, 2**31 - 1, -2**31, 0], np.int32)
    p = row.ctypes.data
    for ps in (16, 48, 4096):
        for i, want in enumerate([3, -1, 99, -1, -1, -1, 0]):
            for pos in (i * ps, i * ps + ps - 1):
                assert host.page_of(p, len(row), 100, pos, ps) == want
        assert host.page_of(p, len(row), 100, len(row) * ps, ps) == -1
        assert host.page_of(p, len(row), 100, -1, ps) == -1
        assert host.page_of(p, len(row), 100, -2**31, ps) == -1
        assert host.page_of(p, len(row), 100, 2**31 - 1, ps) == -1
        assert host.page_of(p, len(row), 100, 2**28, ps) == -1


def test_page_index_is_the_quotient(host):
    """At every page size, positions about each multiple and at the largest."""
    for ps in range(16, 4097, 16):
        last = 2**28 - 1
        for pos in [0, 1, ps - 1, ps, ps + 1, 7 * ps - 1, 7 * ps, last, last - 1, last // ps * ps, last // ps * ps - 1, 2**27 // ps * ps, 2**27 // ps * ps - 1]:
            assert host.page_index_of(pos, ps) == pos // ps, (pos, ps)


def test_ceil_of_a_quotient(host):
    rng = np.random.default_rng(1)
    for d in list(range(1, 1025, 31)) + [2, 3, 64, 512, 1024]:
        for n in [0, 1, d - 1, d, d + 1, 5 * d, 5 * d + 1, 2**30, 2**30 - 1] + rng.integers(0, 2**30, 20).tolist():
            got, want = host.ceil_div_of(n, d), -(-n // d)
            assert want <= got <= want + (n + d >= 2**32 // d), (n, d)


def test_parts_fit_their_slots(host):
    """Whatever the lengths below the host's bound, the parts of all sequences (one of an empty one) are no more than n_seqs +
    extra, and a batch of short sequences is not split."""
    rng = np.random.default_rng(0)
    for rows, hd, dt in ((1, 64, E.F32), (3, 64, E.Q8), (8, 128, E.BF16), (8, 128, E.Q4), (8, 256, E.F16), (40, 128, E.Q8), (1024, 128, E.F32), (16384, 32, E.Q4)):
        for n in (1, 2, 7, 64, 65, 300, 4096):
            for max_len in (1, 31, 128, 512, 513, 4096, 100003, 2**23, 2**28):
                if n * max_len > 2**35:
                    continue
                extra = host.extra(dt, hd, rows, n, max_len)
                assert 1 <= extra <= 1024
                top = -(-max_len // 32)
                for units in (np.full(n, top), rng.integers(0, top + 1, n), np.where(np.arange(n) == n // 2, top, 0), np.zeros(n, int),
                              np.where(rng.random(n) < 0.5, top, 1)):
                    per = host.size(dt, hd, rows, n, max_len, extra, int(units.sum()))
                    parts = [host.count(int(u), per) for u in units]
                    assert per >= 4 and min(parts) >= 1 and sum(parts) <= n + extra, (rows, n, max_len)
                    assert max(parts) <= extra + 1
                    assert max_len > 512 or max(parts) == 1


def test_parts_cover_a_sequence(host):
    """From the first unit to the last, in order, none empty while there are as many units as parts."""
    for units in (1, 2, 4, 5, 13, 100, 999, 4097, 2**18, 2**23 - 1, 2**23):
        for per in (4, 5, 12, 16, 33, 64, 1000, 8192, 2**23):
            parts = host.count(units, per)
            # the quotient is taken 2^-20 low, give or take two roundings of 2^-24; one is added to its floor
            assert parts == -(-units // per) or (units > 2**19 and abs(parts - units / per) <= 1 + units / per * 2.0**-19), (units, per)
            if parts > 1100:
                continue
            at = [host.begin(units, p, parts) for p in range(parts + 1)]
            assert at[0] == 0 and at[-1] == units
            assert all(b > a for a, b in zip(at, at[1:]))
            assert max(b - a for a, b in zip(at, at[1:])) <= max(per, units / parts) + 2
    assert host.count(0, 4) == 1


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 192, 256])
def test_q4_rows(host, hd):
    """Each byte of a row holds two neighbouring values, every byte once."""
    for f in (host.kbyte, host.vbyte):
        assert sorted(f(d, hd) for d in range(0, hd, 2)) == list(range(hd // 2))
        assert all(f(d + 1, hd) == f(d, hd) for d in range(0, hd, 2))
    assert host.kbyte(32 + 8 + 2, hd) == hd // 8 + 5 if hd > 32 else True  # group 1, c = 1, byte 1
    assert host.vbyte(34, hd) == hd // 32 + 1 if hd > 32 else True         # group 1, i = 1


def test_page_bytes():
    assert E.kv_page_bytes(E.F32, 3, 64, 16) == (3 * 16 * 256, 0)
    assert E.kv_page_bytes(E.F16, 8, 96, 32) == E.kv_page_bytes(E.BF16, 8, 96, 32) == (8 * 32 * 192, 0)
    assert E.kv_page_bytes(E.Q8, 8, 128, 48) == (8 * 48 * 128, 8 * 48 * 4)
    assert E.kv_page_bytes(E.Q4, 2, 256, 16) == (2 * 16 * 128, 2 * 16 * 8 * 4)
    for bad in ((3, 8, 128, 16), (E.Q8, 8, 100, 16), (E.Q8, 0, 128, 16), (E.Q8, 8, 128, 20)):
        with pytest.raises(E.ElmhError):
            E.kv_page_bytes(*bad)


def test_scaled_frequencies(host):
    """Against the definitions, in another form than the header's: relative error a few roundings of f64 (2^-53), the blend's
    cancellation at most 32 of them."""
    for rot, th, orig, fac in ((64, 10000.0, 2048, 4.0), (128, 500000.0, 8192, 8.0), (96, 1e6, 32768, 32.0), (2, 10000.0, 100, 2.0)):
        for i in range(rot // 2):
            f = th ** (-2.0 * i / rot)
            lam = 2 * math.pi / f
            want = {None: f, E.ROPE_LINEAR: f / fac}
            lo, hi = 1.0, 4.0
            if lam < orig / hi:
                want[E.ROPE_BANDS] = f
            elif lam > orig / lo:
                want[E.ROPE_BANDS] = f / fac
            else:
                s = (orig / lam - lo) / (hi - lo)
                want[E.ROPE_BANDS] = (1 - s) * f / fac + s * f
            a, b = (rot * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(th)) for t in (32.0, 1.0))
            a, b = max(math.floor(a), 0), min(math.ceil(b), rot - 1)
            r = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            want[E.ROPE_YARN] = f / fac * r + f * (1 - r)
            for kind, w in want.items():
                sc = None if kind is None else E.RopeScaling(kind, fac, orig, lo, hi if kind == E.ROPE_BANDS else 32.0)
                assert abs(host.freq(rot, th, sc, i) / w - 1) <= 64 * 2.0 ** -53, (kind, rot, i)


def test_short_sequences_stay_whole(host):
    """The longest sequence that is not split, in units of 32 positions: sixteen, fewer where a unit takes long and the batch is
    few workgroups, never under a part's least."""
    for dt in (E.F32, E.F16, E.BF16, E.Q8, E.Q4):
        for hd in (32, 64, 96, 128, 192, 256):
            assert host.alone(dt, hd, 65) == 16
            for workgroups in (1, 64):
                assert host.alone(dt, hd, workgroups) == min(16, 2048 // (hd * (2 if dt == E.F32 else 1)))
                assert 4 <= host.alone(dt, hd, workgroups) <= 16

"""The 4-bit paged cache and the plan without a GPU: refusals of the entry
points, descriptor layouts, and the page layout's arithmetic."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from paged_common import HD, f64
from q4_common import BF16_MAX, K_AT, V_AT, bf16_bits_toward, get, put, quantise, values
from test_paged_host import COMMON, P, TOKENS, _append, _attn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _read():
    from vx27_amd import lib as L
    return L.PagedReadDesc(n_kv=4, hd=256, page_size=64, n_pages=9, n_rows=5, slots=P, k_pages=P, v_pages=P, out_dtype=L.F32, k_out=P, v_out=P)


def _plan():
    from vx27_amd import lib as L
    d = L.PagedPlanDesc(B=2, page_size=64, n_pages=9, max_pages=4, n_tok=5)
    for i, n in enumerate(("new_tok", "ended", "len", "next_pos", "table", "free_pages", "n_free", "took", "q_start", "len_out",
                           "next_pos_out", "n_free_out", "slot", "pos", "seq")):
        setattr(d, n, (i + 1) * P)
    return d


MAKE = {"append_q4": _append, "attn_q4": _attn, "read_q4": _read, "plan": _plan}
BIG = {"page_size": 1 << 20, "n_pages": 1 << 19, "max_pages": 1, "n_kv": 1, "n_q": 6}      # 2^34 blocks
CASES = [(k, *c) for k in ("append_q4", "attn_q4") for c in COMMON + TOKENS] + [
    ("append_q4", {"rope_dim": 7}, "rope_dim"), ("append_q4", {"in_dtype": 2}, "in_dtype"), ("append_q4", {"k_new": None}, "null pointer"),
    ("append_q4", {"n_tok": 2 ** 31 - 1, "max_T": 2 ** 25 + 1}, "2^25"), ("append_q4", {"q_head_stride": 258}, "multiples of 4"), ("append_q4", BIG, "2^32 blocks"),
    ("attn_q4", {"n_q": 68}, "k <= 16"), ("attn_q4", {"window": -1}, "negative"), ("attn_q4", {"out_dtype": 3}, "out_dtype"),
    ("attn_q4", {"gate": P + 8}, "aligned"), ("attn_q4", {"acc": P, "acc_stride": 256}, "acc must be NULL"), ("attn_q4", BIG, "2^32 blocks"),
    ("read_q4", {"hd": 128}, "hd must be 256"), ("read_q4", {"n_kv": 0}, "n_kv"), ("read_q4", {"n_kv": 1025}, "n_kv"),
    ("read_q4", {"page_size": 48}, "page_size"), ("read_q4", {"n_pages": 0}, "n_pages"), ("read_q4", {"n_pages": 1 << 25}, "2^31"),
    ("read_q4", {"n_rows": -1}, "n_rows"), ("read_q4", {"n_rows": (1 << 25) + 1}, "n_rows"), ("read_q4", {"out_dtype": 2}, "out_dtype"),
    ("read_q4", {"slots": None}, "null pointer"), ("read_q4", {"k_pages": None}, "null pointer"), ("read_q4", {"v_out": P + 8}, "aligned"),
    ("plan", {"B": 0}, "1 <= B"), ("plan", {"B": 65536}, "1 <= B"), ("plan", {"page_size": 16}, "page_size"), ("plan", {"n_pages": 0}, "n_pages"),
    ("plan", {"max_pages": 0}, "max_pages"), ("plan", {"n_tok": -1}, "n_tok"), ("plan", {"max_pages": 1 << 25}, "2^30"),
    ("plan", {"n_pages": 1 << 25}, "2^31"), ("plan", {"table": None}, "null pointer"), ("plan", {"took": None}, "null pointer"),
    ("plan", {"n_free_out": None}, "null pointer"), ("plan", {"next_pos_out": None}, "go together"), ("plan", {"next_pos": None}, "go together"),
    ("plan", {"took": 9 * P, "len_out": 9 * P}, "overlap"), ("plan", {"q_start": 3 * P}, "overlap"), ("plan", {"slot": 5 * P + 28}, "overlap"),
    ("plan", {"free_pages": 5 * P - 32}, "overlap"), ("plan", {"len_out": 3 * P + 4}, "overlap"), ("plan", {"seq": 14 * P - 4}, "overlap")]


@pytest.mark.parametrize("kind,change,message", CASES)
def test_refusals(kind, change, message):
    """Every check names itself and comes before anything touches a device."""
    from vx27_amd import lib as L
    d = MAKE[kind]()
    for k, v in change.items():
        if hasattr(d, k):
            setattr(d, k, v)
    fn = getattr(L.lib(), "vx27_hip_paged_" + kind)
    assert fn(None, C.byref(d)) == -1
    msg = L.lib().vx27_hip_last_error().decode()
    assert message in msg and "vx27_hip_paged_" + kind in msg, msg


@pytest.mark.parametrize("kind,change", [(k, {}) for k in MAKE] + [
    ("plan", {"len_out": 3 * P, "next_pos_out": 4 * P, "n_free_out": 7 * P}), ("plan", {"ended": None, "slot": None, "pos": None, "seq": None}),
    ("plan", {"next_pos": None, "next_pos_out": None}), ("read_q4", {"v_pages": None, "v_out": None})])
def test_good_descriptors_reach_the_context(kind, change):
    from vx27_amd import lib as L
    d = MAKE[kind]()
    for k, v in change.items():
        setattr(d, k, v)
    fn = getattr(L.lib(), "vx27_hip_paged_" + kind)
    assert fn(None, C.byref(d)) == -1
    assert b"null context" in L.lib().vx27_hip_last_error()
    assert fn(None, None) == -1
    assert b"null descriptor" in L.lib().vx27_hip_last_error()


def test_layouts(tmp_path):
    from vx27_amd import lib as L
    names = {"vx27_paged_read_desc": L.PagedReadDesc, "vx27_paged_plan_desc": L.PagedPlanDesc}
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "vx27_hip.h"', "int main(void) {",
           '    printf("%d\\n%d\\n%d\\n%d\\n", VX27_Q4_BLOCK_BYTES, VX27_Q4_SPLIT_ROWS, VX27_Q4_SPLIT_ROWS_F32, VX27_Q4_SPLIT_TILES);']
    want = [L.Q4_BLOCK_BYTES, L.Q4_SPLIT_ROWS, L.Q4_SPLIT_ROWS_F32, L.Q4_SPLIT_TILES]
    for c, py in names.items():
        src.append(f'    printf("%zu\\n", sizeof({c}));')
        want.append(C.sizeof(py))
        for f, _ in py._fields_:
            src.append(f'    printf("%zu\\n", offsetof({c}, {f}));')
            want.append(getattr(py, f).offset)
    (tmp_path / "l.c").write_text("\n".join(src + ["    return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{ROOT}/include", str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout
    assert [int(x) for x in out.split()] == want


@pytest.mark.parametrize("at", [K_AT, V_AT], ids=["K", "V"])
def test_layout_places(at):
    """Every code, scale and minimum of a block has a place of its own, and all bytes are places."""
    byte, shift, s, m = at
    assert len({(int(b), int(x)) for b, x in zip(byte.ravel(), shift.ravel())}) == 32 * HD and byte.max() == 4095
    places = sorted({int(x) for x in s.ravel()} | {int(x) for x in m.ravel()})
    assert places == list(range(4096, 4608, 2))
    r = np.random.default_rng(1)
    blk = r.integers(0, 256, 4608).astype(np.uint8)
    rows = [(r.integers(0, 16, HD).astype(np.uint8), r.integers(0, 65536, 4).astype(np.uint16), r.integers(0, 65536, 4).astype(np.uint16)) for _ in range(32)]
    for i in r.permutation(32):
        put(blk, at, i, *rows[i])
    for i in range(32):
        assert all(np.array_equal(a, b) for a, b in zip(get(blk, at, i), rows[i]))


def test_quantise_is_the_definition():
    """m and s by search over all bf16 numbers, codes by exact rational arithmetic."""
    from fractions import Fraction as F
    r = np.random.default_rng(2)
    allb = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    v = f64(allb)
    fin = np.isfinite(v)
    order = np.unique(v[fin])
    rows = [r.standard_normal(HD), np.round(r.standard_normal(HD) * 8) / 8, r.integers(-20, 20, HD) / 4.0, 1e-39 * r.standard_normal(HD),
            np.tile([BF16_MAX, -BF16_MAX], 128), np.zeros(HD), np.full(HD, 2.0 ** -140)]
    for x in rows:
        x = x.astype(np.float32).astype(np.float64)
        c, s, m = quantise(x)
        for g in range(4):
            y = x[64 * g:64 * g + 64]
            mm = order[np.searchsorted(order, y.min(), side="right") - 1]
            ss = order[np.searchsorted(order, (y.max() - mm) / 15, side="left")]
            assert f64(m[g]) == mm and f64(s[g]) == ss
            for i, z in enumerate(y):
                t = (F(float(z)) - F(float(mm))) / F(float(ss)) if ss else F(0)
                assert int(c[64 * g + i]) == round(t)       # (Fraction rounds ties to even)
        assert np.all(np.abs(values(c, s, m) - x).reshape(4, 64) <= f64(s)[:, None] / 2 * (1 + 2.0 ** -40))
    assert f64(bf16_bits_toward(np.array([1.001, -1.001, 0.0]), True)).tolist() == [1.0078125, -1.0, 0.0]


def test_launch_of_a_limit():
    """The append's grid at its largest max_T: below 2^32 threads, 256 a workgroup, 12 of them a 32-row block."""
    assert ((2 ** 25 + 30) // 32 + 1) * 12 * 256 < 2 ** 32

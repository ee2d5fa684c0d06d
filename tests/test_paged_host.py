"""The paged cache without a GPU: refusals of the entry points, descriptor
layouts, and the index arithmetic that the kernels share, run on the host."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20      # an aligned address: nothing is dereferenced before the checks are over


def _append():
    from vx27_amd import lib as L
    return L.PagedAppendDesc(B=2, n_q=24, n_kv=4, hd=256, rope_dim=64, rope_theta=1e7, rope_yarn=1.0, page_size=64, n_pages=9,
                             max_pages=4, table=P, len=P, q_start=P, n_tok=5, max_T=3, in_dtype=L.F32, q=P, k_new=P, v_new=P,
                             q_norm_w=P, k_norm_w=P, q_out=P, k_pages=P, v_pages=P)


def _attn():
    from vx27_amd import lib as L
    return L.PagedAttnDesc(B=2, n_q=24, n_kv=4, hd=256, page_size=64, n_pages=9, max_pages=4, table=P, len=P, q_start=P, n_tok=5,
                           max_T=3, q=P, k_pages=P, v_pages=P, out=P)


def _evict():
    from vx27_amd import lib as L
    return L.PagedEvictDesc(B=2, n_kv=4, hd=256, page_size=64, n_pages=9, max_pages=4, table=P, len=P, budget=100, n_sink=4,
                            n_recent=8, acc=P, acc_stride=256, k_pages=P, v_pages=P, dst_table=P, dst_max_pages=2,
                            dst_len=2 * P, acc_out=4 * P, acc_out_stride=100, kept=P)


MAKE = {"append": _append, "attn": _attn, "evict": _evict}
COMMON = [({"hd": 128}, "hd must be 256"), ({"B": 0}, "1 <= B"), ({"B": 65536}, "1 <= B"), ({"n_kv": 0}, "n_kv"),
          ({"page_size": 0}, "page_size"), ({"page_size": 48}, "page_size"), ({"n_pages": 0}, "n_pages"),
          ({"max_pages": 0}, "max_pages"), ({"max_pages": 1 << 25}, "2^30"), ({"table": None}, "null page table"),
          ({"len": None}, "null page table or lengths"), ({"k_pages": None}, "null pointer"), ({"v_pages": None}, "null pointer"),
          ({"k_pages": P + 8}, "aligned"), ({"v_pages": P + 8}, "aligned")]
TOKENS = [({"n_tok": -1}, "max_T <= n_tok"), ({"max_T": 6}, "max_T <= n_tok"), ({"max_T": 0}, "max_T must be"),
          ({"q_start": None}, "q_start may be NULL"), ({"n_q": 26}, "n_q = k"), ({"n_q": 2}, "n_q = k")]
CASES = [(k, *c) for k in MAKE for c in COMMON] + [(k, *c) for k in ("append", "attn") for c in TOKENS] + [
    ("append", {"in_dtype": 2}, "in_dtype"), ("append", {"rope_dim": 7}, "rope_dim"), ("append", {"rope_dim": 258}, "rope_dim"),
    ("append", {"rope_dim": -2}, "rope_dim"), ("append", {"k_new": None}, "null pointer"), ("append", {"v_new": None}, "null pointer"),
    ("append", {"k_norm_w": None}, "null pointer"), ("append", {"q_out": None}, "null pointer"), ("append", {"q_norm_w": None}, "null pointer"),
    ("append", {"q": P + 8}, "16-byte aligned"), ("append", {"q": P + 4, "in_dtype": 1}, "8-byte aligned"),
    ("append", {"q_head_stride": 258}, "multiples of 4"), ("append", {"kv_tok_stride": 1026}, "multiples of 4"),
    ("append", {"q_out": P + 2}, "16-byte aligned"),
    ("attn", {"n_q": 68}, "k <= 16"), ("attn", {"window": -1}, "negative"), ("attn", {"n_sink": -1}, "negative"),
    ("attn", {"q": None}, "null pointer"), ("attn", {"out": None}, "null pointer"), ("attn", {"out_dtype": 3}, "out_dtype"),
    ("attn", {"gate": P, "gate_dtype": -1}, "gate_dtype"), ("attn", {"q": P + 8}, "aligned"), ("attn", {"gate": P + 8}, "aligned"),
    ("attn", {"q_tok_stride": 6148}, "multiples of 8"), ("attn", {"acc": P, "acc_stride": 255}, "acc_stride"),
    ("evict", {"budget": 0}, "budget"), ("evict", {"n_sink": -1}, "n_sink"), ("evict", {"n_recent": 97}, "n_recent"),
    ("evict", {"acc": None}, "null pointer"), ("evict", {"dst_table": None}, "null pointer"), ("evict", {"dst_len": None}, "null pointer"),
    ("evict", {"acc_stride": 255}, "acc_stride"), ("evict", {"acc_out_stride": 99}, "acc_out_stride"),
    ("evict", {"dst_max_pages": 1}, "dst_max_pages"), ("evict", {"dst_max_pages": 0}, "dst_max_pages"),
    ("evict", {"acc_out": P}, "overlap acc"), ("evict", {"dst_len": P}, "overlap len"),
    ("evict", {"dst_len": 8 * P + 16, "table": 8 * P}, "overlap table")]


@pytest.mark.parametrize("kind,change,message", CASES)
def test_refusals(kind, change, message):
    """Every check names itself and comes before anything touches a device."""
    from vx27_amd import lib as L
    d = MAKE[kind]()
    for k, v in change.items():
        setattr(d, k, v)
    fn = getattr(L.lib(), "vx27_hip_paged_" + kind)
    assert fn(None, C.byref(d)) == -1
    msg = L.lib().vx27_hip_last_error().decode()
    assert message in msg and "vx27_hip_paged_" + kind in msg, msg


@pytest.mark.parametrize("kind", list(MAKE))
def test_good_descriptors_reach_the_context(kind):
    from vx27_amd import lib as L
    fn = getattr(L.lib(), "vx27_hip_paged_" + kind)
    assert fn(None, C.byref(MAKE[kind]())) == -1
    assert b"null context" in L.lib().vx27_hip_last_error()
    assert fn(None, None) == -1
    assert b"null descriptor" in L.lib().vx27_hip_last_error()


def test_layouts(tmp_path):
    from vx27_amd import lib as L
    names = {"vx27_paged_append_desc": L.PagedAppendDesc, "vx27_paged_attn_desc": L.PagedAttnDesc,
             "vx27_paged_evict_desc": L.PagedEvictDesc}
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "vx27_hip.h"', "int main(void) {"]
    want = []
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


def test_index_arithmetic(tmp_path):
    """tests/c/paged_host.hip: tile lists against every (token, row) pair, clamps against values from anywhere."""
    from vx27_amd import build as B
    exe = str(tmp_path / "paged_host")
    r = subprocess.run([B.HIPCC, "-O1", f"--offload-arch={B.ARCH}", "-std=c++17", f"-I{B.INC}", f"-I{B.CSRC}", "-Wno-unused-result",
                        os.path.join(ROOT, "tests", "c", "paged_host.hip"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    out = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr


@pytest.mark.parametrize("change,message", [
    ({"n_q": 4097 * 4}, "k <= 4096"), ({"n_q": 32768 * 4}, "k <= 4096"),
    ({"n_tok": 2 ** 31 - 1, "max_T": 2 ** 26 + 1}, "2^26"), ({"n_tok": 2 ** 31 - 1, "max_T": 2 ** 31 - 1}, "2^26")])
def test_append_limits(change, message):
    """Row / group as a high product is exact for 8 tokens of up to 4096 heads (test_group_of_a_row), and a launch holds
    2^32 threads a dimension."""
    from vx27_amd import lib as L
    d = _append()
    for k, v in change.items():
        setattr(d, k, v)
    assert L.lib().vx27_hip_paged_append(None, C.byref(d)) == -1
    assert message in L.lib().vx27_hip_last_error().decode()


def test_group_of_a_row():
    """The kernels' row / group: high 32 bits of row * (floor(2^32 / group) + 1)."""
    def div(r, g):
        return r * (2 ** 32 // g + 1) >> 32
    for g in [*range(2, 300), 1000, 2047, 2048, 4095, 4096]:
        for t in (0, 1, 3, 7):                        # a workgroup of the append: 8 tokens
            assert div(t * g, g) == t and div(t * g + g - 1, g) == t
    for g in range(2, 17):                            # the attention: rows below 2^28
        for t in [*range(100), *((1 << 28) // g - k for k in range(1, 100))]:
            assert div(t * g, g) == t and div(t * g + g - 1, g) == t
    assert div(8 * 32768 - 1, 32768) == 8             # past the limit the last row would be read as a ninth token's


def test_launch_of_a_limit():
    """The append's grid at its largest max_T: below 2^32 threads, 256 a workgroup."""
    assert ((2 ** 26 + 30) // 32 + 1) * 5 * 256 < 2 ** 32


@pytest.mark.parametrize("change,message", [
    ({"acc_out": 4 * P, "kept": 4 * P + 64}, "acc_out must not overlap kept"),
    ({"acc_out": 8 * P, "len": 8 * P + 3196}, "acc_out must not overlap len"),
    ({"acc_out": 8 * P, "table": 8 * P + 3196}, "acc_out must not overlap table"),
    ({"acc_out": 8 * P, "dst_table": 8 * P - 12}, "acc_out must not overlap dst_table"),
    ({"acc_out": 2 * P}, "acc_out must not overlap dst_len"),
    ({"dst_len": 8 * P, "dst_table": 8 * P}, "dst_len must not overlap dst_table"),
    ({"dst_len": 8 * P, "kept": 8 * P - 3196}, "dst_len must not overlap kept"),
    ({"dst_len": 8 * P, "acc": 8 * P - 4}, "dst_len must not overlap acc")])
def test_eviction_outputs_that_overlap(change, message):
    """paged_move reads lengths, tables and kept rows that another workgroup's outputs would change under it."""
    from vx27_amd import lib as L
    d = _evict()
    for k, v in change.items():
        setattr(d, k, v)
    assert L.lib().vx27_hip_paged_evict(None, C.byref(d)) == -1
    assert message in L.lib().vx27_hip_last_error().decode()

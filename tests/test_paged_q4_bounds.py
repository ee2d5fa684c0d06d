"""The bounds of the 4-bit paged attention's GPU tests hold for the kernels'
arithmetic, and for no result with a mistake planted in it."""
import numpy as np
import pytest

import q4_bounds as Q
from paged_common import HD, f64
from q4_common import Batch4, values
from vx27_amd import workloads as W

CASES = [   # kernel, lens, new, n_q, n_kv, page, window, sink
    ("paged_rows_q4", [130, 70, 1, 33], [130, 1, 1, 30], 24, 4, 64, 0, 0),
    ("paged_rows_q4", [1200, 900], [43, 200], 16, 1, 128, 300, 33),
    ("paged_rows_q4", [3, 257], [3, 257], 10, 2, 64, 0, 5),
    ("paged_rows_q4", [1500], [43], 24, 4, 256, 0, 0),
    ("paged_rows_flat", [300, 500, 64], [260, 77, 64], 24, 4, 32, 90, 7),
    ("paged_rows_flat", [1500, 40], [150, 20], 8, 4, 64, 64, 2000),
    ("paged_q4_split", [1000, 7, 257], [1, 0, 1], 24, 4, 64, 0, 0),
    ("paged_q4_split", [900, 40, 64, 3, 700], [1] * 5, 24, 4, 64, 100, 4),
    ("paged_q4_split", [600, 77, 6, 1500], [6, 6, 6, 5], 24, 4, 64, 0, 0),
    ("paged_q4_split", [2500, 5], [9, 5], 24, 4, 96, 700, 40),
]


def batch(i):
    kernel, lens, new, n_q, n_kv, page, window, sink = CASES[i]
    return kernel, Batch4(lens, new, n_q, n_kv, page, window, sink, seed=2100 + i)


def bf16(x):
    return f64(W.bf16_bits(np.asarray(x, np.float32)))


def outputs(bt, kernel, out_bf16, plant=""):
    """The kernel's roundings in float64, of the weights, values and outputs, with a mistake if one is named."""
    out = np.zeros((bt.N, bt.n_q, HD))
    for b in range(bt.B):
        if not bt.lens[b] or not bt.new[b]:
            continue
        see, t0 = bt.seen(b), bt.start[b]
        if plant == "causal":
            see = np.ones_like(see)
        if plant == "next row":
            see = np.concatenate([see[1:], see[-1:]])
        (kc, ks, km), (vc, vs, vm) = bt.held(b)
        k, v = values(kc, ks, km), values(vc, vs, vm)
        if kernel != "paged_q4_split":
            k, v = Q.rounded(k), Q.rounded(v)
        k[np.isnan(k)] = 0                    # (rows that no token sees)
        v[np.isnan(v)] = 0
        for h in range(bt.n_q):
            g = h // bt.qg
            s = np.where(see, f64(bt.q)[t0:t0 + bt.new[b], h] @ k[:, g].T / 16.0, -np.inf)
            with np.errstate(all="ignore"):
                p = np.where(see, np.exp2((s - s.max(1, keepdims=True)) / np.log(2) - 1), 0.0)
            l = p.sum(1, keepdims=True)
            if plant == "part" and bt.lens[b] > 256:
                p[:, :128], l = 0, l           # (a part of the rows that the join leaves out)
            if plant == "tile" and bt.lens[b] > 256:
                p[:, 64:96] = 0
                l = p.sum(1, keepdims=True)
            vg, am = v[:, g], vm[:, g]
            if kernel == "paged_q4_split":
                hi = lambda x: f64((np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)) if out_bf16 else bf16(x)  # noqa: E731
                # weights p s of the codes and p of the minima, each in its two parts (or the first alone)
                parts = lambda x: hi(x) + (0.0 if plant == "one part" else -bf16(x - hi(x)) if plant == "sign" else bf16(x - hi(x)))  # noqa: E731
                o = np.empty((len(p), HD))
                c = vc[:, g].astype(np.float64)
                for e in range(4):
                    d = slice(64 * e, 64 * e + 64)
                    se, me = (np.where(see.any(0), f64(x[:, g, e]), 0.0) for x in (vs, vm))
                    se, me = np.nan_to_num(se), np.nan_to_num(me)
                    o[:, d] = parts(p * se) @ c[:, d] + (parts(p) @ me)[:, None]
            else:
                o = bf16(p) @ vg
            with np.errstate(all="ignore"):
                out[t0:t0 + bt.new[b], h] = np.where(l > 0, o / l, 0.0)
    out /= 1.0 + np.exp(-bt.gate.astype(np.float64))
    if plant == "zero":
        out[:] = 0
    return bf16(out) if out_bf16 else out


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("i", range(len(CASES)))
def test_bounds(i, out_bf16):
    kernel, bt = batch(i)
    res, keys = Q.result(bt, kernel), max(bt.lens)
    most, mean = Q.check(outputs(bt, kernel, out_bf16), res, kernel, keys, out_bf16)
    assert most <= 1 and mean <= 1, (most, mean)
    plants = ["zero"]
    if max(bt.new) > 8:
        plants += ["causal", "next row"]
    if max(bt.lens) > 256 and not bt.window:
        plants += ["part", "tile"]
    if kernel == "paged_q4_split":
        plants += ["one part", "sign"]
    for plant in plants:
        most, mean = Q.check(outputs(bt, kernel, out_bf16, plant), res, kernel, keys, out_bf16)
        assert most > 1 or mean > 1, (plant, most, mean)


def test_the_shapes_reach_every_kernel():
    """The kernels that the GPU tests' shapes run, under the tables that they have and under wide ones; the limits are the
    source's."""
    import os
    import re
    from test_gpu_paged_q4 import SHAPES
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vx27_amd/csrc/vx_paged_rows.h")).read()
    for name in ("FLAT_ROWS", "FLAT_TILES"):
        assert int(re.search(rf"constexpr \w+ {name} = (\d+);", src).group(1)) == getattr(Q, name)
    count = {(k, w): 0 for k in Q.KERNELS for w in (False, True)}
    for lens, new, n_q, n_kv, page, window, sink in SHAPES:
        for wide in (False, True):
            for out_bf16 in (False, True):
                bt = Batch4.__new__(Batch4)
                bt.lens, bt.new, bt.qg, bt.n_kv, bt.page, bt.window, bt.sink, bt.B = lens, new, n_q // n_kv, n_kv, page, window, sink, len(lens)
                bt.N, bt.max_pages = sum(new) + 5, max(1, max(-(-n // page) for n in lens)) + 1 + 2100 * wide
                count[Q.kernel_of(bt, out_bf16), wide] += 1
    assert count["paged_q4_split", False] >= 30 and all(count[k, w] >= 3 for k, w in count if (k, w) != ("paged_rows_q4", False)), count

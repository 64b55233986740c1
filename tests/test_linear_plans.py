"""CPU check that the GPU tests' sizes reach every plan of the linear layers' products, and of the query that says which."""
import ctypes
import json
import math
import os
import random

import pytest

import linear_plans as lp
from chpl_b200 import _lib


def test_the_sizes_reach_every_plan():
    """Layers of random sizes, another draw than the one that the sizes were chosen from: every plan that one of them
    takes is taken by a size under test."""
    tested = {p for s in lp.SIZES + lp.LARGE for p in lp.plans(*s)}
    r = random.Random(2)
    missing = set()
    for _ in range(30000):
        k, n = (int(round(math.exp(r.uniform(math.log(64), math.log(16384))))) for _ in range(2))
        T = max(1, min(int(round(math.exp(r.uniform(0, math.log(8192))))), 8192 * 4096 * 16384 // (k * n)))
        missing.update(p for p in lp.plans(T, k, n) if p not in tested)
    assert not missing


def test_large_sizes_take_several_tiles_of_a_pair():
    for s in lp.LARGE:
        for product, pair, _, _, several in lp.plans(*s):
            assert pair and several, (s, product)


@pytest.mark.parametrize("args", [(3, 64, 64, 64), (-1, 64, 64, 64), (0, 0, 64, 64), (0, 64, 0, 64), (0, 64, 64, -1), (0, -64, 64, 64)])
def test_plan_query_refuses(args):
    out = (ctypes.c_int64 * 4)()
    assert _lib.load().chpl_diag_linear_plan(*args, out) == _lib.CHPL_ERR_INVALID
    assert _lib.load().chpl_diag_linear_plan(0, 64, 64, 64, None) == _lib.CHPL_ERR_INVALID
    assert _lib.load().chpl_diag_linear_plan(0, (1 << 30) + 1, 64, 64, out) == _lib.CHPL_ERR_UNSUPPORTED


def test_the_choice_against_the_recorded_timings():
    """The kernel, tile and split that a product takes, among all that were timed for it: 2 % slower than the best in the
    geometric mean, and in three of 210 products more than a quarter (dW of one k-block)."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "profiles", "linear_plan_timings.json")
    with open(path) as f:
        record = json.load(f)
    assert len(record) == 210 and sum(len(p["us"]) for p in record) == 3553
    over = []
    for p in record:
        T, k, n = p["tokens"], p["k"], p["n"]
        f, r, c = {"fwd": (n, T, k), "dx": (k, T, n), "dw": (k, n, T)}[p["product"]]
        pair, bn, split, _ = lp.plan(("fwd", "dx", "dw").index(p["product"]), f, r, c)
        over.append(p["us"][f"pair {bn}" if pair else f"{bn} split {split}"] / min(p["us"].values()))
    assert math.exp(sum(map(math.log, over)) / len(over)) < 1.02
    assert sum(v > 1.25 for v in over) == 3 and max(over) < 1.62

"""CPU check that the GPU tests' sizes reach every plan of the linear layers' products, and of the query that says which."""
import ctypes
import math
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

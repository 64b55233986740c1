"""CPU check of the ring of stages in which a 4-bit product of a few tokens codes X: a model of its barriers, for every ring that
the products of 1 to 8 tokens have.

A stage is used in turn T (the T-th 256 of the contraction that a CTA takes) by T % stages; its rows come in units, dealt out to
the warps in order, and a unit may be written once the tensor core has read the stage's last use.  A warp learns that from the
parity of the stage's barrier, whose phases are counted here as they complete."""
import ctypes
import random

import pytest

from chpl_b200 import _lib


def overwrites(stages, units, warps, turns, pick):
    """Units that replace what has not been read yet.  pick(coders, reader): which of the warps that can go on goes on (the
    reader, where it can, is one of them)."""
    read = [0] * stages        # phases of a stage's barrier that have completed
    here = [0] * turns         # units of a turn that have been written
    at = list(range(warps))    # the warps' next units
    turn, wrong = 0, 0         # the reader's
    total = turns * units
    while turn < turns:
        can = []
        for w, u in enumerate(at):
            if u < total:
                t = u // units
                if (read[t % stages] & 1) != ((t // stages & 1) ^ 1):
                    can.append(w)
        w = pick(can, here[turn] >= units)
        if w is None:
            assert here[turn] >= units  # something can always go on
            read[turn % stages] += 1
            turn += 1
        else:
            t = at[w] // units
            wrong += read[t % stages] != t // stages
            here[t] += 1
            at[w] += warps
    return wrong


def eager(can, reader):
    """Coding far ahead of the products, as it is where those wait for their weights."""
    return can[0] if can else None


def random_order(seed):
    rng = random.Random(seed)

    def pick(can, reader):
        return rng.choice(can + [None] * reader)

    return pick


def rings():
    """(stages, units of a stage, warps) of products of 1 to 8 tokens, and the products of each."""
    L, found = _lib.load(), {}
    ring = (ctypes.c_int64 * 3)()
    features = sorted({int(1.06 ** i) for i in range(210)} | {128 * 148 + d for d in (-1, 0, 1, 127, 128, 129)} | {19000, 28672, 32000, 128256, 200000})
    for n in features:
        for k in (1, 256, 2560, 2561, 2816, 4096, 8192, 16384, 65536):
            for tokens in range(1, 9):
                assert L.chpl_diag_mx4_ring(n, tokens, k, ring) == 0
                found.setdefault(tuple(ring), []).append((tokens, n, k))
    return found


def test_no_unit_replaces_what_was_not_read():
    """Every ring, far ahead and in random orders, over several turns of it."""
    found = rings()
    assert any(stages == 5 and units == 1 for stages, units, _ in found)  # one and two CTAs to an SM are both among them
    assert any(stages > 6 for stages, _, _ in found)
    for (stages, units, warps), products in found.items():
        assert 0 < warps <= 6 and warps <= stages * units, products[0]
        for pick in (eager, *map(random_order, range(20))):
            assert overwrites(stages, units, warps, 5 * stages + 3, pick) == 0, (stages, units, warps, products[0])


def test_the_model_sees_what_too_many_warps_do():
    """Six warps on five stages of one unit come back more than a turn later, and a parity does not tell them so."""
    assert overwrites(5, 1, 6, 11, eager) > 0 and overwrites(5, 1, 6, 40, eager) > 0
    assert overwrites(5, 1, 6, 10, eager) == 0  # no warp comes back
    assert overwrites(5, 2, 6, 40, eager) == 0 and overwrites(6, 1, 6, 40, eager) == 0


@pytest.mark.parametrize("rows", [9, 4096])
def test_products_that_do_not_code(rows):
    ring = (ctypes.c_int64 * 3)()
    assert _lib.load().chpl_diag_mx4_ring(4096, rows, 4096, ring) == 0
    assert ring[0] >= 2 and ring[1] == ring[2] == 0


def test_refusals():
    L, ring = _lib.load(), (ctypes.c_int64 * 3)()
    for args in ((0, 1, 1, ring), (1, 0, 1, ring), (-1, 1, 1, ring), (1, 1, -1, ring), (1, 1, 1, None)):
        assert L.chpl_diag_mx4_ring(*args) == _lib.CHPL_ERR_INVALID

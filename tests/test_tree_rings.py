"""The model of tests/test_tree_protocol.py with the rings that 16-bit activations have: P in two halves takes a second block of columns at 64 product rows, which costs the ring of V a tile at head
dimensions up to 128."""
import random

import pytest

from tests.test_tree_protocol import KEYS, LIMIT, SMALL, Model


def shape(split, nb, nr):
    """TcTree's numbers."""
    nc, np, mt, box = nr * (2 if split else 1), 2 * nr, nb // 2, KEYS * 128
    parts = 1 if not split or nr > 32 else 2 if nr == 32 else nb
    slot = nb * box
    slots = min((LIMIT - SMALL - nb * nc * 128 - (2 if np > 64 else 1) * box) // slot, 6)
    ks = (slots + 1) // 2
    assert slots >= 2 and 2 * parts * nc + mt * np <= 512 and np <= 128
    return dict(nb=nb, mt=mt, ks=ks, vs=slots - ks)


def test_the_rings_of_64_rows():
    assert shape(False, 2, 64) == dict(nb=2, mt=1, ks=3, vs=2) and shape(False, 4, 64) == dict(nb=4, mt=2, ks=1, vs=1)


@pytest.mark.parametrize("split,nb,nr", [(s, nb, nr) for s in (True, False) for nb in (2, 4) for nr in (16, 32, 64)])
def test_every_schedule_ends_and_nothing_is_overwritten(split, nb, nr):
    s = shape(split, nb, nr)
    rng = random.Random(nb * 100 + nr + split)
    for trial in range(4):
        n = rng.choice((0, 1, 2, 3, 5, 9, 14))
        for masked in {n, max(n - 1, 0), max(n - 3, 0)}:
            for lag in (None, "pipe", "copies", "soft00", "soft11", "issue", "load_k", "load_v"):
                if rng.random() < 0.5:
                    Model(s, n, masked, rng).run(lag)

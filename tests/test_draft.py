"""Drafted tokens over the paged cache, without a device: descriptions that are refused, sizes, and the plain restatements against each other."""
import ctypes as C

import numpy as np
import pytest

import lapid_b200 as lp
from lapid_b200 import _lib
from lapid_b200.paged import Mask, PagedSpec, plan_bytes, tree_bytes

from . import draft_ref as D

OK = dict(dtype=lp.DType.BF16, q_heads=32, kv_heads=8, head_dim=128, page_size=16, pages=1000, requests=4, tokens=40, max_blocks=64, max_new=10, mask=Mask.TREE)


@pytest.mark.parametrize("change,code", [({"max_new": 1025}, "unsupported"), ({"mask": 3}, "invalid_argument"), ({"mask": 5}, "invalid_argument"), ({"mask": -1}, "invalid_argument"),
                                         ({"window": 1 << 31}, "too_large"), ({"mask": Mask.CROSS, "window": 3}, "invalid_argument")])
def test_descriptions_that_are_refused(change, code):
    with pytest.raises(lp.LapidError) as e:
        plan_bytes(PagedSpec(**{**OK, **change}))
    assert e.value.code == code


def test_tree_bytes():
    assert tree_bytes(PagedSpec(**OK)) == 40 * 8 and tree_bytes(PagedSpec(**{**OK, "max_new": 32})) == 40 * 8 and tree_bytes(PagedSpec(**{**OK, "max_new": 33})) == 40 * 12
    assert tree_bytes(PagedSpec(**{**OK, "max_new": 1024, "window": 7})) == 40 * 33 * 4 and tree_bytes(PagedSpec(**{**OK, "tokens": 0})) == 0
    with pytest.raises(lp.LapidError) as e:
        tree_bytes(PagedSpec(**{**OK, "mask": Mask.CAUSAL}))
    assert e.value.code == "invalid_launch"
    n = C.c_uint64(7)
    assert _lib.lib().lapid_b200_paged_tree_bytes(None, C.byref(n)) == 1 and n.value == 7


def test_null_device_is_refused():
    c, lib = PagedSpec(**OK).to_c(), _lib.lib()
    assert lib.lapid_b200_paged_tree(None, C.byref(c), *[None] * 4) == 1
    assert lib.lapid_b200_paged_tree_attention(None, C.byref(c), *[None] * 10) == 1
    assert lib.lapid_b200_paged_verify(None, C.byref(c), None, 0, 10, None, 0, None, 0, *[None] * 8) == 1
    assert lib.lapid_b200_paged_commit(None, C.byref(c), None, None, 0, None, None, None, None, 0, None, None) == 1


def test_the_restated_walk_gives_the_models_distribution():
    """Over all draws of two siblings from 3 tokens and a grid of the random numbers (midpoints of 16 x 16 x 16) the first token has the model's distribution: the rule itself is right. A border moves a
    count by at most one place of 16 in each of the three numbers: 3 / 16 of a token's weight. (The draft's own distribution is 0.3 and more off.)"""
    p, draft = np.array([0.5, 0.3, 0.2]), np.array([[0.2, 0.7, 0.1]] * 3)
    logits, grid, mass = np.log(np.array([p] * 3)), (np.arange(16) + 0.5) / 16, np.zeros(3)
    for x in range(3):
        for y in range(3):
            for a in grid:
                for b in grid:
                    for w in grid:
                        path, nxt = D.verify(logits, [-1, 0, 0], [0, x, y], [0.0, a, b], w, 1.0, draft)
                        mass[[x, y][path[1] - 1] if len(path) > 1 else nxt] += draft[0, x] * draft[0, y] / 16 ** 3
    assert abs(mass.sum() - 1) < 1e-9 and np.all(np.abs(mass - p) <= 3 / 16 * p)


def test_the_restated_tree():
    depth, seen = D.tree([-1, 0, 0, 1, 3, -1])
    assert depth == [0, 1, 1, 2, 3, 0] and seen[4] == {4, 3, 1, 0} and seen[2] == {0, 2} and seen[5] == {5}
    assert D.tree([-1, 0, 1, 2], 2)[1][3] == {3, 2}
    assert D.tree_words([-1] + [0] * 40, 0, 2)[40].tolist() == [1, 1, 1 << 8]

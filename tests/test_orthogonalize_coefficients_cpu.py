"""Coefficients of the iteration in every form that a program may hold them in, and what changes in place between calls."""
import numpy as np
import pytest
import torch

from cuop_b200 import _native as N
from cuop_b200 import muon as M


def schedule(c, steps):
    return list(M._schedule(c, steps, "orthogonalize"))


def test_numbers_that_change_in_place():
    """The same objects with other numbers in them are other coefficients."""
    a = torch.tensor(3.0)
    k = [(a, -4.0, 2.0)] * 2
    assert schedule(k, 2) == [3.0, -4.0, 2.0] * 2
    a.fill_(1.5)
    assert schedule(k, 2) == [1.5, -4.0, 2.0] * 2
    t = torch.tensor([1.0, 2.0, 3.0], dtype=torch.float64)
    assert schedule(t, 1) == [1.0, 2.0, 3.0]
    t[1] = 5.0
    assert schedule(t, 2) == [1.0, 5.0, 3.0] * 2
    k = [[1.0, 2.0, 3.0], [4.0, 5.0, 6.0]]
    assert schedule(k, 2) == [1.0, 2.0, 3.0, 4.0, 5.0, 6.0]
    k[0][0] = 9.0
    assert schedule(k, 2) == [9.0, 2.0, 3.0, 4.0, 5.0, 6.0]


@pytest.mark.parametrize("one", [(3, -4, 2), [3.0, -4.0, 2.0], np.array([3, -4, 2], dtype=np.float32), torch.tensor([3, -4, 2]),
                                 (np.float32(3), np.float64(-4), 2), (torch.tensor(3.0), -4, 2)])
def test_forms(one):
    assert schedule(one, 3) == [3.0, -4.0, 2.0] * 3
    assert schedule([one] * 2, 2) == [3.0, -4.0, 2.0] * 2
    assert schedule([one] * 3, 3) == [3.0, -4.0, 2.0] * 3  # three triples are no triple
    assert len(schedule(one, 0)) == 1 and len(schedule([], 0)) == 1  # nothing is read of them


@pytest.mark.parametrize("bad", [None, 3.0, (1.0, 2.0), (1.0, 2.0, 3.0, 4.0), [(1.0, 2.0, 3.0)], [(1.0, 2.0)] * 2, "abc", ["abc"] * 2,
                                 {1: 2, 3: 4}, [(1.0, 2.0, None)] * 2, [("a", 1.0, 2.0)] * 2, torch.ones(2, 2), torch.ones(3, 2),
                                 [(1.0, 2.0, torch.ones(2))] * 2])
def test_refusals(bad):
    with pytest.raises(N.CuopError):
        schedule(bad, 2)

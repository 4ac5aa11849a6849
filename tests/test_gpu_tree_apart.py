"""A node whose row has no softmax stays out of the weights of slots that it does
not see."""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from test_gpu_tree_attention import ancestors, call, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def with_a_hit(dh, n, L):
    """A forest, one of its nodes, and for each node whether that one is above it (or it)."""
    c = make(dh + n, 2, n, 2, dh, L + n + 20, [L, L + 3], None, "forest")
    hit = n // 2
    below = np.array([any(j == hit for j in ancestors(c["par"][0], i)) for i in range(n)])
    assert 0 < below.sum() < n
    return c, hit, below


SHAPES = [(64, 6, 30), (16, 6, 700), (24, 40, 5), (64, 40, 300), (128, 9, 130), (128, 40, 100), (256, 3, 17)]


@pytest.mark.parametrize("dh,n,L", SHAPES)
@pytest.mark.parametrize("weigh", [3, 256])
def test_a_node_without_a_softmax_weighs_only_what_it_sees(net, dh, n, L, weigh):
    """Its key is NaN or infinite, so its row's weights are NaN: at the slots it
    sees, and nowhere else."""
    c, hit, below = with_a_hit(dh, n, L)
    weigh = min(n, weigh)
    _, want = call(net, c, weigh)
    seen = np.zeros(c["ctx"], bool)  # by a weighing node with such a row
    for i in np.flatnonzero(below[:weigh]):
        seen[:L] = True
        seen[L + np.array(ancestors(c["par"][0], i))] = True
    assert not seen[L:L + n].all()
    for bad in (np.nan, np.inf, -np.inf):
        k = c["k"].copy()
        k[0, :, L + hit] = bad * (1 if bad != bad else np.sign(c["q"][0, hit, 0].real))
        _, w = call(net, dict(c, k=k), weigh)
        assert np.array_equal(w[1], want[1])
        assert np.array_equal(w[0][:, ~seen], want[0][:, ~seen]), bad
        if bad != bad:
            assert np.isnan(w[0][:, seen]).all()

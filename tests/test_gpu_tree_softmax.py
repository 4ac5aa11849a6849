"""The running softmax of a node in a tile it shares with others: its rows bit for
bit whatever the others' scores are, and scores that climb."""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from test_gpu_tree_attention import ancestors, call, close, formula, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


@pytest.mark.parametrize("dh,n", [(16, 6), (64, 6), (16, 40), (64, 40), (128, 20), (256, 3)])
def test_large_scores_of_a_row_that_a_node_does_not_see(net, dh, n):
    """Enough sequences that a wave walks several tiles, scores that rise over
    them: where another node's largest one comes suddenly, this node's sums are
    scaled as they were."""
    B, L = 16, 600
    c = make(dh + n, B, n, 8, dh, L + n + 20, [L] * B, None, "forest")
    c["bias"] += np.linspace(0, 6, c["ctx"])
    want, _ = call(net, c)
    hit = 1 if n < 10 else n // 2
    below = np.array([[any(j == hit for j in ancestors(c["par"][b], i)) for i in range(n)] for b in range(B)])
    for key in (1e3, -1e3, np.inf):
        k = c["k"].copy()
        k[:, :, L + hit] *= key
        got, _ = call(net, dict(c, k=k))
        assert np.array_equal(got[~below], want[~below]), key


def test_scores_that_climb(net):
    """Every node's scores rise by more than 8 from tile to tile, for one node
    sooner than for the others: against the formula."""
    c = make(5, 1, 20, 2, 32, 400, [380], None, "tree")
    step = np.linspace(0, 4, 400)[None, :, None]
    c["k"][0] *= step
    c["q"][0, 7] *= 6.0
    want, tol, w_want, w_tol = formula(c, 20)
    got, w = call(net, c, 20)
    close(got, want, tol)
    close(w, w_want, w_tol)

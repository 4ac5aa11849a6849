"""Lengths and sizes of the serving operators' Python methods: whole numbers that
fit 32 bits, or refused before they reach the library."""
from __future__ import annotations

import numpy as np
import pytest

from test_serving_ops import network

PAR = [[-1, 0]] * 2
BAD = [[1.5, 2.0], np.array([1, 2 ** 32 + 1]), np.array([1, -1]), [1, "2"], [1, 2, 3], np.array([[1, 2]]), [True, False]]


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("call", [
    lambda n, x: n.tree_step([[3, 4]] * 2, PAR, counts=x),
    lambda n, x: n.tree_step_device([[3, 4]] * 2, PAR, 0, counts=x),
    lambda n, x: n.tree_accept([[0, 1]] * 2, x),
    lambda n, x: n.tree_attention_device(0, 0, 0, x, PAR, 1, 1, 4, 0),
    lambda n, x: n.tree_attention_device(0, 0, 0, [1, 1], PAR, 1, 1, 4, 0, counts=x),
])
def test_lengths_that_are_not(call, bad):
    with pytest.raises(ValueError):
        call(network(), bad)


@pytest.mark.parametrize("bad", [x for x in BAD if np.shape(x) != (3,)], ids=str)
def test_lengths_of_an_eviction_that_are_not(bad):
    with pytest.raises(ValueError):
        network().evict_rows_device(0, 0, 0, bad, 1, 1, 4, 2, 0, 0, 0, 0, 0, 4)


@pytest.mark.parametrize("bad", [-1, 2 ** 32, 2 ** 32 + 4, 1.5, np.int64(-1), np.int64(2 ** 32 + 4), np.float64(2)])
@pytest.mark.parametrize("call", [
    lambda n, x: n.tree_step([[3, 4]] * 2, PAR, weigh_nodes=x),
    lambda n, x: n.tree_step_device([[3, 4]] * 2, PAR, 0, weigh_nodes=x),
    lambda n, x: n.tree_attention_device(0, 0, 0, [1, 1], PAR, x, 1, 4, 0),
    lambda n, x: n.tree_attention_device(0, 0, 0, [1, 1], PAR, 1, x, 4, 0),
    lambda n, x: n.tree_attention_device(0, 0, 0, [1, 1], PAR, 1, 1, x, 0),
    lambda n, x: n.tree_attention_device(0, 0, 0, [1, 1], PAR, 1, 1, 4, 0, weigh_nodes=x),
    lambda n, x: n.tree_attention_device(0, 0, 0, [1, 1], PAR, 1, 1, 4, 0, bias_stride=x if x < 0 or isinstance(x, float) else int(x) << 32),
    *(lambda n, x, i=i: n.evict_rows_device(0, 0, 0, [3], *[x if k == i else 2 for k in range(6)], 0, 0, 0, 4) for i in range(6)),
    lambda n, x: n.evict_rows_device(0, 0, 0, [3], 1, 1, 4, 2, 0, 0, 0, 0, 0, x),
    *(lambda n, x, i=i: n.evict_rows(*[x if k == i else 2 for k in range(4)]) for i in range(4)),
    lambda n, x: n.process_logits_device(0, x, 4),
    lambda n, x: n.process_logits_device(0, 4, x),
    lambda n, x: n.process_logits_device(0, 4, 4, max_history=x),
    lambda n, x: n.process_logits_device(0, 4, 4, max_bias=x),
])
def test_sizes_that_are_not(call, bad):
    with pytest.raises((ValueError, TypeError)):
        call(network(), bad)


def test_biases_without_their_ids():
    with pytest.raises(ValueError, match="bias_ids"):
        network().process_logits(np.zeros((1, 7)), bias=[[0.5]])

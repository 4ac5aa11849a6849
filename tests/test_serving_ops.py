"""The operators of a serving loop without a GPU: every entry point refuses a null
network, and the Python methods refuse arrays of wrong shapes and types before
they reach the library."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import rustcrates_amd as ra

NAMES = ["mitok_tree_attention_device", "mitok_tree_step", "mitok_tree_step_device", "mitok_tree_accept",
         "mitok_evict_rows_device", "mitok_evict_rows", "mitok_process_logits_device", "mitok_process_logits"]


@pytest.mark.parametrize("name", NAMES)
def test_a_null_network_is_refused(name):
    lib = ra.load_library()
    args = [None if a is C.c_void_p else 0 for a in ra.SIGNATURES[name][1]]
    assert getattr(lib, name)(*args) == 1
    assert lib.mitok_last_error()


class _Never:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


def network():
    net = ra.Network.__new__(ra.Network)
    net._h, net._lib, net.vocab = None, _Never(), 7
    return net


@pytest.mark.parametrize("call", [
    lambda n: n.tree_step([3, 4], [[-1, 0]]),
    lambda n: n.tree_step([[3, 4]], [[-1]]),
    lambda n: n.tree_step([[3.5, 4.0]], [[-1, 0]]),
    lambda n: n.tree_step([[3, -2]], [[-1, 0]]),
    lambda n: n.tree_step([[3, 2 ** 32]], [[-1, 0]]),
    lambda n: n.tree_step([[3, 4]], [[-1, 0]], counts=[1, 2]),
    lambda n: n.tree_step_device([[3, 4]], [[-1], [0]], 0),
    lambda n: n.tree_accept([0, 1]),
    lambda n: n.tree_accept([[0, 1]], [1, 1]),
    lambda n: n.tree_attention_device(0, 0, 0, [1], [[-1], [-1]], 1, 1, 4, 0),
    lambda n: n.evict_rows_device(0, 0, 0, [[3]], 1, 1, 4, 2, 0, 0, 0, 0, 0, 4),
    lambda n: n.process_logits(np.zeros(7)),
    lambda n: n.process_logits(np.zeros((2, 7)), [[1]], [[1, 0, 0]]),
    lambda n: n.process_logits(np.zeros((2, 7)), [[1], [2]], [[1, 0], [1, 0]]),
    lambda n: n.process_logits(np.zeros((1, 7)), bias_ids=[[1, 2]], bias=[[0.5]]),
    lambda n: n.process_logits(np.zeros((1, 7)), allowed=np.ones((1, 6), bool)),
])
def test_wrong_arrays_are_refused_before_the_library(call):
    with pytest.raises(ValueError):
        call(network())


def test_signed_and_unsigned_ids_are_the_same():
    rows = ra._u32_rows(np.array([[-1, 5]]), "ids")
    assert rows.dtype == np.uint32 and rows.tolist() == [[ra.NO_TOKEN, 5]]
    assert ra._u32_rows(np.array([[0xFFFFFFFF]], np.uint32), "ids")[0, 0] == ra.NO_TOKEN

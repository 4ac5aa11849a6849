"""What a refused mitok_process_logits(_device) leaves behind: nothing for the
next call to take for its own."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import rustcrates_amd as ra

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def test_an_error_is_reported_once(net):
    """A call that ends early, here on the runtime's own last error, takes what
    its kernels found with it."""
    hip = C.CDLL("libamdhip64.so.7")
    x = np.zeros((2, 40))
    good, ids = net.process_logits(x, [[1]] * 2, [[2.0, 1.0, 0.0]] * 2)
    for bad in (dict(history=[[40]] * 2, penalties=[[2.0, 1.0, 0.0]] * 2), dict(history=[[1]] * 2, penalties=[[0.0, 0.0, 0.0]] * 2)):
        assert hip.hipSetDevice(999) != 0  # left as the thread's last error
        with pytest.raises(ra.MitokError):
            net.process_logits(x, **bad)
        hip.hipGetLastError()
        again, ids2 = net.process_logits(x, [[1]] * 2, [[2.0, 1.0, 0.0]] * 2)
        assert np.array_equal(again, good) and np.array_equal(ids2, ids)

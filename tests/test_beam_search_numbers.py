"""Network.beam_search takes 32-bit whole numbers: others are refused before the
library, which would take them cut to size (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest

from host_runtime import run
from test_serving_ops import network


@pytest.mark.parametrize("kw", [
    dict(end_id=2 ** 32 + 7), dict(end_id=-2), dict(end_id=7.9), dict(end_id=2 ** 70), dict(end_id="7"), dict(end_id=[7, 8]),
    dict(prompt=[[3, 2 ** 32 + 4]]), dict(prompt=[[3, -2]]), dict(prompt=[[3.5, 4.0]]), dict(prompt=np.array([[3, -5]])),
    dict(lens=[1.5]), dict(lens=[-1]), dict(lens=np.array([2 ** 32 + 1])),
    dict(beams=2 ** 32 + 2), dict(n_new=-1), dict(n_new=2 ** 32),
])
def test_other_numbers_are_refused(kw):
    with pytest.raises(ValueError):
        network().beam_search(**{**dict(prompt=[[3, 4]], beams=2, n_new=2), **kw})


def test_whole_numbers_of_every_kind_are_taken():
    run("""
net = stack()
for prompt in ([[3, 4, 5]], np.array([[3, 4, 5]], np.int64), np.array([[3, 4, 5]], np.uint8), np.array([[3, 4, 5]], np.uint32)):
    for end in (None, 7, np.uint32(7), np.int64(7), -1, 0xFFFFFFFF, 10**6):
        ids, n, _ = net.beam_search(prompt, lens=np.array([3], np.int16), beams=np.int64(2), n_new=np.uint32(4), end_id=end)
        assert ids.shape == (1, 2, 4) and n.shape == (1, 2)
""")

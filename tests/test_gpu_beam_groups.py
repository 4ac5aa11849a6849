"""mitok_beam_select_device on more groups than one launch holds (2^21)."""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from test_gpu_paged_attention import put

pytestmark = pytest.mark.gpu


def test_more_groups_than_a_launch_holds():
    """Two rows of one token in each group: a row's logit is all of its distribution, so its score stays as it is."""
    B, R = 2 ** 22 - 3, 2
    r = np.random.default_rng(0)
    scores = -r.integers(1, 1000, (B, R)).astype(float)
    d = dict(x=put(r.standard_normal((B, R))), s=put(scores), p=put(np.zeros(B, np.uint32)), t=put(np.ones(B, np.uint32)),
             o=put(np.zeros(B)))
    try:
        with ra.Network(0) as net:
            net.beam_select_device(d["x"], d["s"], B, R, 1, 1, d["p"], d["t"], d["o"])
        best = scores.argmax(1)  # equal scores: the lower row
        assert np.array_equal(d["p"].download((B,), np.uint32), np.arange(B) * R + best)
        assert not d["t"].download((B,), np.uint32).any()
        assert np.array_equal(d["o"].download((B,), float), scores[np.arange(B), best])
    finally:
        for b in d.values():
            b.free()

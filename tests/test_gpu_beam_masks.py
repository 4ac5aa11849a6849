"""mitok_beam_select(_device) where ranks lie far apart: finite masks that shut
whole stretches of the vocabulary, scores and scales at the ends of the doubles,
and a beam search whose length power takes its ranks there.  Tolerances are
test_gpu_beam_select's."""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from conftest import build_explicit, seeded_tensors
from rustcrates_amd import configs, seeded
from test_gpu_beam_select import NONE, check, device, make

pytestmark = pytest.mark.gpu
MOST = np.finfo(float).max


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def masked(seed, B, R, V, K, mask, share=0.3, **kw):
    """One stretch of the vocabulary is allowed in each row, the rest is `mask`: whole quarters of 64 or 128 logits."""
    c = make(seed, B, R, V, K, **kw)
    r = np.random.default_rng(seed + 1)
    wide = max(1, int(share * V))
    for b in range(B):
        for i in range(R):
            at = r.integers(0, V - wide + 1)
            c["x"][b, i, :at] = c["x"][b, i, at + wide:] = mask
    return c


@pytest.mark.parametrize("mask", [-MOST, -1e300, -1e39, -1e30])
@pytest.mark.parametrize("V", [700, 4096, 50280])
@pytest.mark.parametrize("K", [1, 4, 64])
def test_stretches_shut_by_a_finite_mask(net, mask, V, K):
    want = check(net, masked(V + K, 2, 3, V, K, mask))
    assert (want[1] != NONE).all()


@pytest.mark.parametrize("mask", [-MOST, -1e300])
def test_pieces_of_512_logits(net, mask):
    check(net, masked(1, 24, 1, 50280, 5, mask))
    check(net, masked(2, 6, 9, 20000, 24, mask))


@pytest.mark.parametrize("mask", [-MOST, -1e300, -1e39])
def test_fewer_allowed_than_kept(net, mask):
    """The masked tokens of equal logit follow, the lower row and the lower token first."""
    c = masked(3, 2, 2, 3000, 32, mask, share=0.003)
    want = check(net, c)
    assert (c["x"].reshape(4, 3000)[want[0], want[1]] == mask).any(1).all()


@pytest.mark.parametrize("mask", [-MOST, -1e300, -1e39])
@pytest.mark.parametrize("V", [700, 2000])
def test_few_quarters_of_many_continuations(net, mask, V):
    """No more quarters than kept, but a list of more than 512: closer bounds, from a range that the mask opens."""
    check(net, masked(4, 3, 1, V, 64, mask, share=0.85))
    c = masked(5, 3, 1, V, 64, mask, share=0.85)
    c["x"][c["x"] != mask] = 2.5
    check(net, c)


def test_more_quarters_than_the_list_holds(net):
    c = make(6, 1, 1, 400001, 64)
    c["x"][:] = -1.5
    check(net, c)
    c["x"][0, 0, 1::2] = -MOST
    check(net, c)


@pytest.mark.parametrize("score", [-1e39, -1e300, -MOST])
def test_a_row_of_a_very_low_score(net, score):
    c = make(7, 3, 3, 4096, 8)
    c["scores"][:, 1] = score
    c["scores"][2] = score  # none but such rows: what a score swallows is ordered by the logits
    c["scale"][2] = 0.5
    check(net, c)


@pytest.mark.parametrize("scale", [1e-300, 1e-3, 3.0, 1e39, 1e118, 1e300])
@pytest.mark.parametrize("K", [1, 6, 64])
def test_scales_far_from_1(net, scale, K):
    c = make(8, 2, 4, 4096, K)
    c["scale"] = scale * np.random.default_rng(8).uniform(0.5, 2.0, (2, 4))
    check(net, c)
    c["scale"][:] = scale  # ended rows among them
    c["done"][:, 2] = True
    check(net, c)


@pytest.mark.parametrize("mask", [-1e300, -1e39])
def test_masks_and_scales_above_1(net, mask):
    c = masked(9, 2, 3, 4096, 16, mask)
    c["scale"] = np.random.default_rng(9).uniform(1.5, 4.0, (2, 3))
    check(net, c)


def test_ranks_that_pass_the_doubles(net):
    """Below them a continuation is none; above them all are equal, the lower row first."""
    c = masked(10, 1, 2, 900, 8, -1e300, share=0.003)
    c["scale"][:] = 1e200
    p, t, s = device(net, c)
    assert (p[0, :4] != NONE).all() and (s[0, :4] > -1e6).all()
    assert (p[0, 4:] == NONE).all() and (t[0, 4:] == NONE).all() and (s[0, 4:] == -np.inf).all()
    c = make(11, 2, 3, 900, 8)
    c["scores"] += 1e300
    c["scale"][:] = 1e10
    want = check(net, c)
    assert (want[0] == np.array([[0], [3]])).all()


@pytest.mark.parametrize("K", [1, 3])
def test_a_search_whose_ranks_pass_single_precision(K):
    """Hypotheses of equal length are in the same order under any power; one of -16 takes
    ranks of 230 tokens to -1e40 and below."""
    cfg = configs.ModelConfig("bp", layers=1, d=32, heads=2, ffn=48, vocab=400, max_ctx=256, seed=6)
    t = seeded_tensors(cfg)
    prompt = seeded.prompts(90, [7, 12], cfg.vocab)
    with build_explicit(ra.Network(0), cfg, t) as g:
        plain = g.beam_search(prompt, lens=[7, 12], beams=K, n_new=230)
        low = g.beam_search(prompt, lens=[7, 12], beams=K, n_new=230, length_power=-16.0)
    assert (-low[2] * 230.0 ** 16 > 3.5e38).all()
    for x, y in zip(plain, low):
        assert np.array_equal(x, y)
    assert (low[1] == 230).all() and np.isfinite(low[2]).all()

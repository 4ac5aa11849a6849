"""What the caches' next step needs besides their rows, the lengths, position
offsets and next ids on the device, after calls that do not go through the
token loop: a stateless pass of a larger batch, and predict on the caches.

Bar: the same ids and bits as the run without that call between."""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from conftest import seeded_tensors
from rustcrates_amd import configs, seeded
from test_gpu_tree_step import CFG, rope_stack

pytestmark = pytest.mark.gpu

LENS = [9, 6]


@pytest.fixture(scope="module")
def build():
    t = seeded_tensors(CFG)
    return lambda: rope_stack(ra.Network(0), configs.ModelConfig(**{**CFG.__dict__, "rope": True}), t)


def wide_pass(g):
    """A stateless pass of 200 sequences: every workspace of a row per sequence grows."""
    g.predict(seeded.prompts(77, [3] * 200, CFG.vocab), forward_only=False)


@pytest.mark.parametrize("evict", [False, True])
@pytest.mark.parametrize("plan", [None, 0])
def test_a_wide_stateless_pass_between_steps(build, evict, plan):
    prompt = seeded.prompts(8, LENS, CFG.vocab)
    runs = []
    for between in (lambda g: None, wide_pass):
        with build() as g:
            if plan is not None:
                g.set_decode_plan(plan)
            ids = [g.prefill(prompt, lens=LENS)]
            if evict:
                for tok in ([3, 4], [5, 6]):
                    g.tree_step(np.array(tok)[:, None], [[-1]] * 2, weigh_nodes=1)
                    g.tree_accept([[0]] * 2)
                assert g.evict_rows(2, 5, 1, 2).tolist() == [5, 5]
            between(g)
            logits = []
            for _ in range(4):
                i, lg = g.decode_step(want_logits=True)
                ids.append(i)
                logits.append(lg)
            runs.append((np.array(ids), np.array(logits)))
    assert np.array_equal(runs[0][0], runs[1][0]) and np.array_equal(runs[0][1], runs[1][1])


def test_a_wide_stateless_pass_between_accept_and_step(build):
    prompt = seeded.prompts(9, LENS, CFG.vocab)
    runs = []
    for between in (lambda g: None, wide_pass):
        with build() as g:
            g.prefill(prompt, lens=LENS)
            g.tree_step([[3, 4, 5]] * 2, [[-1, 0, 0]] * 2)
            g.tree_accept([[0, 2], [0, 1]], [2, 1])
            between(g)
            runs.append(np.array([g.decode_step(batch=2) for _ in range(3)]))
    assert np.array_equal(runs[0], runs[1])


def test_steps_on_caches_that_predict_used(build):
    """A prompt and a token by predict, then decode steps: as by prefill and steps."""
    prompt = seeded.prompts(10, LENS, CFG.vocab)
    with build() as g:
        g.prefill(prompt, lens=LENS)
        g.decode_step([7, 8])
        want = [g.decode_step([11, 12]), g.decode_step(batch=2)]
    with build() as g:
        g.predict(prompt, lens=LENS)
        with pytest.raises(ra.MitokError, match="without ids") as e:
            g.decode_step(batch=2)
        assert e.value.code == 3
        g.predict([[7], [8]], time_steps=LENS)
        got = [g.decode_step([11, 12]), g.decode_step(batch=2)]
        assert np.array_equal(got, want)
    with build() as g:  # and where the token loop ran on longer caches before
        g.generate(seeded.prompts(11, [20, 30], CFG.vocab), [20, 30], 5)
        g.reset()
        g.predict(prompt, lens=LENS)
        g.decode_step([7, 8])
        got = [g.decode_step([11, 12]), g.decode_step(batch=2)]
        assert np.array_equal(got, want)


def test_accepted_nodes_give_the_next_ids_where_predict_left_none(build):
    prompt = seeded.prompts(12, LENS, CFG.vocab)
    with build() as g:
        g.predict(prompt, lens=LENS)
        g.tree_step([[3, 4]] * 2, [[-1, 0]] * 2)
        g.tree_accept([[0], [0]], [1, 0])  # the second sequence has none
        with pytest.raises(ra.MitokError, match="without ids"):
            g.decode_step(batch=2)
        out = g.tree_step([[3, 4]] * 2, [[-1, 0]] * 2)
        g.tree_accept([[0, 1], [0, 1]])
        a = g.decode_step(batch=2)
    with build() as g:
        g.prefill(prompt, lens=LENS)
        g.tree_step([[3, 4]] * 2, [[-1, 0]] * 2)
        g.tree_accept([[0], [0]], [1, 0])
        g.tree_step([[3, 4]] * 2, [[-1, 0]] * 2)
        g.tree_accept([[0, 1], [0, 1]])
        assert np.array_equal(g.decode_step(out[:, 1]), a)

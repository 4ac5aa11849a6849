"""Tokens past the positions that a RoPE stack's table was made for: a session
that evicts and goes on past max_ctx, through two growths of the table, held to
the plain stack.

Bar: Re-logits within REL_TOL, as in test_gpu_tree_step.py."""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from conftest import REL_TOL, max_rel_err, seeded_tensors
from plain_stack import Sequence
from rustcrates_amd import configs, seeded
from test_gpu_tree_step import rope_stack

pytestmark = pytest.mark.gpu

CFG = configs.ModelConfig("rt", layers=1, d=32, heads=2, ffn=48, vocab=90, max_ctx=48, seed=9)


def test_a_session_past_the_table():
    cfg = configs.ModelConfig(**{**CFG.__dict__, "rope": True})
    t = seeded_tensors(CFG)
    prompt = seeded.prompts(3, [30], cfg.vocab)
    s = Sequence(cfg, t)
    s.prompt(prompt[0])
    r = np.random.default_rng(2)
    with rope_stack(ra.Network(0), cfg, t) as g:
        g.prefill(prompt)
        while s.pos < 1100:
            a, b, c = r.integers(2, cfg.vocab, 3)
            _, lg = g.tree_step([[a, b, c]], [[-1, 0, 1]], weigh_nodes=1, want_logits=True)
            want = [s.step(int(a), weigh=True), s.step(int(b)), s.step(int(c))]
            assert max_rel_err(lg[0], np.array(want)) < REL_TOL, s.pos
            g.tree_accept([[0, 1, 2]])
            for _ in range(9):
                tok = int(r.integers(2, cfg.vocab))
                i, lg = g.decode_step([tok], want_logits=True)
                want = s.step(tok)
                assert max_rel_err(lg[0], want) < REL_TOL and i[0] == np.argmax(want), s.pos
            if len(s.k[0][0]) + 12 > cfg.max_ctx:
                s.evict(20, 2, 4)
                assert g.evict_rows(1, 20, 2, 4)[0] == 20
    assert s.pos > 1024


def test_prompts_and_given_positions_that_need_a_wider_table():
    """predict's own time_steps, first a little past the table, then far."""
    cfg = configs.ModelConfig(**{**CFG.__dict__, "rope": True})
    t = seeded_tensors(CFG)
    prompt = seeded.prompts(4, [7], cfg.vocab)
    with rope_stack(ra.Network(0), cfg, t) as g:
        for p in (511, 512, 513, 1500, 600, 5000):
            s = Sequence(cfg, t)
            s.prompt(prompt[0])
            s.pos = p
            g.reset()
            g.predict(prompt)
            out, _ = g.predict([[5]], time_steps=[p])
            assert max_rel_err(out[0, 0], s.step(5)) < REL_TOL, p

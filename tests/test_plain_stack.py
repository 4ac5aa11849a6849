"""The plain numpy stack against the CPU checker: prompt, cached steps and RoPE."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from conftest import REL_TOL, max_rel_err, seeded_tensors
from plain_stack import Sequence, apply_rules, kept_rows
from rustcrates_amd import configs, seeded


@pytest.mark.parametrize("rope", [False, True])
def test_plain_stack_is_the_checkers(rope):
    cfg = configs.ModelConfig("ps", layers=2, d=32, heads=2, ffn=48, vocab=90, max_ctx=40, seed=4, rope=rope)
    if rope:  # seeded_tensors reads the stack without the RoPE layer: explicit tensors on both sides
        t = seeded_tensors(configs.ModelConfig("ps", layers=2, d=32, heads=2, ffn=48, vocab=90, max_ctx=40, seed=4))
        o = oracle.Network()
        o.add_embedding(90, 32, t[0]["table"])
        o.add_positional_encoding(32, cfg.rope_base)
        for a in range(2):
            n, s, f = t[1 + 3 * a: 4 + 3 * a]
            o.add_norm(32, cfg.norm_eps, n["gamma"], n["beta"])
            o.add_self_attention(2, 32, 40, cfg.attn_eps, s["wq"], s["wk"], s["wv"], s["bias_pos"], s["gamma"], s["beta"])
            o.add_feed_forward(32, 48, f["w1"], f["b1"], f["w2"], f["b2"])
        o.add_linear(32, 90, t[-1]["w"], t[-1]["b"])
        o.add_softmax(1)
    else:
        t = seeded_tensors(cfg)
        o = configs.build_network(oracle.Network(), cfg)
    ids = seeded.prompts(5, [9], 90)
    s = Sequence(cfg, t)
    got = [s.prompt(ids[0])]
    want = [o.predict(ids)[0][0, -1]]
    for k, token in enumerate([7, 1, 33]):
        got.append(s.step(token))
        want.append(o.predict(np.array([[token]], np.uint32), time_steps=[9 + k])[0][0, -1])
    assert max_rel_err(np.array(got), np.array(want)) < REL_TOL
    o.close()


def test_kept_rows_and_rules_by_hand():
    assert kept_rows([5, 1, 3, 3, 9, 2], 4, 1, 1) == [0, 2, 4, 5]
    assert kept_rows([5, 1, 3, 3, 9, 2], 3, 0, 0) == [0, 2, 4]
    assert kept_rows([float("nan"), 1, 0, 0], 2, 0, 0) == [1, 2]
    assert kept_rows([1, 2], 4, 1, 1) == [0, 1]
    x, i = apply_rules([2.0, -1.0, 3.0, 3.0], [2, 2, 1], (2.0, 0.5, 0.25), [(0, 1.0), (0, 5.0)], [True, True, True, False])
    assert np.array_equal(x, [7.0, -2.75, 0.5, -np.inf]) and i == 0
    assert apply_rules([1.0, 1.0])[1] == 1 and apply_rules([1.0], allowed=[False])[1] == -1

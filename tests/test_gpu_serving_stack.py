"""The serving operators through stacks and routes as a server meets them:
create_transformer's default stack (a compressed prompt, layers of 2 and 4
heads) with weights and evictions, trees of many rows, and logits that stay on
the device from the tree to the rules.

Bar: Re-logits within REL_TOL (conftest.max_rel_err) of the plain stacks."""
from __future__ import annotations

import numpy as np
import pytest

import plain_default_stack as pd
import rustcrates_amd as ra
from conftest import REL_TOL, build_explicit, max_rel_err, seeded_tensors
from plain_stack import Sequence, apply_rules
from rustcrates_amd import configs, seeded
from test_gpu_tree_step import CFG, path_to, tree_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S", [(1, 37), (3, 30)])
def test_evictions_on_the_default_stack(B, S):
    V, ctx = 300, 48
    prompt = seeded.prompts(6, [S] * B, V)
    r = np.random.default_rng(4)
    with configs.build_reference_default(ra.Network(0), V, 5, ctx, wavelet_embedding=False) as g:
        t = pd.tensors(g, V, ctx)
        seqs = [pd.Sequence(t) for _ in range(B)]
        first = g.prefill(prompt)
        for b, s in enumerate(seqs):
            assert first[b] == np.argmax(s.prompt(prompt[b]))
        for keep, sinks, recent in [(14, 2, 4), (14, 2, 4), (9, 0, 0)]:
            for _ in range(3):
                # the root, which weighs, a branch that is taken and one that is dropped
                ids = r.integers(2, V, (B, 4)).astype(np.uint32)
                par = [[-1, 0, 0, 2]] * B
                _, lg = g.tree_step(ids, par, weigh_nodes=1, want_logits=True)
                g.tree_accept([[0, 2, 3]] * B)
                for b, s in enumerate(seqs):
                    f = s.fork()
                    want = [s.step(int(ids[b, 0]), weigh=True), None, s.step(int(ids[b, 2])), s.step(int(ids[b, 3]))]
                    f.step(int(ids[b, 0]))
                    want[1] = f.step(int(ids[b, 1]))
                    assert max_rel_err(lg[b], np.array(want)) < REL_TOL, (keep, b)
            tok = r.integers(2, V, B).astype(np.uint32)
            _, lg = g.decode_step(tok, want_logits=True)
            for b, s in enumerate(seqs):
                assert max_rel_err(lg[b], s.step(int(tok[b]))) < REL_TOL, (keep, b)
            assert g.evict_rows(B, keep, sinks, recent).tolist() == [keep] * B
            for s in seqs:
                s.evict(keep, sinks, recent)
        fed = np.full(B, 7, np.uint32)
        for k in range(3):
            i, lg = g.decode_step(None if k else fed, want_logits=True)
            for b, s in enumerate(seqs):
                want = s.step(int(fed[b]))
                assert max_rel_err(lg[b], want) < REL_TOL and i[b] == np.argmax(want), b
            fed = i.copy()
        # a new prompt counts its own positions
        seqs = [pd.Sequence(t) for _ in range(B)]
        first = g.prefill(prompt[:, :11])
        _, lg = g.decode_step([9] * B, want_logits=True)
        for b, s in enumerate(seqs):
            assert first[b] == np.argmax(s.prompt(prompt[b, :11]))
            assert max_rel_err(lg[b], s.step(9)) < REL_TOL


@pytest.mark.parametrize("B,n,counts", [(10, 12, None), (40, 8, True), (3, 40, True), (2, 100, None)])
def test_trees_of_many_rows(B, n, counts):
    cfg = configs.ModelConfig(**{**CFG.__dict__, "max_ctx": 130})
    t = seeded_tensors(cfg)
    r = np.random.default_rng(B)
    lens = [int(x) for x in r.integers(1, 20, B)]
    prompt = seeded.prompts(50 + B, lens, cfg.vocab)
    ids, par = tree_of(r, B, n, cfg.vocab)
    counts = np.full(B, n, np.uint32) if counts is None else r.integers(0, n + 1, B).astype(np.uint32)
    counts[0] = n
    with build_explicit(ra.Network(0), cfg, t) as g:
        g.prefill(prompt, lens=lens)
        out, lg = g.tree_step(ids, par, counts=counts, weigh_nodes=n // 2, want_logits=True)
    for b in {0, 1, B // 2, B - 1}:
        s = Sequence(cfg, t)
        s.prompt(prompt[b, :lens[b]])
        for i in {0, 1, n // 3, n // 2, n - 1}:
            if i >= counts[b]:
                assert out[b, i] == ra.NO_TOKEN
                continue
            f = s.fork()
            want = [f.step(int(ids[b, j])) for j in path_to(par[b], i)][-1]
            assert max_rel_err(lg[b, i], want) < REL_TOL, (b, i)
            assert out[b, i] == np.argmax(want)


def test_logits_that_stay_on_the_device_from_the_tree_to_the_rules():
    """tree_step_device into process_logits_device, in place, over every row of a
    ragged batch: each node's id after its own history, biases and mask."""
    cfg = CFG
    t = seeded_tensors(cfg)
    lens, B, n, V, H = [9, 6, 13], 3, 5, cfg.vocab, 32
    r = np.random.default_rng(8)
    prompt = seeded.prompts(60, lens, V)
    ids, par = tree_of(r, B, n, V)
    counts = np.array([5, 2, 0], np.uint32)
    rows = B * n
    history = np.full((rows, H), -1, np.int32)
    for b in range(B):
        for i in range(n):
            h = [*prompt[b, :lens[b]], *(int(ids[b, j]) for j in path_to(par[b], i))]
            history[b * n + i, :len(h)] = h
    pen = np.tile([1.4, 0.3, 0.2], (rows, 1))
    bias_ids, bias = np.tile([4, 8], (rows, 1)).astype(np.int32), np.tile([0.7, -0.4], (rows, 1))
    allowed = np.zeros((rows, -(-V // 32) * 32), bool)
    allowed[:, :V] = r.random((rows, V)) < 0.5
    host = dict(history=history, penalties=pen, bias_ids=bias_ids, bias=bias,
                allowed=np.ascontiguousarray(np.packbits(allowed, axis=1, bitorder="little")))
    with build_explicit(ra.Network(0), cfg, t) as g:
        g.prefill(prompt, lens=lens)
        d = {k: ra.DeviceBuffer(a.nbytes) for k, a in host.items()}
        for k, a in host.items():
            d[k].upload(a)
        lg, best = ra.DeviceBuffer(rows * V * 8), ra.DeviceBuffer(rows * 4)
        g.tree_step_device(ids, par, lg, counts=counts, weigh_nodes=1)
        g.process_logits_device(lg, rows, V, out=lg, ids=best, max_history=H, max_bias=2, **d)
        got, nxt = lg.download((B, n, V), float), best.download((B, n), np.uint32)
        g.tree_accept([[0], [0], [0]], [1, 1, 0])
        for x in [lg, best, *d.values()]:
            x.free()
    for b in range(B):
        s = Sequence(cfg, t)
        s.prompt(prompt[b, :lens[b]])
        for i in range(int(counts[b])):
            f, k = s.fork(), b * n + i
            plain = [f.step(int(ids[b, j])) for j in path_to(par[b], i)][-1]
            want, top = apply_rules(plain, history[k], pen[k], list(zip(bias_ids[k].tolist(), bias[k])), allowed[k, :V])
            m = ~np.isneginf(want)
            assert np.array_equal(np.isneginf(got[b, i]), ~m)
            assert max_rel_err(got[b, i][m], want[m]) < REL_TOL and nxt[b, i] == top, (b, i)

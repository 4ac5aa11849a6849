"""Beam search through the stack (mitok_beam_search) against one written out over
the plain stacks, every hypothesis a sequence of its own; and the three operators
in the order in which a caller uses them on caches of its own.

A score is a sum of log probabilities, each of logits within REL_TOL of their row's
largest: within 2 REL_TOL max|logit| a token.  Ids are compared where the plain
search's ranks lie further apart than that, which each test asserts of its inputs."""
from __future__ import annotations

import numpy as np
import pytest

import plain_default_stack as pd
import rustcrates_amd as ra
from conftest import REL_TOL, build_explicit, seeded_tensors
from plain_stack import Sequence
from rustcrates_amd import configs, seeded
from test_gpu_paged_attention import put
from test_gpu_tree_step import rope_stack

pytestmark = pytest.mark.gpu
CFG = configs.ModelConfig("bs", layers=2, d=32, heads=2, ffn=48, vocab=90, max_ctx=64, seed=4)
NONE = ra.NO_TOKEN


def log_softmax(x):
    x = x - x.max()
    return x - np.log(np.exp(x).sum())


def plain_search(seq, logits, K, n_new, end=None, power=0.0):
    """([(tokens, score)], the least distance between two ranks at or before the first that was not kept, the largest |logit|)"""
    hyps, gap, big = [([], 0.0, False, seq, logits)], np.inf, 0.0
    for s in range(n_new):
        found = []
        for r, (toks, score, done, _, x) in enumerate(hyps):
            if done:
                found.append((score / len(toks) ** power, r, None, score))
                continue
            big = max(big, np.abs(x).max())
            lp = log_softmax(x)
            for t in np.argsort(-lp, kind="stable")[:K + 1]:
                found.append(((score + lp[t]) / (len(toks) + 1) ** power, r, int(t), score + lp[t]))
        found.sort(key=lambda a: -a[0])
        ranks = np.array([f[0] for f in found[:K + 1]])
        gap = min(gap, np.min(-np.diff(ranks), initial=np.inf))
        new = []
        for _, r, t, score in found[:K]:
            toks, _, _, q, x = hyps[r]
            if t is None:
                new.append((toks, score, True, None, None))
                continue
            over = t == end
            q = None if over or s + 1 == n_new else q.fork()
            new.append((toks + [t], score, over, q, None if q is None else q.step(t)))
        hyps = new
    return [(h[0], h[1]) for h in hyps], gap, big


def check(got, b, want, gap, big, n_new):
    ids, lens, scores = (a[b] for a in got)
    tol = 2 * REL_TOL * big * n_new
    assert gap > 4 * tol, "the inputs leave the order open"
    for k, (toks, score) in enumerate(want):
        assert lens[k] == len(toks) and ids[k, :len(toks)].tolist() == toks, (b, k, ids[k], toks)
        assert (ids[k, len(toks):] == NONE).all() and abs(scores[k] - score) <= tol, (b, k)


@pytest.fixture(scope="module", params=[False, True], ids=["plain", "rope"])
def model(request):
    cfg = CFG if not request.param else configs.ModelConfig(**{**CFG.__dict__, "rope": True})
    t = seeded_tensors(CFG)
    build = (lambda net: rope_stack(net, cfg, t)) if request.param else (lambda net: build_explicit(net, cfg, t))
    return cfg, t, build


@pytest.mark.parametrize("K,n_new,power", [(1, 6, 0.0), (3, 20, 0.0), (5, 18, 1.0), (8, 3, 0.5), (4, 1, 0.0)])
def test_against_a_search_written_out(model, K, n_new, power):
    cfg, t, build = model
    lens = [13, 5, 16, 1]
    prompt = seeded.prompts(70 + K, lens, cfg.vocab)
    with build(ra.Network(0)) as g:
        got = g.beam_search(prompt, lens=lens, beams=K, n_new=n_new, length_power=power)
    for b in range(len(lens)):
        s = Sequence(cfg, t)
        first = s.prompt(prompt[b, :lens[b]])
        check(got, b, *plain_search(s, first, K, n_new, power=power), n_new)


@pytest.mark.parametrize("power", [0.0, 0.8])
def test_hypotheses_that_end(model, power):
    """The end is a token that the search without one chooses often, so some end early and some on the last step."""
    cfg, t, build = model
    lens, K, n_new = [9, 17], 4, 12
    prompt = seeded.prompts(80, lens, cfg.vocab)
    plain = []
    for b in range(2):
        s = Sequence(cfg, t)
        plain.append((s, s.prompt(prompt[b, :lens[b]])))
    free = [plain_search(s.fork(), x, K, n_new)[0] for s, x in plain]
    toks = np.concatenate([h[0][2:] for f in free for h in f])
    end = int(np.bincount(toks).argmax())
    with build(ra.Network(0)) as g:
        got = g.beam_search(prompt, lens=lens, beams=K, n_new=n_new, end_id=end, length_power=power)
    assert (got[1] < n_new).any()
    for b, (s, x) in enumerate(plain):
        check(got, b, *plain_search(s, x, K, n_new, end=end, power=power), n_new)


def test_all_ended_long_before_the_last_token(model):
    cfg, t, build = model
    prompt = seeded.prompts(81, [8], cfg.vocab)
    t = [dict(x) for x in t]
    t[-1]["b"] = np.array(t[-1]["b"])
    t[-1]["b"][7] += 60.0  # every beam but the ended ones chooses 7
    build = (lambda net: rope_stack(net, cfg, t)) if cfg.rope else (lambda net: build_explicit(net, cfg, t))
    with build(ra.Network(0)) as g:
        ids, lens, scores = g.beam_search(prompt, beams=3, n_new=50, end_id=7)
        assert lens[0].tolist() == [1, 2, 2] and ids[0, 0, 0] == 7 and (ids[0, 1:, 1] == 7).all()
        assert (ids[0, :, 2:] == NONE).all() and (np.diff(scores[0]) <= 0).all()


def test_one_beam_is_the_token_loop(model):
    cfg, t, build = model
    lens = [20, 3, 11, 7, 30]
    prompt = seeded.prompts(82, lens, cfg.vocab)
    with build(ra.Network(0)) as g:
        want = g.generate(prompt, lens=lens, n_new=34)
        ids, n, scores = g.beam_search(prompt, lens=lens, beams=1, n_new=34)
        assert np.array_equal(ids[:, 0], want) and (n == 34).all() and (scores < 0).all()
        again = g.beam_search(prompt, lens=lens, beams=1, n_new=34)
        assert all(np.array_equal(x, y) for x, y in zip((ids, n, scores), again))
        assert np.array_equal(g.generate(prompt, lens=lens, n_new=34), want)  # and leaves nothing behind


def test_more_beams_than_tokens():
    """The first step has fewer continuations than beams; empty ones stay last."""
    cfg = configs.ModelConfig("bv", layers=1, d=16, heads=2, ffn=24, vocab=5, max_ctx=32, seed=2)
    t = seeded_tensors(cfg)
    prompt = np.array([[2, 3, 4]], np.uint32)
    with build_explicit(ra.Network(0), cfg, t) as g:
        ids, lens, scores = g.beam_search(prompt, beams=12, n_new=1)
        assert lens[0].tolist() == [1] * 5 + [0] * 7 and sorted(ids[0, :5, 0]) == list(range(5))
        assert (scores[0, 5:] == -np.inf).all() and (ids[0, 5:] == NONE).all()
        ids, lens, scores = g.beam_search(prompt, beams=12, n_new=2)
        got = g.beam_search(prompt, beams=12, n_new=7)
    s = Sequence(cfg, t)
    first = s.prompt(prompt[0])
    check((ids, lens, scores), 0, *plain_search(s.fork(), first, 12, 2), 2)
    check(got, 0, *plain_search(s, first, 12, 7), 7)


@pytest.mark.parametrize("B,S", [(1, 37), (3, 30)])
def test_the_default_stack(B, S):
    """A compressed prompt, RoPE at the uncompressed positions, layers of 2 and 4 heads."""
    V, ctx = 300, 64
    prompt = seeded.prompts(6, [S] * B, V)
    with configs.build_reference_default(ra.Network(0), V, 5, ctx, wavelet_embedding=False) as g:
        t = pd.tensors(g, V, ctx)
        got = g.beam_search(prompt, beams=4, n_new=20)
        assert np.array_equal(g.beam_search(prompt, beams=1, n_new=20)[0][:, 0], g.generate(prompt, n_new=20))
    for b in range(B):
        s = pd.Sequence(t)
        first = s.prompt(prompt[b])
        check(got, b, *plain_search(s, first, 4, 20), 20)


def test_many_prompts_and_a_wide_vocabulary():
    """More rows than a launch's arguments hold, more than one block of logits to a row."""
    cfg = configs.ModelConfig("bw", layers=1, d=16, heads=1, ffn=16, vocab=1500, max_ctx=40, seed=9)
    t = seeded_tensors(cfg)
    r = np.random.default_rng(1)
    lens = [int(x) for x in r.integers(1, 25, 70)]
    prompt = seeded.prompts(90, lens, cfg.vocab)
    with build_explicit(ra.Network(0), cfg, t) as g:
        got = g.beam_search(prompt, lens=lens, beams=5, n_new=6)
    for b in (0, 1, 33, 69):
        s = Sequence(cfg, t)
        first = s.prompt(prompt[b, :lens[b]])
        check(got, b, *plain_search(s, first, 5, 6), 6)


def test_up_to_the_last_row_of_the_context(model):
    cfg, t, build = model
    prompt = seeded.prompts(83, [44], cfg.vocab)
    with build(ra.Network(0)) as g:
        ids, lens, _ = g.beam_search(prompt, beams=2, n_new=21)  # the last token is not fed
        assert (lens == 21).all() and (ids < cfg.vocab).all()
        with pytest.raises(ra.MitokError, match="max context"):
            g.beam_search(prompt, beams=2, n_new=22)
        assert np.array_equal(g.beam_search(prompt, beams=2, n_new=21)[0], ids)


def test_an_error_leaves_the_network_usable(model):
    cfg, t, build = model
    prompt = seeded.prompts(84, [6], cfg.vocab)
    with build(ra.Network(0)) as g:
        want = g.beam_search(prompt, beams=3, n_new=5)
        with pytest.raises(ra.MitokError, match="No token embedding found"):
            g.beam_search(np.array([[cfg.vocab]]), beams=3, n_new=5)
        for a, b in zip(g.beam_search(prompt, beams=3, n_new=5), want):
            assert np.array_equal(a, b)


def test_the_operators_on_a_callers_own_caches():
    """Two prompts in two chunks each, then beams: selection, fork and attention on
    device arrays from step to step, against hypotheses that keep rows of their own."""
    r = np.random.default_rng(12)
    G, K, H, dh, ps, V, P, pages, steps = 2, 3, 2, 16, 16, 400, 8, 64, 30
    d, N = H * dh, G * K
    c = lambda *s: r.standard_normal(s) + 1j * r.standard_normal(s)  # noqa: E731
    qkv, head, bias = c(3, V, d), c(d, V) / 4, 0.3 * r.standard_normal((H, P * ps))
    prompts = [r.integers(0, V, n) for n in (37, 21)]

    def attend(rows, tok):
        out = np.zeros(d, complex)
        for h in range(H):
            s = slice(h * dh, (h + 1) * dh)
            K_, V_ = (np.array([qkv[i, t, s] for t in rows]) for i in (1, 2))
            x = (K_ @ qkv[0, tok, s]).real / (1e-8 + np.sqrt(dh)) + bias[h, :len(rows)]
            w = np.exp(x - x.max())
            out[s] = (w / w.sum()) @ V_
        return out

    with ra.Network(0) as net:
        pool = [put(np.zeros((pages, H, ps, dh), complex)) for _ in range(2)]
        bias_d = put(bias)
        table, lens_d = put(np.zeros((N, P), np.uint32)), put(np.zeros(N, np.uint32))
        parents, tokens, scores = put(np.zeros(N, np.uint32)), put(np.zeros(N, np.uint32)), put(np.zeros(N))

        def attention(rows, lens, counts):
            n = rows.shape[1]
            b = [put(qkv[i][rows]) for i in range(3)]
            o = put(np.zeros((len(rows), n, d), complex))
            net.paged_attention_device(*b, *pool, table, lens, n, H, dh, ps, pages, P, o, counts=counts, bias=bias_d, bias_stride=P * ps)
            out = o.download((len(rows), n, d), complex)
            for x in [*b, o]:
                x.free()
            return out

        def fork(old, new, grow):
            g = put(np.asarray(grow, np.uint32))
            net.fork_pages_device(*pool, 1, pages, H, ps, dh, table, lens_d, old, P, parents, new, table, lens_d, grow=g)
            g.free()

        lens = np.zeros(G, np.int64)
        for lo, hi in ((0, 16), (16, 99)):  # the prompts in two chunks
            part = [p[lo:hi] for p in prompts]
            n = np.array([len(p) for p in part])
            rows = np.array([np.r_[p, np.zeros(n.max() - len(p), int)] for p in part])
            parents.upload(np.arange(G, dtype=np.uint32))
            lens_d.upload(lens.astype(np.uint32))
            fork(G, G, n)
            out = attention(rows, lens, n)
            lens = lens + n
        logits = np.array([(out[b, n[b] - 1] @ head).real for b in range(G)])
        hyps = [[(list(p), 0.0)] for p in prompts]
        for b in range(G):
            assert np.allclose(out[b, n[b] - 1], attend(prompts[b], prompts[b][-1]), rtol=1e-12, atol=1e-12)
        old, had = G, [np.zeros((G, 1))]
        for step in range(steps):
            x = put(logits)
            s0 = put(had[0])
            net.beam_select_device(x, s0, G, old // G, V, K, parents, tokens, scores)
            x.free(), s0.free()
            pr, tk, sc = parents.download(N, np.uint32), tokens.download(N, np.uint32), scores.download(N, float)
            for b in range(G):  # the same, written out
                found = [(score + lp, r_, t) for r_, (rows, score) in enumerate(hyps[b])
                         for t, lp in enumerate(log_softmax((attend(rows, rows[-1]) @ head).real))]
                found = sorted(found, key=lambda a: -a[0])[:K + 1]
                assert np.min(-np.diff([f[0] for f in found])) > 1e-8, "the inputs leave the order open"
                assert [(int(p) - b * (old // G), int(t)) for p, t in zip(pr[b * K:(b + 1) * K], tk[b * K:(b + 1) * K])] == \
                    [(f[1], f[2]) for f in found[:K]], (step, b)
                assert np.allclose(sc[b * K:(b + 1) * K], [f[0] for f in found[:K]], rtol=0, atol=1e-10)
                hyps[b] = [(hyps[b][f[1]][0] + [f[2]], f[0]) for f in found[:K]]
            lens_d.upload(np.asarray(lens, np.uint32))
            fork(old, N, np.ones(N))
            lens = lens[pr]
            assert np.array_equal(lens_d.download(N, np.uint32), lens)
            out = attention(tk[:, None].astype(np.int64), lens, None)
            lens = lens + 1
            logits, had, old = (out[:, 0] @ head).real, [sc], N
        for x in [*pool, bias_d, table, lens_d, parents, tokens, scores]:
            x.free()

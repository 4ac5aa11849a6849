"""Trees of drafted tokens through a whole stack: mitok_tree_step, mitok_tree_accept
and mitok_evict_rows against the CPU checker and the plain stack, and all of the
serving operators together as a decoding loop uses them.

Bar: Re-logits within REL_TOL of single steps along each node's path, greedy ids equal."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
import rustcrates_amd as ra
from conftest import REL_TOL, build_explicit, max_rel_err, seeded_tensors
from plain_stack import Sequence, apply_rules, kept_rows
from rustcrates_amd import configs, seeded

pytestmark = pytest.mark.gpu

CFG = configs.ModelConfig("ts", layers=2, d=64, heads=4, ffn=96, vocab=300, max_ctx=64, seed=6)


def rope_stack(net, cfg, t):
    net.add_embedding(cfg.vocab, cfg.d, t[0]["table"])
    net.add_positional_encoding(cfg.d, cfg.rope_base)
    for a in range(cfg.layers):
        n, s, f = t[1 + 3 * a: 4 + 3 * a]
        net.add_norm(cfg.d, cfg.norm_eps, n["gamma"], n["beta"])
        net.add_self_attention(cfg.heads, cfg.d, cfg.max_ctx, cfg.attn_eps, s["wq"], s["wk"], s["wv"], s["bias_pos"],
                               s["gamma"], s["beta"])
        net.add_feed_forward(cfg.d, cfg.ffn, f["w1"], f["b1"], f["w2"], f["b2"])
    net.add_linear(cfg.d, cfg.vocab, t[-1]["w"], t[-1]["b"])
    net.add_softmax(1)
    return net


@pytest.fixture(scope="module", params=[False, True], ids=["plain", "rope"])
def model(request):
    """(cfg, tensors, a function that builds a network of them)"""
    cfg = CFG if not request.param else configs.ModelConfig(**{**CFG.__dict__, "rope": True})
    t = seeded_tensors(CFG)
    build = (lambda net: rope_stack(net, cfg, t)) if request.param else (lambda net: build_explicit(net, cfg, t))
    return cfg, t, build


def tree_of(r, B, n, V):
    par = np.full((B, n), -1)
    for b in range(B):
        for i in range(1, n):
            par[b, i] = r.integers(max(-1, i // 2 - 2), i)
    return r.integers(0, V, (B, n)).astype(np.uint32), par


def path_to(par, i):
    p = []
    while i >= 0:
        p.append(int(i))
        i = par[i]
    return p[::-1]


@pytest.mark.parametrize("lens,n", [([7], 1), ([5, 11, 9], 6), ([3 + b % 9 for b in range(10)], 8)])
def test_nodes_are_the_checkers_steps_along_their_paths(model, lens, n):
    cfg, t, build = model
    r = np.random.default_rng(n)
    B = len(lens)
    prompt = seeded.prompts(30 + n, lens, cfg.vocab)
    ids, par = tree_of(r, B, n, cfg.vocab)
    ids[0, n // 2] = 1  # PAD: the zero embedding
    counts = np.array([max(1, n - b % 3) for b in range(B)], np.uint32)
    with build(ra.Network(0)) as g:
        g.prefill(prompt, lens=lens)
        out, lg = g.tree_step(ids, par, counts=counts, want_logits=True)
        again, lg2 = g.tree_step(ids, par, counts=counts, weigh_nodes=n, want_logits=True)  # nothing was committed
        assert np.array_equal(out, again) and np.array_equal(lg[0, 0], lg2[0, 0])
    o = build(oracle.Network())
    for b in range(B if B < 4 else 2):
        for i in range(int(counts[b])):
            o.reset()
            o.predict(prompt[b:b + 1, :lens[b]])
            for k, j in enumerate(path_to(par[b], i)):
                want, _ = o.predict(ids[b:b + 1, j:j + 1], time_steps=[lens[b] + k])
            err = max_rel_err(lg[b, i], want[0, 0])
            assert err < REL_TOL, (b, i, err)
            assert out[b, i] == oracle.greedy_row(want[0, 0])
        assert (out[b, int(counts[b]):] == ra.NO_TOKEN).all()
    o.close()


@pytest.mark.parametrize("path", [[0], [0, 2, 5], [0, 1, 3], []])
def test_accepted_nodes_are_the_cache_of_single_steps(model, path):
    cfg, t, build = model
    prompt = seeded.prompts(8, [9, 6], cfg.vocab)
    par = np.array([[-1, 0, 0, 1, 0, 2], [-1, 0, 1, 2, 3, 4]])
    r = np.random.default_rng(3)
    ids = r.integers(2, cfg.vocab, (2, 6)).astype(np.uint32)
    paths = np.zeros((2, 3), np.uint32)
    paths[0, :len(path)] = path
    paths[1] = [0, 1, 2]
    s = [Sequence(cfg, t) for _ in range(2)]
    after = []
    for b, p in enumerate((path, [0, 1])):
        lg = s[b].prompt(prompt[b, :[9, 6][b]])
        for i in p:
            lg = s[b].step(int(ids[b, i]))
        after.append(lg)
    with build(ra.Network(0)) as g:
        first = g.prefill(prompt, lens=[9, 6])
        g.tree_step(ids, par)
        g.tree_accept(paths, [len(path), 2])
        fed, lg = g.decode_step(want_logits=True)  # feeds the greedy id after the last accepted node
        for b in range(2):
            tok = int(first[b]) if b == 0 and not path else int(np.argmax(after[b]))
            want = s[b].step(tok)
            assert max_rel_err(lg[b], want) < REL_TOL, b
            assert fed[b] == np.argmax(want)
        with pytest.raises(ra.MitokError, match="without a tree_step"):
            g.tree_accept(paths, [1, 1])


def test_a_chain_on_the_default_stack_counts_positions_of_the_uncompressed_prompt():
    """create_transformer's stack compresses the prompt before RoPE: a chain of
    nodes gives what decode steps give."""
    build = lambda net: configs.build_reference_default(net, 400, 3, 96, wavelet_embedding=False)  # noqa: E731
    prompt = seeded.prompts(2, [21], 400)
    with build(ra.Network(0)) as g:
        a = [int(g.prefill(prompt)[0])]
        logits = []
        for _ in range(4):
            i, lg = g.decode_step(want_logits=True)
            a.append(int(i[0]))
            logits.append(lg[0])
        g.prefill(prompt)
        out, lg = g.tree_step([a[:4]], [[-1, 0, 1, 2]], want_logits=True)
        assert out[0].tolist() == a[1:] and max_rel_err(lg[0], np.array(logits)) < REL_TOL
        g.tree_accept([[0, 1]])
        assert g.decode_step([a[2]])[0] == a[3]


@pytest.mark.parametrize("steps", [1, 5])
def test_eviction_in_a_stack(model, steps):
    """Steps that weigh, an eviction, further steps, another eviction: the plain
    stack that takes the same rows out of its lists."""
    cfg, t, build = model
    lens = [22, 13, 30]
    prompt = seeded.prompts(14, lens, cfg.vocab)
    seqs = [Sequence(cfg, t) for _ in lens]
    with build(ra.Network(0)) as g:
        g.prefill(prompt, lens=lens)
        with pytest.raises(ra.MitokError, match="no tree_step"):
            g.evict_rows(3, 16, 2, 4)
        for b, s in enumerate(seqs):
            s.prompt(prompt[b, :lens[b]])
        r = np.random.default_rng(5)
        for rnd, (keep, sinks, recent) in enumerate([(16, 2, 4), (12, 0, 3)]):
            for _ in range(steps):
                tok = r.integers(2, cfg.vocab, 3).astype(np.uint32)
                _, lg = g.tree_step(tok[:, None], [[-1]] * 3, weigh_nodes=1, want_logits=True)
                g.tree_accept([[0]] * 3)
                for b, s in enumerate(seqs):
                    assert max_rel_err(lg[b, 0], s.step(int(tok[b]), weigh=True)) < REL_TOL, (rnd, b)
            tok = r.integers(2, cfg.vocab, 3).astype(np.uint32)  # a step that does not weigh
            _, lg = g.decode_step(tok, want_logits=True)
            for b, s in enumerate(seqs):
                assert max_rel_err(lg[b], s.step(int(tok[b]))) < REL_TOL, (rnd, b)
            left = g.evict_rows(3, keep, sinks, recent)
            for b, s in enumerate(seqs):
                s.evict(keep, sinks, recent)
                assert left[b] == len(s.k[0][0])
        for _ in range(3):  # ordinary decode steps go on from the packed cache
            tok = r.integers(2, cfg.vocab, 3).astype(np.uint32)
            i, lg = g.decode_step(tok, want_logits=True)
            for b, s in enumerate(seqs):
                want = s.step(int(tok[b]))
                assert max_rel_err(lg[b], want) < REL_TOL and i[b] == np.argmax(want)


def test_weights_of_an_accepted_path_move_with_its_rows(model):
    """Several nodes weigh, a rejected one among them, and the path's rows do not
    lie together: each keeps its own weight, which the next eviction goes by."""
    cfg, t, build = model
    lens, path, weigh = [11, 17], [0, 2, 4, 5], 5
    par = np.array([[-1, 0, 0, 1, 2, 4]] * 2)
    prompt = seeded.prompts(41, lens, cfg.vocab)
    ids = np.random.default_rng(19).integers(2, cfg.vocab, (2, 6)).astype(np.uint32)
    keep, seqs, unmoved = 10, [], False
    for b, L in enumerate(lens):
        s = Sequence(cfg, t)
        s.prompt(prompt[b, :L])
        slots = np.zeros((cfg.layers, cfg.heads, L + 6))  # committed rows, then nodes
        for i in range(weigh):
            f, way = s.fork(), path_to(par[b], i)
            for j in way:
                f.step(int(ids[b, j]), weigh=j == i)
            slots[:, :, [*range(L), *(L + j for j in way)]] += np.array(f.weights)
        for j in path:
            s.step(int(ids[b, j]))
        for layer in range(cfg.layers):
            for h in range(cfg.heads):
                own = slots[layer, h, [*range(L), *(L + j for j in path)]]
                s.weights[layer][h] = list(own)
                unmoved |= kept_rows(list(slots[layer, h, :L + 4]), keep, 0, 0) != kept_rows(list(own), keep, 0, 0)
        seqs.append(s)
    assert unmoved  # weights left where they were would keep other rows
    with build(ra.Network(0)) as g:
        g.prefill(prompt, lens=lens)
        g.tree_step(ids, par, weigh_nodes=weigh)
        g.tree_accept([path] * 2)
        assert g.evict_rows(2, keep, 0, 0).tolist() == [keep, keep]
        for s in seqs:
            s.evict(keep, 0, 0)
        for tok in (7, 12):
            _, lg = g.decode_step(np.array([tok, tok + 1], np.uint32), want_logits=True)
            for b, s in enumerate(seqs):
                assert max_rel_err(lg[b], s.step(tok + b)) < REL_TOL, (tok, b)


def test_a_prompt_starts_weights_anew_and_generate_is_what_it_was(model):
    cfg, t, build = model
    prompt = seeded.prompts(15, [20, 12], cfg.vocab)
    with build(ra.Network(0)) as fresh:
        want = [fresh.generate(prompt, [20, 12], 12)]
        fresh.set_decode_plan(0)
        want.append(fresh.generate(prompt, [20, 12], 12))
    with build(ra.Network(0)) as g:
        g.prefill(prompt, lens=[20, 12])
        for _ in range(3):
            g.tree_step([[5], [6]], [[-1], [-1]], weigh_nodes=1)
            g.tree_accept([[0], [0]])
        g.evict_rows(2, 8, 1, 2)
        assert np.array_equal(g.generate(prompt, [20, 12], 12), want[0])
        g.set_decode_plan(0)
        assert np.array_equal(g.generate(prompt, [20, 12], 12), want[1])
        g.prefill(prompt, lens=[20, 12])
        with pytest.raises(ra.MitokError, match="no tree_step"):
            g.evict_rows(2, 8, 1, 2)


def test_a_drafting_loop_with_rules_and_evictions(model):
    """The loop a server runs: drafts (some right, some wrong) in one pass, rules
    on every node's logits with its own history, the longest agreeing path
    committed, the cache packed whenever it is nearly full, past max_ctx tokens
    in all.  The plain stack generates the same tokens one by one."""
    cfg, t, build = model
    r = np.random.default_rng(17)
    prompt = seeded.prompts(21, [18], cfg.vocab)[0]
    pen = (1.3, 0.4, 0.1)
    banned = np.ones(cfg.vocab, bool)
    banned[::3] = False  # only these tokens
    allowed = ~banned

    def rule(lg, history):
        return apply_rules(lg, history, pen, [(6, 0.5)], allowed)[1]

    s = Sequence(cfg, t)
    keep, sinks, recent = 24, 2, 8
    got, evicted, committed = [rule(s.prompt(prompt), prompt)], 0, 0
    with build(ra.Network(0)) as g:
        _, lg = g.prefill(prompt[None], want_logits=True)
        _, ids = g.process_logits(lg, [prompt], [pen], [[6]], [[0.5]], [allowed])
        assert ids[0] == got[0]
        with ra.DeviceBuffer(7 * cfg.vocab * 8) as d_lg:
            while len(got) < 90:
                # what comes next, for drafting and for the check
                ahead, truth = s.fork(), []
                for _ in range(4):
                    truth.append(rule(ahead.step([got[-1], *truth][-1]), [*prompt, *got, *truth]))
                right = int(r.integers(0, 4))  # how many of the drafted ones agree
                wrong = [next(w for w in (6, 9, 12) if w != x) for x in truth]
                chain = truth[:right] + wrong[right:3]
                ids = [got[-1], *chain, wrong[0], wrong[1], chain[0]]
                par = [-1, 0, 1, 2, 0, 1, 5]
                n = len(ids)
                g.tree_step_device([ids], [par], d_lg, weigh_nodes=1)
                hist = np.full((n, 128), -1, np.int64)
                for i in range(n):
                    h = [*prompt, *got, *[ids[j] for j in path_to(par, i)[1:]]]
                    hist[i, :len(h)] = h
                _, nxt = g.process_logits(d_lg.download((n, cfg.vocab), float), hist, [pen] * n, [[6]] * n, [[0.5]] * n,
                                          [allowed] * n)
                path = [0]
                while True:
                    kids = [j for j in range(n) if par[j] == path[-1] and ids[j] == nxt[path[-1]]]
                    if not kids:
                        break
                    path.append(kids[0])
                g.tree_accept([path])
                new = [ids[j] for j in path[1:]] + [int(nxt[path[-1]])]
                assert new == truth[:len(new)] and len(new) == right + 1
                s.step(got[-1], weigh=True)
                for j in path[1:]:
                    s.step(ids[j])
                got += new
                committed += len(path)
                if len(s.k[0][0]) + 7 > cfg.max_ctx:
                    assert g.evict_rows(1, keep, sinks, recent)[0] == keep
                    s.evict(keep, sinks, recent)
                    evicted += 1
    assert evicted >= 2 and len(prompt) + committed > cfg.max_ctx


def test_trees_on_a_cache_that_predict_filled_with_launches_timed(model):
    """A forward_only predict leaves the caches too; attention launches are timed
    like the others."""
    cfg, t, build = model
    prompt = seeded.prompts(9, [12, 8], cfg.vocab)
    with build(ra.Network(0)) as g:
        g.prefill(prompt, lens=[12, 8])
        want, lg = g.tree_step([[5, 6], [7, 8]], [[-1, 0], [-1, -1]], want_logits=True)
        g.reset()
        g.predict(prompt, lens=[12, 8])
        g.timing_enable(ra.TIME_ATTENTION)
        got, lg2 = g.tree_step([[5, 6], [7, 8]], [[-1, 0], [-1, -1]], want_logits=True)
        timed = g.timing_read()
        g.timing_enable(0)
        assert np.array_equal(got, want) and np.array_equal(lg, lg2)
        assert timed["launches"] == cfg.layers and timed["total_ms"] > 0
        g.tree_accept([[0, 1], [1, 0]], [2, 1])
        assert np.array_equal(g.decode_step([3, 4]), g_steps(build, prompt, [12, 8], [[5, 6], [8]], [3, 4]))


def g_steps(build, prompt, lens, fed, last):
    """The same tokens one step at a time, each sequence in a network of its own: the ids after the last."""
    out = []
    for b in range(2):
        with build(ra.Network(0)) as g:
            g.prefill(prompt[b:b + 1, :lens[b]])
            for tok in fed[b]:
                g.decode_step([tok])
            out.append(int(g.decode_step([last[b]])[0]))
    return np.array(out, np.uint32)


def test_refusals(model):
    cfg, t, build = model

    def go(match, code, f):
        with pytest.raises(ra.MitokError, match=match) as e:
            f()
        assert e.value.code == code, e.value

    with build(ra.Network(0)) as g:
        go("before prefill", 3, lambda: g.tree_step([[3]], [[-1]]))
        go("before prefill", 3, lambda: g.evict_rows(1, 4))
        prompt = seeded.prompts(4, [60, 50], cfg.vocab)
        g.prefill(prompt, lens=[60, 50])
        two = [[3, 4]] * 2
        go("prefill first", 3, lambda: g.tree_step([[3, 4]], [[-1, 0]]))
        go("parents come before", 1, lambda: g.tree_step(two, [[-1, 1], [-1, 0]]))
        go("token id", 1, lambda: g.tree_step([[3, cfg.vocab], [3, 4]], [[-1, 0]] * 2))
        go("exceed max context", 1, lambda: g.tree_step([[3] * 5] * 2, [[-1] * 5] * 2))
        go("above", 1, lambda: g.tree_step(two, [[-1, 0]] * 2, counts=[2, 3]))
        go("weigh_nodes", 1, lambda: g.tree_step(two, [[-1, 0]] * 2, weigh_nodes=3))
        go("without a tree_step", 3, lambda: g.tree_accept([[0], [0]]))
        a = g.tree_step(two, [[-1, 0], [-1, -1]])
        go("does not follow", 1, lambda: g.tree_accept([[1], [0]]))
        go("does not follow", 1, lambda: g.tree_accept([[0, 1], [0, 1]]))
        go("node 2 of 2", 1, lambda: g.tree_accept([[2], [0]]))
        go("above", 1, lambda: g.tree_accept([[0], [0]], [1, 2]))
        go("cached batch", 3, lambda: g.tree_accept([[0]]))
        go("exceed keep", 1, lambda: g.evict_rows(2, 4, 3, 2))
        go("no tree_step", 3, lambda: g.evict_rows(2, 4, 1, 2))
        with ra.DeviceBuffer(2 * 2 * cfg.vocab * 8 - 8) as d:
            go("exceed its allocation", 1, lambda: g.tree_step_device(two, [[-1, 0]] * 2, d))
        # refusals leave the caches and the pending tree as they were
        g.tree_accept([[0, 1], [1, 0]], [2, 1])
        b = g.tree_step(two, [[-1, 0], [-1, -1]])
        assert a.shape == b.shape
        g.decode_step([3, 4])
        go("without a tree_step", 3, lambda: g.tree_accept([[0], [0]]))
        for bad in (dict(ids=[3, 4], parents=[[-1, 0]]), dict(ids=two, parents=[[-1, 0]]),
                    dict(ids=two, parents=[[-1, 0]] * 2, counts=[1])):
            with pytest.raises(ValueError):
                g.tree_step(**bad)

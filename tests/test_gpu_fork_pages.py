"""mitok_fork_pages_device against its definition, page by page."""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from test_gpu_paged_attention import put

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def make(seed, lens, parents, grow, H=2, dh=8, ps=16, layers=2, spare=None, share=0, width=None):
    """`share`: the sequences' first so many pages are the first one's."""
    r = np.random.default_rng(seed)
    lens, parents, grow = np.asarray(lens, np.uint32), np.asarray(parents, np.int64), np.asarray(grow, np.uint32)
    grow = np.broadcast_to(grow, parents.shape).astype(np.uint32)
    used = -(-lens.astype(np.int64) // ps)
    P = int(used.max() + -(-int(grow.max(initial=0)) // ps)) + 1 if width is None else width
    pages = int(used.sum()) + (len(parents) * (2 + int(grow.max(initial=0)) // ps) if spare is None else spare)
    order = iter(r.permutation(pages).tolist())
    table = np.full((len(lens), P), 0xFFFFFFF0, np.uint32)
    for i in range(len(lens)):
        for j in range(used[i]):
            table[i, j] = table[0, j] if i and j < min(share, used[0]) else next(order)
    c = lambda *s: r.standard_normal(s) + 1j * r.standard_normal(s)  # noqa: E731
    return dict(table=table, lens=lens, parents=(parents & NONE).astype(np.uint32), grow=grow, k=c(layers, pages, H, ps, dh),
                v=c(layers, pages, H, ps, dh), H=H, dh=dh, ps=ps, layers=layers, pages=pages, P=P)


def formula(c):
    """(table, lens, k, v), or None where there are too few pages"""
    ps, N, k, v = c["ps"], len(c["parents"]), c["k"].copy(), c["v"].copy()
    n = [0 if p == NONE else int(c["lens"][p]) for p in c["parents"]]
    g = [0 if p == NONE else int(x) for p, x in zip(c["parents"], c["grow"])]
    new = [[] if p == NONE else c["table"][p, :-(-n[i] // ps)].tolist() for i, p in enumerate(c["parents"])]
    holders = {}
    for i in range(N):
        for j, page in enumerate(new[i]):
            holders.setdefault(page, []).append((i, bool(g[i] and n[i] % ps and j == len(new[i]) - 1)))
    free = [p for p in range(c["pages"]) if p not in holders][::-1]
    table = np.full((N, c["P"]), NONE, np.uint32)
    try:
        for i in range(N):
            if g[i] and n[i] % ps:
                those = holders[new[i][-1]]
                if not all(w for _, w in those) or those[0][0] != i:
                    to = free.pop()
                    for x in (k, v):
                        x[:, to, :, :n[i] % ps] = x[:, new[i][-1], :, :n[i] % ps]
                    new[i][-1] = to
            while len(new[i]) * ps < n[i] + g[i]:
                new[i].append(free.pop())
            table[i, :len(new[i])] = new[i]
    except IndexError:
        return None
    return table, np.array(n, np.uint32), k, v


def call(net, c, in_place=False, grow=True):
    d = {x: put(c[x]) for x in ("table", "lens", "parents", "grow", "k", "v")}
    N = len(c["parents"])
    d["t2"] = put(np.full((N, c["P"]), 77, np.uint32))
    d["l2"] = put(np.full(N, 77, np.uint32))
    t2, l2 = ("table", "lens") if in_place else ("t2", "l2")
    error = None
    try:
        try:
            net.fork_pages_device(d["k"], d["v"], c["layers"], c["pages"], c["H"], c["ps"], c["dh"], d["table"], d["lens"],
                                  len(c["lens"]), c["P"], d["parents"], N, d[t2], d[l2], grow=d["grow"] if grow else None)
        except ra.MitokError as e:
            error = e
        got = (d[t2].download((N, c["P"]), np.uint32), d[l2].download(N, np.uint32), d["k"].download(c["k"].shape, complex),
               d["v"].download(c["v"].shape, complex))
        if not in_place:
            assert np.array_equal(d["table"].download(c["table"].shape, np.uint32), c["table"])
            assert np.array_equal(d["lens"].download(c["lens"].shape, np.uint32), c["lens"])
        return got, error
    finally:
        for b in d.values():
            b.free()


def check(net, c, **kw):
    got, error = call(net, c, **kw)
    assert error is None, error
    for name, a, b in zip(("table", "lens", "k", "v"), got, formula(c)):
        assert np.array_equal(a, b), name


@pytest.mark.parametrize("grow", [0, 1, 5, 16, 40])
@pytest.mark.parametrize("in_place", [False, True])
def test_beams_that_take_over_one_another(net, grow, in_place):
    check(net, make(grow, [37, 37, 37, 37], [1, 1, 3, 1], grow, share=2), in_place=in_place)
    check(net, make(grow, [32, 37, 1, 16], [3, 0, 1, 2], grow), in_place=in_place)
    check(net, make(grow, [7, 8, 9], [2, -1, 2], grow), in_place=in_place)


def test_more_and_fewer_sequences_than_before(net):
    check(net, make(1, [20, 0, 31], [0, 0, 0, 0, 1, 1, 2, 2, -1], 1))
    check(net, make(2, [20, 5, 31, 40], [2], 3))
    check(net, make(3, [0], [0, 0, 0], 17))


def test_one_that_stays_and_one_that_grows(net):
    """Nobody writes to a page that a sequence without room holds too."""
    check(net, make(4, [21, 21], [0, 0], [0, 1]))
    check(net, make(5, [21, 21], [0, 0], [1, 0]))
    check(net, make(6, [21, 21], [0, 0, 0], [4, 0, 4]))


def test_a_shorter_sequence_on_anothers_full_page(net):
    c = make(7, [32, 20], [0, 1], [0, 1])
    c["table"][1, :2] = c["table"][0, :2]  # it went back to 20 rows
    check(net, c)
    c["grow"][:] = 1
    check(net, c)


def test_a_page_twice_in_one_sequence(net):
    c = make(8, [40], [0], 1)
    c["table"][0, 2] = c["table"][0, 0]
    check(net, c)


def test_no_room_anywhere_without_grow(net):
    c = make(9, [37, 5], [0, 0], 0, spare=0)
    check(net, c, grow=False)


@pytest.mark.parametrize("seed", range(12))
def test_random_forks(net, seed):
    r = np.random.default_rng(100 + seed)
    old, new, ps = int(r.integers(1, 40)), int(r.integers(1, 60)), int(r.choice([16, 32, 48]))
    c = make(seed, r.integers(0, 6 * ps, old), r.integers(-1, old, new), r.choice([0, 0, 1, 1, 3, 50], new),
             H=int(r.integers(1, 5)), dh=int(r.choice([1, 8, 24, 64])), ps=ps, layers=int(r.integers(1, 4)))
    check(net, c)


def test_many_sequences_and_pages(net):
    r = np.random.default_rng(5)
    check(net, make(10, r.integers(0, 80, 1500), r.integers(-1, 1500, 2300), r.choice([0, 1, 20], 2300), H=1, dh=2, layers=1))
    check(net, make(11, r.integers(900, 1000, 64), r.integers(0, 64, 64), 1, H=1, dh=2, layers=1, share=50, width=300))


def test_forks_of_forks(net):
    """A chain of in-place forks: what each sequence's pages hold is its history."""
    r = np.random.default_rng(9)
    N, ps, H, dh, pages, P = 6, 16, 2, 4, 64, 8
    d = dict(k=put(np.zeros((1, pages, H, ps, dh), complex)), v=put(np.zeros((1, pages, H, ps, dh), complex)),
             table=put(np.zeros((N, P), np.uint32)), lens=put(np.zeros(N, np.uint32)), parents=put(np.zeros(N, np.uint32)),
             grow=put(np.ones(N, np.uint32)))
    rows = [[] for _ in range(N)]
    for step in range(60):
        parents = r.integers(-1, N, N) if step % 9 == 5 else np.sort(r.integers(0, N, N))
        rows = [[] if p < 0 else list(rows[p]) for p in parents]
        d["parents"].upload((parents & NONE).astype(np.uint32))
        net.fork_pages_device(d["k"], d["v"], 1, pages, H, ps, dh, d["table"], d["lens"], N, P, d["parents"], N, d["table"],
                              d["lens"], grow=d["grow"])
        table, lens = d["table"].download((N, P), np.uint32), d["lens"].download(N, np.uint32)
        k = d["k"].download((1, pages, H, ps, dh), complex)
        for i in range(N):
            if parents[i] < 0:
                continue
            rows[i].append(complex(step, i))
            k[0, table[i, lens[i] // ps], :, lens[i] % ps] = rows[i][-1]
            lens[i] += 1
        d["k"].upload(k)
        d["lens"].upload(lens)
        for i in range(N):
            got = [k[0, table[i, t // ps], 1, t % ps, 3] for t in range(lens[i])]
            assert got == rows[i], (step, i)
    for b in d.values():
        b.free()


@pytest.mark.parametrize("what,code,match", [("parent", 1, "parent"), ("page", 1, "outside the pool"), ("length", 1, "max_pages"),
                                             ("grow", 1, "max_pages"), ("pages", 5, "free pages")])
@pytest.mark.parametrize("in_place", [False, True])
def test_what_is_refused_changes_nothing(net, what, code, match, in_place):
    c = make(12, [37, 20, 50], [0, 0, 2], 1, spare=1 if what == "pages" else None)
    good = {k: v.copy() for k, v in c.items() if isinstance(v, np.ndarray)}
    if what == "parent":
        c["parents"][1] = 3
    if what == "page":
        c["table"][0, 1] = c["pages"]
    if what == "length":
        c["lens"][2] = 0xFFFFFFF0
    if what == "grow":
        c["grow"][1] = 0xFFFFFFFF
    if what == "pages":
        c["parents"][:] = [0, 0, 0]  # pages of 1 and 2 come free
        c["grow"][:] = [1, 90, 90]
        c["P"] = 10
        c["table"] = np.pad(c["table"], ((0, 0), (0, 10 - c["table"].shape[1])))
        assert formula(c) is None
    got, error = call(net, c, in_place=in_place)
    assert error is not None and error.code == code and match in str(error)
    before = (c["table"], c["lens"]) if in_place else (np.full_like(c["table"], 77), np.full_like(c["lens"], 77))
    for a, b in zip(got, (*before, c["k"], c["v"])):
        assert np.array_equal(a, b)
    c.update({k: v for k, v in good.items()})
    if what == "pages":
        c["P"] = c["table"].shape[1]
        c["parents"][:], c["grow"][:] = [0, 0, 1], [1, 1, 1]
    check(net, c)  # the counts that a refused call left are none

"""mitok_beam_select(_device) against its definition.

Tolerance of a score, u = 2^-53: the sum of V exponentials is within (V + 8) u of
itself on either side (each exponential within 2 u, and the error u |x - m| of
its argument times its weight below u), so its logarithm within as much and
u |log s|; the subtractions and the sum round to u of what they give.  The two sides
are within 2 ((V + 8) + 2 (|m| + |lse| + |x - lse| + |score|)) u.
"""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from test_gpu_paged_attention import put

pytestmark = pytest.mark.gpu
U = 2.0 ** -53
NONE = 0xFFFFFFFF


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def make(seed, B, R, V, K, done=0.0, scaled=True, spread=3.0):
    r = np.random.default_rng(seed)
    n = r.integers(1, 40, (B, R))
    return dict(x=spread * r.standard_normal((B, R, V)), scores=-2.0 * n * r.uniform(0.9, 1.1, (B, R)), done=r.random((B, R)) < done,
                scale=(n + 1.0) ** -0.7 if scaled else None, K=K)


def formula(c):
    """(parents, tokens, scores, tolerance)"""
    B, R, V = c["x"].shape
    K = c["K"]
    parents, tokens = np.full((B, K), NONE, np.uint32), np.full((B, K), NONE, np.uint32)
    best, tol = np.full((B, K), -np.inf), np.zeros((B, K))
    for b in range(B):
        found = []
        for r in range(R):
            had, f = c["scores"][b, r], 1.0 if c["scale"] is None else c["scale"][b, r]
            if had == -np.inf:
                continue
            if c["done"] is not None and c["done"][b, r]:
                found.append((-had * f, r, 0.0, NONE, had, 0.0))
                continue
            x = c["x"][b, r]
            m = x.max()
            if m == -np.inf:
                continue
            lse = m + np.log(np.exp(x - m).sum())
            for t in np.lexsort((np.arange(V), -x))[:K]:
                if x[t] > -np.inf:
                    y = had + (x[t] - lse)
                    err = 2 * U * (V + 8 + 2 * (abs(m) + abs(lse) + abs(x[t] - lse) + abs(y)))
                    found.append((-y * f, r, -x[t], int(t), y, err))
        for j, (_, r, _, t, y, err) in enumerate(sorted(found, key=lambda a: a[:4])[:K]):
            parents[b, j], tokens[b, j], best[b, j], tol[b, j] = b * R + r, t, y, err
    return parents, tokens, best, tol


def device(net, c):
    B, R, V = c["x"].shape
    K = c["K"]
    d = {k: put(np.ascontiguousarray(c[k], np.uint32 if k == "done" else float)) for k in ("x", "scores", "done", "scale") if c[k] is not None}
    d.update(p=put(np.full((B, K), 9, np.uint32)), t=put(np.full((B, K), 9, np.uint32)), s=put(np.full((B, K), 9.0)))
    try:
        net.beam_select_device(d["x"], d["scores"], B, R, V, K, d["p"], d["t"], d["s"], done=d.get("done"), scale=d.get("scale"))
        return d["p"].download((B, K), np.uint32), d["t"].download((B, K), np.uint32), d["s"].download((B, K), float)
    finally:
        for b in d.values():
            b.free()


def check(net, c):
    want = formula(c)
    host = net.beam_select(c["x"], c["scores"], c["K"], done=c["done"], scale=c["scale"])
    for p, t, s in (device(net, c), host):
        assert np.array_equal(p, want[0]), (p, want[0])
        assert np.array_equal(t, want[1])
        off = ~((s == want[2]) | (np.abs(s - want[2]) <= want[3]))
        assert not off.any(), (s[off], want[2][off], want[3][off])
    return want


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 511, 512, 513, 1000, 4097])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 5), (3, 3), (4, 8)])
def test_sizes(net, V, R, K):
    check(net, make(V + R, 3, R, V, K))


@pytest.mark.parametrize("B,R,V,K", [(1, 4, 32000, 4), (9, 5, 31999, 64), (2, 64, 5000, 64), (33, 2, 50280, 17), (1, 1024, 70, 40),
                                     (700, 1, 300, 2), (1, 1, 400001, 30)])
def test_larger(net, B, R, V, K):
    check(net, make(V, B, R, V, K))


def test_ended_and_dead_rows(net):
    for seed in range(6):
        c = make(seed, 6, 5, 700, 6, done=0.5)
        c["scores"][np.random.default_rng(seed).random((6, 5)) < 0.3] = -np.inf
        c["scores"][3] = -np.inf  # nothing goes on
        c["x"][c["done"] | (c["scores"] == -np.inf)] = np.nan  # not read
        check(net, c)


def test_first_step(net):
    c = make(3, 4, 6, 5000, 6, scaled=False)
    c["scores"][:] = -np.inf
    c["scores"][:, 0] = 0.0
    assert (check(net, c)[0] % 6 == 0).all()


def test_fewer_continuations_than_asked_for(net):
    c = make(4, 3, 2, 900, 12)
    shut = np.random.default_rng(1).random(c["x"].shape) > 0.004
    c["x"][shut] = -np.inf
    c["x"][1, 0] = -np.inf  # a row that allows nothing
    want = check(net, c)
    assert (want[0] == NONE).any()
    check(net, make(5, 2, 3, 2, 20))


def test_equal_logits(net):
    """The lower token and the lower row first, whole rows of one value too."""
    c = make(6, 3, 4, 3000, 9)
    c["x"] = np.round(c["x"])
    c["scores"][:], c["scale"][:] = -7.0, 0.5
    c["x"][:, 2] = c["x"][:, 1]  # equal ranks between rows
    c["x"][1] = 2.0
    want = check(net, c)
    assert want[0][1].tolist() == [4] * 9 and want[1][1].tolist() == list(range(9))
    c = make(7, 1, 1, 200000, 64)
    c["x"][:] = -1.5
    check(net, c)


def test_logits_far_apart(net):
    c = make(8, 2, 3, 2000, 8)
    c["x"] *= 300.0
    check(net, c)
    c["x"] = np.where(c["x"] > 0, 700.0, -1e300)
    check(net, c)


@pytest.mark.parametrize("what", ["nan", "inf", "score nan", "score inf"])
def test_what_has_no_order_is_refused(net, what):
    c = make(9, 2, 3, 800, 4)
    good = {k: None if v is None else np.copy(v) for k, v in c.items()}
    if what == "nan":
        c["x"][1, 2, 799] = np.nan
    if what == "inf":
        c["x"][0, 0, 5] = np.inf
    if what.startswith("score"):
        c["scores"][1, 1] = float(what.split()[1])
    for f in (device, lambda n, c: n.beam_select(c["x"], c["scores"], c["K"], scale=c["scale"])):
        with pytest.raises(ra.MitokError, match="NaN") as e:
            f(net, c)
        assert e.value.code == 4
    good["K"] = 4
    check(net, good)


@pytest.mark.parametrize("scale", [0.0, -1.0, np.nan, np.inf])
def test_scales_that_are_none_are_refused(net, scale):
    c = make(10, 2, 3, 800, 4)
    c["scale"][1, 0] = scale
    with pytest.raises(ra.MitokError, match="scales") as e:
        device(net, c)
    assert e.value.code == 1

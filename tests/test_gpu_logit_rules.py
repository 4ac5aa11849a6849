"""mitok_process_logits(_device) against apply_rules (plain_stack.py).

Tolerance.  The rules are a division or a product, frequency * c + presence, a
subtraction and an addition, each rounded once on either side (a fused
multiply-add rounds fewer): within 5 u of the magnitudes that enter them, u =
2^-53, and twice that between the two.  Logits that no rule touches and -inf are
equal bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from plain_stack import apply_rules

pytestmark = pytest.mark.gpu
U = 2.0 ** -53


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def make(seed, R, V, H=0, nb=0, mask=False):
    r = np.random.default_rng(seed)
    c = dict(x=3 * r.standard_normal((R, V)), hist=None, pen=None, bi=None, bv=None, ok=None)
    if H:
        c["hist"] = (V * r.random((R, H)) ** 3).astype(np.int64)
        c["hist"][r.random((R, H)) < 0.2] = -1
        c["pen"] = np.stack([r.uniform(0.7, 1.6, R), r.uniform(-1, 1, R), r.uniform(-0.2, 0.4, R)], 1)
    if nb:
        c["bi"] = r.integers(-1, V, (R, nb))
        c["bv"] = 2 * r.standard_normal((R, nb))
    if mask:
        c["ok"] = r.random((R, V)) < 0.1
        c["ok"][::2] = True
    return c


def formula(c):
    R = len(c["x"])
    rows = [apply_rules(c["x"][r], () if c["hist"] is None else c["hist"][r], (1, 0, 0) if c["pen"] is None else c["pen"][r],
                        () if c["bi"] is None else list(zip(c["bi"][r].tolist(), c["bv"][r])),
                        None if c["ok"] is None else c["ok"][r]) for r in range(R)]
    return np.array([x for x, _ in rows]), np.array([i for _, i in rows], np.int64)


def check(c, out, ids, want=None):
    x, best = formula(c) if want is None else want
    R, V = x.shape
    if out is not None:
        big = np.abs(c["x"])
        if c["pen"] is not None:
            n = np.stack([np.bincount(h[h >= 0], minlength=V) for h in c["hist"]])
            th, pr, fr = (np.abs(c["pen"][:, i:i + 1]) for i in range(3))
            big = np.where(n > 0, big * np.maximum(th, 1 / th) + fr * n + pr, big)
        if c["bi"] is not None:
            for r in range(R):
                for t, v in zip(c["bi"][r], c["bv"][r]):
                    if t >= 0:
                        big[r, t] += abs(v)
        assert np.array_equal(np.isneginf(out), np.isneginf(x))
        m = ~np.isneginf(x)
        assert np.all(np.abs(out[m] - x[m]) <= 10 * U * big[m])
        ruled = np.zeros((R, V), bool)
        if c["hist"] is not None:
            for r in range(R):
                ruled[r, c["hist"][r][c["hist"][r] >= 0]] = True
        if c["bi"] is not None:
            for r in range(R):
                ruled[r, c["bi"][r][c["bi"][r] >= 0]] = True
        assert np.array_equal(out[m & ~ruled], c["x"][m & ~ruled])
    got = np.where(ids == ra.NO_TOKEN, -1, ids.astype(np.int64))
    for r in range(R):
        if got[r] != best[r]:  # only where the two largest are within the rounding
            assert got[r] >= 0 and abs(x[r, got[r]] - x[r, best[r]]) <= 20 * U * (np.abs(x[r, best[r]]) + 8), r


def run(net, c, want_logits=True):
    return net.process_logits(c["x"], c["hist"], c["pen"], c["bi"], c["bv"], c["ok"], want_logits=want_logits)


CASES = [(1, 1, 0, 0, False), (1, 1, 3, 2, True), (2, 2, 5, 0, False), (3, 31, 4, 3, True), (3, 32, 4, 3, True),
         (3, 33, 4, 3, True), (1, 4096, 48, 3, True), (5, 4095, 300, 64, True), (5, 4097, 300, 64, True),
         (2, 8192, 5000, 0, False), (32, 32000, 256, 16, True), (7, 31999, 2000, 0, False), (3, 50280, 512, 40, True),
         (300, 2001, 9, 5, True), (4, 9000, 0, 7, False), (4, 9000, 0, 0, True), (2, 200001, 33, 9, True)]


@pytest.mark.parametrize("R,V,H,nb,mask", CASES)
def test_formula(net, R, V, H, nb, mask):
    c = make(R + V, R, V, H, nb, mask)
    want = formula(c)
    out, ids = run(net, c)
    check(c, out, ids, want)
    none, ids2 = run(net, c, want_logits=False)
    assert none is None and np.array_equal(ids, ids2)


@pytest.mark.parametrize("R,V,H,nb,mask", [(600, 2001, 9, 5, True), (300, 4097, 30, 3, True), (40, 27001, 300, 0, False)])
def test_many_rows_of_odd_sizes(net, R, V, H, nb, mask):
    """Rows that start between two 16-byte words, chunks that end in one token."""
    test_formula(net, R, V, H, nb, mask)


@pytest.mark.parametrize("R,V", [(2, 5000), (200, 6001)])
def test_logits_that_start_between_two_words(net, R, V):
    c = make(R, R, V, 20)
    want = formula(c)
    host = [np.concatenate([[7.0], c["x"].ravel(), [7.0]]), c["hist"].astype(np.int32), c["pen"]]
    d = [ra.DeviceBuffer(a.nbytes) for a in host]
    ids = ra.DeviceBuffer(4 * R)
    for b, a in zip(d, host):
        b.upload(a)
    net.process_logits_device(d[0].ptr + 8, R, V, out=d[0].ptr + 8, ids=ids, history=d[1], max_history=20, penalties=d[2])
    got = d[0].download(R * V + 2, float)
    assert got[0] == got[-1] == 7.0
    check(c, got[1:-1].reshape(R, V), ids.download(R, np.uint32), want)
    for b in [*d, ids]:
        b.free()


def test_no_rules_is_greedy_decoding(net):
    x = np.round(np.random.default_rng(1).standard_normal((40, 5003)) * 4) / 4  # ties: the last one
    out, ids = net.process_logits(x)
    assert np.array_equal(out, x) and np.array_equal(ids, net.greedy_decoding(x))


def test_in_place_on_the_device_and_each_output_alone(net):
    c = make(8, 6, 5000, 40, 5, True)
    want = formula(c)
    bits = np.zeros((6, 157 * 32), bool)
    bits[:, :5000] = c["ok"]
    host = [c["x"], c["hist"].astype(np.int32), c["pen"], c["bi"].astype(np.int32), c["bv"],
            np.ascontiguousarray(np.packbits(bits, axis=1, bitorder="little"))]
    d = [ra.DeviceBuffer(a.nbytes) for a in host]
    ids = ra.DeviceBuffer(24)

    def go(out, i):
        for b, a in zip(d, host):
            b.upload(a)
        ids.upload(np.full(6, 99, np.uint32))
        net.process_logits_device(d[0], 6, 5000, out=out, ids=i, history=d[1], max_history=40, penalties=d[2],
                                  bias_ids=d[3], bias=d[4], max_bias=5, allowed=d[5])
        return d[0].download((6, 5000), float), ids.download(6, np.uint32)

    x, i = go(d[0], ids)
    check(c, x, i, want)
    x, i2 = go(None, ids)
    assert np.array_equal(x, c["x"]) and np.array_equal(i, i2)  # logits left as they were
    x, i3 = go(d[0], None)
    check(c, x, i, want)
    assert (i3 == 99).all()
    for b in [*d, ids]:
        b.free()


def test_rows_with_nothing_left_and_masked_values(net):
    x = np.array([[1.0, np.nan, 3.0, -np.inf], [1.0, 2.0, 3.0, 4.0], [-np.inf] * 4, [np.inf, 1.0, np.inf, 0.0]])
    ok = np.array([[1, 0, 1, 1], [0, 0, 0, 0], [1, 1, 1, 1], [1, 1, 1, 0]], bool)
    out, ids = net.process_logits(x, allowed=ok)
    assert ids.tolist() == [2, ra.NO_TOKEN, ra.NO_TOKEN, 2]
    assert np.isneginf(out[0, 1]) and np.isneginf(out[1]).all() and np.isneginf(out[3, 3])
    assert np.array_equal(out[3, :3], x[3, :3])
    # -inf stays, +inf stays under a penalty
    out, ids = net.process_logits(np.array([[-np.inf, np.inf, 0.0, -0.0]]), [[0, 1, 2, 3]], [[1.5, 0.5, 0.25]])
    assert np.isneginf(out[0, 0]) and np.isposinf(out[0, 1]) and (out[0, 2:] == -0.75).all() and ids.tolist() == [1]


def test_repeated_entries(net):
    """A token that comes five times counts five times; of equal bias ids the last counts."""
    x = np.zeros((1, 70))
    x[0, 5], x[0, 6] = 2.0, -2.0
    out, _ = net.process_logits(x, [[5, 5, 6, 5, -1, 5, 5]], [[2.0, 0.5, 0.25]], [[7, 7, 5, 7]], [[1.0, 2.0, 10.0, 3.0]])
    assert out[0, 5] == 1.0 - (0.25 * 5 + 0.5) + 10.0 and out[0, 6] == -4.0 - 0.75 and out[0, 7] == 3.0
    assert np.count_nonzero(out) == 3


@pytest.mark.parametrize("big", ["rows", "vocab", "max_history", "max_bias"])
def test_sizes_past_the_kernels_indices(net, big):
    """A step past the last entry would wrap 31 bits: refused before any array is looked at."""
    with ra.DeviceBuffer(64) as d:
        with pytest.raises(ra.MitokError, match="2\\^30") as e:
            net.process_logits_device(d, ids=d.ptr + 32, **{**dict(rows=1, vocab=2), big: 2 ** 30 + 1})
        assert e.value.code == 1


def test_refusals(net):
    c = make(2, 2, 50, 4, 3, True)

    def go(match, code=1, **kw):
        with pytest.raises(ra.MitokError, match=match) as e:
            run(net, {**c, **kw})
        assert e.value.code == code

    bad = c["x"].copy()
    bad[1, 0] = np.nan
    ok = c["ok"].copy()
    ok[1, 0] = True
    go("NaN", code=4, x=bad, ok=ok)
    hist = c["hist"].copy()
    hist[1, 2] = 50
    go("outside the vocabulary", hist=hist)
    bi = c["bi"].copy()
    bi[0, 1] = 0xFFFFFFFE
    go("outside the vocabulary", bi=bi)
    for v in (0.0, -1.0, np.nan, np.inf):
        pen = c["pen"].copy()
        pen[0, 0] = v
        go("penalties", pen=pen)
    for i in (1, 2):
        pen = c["pen"].copy()
        pen[1, i] = np.inf
        go("penalties", pen=pen)
    for kw in (dict(hist=c["hist"][:1]), dict(pen=c["pen"][:1]), dict(bv=c["bv"][:, :2]), dict(ok=c["ok"][:, :49]),
               dict(hist=c["hist"].astype(float))):
        with pytest.raises(ValueError):
            run(net, {**c, **kw})
    d, i = ra.DeviceBuffer(2 * 50 * 8), ra.DeviceBuffer(64)

    def dev(match, d_x=d, rows=2, vocab=50, out=d, ids=i, **kw):
        with pytest.raises(ra.MitokError, match=match) as e:
            net.process_logits_device(d_x, rows, vocab, out=out, ids=ids, **kw)
        assert e.value.code == 1

    dev("neither", out=None, ids=None)
    dev("bad arguments", vocab=0)
    dev("exceed its allocation", vocab=51)
    dev("a history needs", max_history=3)
    dev("biases need", max_bias=3, bias=d)
    dev("overlap", ids=d)
    dev("overlap", out=d, d_x=d.ptr + 8, rows=1)
    dev("aligned", d_x=d.ptr + 4, rows=1)
    dev("aligned", ids=i.ptr + 2)
    dev("31 bits", rows=2 ** 31)
    out, ids = run(net, c)
    check(c, out, ids)
    d.free(), i.free()

"""mitok_tree_attention_device against the formula in 64 bits (numpy).

Tolerance.  Half a step of a double is u = 2^-53.  A score is a sum of 2 dh
products, a scale and a bias, off by at most
  ds = (2 dh + 4) u (sum |q||k| scale + |bias|),
and exp turns a score's error into a relative one of its weight; exp itself is
within 2 u, a sum of T weights or weighted values within T u of the sum of
magnitudes, the running maximum's and the splits' rescalings within 2 u each, at
most T / 16 + 8 of them on any value.  (A key whose weight is 0, its score at
least 745 below the largest, adds nothing on either side: ds is the largest of
the others.)  So either side is within
  (2 ds + (9 T / 8 + 40) u) sum_t w_t |v_t|
of the formula, and the two within twice that.  Weights: the same without v.
"""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra

pytestmark = pytest.mark.gpu
U = 2.0 ** -53


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def make(seed, B, n, H, dh, ctx, lens, counts=None, shape="tree", bias=True):
    r = np.random.default_rng(seed)
    c = lambda *s: r.standard_normal(s) + 1j * r.standard_normal(s)  # noqa: E731
    par = np.full((B, n), -1, np.int64)
    for b in range(B):
        for i in range(1, n):
            par[b, i] = {"chain": i - 1, "star": 0, "roots": -1, "forest": r.integers(-1, i),
                         "tree": r.integers(max(0, i // 2 - 1), i)}[shape]
    return dict(q=c(B, n, H * dh), k=c(B, H, ctx, dh), v=c(B, H, ctx, dh), par=par, lens=np.asarray(lens, np.uint32),
                counts=None if counts is None else np.asarray(counts, np.uint32), H=H, dh=dh, ctx=ctx,
                bias=0.5 * r.standard_normal((H, ctx)) if bias else None, w=r.random((B, H, ctx)))


def ancestors(par, i):
    out = []
    while i >= 0:
        out.append(int(i))
        i = par[i]
    return out[::-1]


def formula(c, weigh=0):
    """(out, its tolerance, weights, their tolerance)"""
    B, n = c["par"].shape
    H, dh = c["H"], c["dh"]
    out, tol = np.zeros((B, n, H * dh), complex), np.zeros((B, n, H * dh))
    w_out, w_tol = c["w"].copy(), np.zeros_like(c["w"])
    sc = 1.0 / (1e-8 + np.sqrt(dh))
    for b in range(B):
        L, cnt = int(c["lens"][b]), n if c["counts"] is None else int(c["counts"][b])
        if weigh:
            w_out[b, :, L:L + cnt] = 0
        for i in range(cnt):
            up = ancestors(c["par"][b], i)
            slots = np.r_[np.arange(L), L + np.array(up, np.int64)].astype(np.int64)
            cols = np.r_[np.arange(L), L + np.arange(len(up))].astype(np.int64)
            for h in range(H):
                q, K, V = c["q"][b, i, h * dh:(h + 1) * dh], c["k"][b, h, slots], c["v"][b, h, slots]
                bias = c["bias"][h, cols] if c["bias"] is not None else 0.0
                s = (K @ q).real * sc + bias
                e = np.exp(s - s.max())
                w = e / e.sum()
                out[b, i, h * dh:(h + 1) * dh] = w @ V
                ds = (2 * dh + 4) * U * np.max((np.abs(K) @ np.abs(q) * sc + np.abs(bias))[w != 0])
                rel = 2 * (2 * ds + (1.125 * len(slots) + 40) * U)
                tol[b, i, h * dh:(h + 1) * dh] = rel * (w @ (np.abs(V.real) + np.abs(V.imag)))
                if i < weigh:
                    w_out[b, h, slots] += w
                    w_tol[b, h, slots] += rel * w + 2 * weigh * U * w_out[b, h, slots]
    return out, tol, w_out, w_tol


def close(got, want, tol):
    """Within tol, and NaN exactly where the formula is."""
    for g, w in ((got.real, want.real), (got.imag, want.imag)):
        off = np.abs(g - w) > tol
        nan = np.isnan(g) != np.isnan(w)
        if off.any() or nan.any():
            at = np.argwhere(off | nan)[0]
            raise AssertionError(f"{off.sum()} values off, {nan.sum()} NaN or not, first at {at}: {g[tuple(at)]} "
                                 f"for {w[tuple(at)]}, tolerance {tol[tuple(at)]}")


def call(net, c, weigh=0, want_w=True, fill=7.0):
    B, n = c["par"].shape
    bufs = {}
    for name in ("q", "k", "v", "bias", "w"):
        if c[name] is not None:
            bufs[name] = ra.DeviceBuffer(max(c[name].nbytes, 16))
            bufs[name].upload(c[name])
    o = bufs["o"] = ra.DeviceBuffer(c["q"].nbytes)
    o.upload(np.full(c["q"].shape, fill, complex))
    try:
        net.tree_attention_device(bufs["q"], bufs["k"], bufs["v"], c["lens"], c["par"], c["H"], c["dh"], c["ctx"], o,
                                  counts=c["counts"], bias=bufs.get("bias"), bias_stride=c["ctx"],
                                  weights=bufs["w"] if weigh else None, weigh_nodes=weigh)
        for name in ("k", "v", "q"):
            assert np.array_equal(bufs[name].download(c[name].shape, complex), c[name], equal_nan=True), name
        return o.download(c["q"].shape, complex), bufs["w"].download(c["w"].shape, float)
    finally:
        for b in bufs.values():
            b.free()


CASES = [
    # B, n, H, dh, ctx, lens, counts, shape, weigh, bias
    (1, 1, 1, 16, 16, [0], None, "chain", 1, True),          # nothing cached: a token sees itself alone
    (1, 1, 2, 64, 64, [1], None, "chain", 1, True),
    (1, 1, 8, 64, 512, [160], None, "chain", 1, True),
    (2, 1, 3, 8, 70, [15, 17], None, "chain", 0, False),
    (3, 5, 2, 24, 80, [0, 16, 75], None, "tree", 5, True),   # the last one fills its cache
    (5, 7, 4, 64, 200, [37, 171, 64, 63, 65], None, "chain", 1, True),
    (4, 9, 2, 32, 100, [10, 20, 30, 40], [9, 0, 1, 4], "tree", 3, True),  # unused nodes, a sequence without any
    (2, 16, 2, 16, 300, [128, 250], None, "star", 16, True),
    (2, 17, 3, 40, 130, [31, 33], None, "roots", 17, True),  # every node a root
    (2, 33, 2, 128, 90, [50, 3], None, "forest", 1, True),
    (1, 64, 2, 64, 700, [600], None, "tree", 64, True),
    (2, 65, 1, 64, 140, [64, 75], [65, 40], "chain", 2, True),
    (1, 256, 2, 32, 300, [40], None, "forest", 256, True),
    (1, 3, 2, 256, 60, [40], None, "tree", 3, True),
    (2, 4, 2, 100, 60, [17, 40], None, "tree", 1, False),
    (2, 3, 5, 1, 40, [5, 33], None, "tree", 3, True),        # one complex number a head
    (1, 2, 2, 7, 20, [9], None, "chain", 2, True),
    (2, 20, 12, 64, 2048, [2028, 1500], None, "tree", 1, True),
    (1, 40, 2, 24, 90, [33], None, "tree", 7, True),         # 33 nodes and more, odd widths
    (2, 50, 1, 100, 120, [61, 8], [50, 37], "forest", 50, True),
    (1, 70, 3, 7, 200, [127], None, "tree", 1, False),
    (3, 34, 2, 128, 600, [566, 300, 16], None, "tree", 5, True),
    (1, 20, 2, 200, 100, [70], None, "tree", 20, True),
    (2, 24, 3, 128, 1100, [1076, 513], None, "tree", 24, True),
    (9, 64, 12, 64, 1200, [1100, 1136, 5, 700, 300, 64, 0, 999, 1000], None, "tree", 64, True),  # several chunks each
    (33, 16, 8, 32, 600, [(37 * b) % 584 for b in range(33)], None, "tree", 2, True),
    (70, 2, 1, 16, 40, [(7 * b) % 38 for b in range(70)], None, "chain", 2, True),
]


@pytest.mark.parametrize("B,n,H,dh,ctx,lens,counts,shape,weigh,bias", CASES)
def test_formula(net, B, n, H, dh, ctx, lens, counts, shape, weigh, bias):
    c = make(B * 1000 + n, B, n, H, dh, ctx, lens, counts, shape, bias)
    want, tol, w_want, w_tol = formula(c, weigh)
    got, w = call(net, c, weigh)
    close(got, want, tol)
    close(w, w_want, w_tol)  # slots that nobody attends: unchanged


def test_the_same_call_gives_the_same_bits(net):
    c = make(5, 3, 12, 4, 64, 900, [800, 555, 801])
    a, wa = call(net, c, 12)
    with ra.Network(0) as other:
        b, wb = call(other, c, 12)
    assert np.array_equal(a, b) and np.array_equal(wa, wb)


@pytest.mark.parametrize("dh,n,L", [(64, 6, 30), (64, 1, 100), (24, 40, 5), (256, 3, 17)])
def test_rows_that_a_node_does_not_see_have_no_part(net, dh, n, L):
    """Slots behind the last node, unused nodes and other branches may hold
    infinities and NaN."""
    c = make(dh, 2, n, 2, dh, 160, [L, L + 3], [n, max(1, n - 2)], "forest")
    want, w_want = call(net, c, n)
    bad = [np.nan, np.inf, -np.inf, complex(np.nan, np.inf)]
    for b in range(2):
        used = int(c["lens"][b] + c["counts"][b])
        for x in (c["k"], c["v"]):
            x[b, :, used:] = np.resize(bad, x[b, :, used:].shape)
    got, w = call(net, c, n)
    assert np.array_equal(got, want) and np.array_equal(w, w_want)
    # one node's rows are not finite: it and its descendants alone are touched
    if n > 3:
        hit = 1
        below = [any(j == hit for j in ancestors(c["par"][0], i)) for i in range(n)]
        assert 0 < sum(below) < n
        for x in bad:
            c["v"][0, :, L + hit] = x
            got, _ = call(net, c, 0)
            assert np.array_equal(got[0, ~np.array(below)], want[0, ~np.array(below)]), x
            assert np.array_equal(got[1], want[1])
            assert not np.isfinite(got[0, hit]).any(), x
        c["k"][0, :, L + hit] = np.nan
        got, _ = call(net, c, 0)
        assert np.array_equal(got[0, ~np.array(below)], want[0, ~np.array(below)])
        assert np.isnan(got[0, below]).all()


def test_values_of_a_seen_row_that_are_not_finite(net):
    """An infinite value column gives an infinite output column in the rows that
    see it, the others stay."""
    c = make(9, 1, 4, 1, 32, 64, [20], None, "star")
    c["par"][0] = [-1, 0, 0, 2]
    c["v"][0, 0, 22, 3] = complex(np.inf, 1.0)   # node 2
    c["v"][0, 0, 23, 5] = complex(1.0, np.nan)   # node 3
    got, _ = call(net, c)
    g = got[0]
    assert np.isposinf(g[2:, 3].real).all() and np.isfinite(g[:2]).all() and np.isfinite(g[2:, 3].imag).all()
    assert np.isnan(g[3, 5].imag) and np.isfinite(g[2, 5])
    rest = np.ones(32, bool)
    rest[[3, 5]] = False
    assert np.isfinite(g[:, rest]).all()


def test_biases_of_minus_infinity_and_the_least_number(net):
    c = make(11, 2, 3, 2, 16, 80, [40, 33], None, "chain")
    c["bias"][0, :35] = -np.inf          # a stretch of no weight
    c["bias"][1, 3:60] = np.finfo(float).min
    want, tol, w_want, w_tol = formula(c, 3)
    got, w = call(net, c, 3)
    close(got, want, tol)
    close(w, w_want, w_tol + 1e-300)
    c["bias"][0] = -np.inf               # nothing left: 0 / 0, as the formula
    got, _ = call(net, c, 0)
    assert np.isnan(got[:, :, :16]).all()
    assert np.array_equal(got[:, :, 16:], call(net, c, 0)[0][:, :, 16:]) and np.isfinite(got[:, :, 16:]).all()


def test_large_scores_and_one_dominant_row(net):
    c = make(12, 1, 4, 2, 64, 400, [390], None, "tree")
    c["k"][0, :, 77] *= 60.0
    c["q"] *= 20.0
    want, tol, _, _ = formula(c)
    got, _ = call(net, c)
    close(got, want, tol)


def test_weights_add_up_over_calls(net):
    c = make(13, 2, 5, 2, 32, 90, [50, 70], [5, 3])
    _, w1 = call(net, c, 5)
    c2 = dict(c, w=w1)
    _, w2 = call(net, c2, 5)
    for b in range(2):
        L = int(c["lens"][b])
        assert np.allclose(w2[b, :, :L] - w1[b, :, :L], w1[b, :, :L] - c["w"][b, :, :L], rtol=0, atol=1e-12)
        assert np.array_equal(w2[b, :, L:], w1[b, :, L:])  # drafted slots are set, the rest left
        assert abs((w1 - c["w"])[b, :, :L].sum() + w1[b, :, L:L + c["counts"][b]].sum() - 2 * c["counts"][b]) < 1e-10


def test_offsets_past_32_bits(net):
    """A cache of 6.4 GB of keys: the last sequence's heads begin past 2^32 bytes."""
    c = make(21, 2, 5, 3, 64, 60, [0, 50], [0, 5])
    ctx = 1 << 20
    q, o, w = ra.DeviceBuffer(c["q"].nbytes), ra.DeviceBuffer(c["q"].nbytes), ra.DeviceBuffer(2 * 3 * ctx * 8)
    k, v, b = ra.DeviceBuffer(2 * 3 * ctx * 64 * 16), ra.DeviceBuffer(2 * 3 * ctx * 64 * 16), ra.DeviceBuffer(c["bias"].nbytes)

    def part(buf, row, a):
        x = ra.DeviceBuffer.__new__(ra.DeviceBuffer)
        x._hip, x.nbytes, x.device = buf._hip, a.nbytes, 0
        x._p = type(buf._p)(buf.ptr + row * a.itemsize * (a.shape[-1] if a.ndim > 1 else 1))
        return x

    q.upload(c["q"])
    b.upload(c["bias"])
    for h in range(3):
        part(k, (3 + h) * ctx, c["k"][1, h]).upload(c["k"][1, h])
        part(v, (3 + h) * ctx, c["v"][1, h]).upload(c["v"][1, h])
        part(w, (3 + h) * ctx, c["w"][1, h]).upload(c["w"][1, h])
    net.tree_attention_device(q, k, v, c["lens"], c["par"], 3, 64, ctx, o, counts=c["counts"], bias=b, bias_stride=60,
                              weights=w, weigh_nodes=5)
    want, tol, w_want, w_tol = formula(c, 5)
    close(o.download(c["q"].shape, complex), want, tol)
    for h in range(3):
        close(part(w, (3 + h) * ctx, c["w"][1, h]).download((60,), float), w_want[1, h], w_tol[1, h])
    # and an eviction of the same rows, to a small cache and in place
    ko, vo, wo = ra.DeviceBuffer(2 * 3 * 20 * 64 * 16), ra.DeviceBuffer(2 * 3 * 20 * 64 * 16), ra.DeviceBuffer(2 * 3 * 20 * 8)
    kept = ra.DeviceBuffer(2 * 3 * 20 * 4)
    assert net.evict_rows_device(k, v, w, [0, 55], 3, 64, ctx, 20, 2, 6, ko, vo, wo, 20, kept=kept).tolist() == [0, 20]
    rows = kept.download((2, 3, 20), np.uint32)[1]
    assert net.evict_rows_device(k, v, w, [0, 55], 3, 64, ctx, 20, 2, 6, k, v, w, ctx).tolist() == [0, 20]
    for h in range(3):
        x = ko.download((2, 3, 20, 64), complex)[1, h]
        assert np.array_equal(x, c["k"][1, h, rows[h]])
        assert np.array_equal(part(k, (3 + h) * ctx, x).download(x.shape, complex), x)
        y = vo.download((2, 3, 20, 64), complex)[1, h]
        assert np.array_equal(part(v, (3 + h) * ctx, y).download(y.shape, complex), y)
    for x in (q, o, w, k, v, b, ko, vo, wo, kept):
        x.free()


def test_work_queued_on_the_default_stream_comes_first(net):
    """The queries arrive by a copy that the default stream still has before it
    when the call is made."""
    c = make(22, 2, 5, 3, 64, 200, [150, 40])
    want, _ = call(net, c)
    big = [ra.DeviceBuffer(1 << 30) for _ in range(2)]
    bufs = {x: ra.DeviceBuffer(c[x].nbytes) for x in ("q", "k", "v", "bias")}
    late, o = ra.DeviceBuffer(c["q"].nbytes), ra.DeviceBuffer(c["q"].nbytes)
    for x in bufs:
        bufs[x].upload(c[x])
    late.upload(np.zeros_like(c["q"]))
    hip = late._hip
    size = __import__("ctypes").c_size_t
    for i in range(16):  # about 6 ms of copies
        assert hip.hipMemcpyAsync(big[i % 2]._p, big[1 - i % 2]._p, size(1 << 30), 3, None) == 0
    assert hip.hipMemcpyAsync(late._p, bufs["q"]._p, size(c["q"].nbytes), 3, None) == 0
    net.tree_attention_device(late, bufs["k"], bufs["v"], c["lens"], c["par"], 3, 64, 200, o, bias=bufs["bias"], bias_stride=200)
    assert np.array_equal(o.download(c["q"].shape, complex), want)
    for x in [*big, *bufs.values(), late, o]:
        x.free()


def test_two_networks_at_once():
    """Two threads, each with a network of its own: every call gives its own result."""
    import threading

    cases = [make(30 + i, 3, 9 + 30 * i, 4, 64, 400, [300, 200 + i, 17]) for i in range(2)]
    wants, bad = [None, None], []
    with ra.Network(0) as one:
        for i, c in enumerate(cases):
            wants[i] = call(one, c, 2)

    def loop(i):
        try:
            with ra.Network(0) as n:
                for _ in range(10):
                    o, w = call(n, cases[i], 2)
                    if not (np.array_equal(o, wants[i][0]) and np.array_equal(w, wants[i][1])):
                        bad.append(i)
        except Exception as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("B,H", [(5, 65535), (65536, 1), (1, 65536), (513, 512)])
def test_batches_and_heads_that_a_launch_cannot_hold(net, B, H):
    with ra.DeviceBuffer(4096) as x, ra.DeviceBuffer(4096) as y:
        with pytest.raises(ra.MitokError, match="their product 262144") as e:
            net.tree_attention_device(x, x, x, np.zeros(B, np.uint32), np.full((B, 1), -1), H, 1, 1, y)
        assert e.value.code == 1


def test_refusals(net):
    c = make(1, 2, 4, 2, 16, 32, [3, 28])
    good = dict(par=c["par"], lens=c["lens"], H=2, dh=16, ctx=32, counts=None, weigh=0, stride=32)
    qb, kb, vb, wb, ob, bb = (ra.DeviceBuffer(x) for x in (c["q"].nbytes, c["k"].nbytes, c["v"].nbytes, c["w"].nbytes,
                                                           c["q"].nbytes, 32 * 2 * 8))

    def go(match, q=qb, k=kb, v=vb, o=ob, w=wb, bias=bb, **kw):
        a = {**good, **kw}
        with pytest.raises(ra.MitokError, match=match) as e:
            net.tree_attention_device(q, k, v, a["lens"], a["par"], a["H"], a["dh"], a["ctx"], o, counts=a["counts"],
                                      bias=bias, bias_stride=a["stride"], weights=w, weigh_nodes=a["weigh"])
        assert e.value.code == 1, e.value

    par = c["par"].copy()
    par[1, 2] = 2
    go("parents come before", par=par)
    par[1, 2] = 3
    go("parents come before", par=par)
    go("exceed max_ctx", lens=np.array([3, 29], np.uint32))
    go("exceed max_ctx", lens=np.array([3, 0xFFFFFFFF], np.uint32))
    go("counts", counts=[4, 5])
    go("head dim", dh=257)
    go("bad shape", H=0)
    go("256", par=np.full((2, 257), -1))
    go("weigh_nodes", weigh=5)
    go("weigh_nodes without", weigh=1, w=None)
    go("bias_stride", stride=31)
    go("null", q=None)
    go("not device memory", q=c["q"].ctypes.data)
    go("exceed its allocation", H=3)
    go("exceed its", H=65535, dh=256, ctx=2 ** 30, weigh=1)
    go("bad shape", ctx=2 ** 30 + 1)
    go("aligned", q=qb.ptr + 8)
    go("overlap", o=qb)
    go("overlap", o=vb)
    go("exceed its allocation", bias=bb, stride=40)
    with pytest.raises(ValueError):
        net.tree_attention_device(qb, kb, vb, [3], c["par"], 2, 16, 32, ob)
    with pytest.raises(ValueError):
        net.tree_attention_device(qb, kb, vb, c["lens"], c["par"].astype(float), 2, 16, 32, ob)
    got, _ = call(net, c)  # and the network still works
    want, tol, _, _ = formula(c)
    close(got, want, tol)
    for x in (qb, kb, vb, wb, ob, bb):
        x.free()

"""mitok_evict_rows_device against kept_rows (plain_stack.py): which rows stay,
their order, the moved keys, values and weights bit for bit, and everything
else left as it was."""
from __future__ import annotations

import numpy as np
import pytest

import rustcrates_amd as ra
from plain_stack import kept_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def make(seed, B, H, dh, ctx, lens, values="plain"):
    r = np.random.default_rng(seed)
    c = lambda: r.standard_normal((B, H, ctx, dh)) + 1j * r.standard_normal((B, H, ctx, dh))  # noqa: E731
    w = r.random((B, H, ctx)) ** 4
    if values == "ties":
        w = r.integers(0, 4, w.shape) / 4.0
    if values == "same":
        w[:] = 0.5
    if values == "odd":
        w.reshape(-1)[:] = np.resize([0.0, -0.0, np.nan, np.inf, -np.inf, 1.0, -1.0, 5e-324, 1.0, np.nan, -np.nan], w.size)
        w = r.permuted(w, axis=2)
    if values == "close":  # differing in the last bits only
        w = 1.0 + r.integers(0, 64, w.shape) * 2.0 ** -52
    return dict(k=c(), v=c(), w=w, lens=np.asarray(lens, np.uint32))


def call(net, c, keep, sinks, recent, out_ctx=None, in_place=False, want_kept=True):
    B, H, ctx, dh = c["k"].shape
    oc = ctx if in_place else out_ctx or keep
    dev = {x: ra.DeviceBuffer(c[x].nbytes) for x in "kvw"}
    for x in "kvw":
        dev[x].upload(c[x])
    shapes = dict(k=(B, H, oc, dh), v=(B, H, oc, dh), w=(B, H, oc))
    start = {x: c[x].copy() if in_place else np.full(shapes[x], 3.0, c[x].dtype) for x in "kvw"}
    out = dev if in_place else {x: ra.DeviceBuffer(start[x].nbytes) for x in "kvw"}
    if not in_place:
        for x in "kvw":
            out[x].upload(start[x])
    kept = ra.DeviceBuffer(B * H * keep * 4)
    lens = net.evict_rows_device(dev["k"], dev["v"], dev["w"], c["lens"], H, dh, ctx, keep, sinks, recent, out["k"],
                                 out["v"], out["w"], oc, kept=kept if want_kept else None)
    got = {x: out[x].download(shapes[x], c[x].dtype) for x in "kvw"}
    ids = kept.download((B, H, keep), np.uint32) if want_kept else None
    if not in_place:
        for x in "kvw":
            assert np.array_equal(dev[x].download(c[x].shape, c[x].dtype), c[x], equal_nan=True)
    for b in {id(x): x for x in [*dev.values(), *out.values(), kept]}.values():
        b.free()
    return got, ids, lens, start


def check(c, keep, sinks, recent, got, ids, lens, start):
    B, H = c["w"].shape[:2]
    assert np.array_equal(lens, np.minimum(c["lens"], keep))
    for b in range(B):
        L = int(c["lens"][b])
        for h in range(H):
            stay = kept_rows(list(c["w"][b, h, :L]), keep, sinks, recent)
            n = len(stay)
            if ids is not None:
                assert ids[b, h, :n].tolist() == stay
                assert (ids[b, h, n:] == ra.NO_ROW).all()
            for x in "kvw":
                assert np.array_equal(got[x][b, h, :n], c[x][b, h, stay], equal_nan=True), x
                assert np.array_equal(got[x][b, h, n:], start[x][b, h, n:], equal_nan=True), x


CASES = [
    # B, H, dh, ctx, lens, keep, sinks, recent, weights
    (1, 1, 16, 16, [1], 1, 0, 0, "plain"),
    (1, 2, 16, 64, [64], 1, 0, 0, "plain"),
    (1, 4, 16, 512, [320], 256, 4, 32, "plain"),
    (3, 2, 64, 100, [0, 57, 100], 57, 3, 5, "plain"),       # empty, exactly full, over
    (2, 3, 24, 130, [129, 66], 65, 0, 65, "plain"),         # the recent ones alone
    (2, 3, 24, 130, [129, 66], 65, 65, 0, "plain"),         # the first ones alone
    (2, 3, 24, 130, [129, 66], 65, 30, 35, "plain"),        # both, none by weight
    (5, 2, 8, 300, [300, 299, 257, 256, 255], 255, 1, 1, "plain"),
    (2, 2, 1, 200, [200, 190], 99, 4, 8, "ties"),
    (2, 2, 3, 200, [200, 190], 99, 4, 8, "same"),
    (2, 2, 7, 200, [200, 190], 99, 0, 0, "odd"),
    (2, 2, 7, 200, [200, 190], 150, 2, 3, "odd"),
    (1, 2, 100, 700, [700], 333, 4, 8, "close"),
    (1, 2, 256, 150, [150], 70, 4, 8, "plain"),
    (2, 3, 64, 2048, [2048, 2047], 1024, 4, 256, "plain"),
    (1, 2, 2, 5000, [4999], 1, 0, 0, "ties"),
    (1, 2, 2, 20000, [20000], 19999, 4, 8, "plain"),
    (1, 1, 2, 20000, [20000], 7000, 4, 8, "close"),
    (70, 1, 4, 40, [(11 * b) % 41 for b in range(70)], 20, 2, 6, "plain"),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,H,dh,ctx,lens,keep,sinks,recent,values", CASES)
def test_kept_and_moved(net, B, H, dh, ctx, lens, keep, sinks, recent, values, in_place):
    c = make(B * 1000 + keep, B, H, dh, ctx, lens, values)
    check(c, keep, sinks, recent, *call(net, c, keep, sinks, recent, in_place=in_place))


def test_a_wider_output_cache_and_no_list_wanted(net):
    c = make(3, 2, 2, 16, 90, [90, 40])
    check(c, 50, 2, 10, *call(net, c, 50, 2, 10, out_ctx=77))
    check(c, 50, 2, 10, *call(net, c, 50, 2, 10, want_kept=False))
    check(c, 5000, 2, 10, *call(net, c, 5000, 2, 10, out_ctx=90))  # more than there is


def test_evicting_twice(net):
    c = make(4, 2, 3, 32, 300, [300, 280])
    got, _, lens, _ = call(net, c, 200, 4, 50, in_place=True)
    again = dict(got, lens=lens)
    check(again, 90, 4, 50, *call(net, again, 90, 4, 50, in_place=True))


@pytest.mark.parametrize("B,H", [(5, 65535), (65536, 1), (1, 65536), (513, 512)])
def test_batches_and_heads_that_a_launch_cannot_hold(net, B, H):
    b = [ra.DeviceBuffer(256) for _ in range(6)]
    with pytest.raises(ra.MitokError, match="their product 262144") as e:
        net.evict_rows_device(*b[:3], np.zeros(B, np.uint32), H, 1, 1, 1, 0, 0, *b[3:], 1)
    assert e.value.code == 1
    for x in b:
        x.free()


def test_a_list_of_kept_slots_past_the_kernels_indices(net):
    with ra.DeviceBuffer(4096) as x, pytest.raises(ra.MitokError, match="2\\^30") as e:
        net.evict_rows_device(x, x, x, [1], 1, 1, 1, 2 ** 30 + 1, 0, 0, x, x, x, 1, kept=x)
    assert e.value.code == 1


def test_refusals(net):
    c = make(1, 2, 2, 8, 40, [40, 30])
    dev = {x: ra.DeviceBuffer(c[x].nbytes) for x in "kvw"}
    out = {x: ra.DeviceBuffer(c[x].nbytes) for x in "kvw"}
    kept = ra.DeviceBuffer(2 * 2 * 20 * 4)

    def go(match, k=dev["k"], w=dev["w"], ko=out["k"], vo=out["v"], wo=out["w"], lens=c["lens"], H=2, dh=8, ctx=40, keep=20,
           sinks=2, recent=3, oc=20, kept=kept):
        with pytest.raises(ra.MitokError, match=match) as e:
            net.evict_rows_device(k, dev["v"], w, lens, H, dh, ctx, keep, sinks, recent, ko, vo, wo, oc, kept=kept)
        assert e.value.code == 1

    go("keep", keep=0)
    go("exceed keep", sinks=10, recent=11)
    go("exceed keep", sinks=0xFFFFFFFF, recent=2)
    go("exceeds max_ctx", lens=[41, 1])
    go("do not fit", oc=19)
    go("bad shape", H=0)
    go("head dim", dh=300)
    go("null", w=None)
    go("overlap", ko=dev["k"])                 # in place in part
    go("overlap", ko=out["v"])
    go("overlap", ko=dev["k"], vo=dev["v"], wo=dev["w"], oc=20)  # in place needs out_ctx == max_ctx
    go("overlap", kept=dev["k"])
    go("exceed its allocation", keep=41, kept=kept, oc=40)
    go("not device memory", k=c["k"].ctypes.data)
    go("aligned", k=dev["k"].ptr + 8)
    for b in [*dev.values(), *out.values(), kept]:
        b.free()

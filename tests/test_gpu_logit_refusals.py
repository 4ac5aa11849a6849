"""What a refused mitok_process_logits(_device) leaves behind: in-place logits as
they were, and nothing for the next call to take for its own."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import rustcrates_amd as ra
from test_gpu_logit_rules import check, formula, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def on_device(c):
    R, V = c["x"].shape
    bits = np.zeros((R, -(-V // 32) * 32), bool)
    bits[:, :V] = c["ok"]
    host = dict(x=c["x"], history=c["hist"].astype(np.int32), penalties=c["pen"], bias_ids=c["bi"].astype(np.int32),
                bias=c["bv"], allowed=np.ascontiguousarray(np.packbits(bits, axis=1, bitorder="little")))
    d = {k: ra.DeviceBuffer(a.nbytes) for k, a in host.items()}
    for k, a in host.items():
        d[k].upload(a)
    return d


def rules(net, d, c, out):
    R, V = c["x"].shape
    ids = ra.DeviceBuffer(4 * R)
    try:
        net.process_logits_device(d["x"], R, V, out=out, ids=ids, max_history=c["hist"].shape[1], max_bias=c["bi"].shape[1],
                                  **{k: d[k] for k in ("history", "penalties", "bias_ids", "bias", "allowed")})
        return ids.download(R, np.uint32)
    finally:
        ids.free()


@pytest.mark.parametrize("R,V", [(1, 70), (6, 5000), (300, 4097)])
def test_a_refused_call_leaves_logits_in_place_as_they_were(net, R, V):
    """A bad id or penalty in one row: no row is changed, so the mended call gives
    the rules once."""
    c = make(R, R, V, 9, 4, True)
    want = formula(c)
    d = on_device(c)
    row = R // 2
    for name, at, bad in [("hist", (row, 8), V), ("bi", (row, 0), V + 7), ("pen", (row, 0), 0.0), ("pen", (row, 1), np.nan),
                          ("pen", (row, 2), np.inf)]:
        key = dict(hist="history", bi="bias_ids", pen="penalties")[name]
        broken = c[name].copy()
        broken[at] = bad
        kind = np.float64 if name == "pen" else np.int32
        d[key].upload(broken.astype(kind))
        with pytest.raises(ra.MitokError, match="outside the vocabulary|penalties") as e:
            rules(net, d, c, d["x"])
        assert e.value.code == 1
        assert np.array_equal(d["x"].download((R, V), float), c["x"]), name
        d[key].upload(c[name].astype(kind))
    ids = rules(net, d, c, d["x"])
    check(c, d["x"].download((R, V), float), ids, want)
    d["x"].upload(c["x"])
    out = ra.DeviceBuffer(c["x"].nbytes)
    assert np.array_equal(rules(net, d, c, out), ids)
    assert np.array_equal(d["x"].download((R, V), float), c["x"])
    for b in [out, *d.values()]:
        b.free()


def test_an_error_is_reported_once(net):
    """Also where the runtime holds an older error of the thread."""
    hip = C.CDLL("libamdhip64.so.7")
    x = np.zeros((2, 40))
    good, ids = net.process_logits(x, [[1]] * 2, [[2.0, 1.0, 0.0]] * 2)
    for bad in (dict(history=[[40]] * 2, penalties=[[2.0, 1.0, 0.0]] * 2), dict(history=[[1]] * 2, penalties=[[0.0, 0.0, 0.0]] * 2)):
        assert hip.hipSetDevice(999) != 0  # left as the thread's last error
        with pytest.raises(ra.MitokError):
            net.process_logits(x, **bad)
        hip.hipGetLastError()
        again, ids2 = net.process_logits(x, [[1]] * 2, [[2.0, 1.0, 0.0]] * 2)
        assert np.array_equal(again, good) and np.array_equal(ids2, ids)

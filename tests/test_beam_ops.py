"""The operators of beams on a paged cache without a GPU: refusals of the entry
points and of the Python methods, and what a failing runtime call leaves behind
(host_runtime.py)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import rustcrates_amd as ra
from host_runtime import run
from test_serving_ops import network

NAMES = ["mitok_paged_attention_device", "mitok_fork_pages_device", "mitok_beam_select_device", "mitok_beam_select",
         "mitok_beam_search"]


@pytest.mark.parametrize("name", NAMES)
def test_a_null_network_is_refused(name):
    lib = ra.load_library()
    args = [None if a is C.c_void_p else 0 for a in ra.SIGNATURES[name][1]]
    assert getattr(lib, name)(*args) == 1
    assert lib.mitok_last_error()


@pytest.mark.parametrize("call", [
    lambda n: n.paged_attention_device(0, 0, 0, 0, 0, 0, [[1]], 1, 1, 1, 16, 1, 1, 0),
    lambda n: n.paged_attention_device(0, 0, 0, 0, 0, 0, [1.5], 1, 1, 1, 16, 1, 1, 0),
    lambda n: n.paged_attention_device(0, 0, 0, 0, 0, 0, [-1], 1, 1, 1, 16, 1, 1, 0),
    lambda n: n.paged_attention_device(0, 0, 0, 0, 0, 0, [1], 1, 1, 1, 16, 1, 1, 0, counts=[1, 1]),
    lambda n: n.paged_attention_device(0, 0, 0, 0, 0, 0, [1], -1, 1, 1, 16, 1, 1, 0),
    lambda n: n.paged_attention_device(0, 0, 0, 0, 0, 0, [1], 1, 1, 1, 16, 1, 1, 0, bias_row_stride=-1),
    lambda n: n.fork_pages_device(0, 0, 1, 2 ** 32, 1, 16, 1, 0, 0, 1, 1, 0, 1, 0, 0),
    lambda n: n.beam_select_device(0, 0, 1, 1, 1, -1, 0, 0, 0),
    lambda n: n.beam_select(np.zeros((2, 7)), np.zeros(2), 1),
    lambda n: n.beam_select(np.zeros((1, 2, 7)), np.zeros(2), 1),
    lambda n: n.beam_select(np.zeros((1, 2, 7)), None, 1),
    lambda n: n.beam_select(np.zeros((1, 2, 7)), np.zeros((1, 2)), 1, done=[0, 1]),
    lambda n: n.beam_select(np.zeros((1, 2, 7)), np.zeros((1, 2)), 1, scale=np.ones((2, 1))),
    lambda n: n.beam_search([3, 4]),
    lambda n: n.beam_search([[3, 4]], lens=[1, 2]),
    lambda n: n.beam_search([[3, 4]], beams=-1),
])
def test_wrong_arrays_are_refused_before_the_library(call):
    with pytest.raises(ValueError):
        call(network())


PAGED = """
net = ra.Network(0)
a = dict(q=device(65536), k_new=device(65536), v_new=device(65536), k=device(65536), v=device(65536), table=device(64), out=device(65536), bias=device(65536))
def paged(lens=[20], rows=2, heads=2, dh=8, page_rows=16, pages=4, max_pages=4, counts=None, bias=None, bias_stride=0, bias_row=0, **swap):
    b = {**a, **swap}
    net.paged_attention_device(b["q"], b["k_new"], b["v_new"], b["k"], b["v"], b["table"], lens, rows, heads, dh, page_rows, pages,
                               max_pages, b["out"], counts=counts, bias=bias, bias_stride=bias_stride, bias_row_stride=bias_row)
paged()
assert launches("k_paged_split") == 1
"""


def test_paged_attention_refuses():
    run(PAGED + """
bad = lambda match, **kw: refused(1, match, lambda: paged(**kw))
for kw in (dict(rows=0), dict(rows=65537)): bad("new rows", **kw)
for kw in (dict(heads=0), dict(dh=0), dict(pages=0), dict(max_pages=0), dict(lens=np.zeros(0, np.uint32))): bad("bad shape", **kw)
for ps in (0, 8, 24, 1040): bad("rows of a page", page_rows=ps)
bad("head dim", dh=257)
bad("2\\^24|pages", pages=2**24 + 1)
bad("2\\^30", heads=65536)
bad("2\\^30", heads=65535, page_rows=1024, dh=256)
bad("sequences", max_pages=2**27)
bad("exceed", lens=[63])
bad("exceed", lens=[0xFFFFFFFF])
bad("above", counts=[3])
bad("2\\^20", lens=[0] * 300, rows=65536, max_pages=4)
bad("bias_stride", bias=a["bias"], bias_stride=21)
bad("bias_stride", bias=a["bias"], bias_stride=30, bias_row=22)
bad("stride", bias=a["bias"], bias_stride=2**62)
bad("exceed its allocation|64 bits", bias=a["bias"], bias_stride=2**58, bias_row=0)
bad("exceed its allocation|64 bits|bias_stride", bias=a["bias"], bias_stride=2**58, bias_row=2**58)
paged(bias=a["bias"], bias_stride=22)
paged(bias=a["bias"], bias_stride=21 * 22 + 22, bias_row=22)
for x in ("q", "k_new", "v_new", "k", "v", "table", "out"):
    bad("not device memory|exceed", **{x: 4096})
    bad("aligned", **{x: a[x] + 2})
    bad("exceed", **{x: a[x] + 65536 - (64 if x != "table" else 65536 - 60)})
    refused(1, "null", lambda: paged(**{x: None}))
for x in ("q", "k_new", "v_new", "k", "v"): bad("overlap", out=a[x])
for x in ("q", "k_new", "v_new"): bad("overlap", k=a[x]); bad("overlap", v=a[x])
bad("overlap", v=a["k"])
bad("overlap", bias=a["k"], bias_stride=22)
n = launches("k_paged")
paged(k_new=a["q"], v_new=a["q"])  # inputs may be one
assert launches("k_paged") == n + 1
""")


FORK = """
net = ra.Network(0)
a = dict(k=device(65536), v=device(65536), table=device(64), lens=device(64), parents=device(64), grow=device(64), table_out=device(64), lens_out=device(64))
def fork(layers=1, pages=4, heads=2, page_rows=16, dh=8, old=2, max_pages=4, new=3, **swap):
    b = {**a, **swap}
    net.fork_pages_device(b["k"], b["v"], layers, pages, heads, page_rows, dh, b["table"], b["lens"], old, max_pages, b["parents"], new,
                          b["table_out"], b["lens_out"], grow=b["grow"])
fork()
fork(grow=None)
fork(old=3, table_out=a["table"], lens_out=a["lens"])
fork(parents=a["grow"])
assert launches("k_fork_assign") == launches("k_fork_commit") == 4
"""


def test_forks_refuse():
    run(FORK + """
bad = lambda match, **kw: refused(1, match, lambda: fork(**kw))
for kw in (dict(heads=0), dict(dh=0), dict(pages=0), dict(max_pages=0), dict(old=0), dict(new=0)): bad("bad shape", **kw)
for kw in (dict(layers=0), dict(layers=16385)): bad("layers", **kw)
for ps in (0, 8, 24, 1040): bad("rows of a page", page_rows=ps)
for kw in (dict(old=65536), dict(new=65536)): bad("sequences", **kw)
bad("exceed", layers=17)
for x in a:
    bad("not device memory|exceed", **{x: 4096})
    bad("aligned", **{x: a[x] + 2})
    if x != "grow": refused(1, "null", lambda: fork(**{x: None}))
for x in ("table_out", "lens_out"):
    for y in ("k", "v", "parents", "grow"): bad("overlap", **{x: a[y]})
bad("overlap", table_out=a["lens"])
bad("overlap", lens_out=a["table"])
bad("overlap", table_out=a["table"] + 16)
bad("overlap", lens_out=a["lens"] + 4)
bad("overlap", lens_out=a["table_out"])
bad("overlap", v=a["k"])
assert launches("k_fork_assign") == 4
""")


def test_a_fork_that_failed_half_way_does_not_leave_its_counts():
    """The counts start at zero again: filled once when made, once after the failure."""
    run(FORK + """
fills = launches("k_fill")
fork()
assert launches("k_fill") == fills
fail("launch", 2)
refused(2, "", fork)
fork()
assert launches("k_fill") == fills + 1
fork()
assert launches("k_fill") == fills + 1
""")


SELECT = """
net = ra.Network(0)
a = dict(x=device(8192), scores=device(512), done=device(512), scale=device(512), parents=device(512), tokens=device(512), best=device(512))
def select(batch=2, beams=3, vocab=10, keep=4, **swap):
    b = {**a, **swap}
    net.beam_select_device(b["x"], b["scores"], batch, beams, vocab, keep, b["parents"], b["tokens"], b["best"], done=b["done"], scale=b["scale"])
select()
select(done=None, scale=None)
select(batch=1, beams=1, vocab=1, keep=64)
assert launches("k_beam_pick") == 3
"""


def test_selections_refuse():
    run(SELECT + """
bad = lambda match, **kw: refused(1, match, lambda: select(**kw))
for kw in (dict(batch=0), dict(beams=0), dict(vocab=0)): bad("bad shape", **kw)
for k in (0, 65): bad("kept", keep=k)
for kw in (dict(beams=1025), dict(beams=1024, vocab=2**21), dict(batch=2**22, beams=3)): bad("at most", **kw)
bad("exceed", vocab=500)
for x in a:
    bad("not device memory|exceed", **{x: 4096})
    bad("aligned", **{x: a[x] + 2})
    if x not in ("done", "scale"): refused(1, "null", lambda: select(**{x: None}))
for x in ("parents", "tokens", "best"):
    for y in ("x", "scores", "done", "scale"): bad("overlap", **{x: a[y]})
bad("overlap", tokens=a["parents"])
bad("overlap", best=a["tokens"])
assert launches("k_beam_pick") == 3
refused(1, "kept", lambda: net.beam_select(np.zeros((1, 2, 7)), np.zeros((1, 2)), 65))
""")


def test_a_beam_search_refuses():
    run("""
net = stack()
prompt = [[3, 4, 5]]
bad = lambda code, match, **kw: refused(code, match, lambda: net.beam_search(**{**dict(prompt=prompt, beams=2, n_new=3), **kw}))
bad(1, "new tokens", n_new=0)
for k in (0, 65): bad(1, "beams", beams=k)
bad(1, "max context", n_new=39)
bad(1, "outside", lens=[4])
for p in (np.nan, 17.0, -17.0): bad(1, "length_power", length_power=p)
bad(1, "sequences", prompt=[[3]] * 1100, beams=60)
net.prefill(prompt)
net.beam_search(prompt, beams=2, n_new=3)
refused(3, "before prefill", lambda: net.decode_step([3]))  # it dropped the caches
empty = ra.Network(0)
refused(3, "Embedding", lambda: empty.beam_search(prompt))
flat = ra.Network(0)
flat.add_embedding(9, 4), flat.add_linear(4, 9), flat.add_softmax(1)
refused(3, "no attention", lambda: flat.beam_search(prompt, n_new=2))
refused(1, "all hypotheses", lambda: flat.beam_search([[3]] * 1000, beams=60, n_new=2000))
""")


@pytest.mark.parametrize("k", [1, 3, 9, 20, 33])
def test_a_beam_search_that_fails_half_way(k):
    """Nothing of it is left: the error words are clear and the next search starts anew."""
    run(f"""
net = stack()
net.beam_search([[3, 4, 5]], beams=2, n_new=4)
fail("launch", {k})
with pytest.raises(ra.MitokError):
    net.beam_search([[3, 4, 5]], beams=2, n_new=4)
fail("launch", 0)
net.beam_search([[3, 4, 5]], beams=2, n_new=4)
""")

"""mitok_paged_attention_device against the formula in 64 bits (numpy).

Tolerance: as test_gpu_tree_attention derives it.  A score is off by at most
  ds = (2 dh + 4) u (sum |q||k| scale + |bias|),  u = 2^-53,
exp turns that into a relative error of the weight, and sums of T weights or
weighted values with the rescalings of T / 16 + 8 maxima are within
(9 T / 8 + 40) u of the sum of magnitudes, so the two sides are within
  2 (2 ds + (9 T / 8 + 40) u) sum_t w_t |v_t|
of one another.
"""
from __future__ import annotations

import ctypes as C
import threading

import numpy as np
import pytest

import rustcrates_amd as ra
from test_gpu_tree_attention import close

pytestmark = pytest.mark.gpu
U = 2.0 ** -53


@pytest.fixture(scope="module")
def net():
    with ra.Network(0) as n:
        yield n


def make(seed, lens, n, H, dh, ps, counts=None, bias="decode", share=0, spare=2, width=None):
    """A case; `share`: the sequences' first so many pages are the first one's."""
    r = np.random.default_rng(seed)
    c = lambda *s: r.standard_normal(s) + 1j * r.standard_normal(s)  # noqa: E731
    lens = np.asarray(lens, np.int64)
    B = len(lens)
    counts = np.full(B, n) if counts is None else np.asarray(counts, np.int64)
    used = -(-(lens + counts) // ps)
    P = int(used.max()) + 1 if width is None else width
    pages = int(used.sum()) + spare
    order = iter(r.permutation(pages).tolist())
    table = np.full((B, P), 0xFFFFFFF0, np.uint32)  # entries behind the used ones are not read
    for b in range(B):
        for j in range(used[b]):
            table[b, j] = table[0, j] if b and j < share else next(order)
    T = int((lens + counts).max())
    ctx = T + 3
    return dict(q=c(B, n, H * dh), kn=c(B, n, H * dh), vn=c(B, n, H * dh), k=c(pages, H, ps, dh), v=c(pages, H, ps, dh),
                table=table, lens=lens, counts=counts, H=H, dh=dh, ps=ps, pages=pages, P=P, ctx=ctx, by_row=bias == "rows",
                bias=None if bias is None else 0.5 * r.standard_normal((H, ctx, ctx) if bias == "rows" else (H, ctx)))


def formula(c):
    """(out, its tolerance, the pools after the call)"""
    B, n = c["q"].shape[:2]
    H, dh, ps = c["H"], c["dh"], c["ps"]
    k, v = c["k"].copy(), c["v"].copy()
    out, tol = np.zeros((B, n, H * dh), complex), np.zeros((B, n, H * dh))
    sc = 1.0 / (1e-8 + np.sqrt(dh))
    for b in range(B):
        L, cnt = int(c["lens"][b]), int(c["counts"][b])
        for i in range(cnt):
            page, row = c["table"][b, (L + i) // ps], (L + i) % ps
            k[page, :, row] = c["kn"][b, i].reshape(H, dh)
            v[page, :, row] = c["vn"][b, i].reshape(H, dh)
        whole = c["table"][b, :-(-(L + cnt) // ps)].astype(np.int64)
        for h in range(H):
            K, V = k[whole, h].reshape(-1, dh), v[whole, h].reshape(-1, dh)
            for i in range(cnt):
                T = L + i + 1
                q = c["q"][b, i, h * dh:(h + 1) * dh]
                bias = 0.0 if c["bias"] is None else c["bias"][h, L + i, :T] if c["by_row"] else c["bias"][h, :T]
                with np.errstate(invalid="ignore"):
                    s = (K[:T] @ q).real * sc + bias
                    e = np.exp(s - s.max())
                    w = e / e.sum()
                    o = out[b, i, h * dh:(h + 1) * dh]  # real weights: numpy's complex product would make 0 inf of an infinity's other part
                    o.real, o.imag = w @ V[:T].real, w @ V[:T].imag
                    ds = (2 * dh + 4) * U * np.max((np.abs(K[:T]) @ np.abs(q) * sc + np.abs(bias))[w != 0], initial=0.0)
                    rel = 2 * (2 * ds + (1.125 * T + 40) * U)
                    tol[b, i, h * dh:(h + 1) * dh] = rel * (w @ (np.abs(V[:T].real) + np.abs(V[:T].imag)))
    return out, tol, k, v


def put(a):
    d = ra.DeviceBuffer(max(a.nbytes, 16))
    d.upload(a)
    return d


def call(net, c, counts=True, fill=7.0):
    names = [x for x in ("q", "kn", "vn", "k", "v", "table", "bias") if c[x] is not None]
    d = {x: put(c[x]) for x in names}
    d["out"] = put(np.full(c["q"].shape, fill, complex))
    try:
        net.paged_attention_device(d["q"], d["kn"], d["vn"], d["k"], d["v"], d["table"], c["lens"], c["q"].shape[1], c["H"],
                                   c["dh"], c["ps"], c["pages"], c["P"], d["out"], counts=c["counts"] if counts else None,
                                   bias=d.get("bias"), bias_stride=0 if c["bias"] is None else c["bias"][0].size,
                                   bias_row_stride=c["ctx"] if c["by_row"] else 0)
        for x in ("q", "kn", "vn", "table"):
            assert np.array_equal(d[x].download(c[x].shape, c[x].dtype), c[x], equal_nan=True), x
        return tuple(d[x].download(c[y].shape, complex) for x, y in (("out", "q"), ("k", "k"), ("v", "v")))
    finally:
        for b in d.values():
            b.free()


def check(net, c, **kw):
    out, k, v = call(net, c, **kw)
    want, tol, wk, wv = formula(c)
    assert np.array_equal(k, wk, equal_nan=True) and np.array_equal(v, wv, equal_nan=True)
    close(out, want, tol)
    return out


@pytest.mark.parametrize("dh", [1, 3, 16, 17, 24, 32, 48, 64, 65, 96, 128, 160, 256])
def test_one_token_of_every_width(net, dh):
    check(net, make(dh, [0, 1, 15, 16, 37, 130], 1, 3, dh, 16))


@pytest.mark.parametrize("n", [2, 7, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 130])
@pytest.mark.parametrize("bias", ["decode", "rows", None])
def test_chunks(net, n, bias):
    check(net, make(n, [0, 5, 64, 83], n, 2, 32, 32, bias=bias))


@pytest.mark.parametrize("dh", [5, 16, 31, 64, 100, 128, 130, 256])
@pytest.mark.parametrize("n", [20, 70])
def test_chunks_of_every_width(net, dh, n):
    check(net, make(dh + n, [0, 30], n, 2, dh, 16, bias="rows"))


@pytest.mark.parametrize("ps", [16, 32, 48, 80, 256, 1008, 1024])
@pytest.mark.parametrize("n", [1, 40])
def test_page_sizes(net, ps, n):
    check(net, make(ps, [ps - 1, ps, ps + 1, max(0, 2 * ps - n), 3], n, 2, 16, ps))


@pytest.mark.parametrize("n,lens", [(1, [3000]), (1, [2047, 5]), (9, [1500, 0, 700]), (30, [2500]), (40, [2900]), (200, [900, 17])])
def test_long_caches_in_chunks(net, n, lens):
    check(net, make(n, lens, n, 1, 64, 64, bias="rows" if n > 64 else "decode"))


@pytest.mark.parametrize("n,counts", [(3, [3, 0, 1, 2]), (20, [0, 20, 1, 17]), (70, [1, 64, 0, 70]), (150, [65, 150, 128, 3])])
def test_ragged_counts(net, n, counts):
    """Rows past a sequence's count are zero and store nothing; one of 0 rows has no slots at all."""
    check(net, make(n, [0, 40, 7, 16], n, 2, 32, 16, counts=counts))


def test_all_rows_without_counts(net):
    check(net, make(5, [3, 9], 6, 2, 24, 16), counts=False)


def test_sequences_that_share_pages(net):
    check(net, make(6, [70] * 5 + [40], 1, 4, 64, 16, share=2))
    check(net, make(7, [64] * 3, 33, 2, 16, 32, share=2))


@pytest.mark.parametrize("n", [1, 5, 40])
def test_what_a_row_does_not_see_has_no_part_in_it(net, n):
    """Infinities and NaN behind the rows, in unused pages and in later new rows."""
    c = make(11, [21, 0, 48], n, 2, 32, 16)
    for pool in (c["k"], c["v"]):
        for b, L in enumerate(c["lens"]):
            for j in range(-(-(L + n) // 16)):
                x = pool[c["table"][b, j]]
                x[:, max(0, L - 16 * j):] = np.nan  # where the new rows go
        pool[np.setdiff1d(np.arange(c["pages"]), c["table"])] = np.inf
    plain, _, _ = call(net, c)
    assert np.isfinite(plain).all()
    check(net, c)
    c["vn"][0, n // 2] = np.inf
    c["kn"][2, n // 2] = np.nan
    c["vn"][1, n - 1, ::3] = -np.inf
    out = check(net, c)
    assert np.array_equal(out[:, :n // 2], plain[:, :n // 2])
    assert np.isnan(out[2, n // 2:]).all() and not np.isfinite(out[0, n // 2:]).any()


@pytest.mark.parametrize("n", [1, 20, 70])
def test_biases_of_minus_infinity_and_the_least_number(net, n):
    c = make(13, [40, 70], n, 2, 16, 16)
    c["bias"][0, 3:39] = -np.inf
    c["bias"][1, ::2] = np.finfo(float).min
    check(net, c)
    c["bias"][0, :] = -np.inf  # nothing left: no softmax
    out = check(net, c)
    assert np.isnan(out[:, :, :16]).all() and np.isfinite(out[:, :, 16:]).all()


def test_scores_far_apart(net):
    c = make(14, [600], 3, 2, 16, 32)
    c["q"] *= 200.0
    check(net, c)


@pytest.mark.parametrize("n", [1, 17, 65])
def test_the_same_bits_each_time_and_whatever_lies_beside(net, n):
    c = make(15, [700, 1203, 12], n, 3, 64, 16)
    a = call(net, c)
    for x, y in zip(a, call(net, c)):
        assert np.array_equal(x, y)


def test_more_sequences_than_the_arguments_hold(net):
    lens = (np.arange(300) * 7 % 90).tolist()
    check(net, make(16, lens, 1, 2, 16, 16))
    check(net, make(17, lens[:120], 18, 1, 16, 16))


def beams(seed, G, K, L, H, dh, ps, shared, bias="decode"):
    """G prompts of K sequences of one row each: sequence k of a prompt holds the prompt's first shared[k] pages."""
    c = make(seed, np.repeat(L, K) if np.ndim(L) else [L] * (G * K), 1, H, dh, ps, bias=bias)
    for b in range(G * K):
        j = min(shared[b % K], int(c["lens"][b]) // ps)
        c["table"][b, :j] = c["table"][b - b % K, :j]
    return c


@pytest.mark.parametrize("L", [0, 5, 15, 16, 17, 47, 48, 100, 128])
def test_beams_of_many_prompts(net, L):
    """Bunches of sequences of equal length, which share all, some or none of their pages."""
    check(net, beams(L, 20, 4, L, 16, 16, 16, [9, 9, 9, 9]))
    check(net, beams(L + 1, 20, 4, L, 16, 16, 16, [9, 1, 2, 0]))


@pytest.mark.parametrize("dh", [3, 16, 24, 32, 40, 64])
@pytest.mark.parametrize("K", [2, 3, 7, 16, 20])
def test_beams_of_every_width(net, dh, K):
    r = np.random.default_rng(K)
    G = -(-70 // K)
    check(net, beams(K, G, K, r.integers(0, 90, G), 8 * 4, dh, 16, r.integers(0, 6, K), bias="rows" if dh == 24 else "decode"))


@pytest.mark.parametrize("K", [2, 4])
@pytest.mark.parametrize("G", [24, 40])
def test_beams_in_blocks_of_either_size(net, G, K):
    """Prompts of their own lengths each, 10 heads: 240 blocks, one a CU, and 400."""
    for dh in (16, 24, 64):
        lens = np.random.default_rng(G + K + dh).permutation(np.arange(0, 6 * G, 6))
        check(net, beams(G + K, G, K, lens, 10, dh, 16, [14, 3, 0, 9][:K]))


def test_equal_lengths_that_share_nothing(net):
    check(net, make(30, [77] * 96, 1, 8, 16, 32))
    c = beams(31, 24, 4, 130, 8, 16, 80, [1, 1, 1, 1])  # pages of five tiles
    check(net, c)


def test_what_a_beam_does_not_see_has_no_part_in_it(net):
    """Values that are not finite in one beam's own rows leave the others' alone, those
    of shared rows reach all that see them, and what lies behind a row reaches none."""
    c = beams(32, 24, 4, 43, 16, 16, 16, [2, 2, 2, 2])
    plain, _, _ = call(net, c)
    for pool in (c["k"], c["v"]):
        for b in range(96):
            pool[c["table"][b, 2], :, 43 % 16:] = np.nan  # where the new row goes and behind it
    out = check(net, c)
    assert np.array_equal(out, plain)
    c["v"][c["table"][5, 2], :, 3] = np.inf  # beam 1 of prompt 1
    c["k"][c["table"][10, 2], :, 0] = np.nan  # beam 2 of prompt 2
    c["v"][c["table"][12, 1], 3, 7, 2] = -np.inf  # a shared row of prompt 3
    c["vn"][17] = np.nan
    out = check(net, c)
    touched = [5, 10, 12, 13, 14, 15, 17]
    rest = np.setdiff1d(np.arange(96), touched)
    assert np.array_equal(out[rest], plain[rest])


def test_pages_of_beams_that_are_none_are_refused(net):
    c = beams(33, 24, 4, 43, 16, 16, 16, [2, 2, 2, 2])
    good = c["table"].copy()
    for at in ((3, 2), (4, 1)):
        c["table"] = good.copy()
        c["table"][at] = c["pages"]
        with pytest.raises(ra.MitokError, match="outside the pool"):
            call(net, c)
    c["table"] = good.copy()
    c["table"][1, 2] = c["table"][0, 2]
    with pytest.raises(ra.MitokError, match="one page"):
        call(net, c)
    c["table"] = good
    check(net, c)


def part(buf, nbytes, offset):
    """`nbytes` of a buffer at `offset`, as a buffer that does not own them"""
    x = ra.DeviceBuffer.__new__(ra.DeviceBuffer)
    x._hip, x.nbytes, x.device, x._p = buf._hip, nbytes, buf.device, C.c_void_p(buf.ptr + offset)
    return x


@pytest.mark.parametrize("n", [3, 40])
def test_offsets_past_32_bits(net, n):
    """The sequence lies in the last pages of a pool of 4.6 GB."""
    H, dh, ps, pages, L = 4, 64, 16, 70000, 40
    c = make(18, [L], n, H, dh, ps, spare=0)
    page, last = H * ps * dh * 16, c["pages"]
    pools = [ra.DeviceBuffer(pages * page) for _ in range(2)]
    ends = [part(p, last * page, (pages - last) * page) for p in pools]
    for e, x in zip(ends, ("k", "v")):
        e.upload(c[x])
    d = {x: put(c[x]) for x in ("q", "kn", "vn", "bias")}
    d["table"], d["out"] = put(np.where(c["table"] < last, c["table"] + (pages - last), 0).astype(np.uint32)), put(c["q"])
    net.paged_attention_device(d["q"], d["kn"], d["vn"], *pools, d["table"], [L], n, H, dh, ps, pages, c["P"], d["out"],
                               bias=d["bias"], bias_stride=c["ctx"])
    want, tol, wk, wv = formula(c)
    close(d["out"].download(c["q"].shape, complex), want, tol)
    for e, w in zip(ends, (wk, wv)):
        assert np.array_equal(e.download(w.shape, complex), w)
    for x in [*pools, *d.values()]:
        x.free()


def test_behind_work_still_queued_on_the_default_stream(net):
    """The queries arrive by a copy that the default stream still has before it
    when the call is made."""
    c = make(19, [150, 40], 5, 3, 64, 16)
    want, _, _ = call(net, c)
    big = [ra.DeviceBuffer(1 << 30) for _ in range(2)]
    d = {x: put(c[x]) for x in ("q", "kn", "vn", "k", "v", "table", "bias")}
    late, o = put(np.zeros_like(c["q"])), ra.DeviceBuffer(c["q"].nbytes)
    hip = late._hip
    for i in range(16):  # about 6 ms of copies
        assert hip.hipMemcpyAsync(big[i % 2]._p, big[1 - i % 2]._p, C.c_size_t(1 << 30), 3, None) == 0
    assert hip.hipMemcpyAsync(late._p, d["q"]._p, C.c_size_t(c["q"].nbytes), 3, None) == 0
    net.paged_attention_device(late, d["kn"], d["vn"], d["k"], d["v"], d["table"], c["lens"], 5, 3, 64, 16, c["pages"], c["P"], o,
                               bias=d["bias"], bias_stride=c["ctx"])
    assert np.array_equal(o.download(c["q"].shape, complex), want)
    for x in [*big, *d.values(), late, o]:
        x.free()


def test_two_networks_at_once():
    cases = [make(20, [300, 40], 1, 2, 32, 16), make(21, [500], 40, 2, 64, 32)]
    want = [formula(c) for c in cases]
    errors = []

    def work(c, w):
        try:
            with ra.Network(0) as n:
                for _ in range(20):
                    out, k, v = call(n, c)
                    close(out, w[0], w[1])
                    assert np.array_equal(k, w[2]) and np.array_equal(v, w[3])
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_pages_that_are_none_are_refused(net):
    for n in (1, 40):
        c = make(22, [50, 20], n, 2, 16, 16)
        good = c["table"].copy()
        for at in ((0, 1), (1, (20 + n - 1) // 16)):
            c["table"] = good.copy()
            c["table"][at] = c["pages"]
            with pytest.raises(ra.MitokError, match="outside the pool") as e:
                call(net, c)
            assert e.value.code == 1
        c["table"] = good
        check(net, c)  # the next call is none the worse


def test_two_sequences_that_store_to_one_page_are_refused(net):
    c = make(23, [20, 40, 3], 2, 2, 16, 16)
    c["table"][1, 2] = c["table"][0, 1]
    with pytest.raises(ra.MitokError, match="one page") as e:
        call(net, c)
    assert e.value.code == 1
    c = make(24, [10], 40, 2, 16, 16)
    c["table"][0, 3] = c["table"][0, 1]  # one sequence's page twice
    with pytest.raises(ra.MitokError, match="one page"):
        call(net, c)
    check(net, make(25, [20, 40, 3], 2, 2, 16, 16))

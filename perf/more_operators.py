"""What is timed of the operators of a beam search on a paged cache: attention
of a chunk of new tokens over pages that sequences may share, forking of
sequences with their pages, and the selection over beams and vocabulary.

Everything is complex double precision (logits and scores real double), the
model's own types; there are no others.  A case is one of

  attention  a chunk of `rows` new tokens per sequence is appended to its pages
             and attends over `lo`..`hi` rows before it and causally over its
             own.  `beams` consecutive sequences share the pages of their first
             `prompt` rows.  `by_row`: the bias row goes by the query's
             position (a prompt), otherwise it is the same for all (decoding).
  fork       every sequence takes the pages of its parent and room for `grow`
             more rows: part-filled pages that are shared are copied in every
             layer.  All hold `system` rows in common, each group of `beams`
             `prompt` more.
  beams      of `beams` x `vocab` continuations per prompt the best `keep`.

With `own` the framework's entry points run, otherwise elementary torch
operations.  Both read the same tensors.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-8  # the attention's scale is 1 / (EPS + sqrt(head width))
NONE = -1   # no parent, no token, no page (0xFFFFFFFF)


def listed():
    return [
        # one user, one token: launches and latency
        dict(name="attention one token b1", kind="attention", batch=1, rows=1, heads=8, dh=64, page=16, ctx=512, lo=160, hi=160,
             beams=1, prompt=0, by_row=False),
        # the wide batch, one token each, over caches near their end: the pages are streamed once
        dict(name="attention one token b64", kind="attention", batch=64, rows=1, heads=12, dh=64, page=16, ctx=512, lo=400,
             hi=511, beams=1, prompt=0, by_row=False),
        # the headline batch with four beams each on their prompt's pages
        dict(name="attention beams b32x4", kind="attention", batch=128, rows=1, heads=8, dh=64, page=16, ctx=512, lo=200,
             hi=248, beams=4, prompt=128, by_row=False),
        # long context, a chunk of a turn's tokens, ragged
        dict(name="attention 64 on long b4", kind="attention", batch=4, rows=64, heads=12, dh=64, page=64, ctx=2048, lo=1801,
             hi=1984, beams=1, prompt=0, by_row=False),
        # a long prompt's next chunk behind an earlier one
        dict(name="attention prompt 700 b3", kind="attention", batch=3, rows=700, heads=12, dh=64, page=32, ctx=2048, lo=512,
             hi=1024, beams=1, prompt=0, by_row=True),
        # one user's beams on the smallest model
        dict(name="fork tiny b1x4", kind="fork", groups=1, beams=4, layers=2, heads=4, dh=16, page=16, ctx=512, system=0,
             prompt=16, lo=23, hi=47, grow=1),
        # every step of the headline batch's beams
        dict(name="fork b32x4", kind="fork", groups=32, beams=4, layers=6, heads=8, dh=64, page=16, ctx=512, system=0,
             prompt=128, lo=150, hi=190, grow=1),
        # a system prompt in common, wide pages, room for a drafted chunk
        dict(name="fork long b16x4", kind="fork", groups=16, beams=4, layers=12, heads=12, dh=64, page=32, ctx=2048, system=1536,
             prompt=0, lo=1580, hi=1620, grow=8),
        # one user of the smallest model
        dict(name="beams b1x4", kind="beams", batch=1, beams=4, vocab=4096, keep=4, mask=False, first=False),
        # every step of the headline batch's beams, half of it under a grammar
        dict(name="beams b32x4", kind="beams", batch=32, beams=4, vocab=32000, keep=4, mask=True, first=False),
        # many beams on the default stack's odd vocabulary, twice as many kept
        dict(name="beams b16x12", kind="beams", batch=16, beams=12, vocab=50280, keep=24, mask=False, first=False),
        # the step after the prompt: one beam lives
        dict(name="beams first step b7x5", kind="beams", batch=7, beams=5, vocab=31999, keep=5, mask=False, first=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return w["bytes"] / 4e12 + w["flops"] / 40e12


def _pool(c):
    """bytes of the pages that a case holds"""
    return 32 * c.get("layers", 1) * c["heads"] * c["dh"] * _pages(c) * c["page"] if c["kind"] != "beams" else 0


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    while True:
        kind = rng.choice(["attention", "attention", "fork", "beams"])
        if kind == "attention":
            ctx = rng.choice([512, 512, 2048])
            rows = rng.choice([1, 1, _log(rng, 1, 64), _log(rng, 16, 800)])
            if rows > ctx // 2:
                continue
            hi = _log(rng, 8, ctx - rows)
            beams = rng.choice([1, 1, 3, 4]) if rows == 1 else 1
            lo = rng.choice([hi, rng.randint(0, hi)])
            c = dict(kind=kind, batch=beams * _log(rng, 1, 64 // beams), rows=rows, heads=rng.randint(1, 12),
                     dh=rng.choice([16, 24, 32, 64, 64, 128]), page=rng.choice([16, 16, 32, 48, 64]), ctx=ctx, lo=lo, hi=hi,
                     beams=beams, prompt=lo // 2 if beams > 1 else 0, by_row=rows > 1 and rng.choice([True, False]))
        elif kind == "fork":
            ctx = rng.choice([512, 512, 2048])
            hi = _log(rng, 8, ctx - 16)
            lo = rng.choice([hi, rng.randint(1, hi)])
            system = rng.choice([0, lo // 2])
            c = dict(kind=kind, groups=_log(rng, 1, 32), beams=rng.randint(1, 8), layers=_log(rng, 1, 12), heads=rng.randint(1, 12),
                     dh=rng.choice([16, 24, 32, 64, 64, 128]), page=rng.choice([16, 16, 32, 48, 64]), ctx=ctx, system=system,
                     prompt=rng.randint(0, lo - system), lo=lo, hi=hi, grow=rng.choice([1, 1, 1, 0, 3, 16]))
        else:
            beams = _log(rng, 1, 16)
            c = dict(kind=kind, batch=_log(rng, 1, 64), beams=beams, vocab=_log(rng, 2000, 50280),
                     keep=rng.choice([beams, beams, 2 * beams, rng.randint(1, 32)]), mask=rng.choice([True, False]),
                     first=rng.choice([True, False, False]))
        if _cost(c) <= most[kind] and _pool(c) <= 1.3e9:
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _pages(c):
    """pages of a pool: enough for every sequence, and a fork's copies and room"""
    if c["kind"] == "attention":
        return c["batch"] * -(-(c["hi"] + c["rows"]) // c["page"]) - (c["batch"] - c["batch"] // c["beams"]) * (c["prompt"] // c["page"])
    own_pages = -(-c["hi"] // c["page"]) - (c["system"] + c["prompt"]) // c["page"] + 1
    n = c["groups"] * c["beams"]
    return -(-c["system"] // c["page"]) + c["groups"] * -(-c["prompt"] // c["page"]) + n * (own_pages + 2 + -(-c["grow"] // c["page"]))


def _lens(c, r, n):
    x = r.integers(c["lo"], c["hi"] + 1, n)
    x[0] = c["hi"]  # one is as long as declared
    return x


def prepare(case, seed):
    r = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    real = dict(dtype=torch.float64, device="cuda", generator=g)
    rows = lambda *s: torch.randn(*s, dtype=torch.complex128, device="cuda", generator=g) * math.sqrt(2.0)  # noqa: E731
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    c = case
    if c["kind"] == "beams":
        B, R, V, K = c["batch"], c["beams"], c["vocab"], c["keep"]
        s = dict(case=c, logits=3.0 * torch.randn(B, R, V, **real), parents=torch.empty(B, K, dtype=torch.int32, device="cuda"),
                 tokens=torch.empty(B, K, dtype=torch.int32, device="cuda"), best=torch.empty(B, K, dtype=torch.float64, device="cuda"))
        if c["mask"]:  # every second prompt's rows allow about one token in 30
            shut = (torch.rand(B, R, V, **real) > 0.03) & (torch.arange(B, device="cuda") % 2 == 1)[:, None, None]
            s["logits"].masked_fill_(shut, -math.inf)
        n = r.integers(4, 60, (B, R))  # tokens of each beam so far
        scores = -2.5 * n * r.uniform(0.9, 1.1, (B, R))
        done = r.random((B, R)) < 0.15  # some have ended
        done[:, 0] = False
        if c["first"]:
            scores[:], done[:] = -np.inf, False
            scores[:, 0] = 0.0
        s.update(scores=put(scores), done=put(done.astype(np.int32)), scale=put((n + 1.0) ** -0.7))
        return s
    H, dh, ps = c["heads"], c["dh"], c["page"]
    P = -(-c["ctx"] // ps)
    if c["kind"] == "attention":
        B, n = c["batch"], c["rows"]
        lens = np.repeat(_lens(c, r, B // c["beams"]), c["beams"])
        counts = np.full(B, n)
        if n > 1:  # ragged
            counts = r.integers(-(-n // 4), n + 1, B)
            counts[0] = n
        used = -(-(lens + n) // ps)
        pages = _pages(c)
        order = iter(r.permutation(pages).tolist())  # pages lie anywhere
        table = np.full((B, P), NONE, np.int32)
        for b in range(B):
            for j in range(used[b]):
                share = b % c["beams"] and (j + 1) * ps <= c["prompt"]
                table[b, j] = table[b - 1, j] if share else next(order)
        s = dict(case=c, q=rows(B, n, H * dh), k_new=rows(B, n, H * dh), v_new=rows(B, n, H * dh), k=rows(pages, H, ps, dh),
                 v=rows(pages, H, ps, dh), table=put(table), lens=lens.astype(np.uint32), counts=counts.astype(np.uint32),
                 lens_d=put(lens.astype(np.int64)), counts_d=put(counts.astype(np.int64)), pages=pages, table_width=P)
        s["bias"] = 0.1 * torch.randn(*((H, c["ctx"], c["ctx"]) if c["by_row"] else (H, c["ctx"])), **real)
        s["out"] = torch.empty_like(s["q"])
        return s
    G, N = c["groups"], c["groups"] * c["beams"]
    lens = np.repeat(_lens(c, r, G), c["beams"])
    pages = _pages(c)
    order = iter(r.permutation(pages).tolist())
    table = np.full((N, P), NONE, np.int32)
    for i in range(N):
        for j in range(-(-lens[i] // ps)):
            end = (j + 1) * ps
            if i and end <= c["system"]:
                table[i, j] = table[0, j]
            elif i % c["beams"] and end <= c["system"] + c["prompt"]:
                table[i, j] = table[i - 1, j]
            else:
                table[i, j] = next(order)
    # a few beams of a group live on, some hypotheses are dropped
    parents = np.arange(N) // c["beams"] * c["beams"] + (c["beams"] * r.random(N) ** 2).astype(int)
    parents = np.where(r.random(N) < 0.06, NONE, parents)
    return dict(case=c, k=rows(c["layers"], pages, H, ps, dh), v=rows(c["layers"], pages, H, ps, dh), table=put(table),
                lens=put(lens.astype(np.int32)), parents=put(parents.astype(np.int32)),
                grow=put(np.full(N, c["grow"], np.int32)), table_out=torch.empty(N, P, dtype=torch.int32, device="cuda"),
                lens_out=torch.empty(N, dtype=torch.int32, device="cuda"), pages=pages, table_width=P)


_handle = None


def _network():
    """The handle that a program keeps for its whole life."""
    global _handle
    if _handle is None:
        import rustcrates_amd

        _handle = rustcrates_amd.Network(0)
    return _handle


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"attention": _attention, "fork": _fork, "beams": _beams}[c["kind"]](s)
    net = _network()
    at = lambda name: s[name].data_ptr()  # noqa: E731
    if c["kind"] == "attention":
        net.paged_attention_device(at("q"), at("k_new"), at("v_new"), at("k"), at("v"), at("table"), s["lens"], c["rows"],
                                   c["heads"], c["dh"], c["page"], s["pages"], s["table_width"], at("out"), counts=s["counts"],
                                   bias=at("bias"), bias_stride=s["bias"].stride(0),
                                   bias_row_stride=c["ctx"] if c["by_row"] else 0)
        return dict(out=s["out"], k=s["k"], v=s["v"])
    if c["kind"] == "fork":
        N = c["groups"] * c["beams"]
        net.fork_pages_device(at("k"), at("v"), c["layers"], s["pages"], c["heads"], c["page"], c["dh"], at("table"), at("lens"),
                              N, s["table_width"], at("parents"), N, at("table_out"), at("lens_out"), grow=at("grow"))
        return dict(table=s["table_out"], lens=s["lens_out"], k=s["k"], v=s["v"])
    net.beam_select_device(at("logits"), at("scores"), c["batch"], c["beams"], c["vocab"], c["keep"], at("parents"), at("tokens"),
                           at("best"), done=at("done"), scale=at("scale"))
    return dict(parents=s["parents"], tokens=s["tokens"], scores=s["best"])


# ---------------------------------------------------------------------------
# the plain forms (64 bits throughout: the types are double)
# ---------------------------------------------------------------------------
def _attention(s):
    c = s["case"]
    B, n, H, dh, ps = c["batch"], c["rows"], c["heads"], c["dh"], c["page"]
    T = -(-(c["hi"] + n) // ps) * ps
    L, cnt = s["lens_d"], s["counts_d"]
    b = torch.arange(B, device="cuda")[:, None]
    i = torch.minimum(torch.arange(n, device="cuda")[None], cnt[:, None] - 1)  # an unused row repeats the last one
    slot = L[:, None] + i
    page = s["table"].gather(1, slot // ps).long()
    s["k"][page, :, slot % ps] = s["k_new"][b, i].view(B, n, H, dh)
    s["v"][page, :, slot % ps] = s["v_new"][b, i].view(B, n, H, dh)
    whole = s["table"][:, :T // ps].clamp(min=0).long()
    u = torch.view_as_real(s["q"].conj().resolve_conj()).reshape(B, n, H, 2 * dh).permute(0, 2, 3, 1).reshape(B * H, 2 * dh, n)
    k = torch.view_as_real(s["k"][whole].transpose(1, 2).reshape(B * H, T, dh)).view(B * H, T, 2 * dh)
    v = torch.view_as_real(s["v"][whole].transpose(1, 2).reshape(B * H, T, dh)).view(B * H, T, 2 * dh)
    t = torch.arange(T, device="cuda")
    seen = t[None, :, None] <= slot[:, None]  # [B][T][n]
    if c["by_row"]:
        bias = torch.nn.functional.pad(s["bias"], (0, max(0, T - c["ctx"])))[:, slot, :T].permute(1, 0, 3, 2)  # [B][H][T][n]
    else:
        bias = torch.nn.functional.pad(s["bias"], (0, max(0, T - c["ctx"])))[None, :, :T, None]
    x = torch.bmm(k, u).view(B, H, T, n) / (EPS + math.sqrt(dh)) + bias
    x = x.masked_fill(~seen[:, None], -math.inf)
    e = torch.exp(x - x.amax(2, keepdim=True))
    w = e / e.sum(2, keepdim=True)
    o = torch.bmm(w.view(B * H, T, n).transpose(1, 2).contiguous(), v).view(B, H, n, dh, 2).transpose(1, 2)
    o = o.masked_fill((torch.arange(n, device="cuda")[None] >= cnt[:, None])[..., None, None, None], 0.0)
    return dict(out=torch.view_as_complex(o.contiguous()).reshape(B, n, H * dh), k=s["k"], v=s["v"])


def _fork(s):
    c = s["case"]
    ps, N, P, pages = c["page"], c["groups"] * c["beams"], s["table_width"], s["pages"]
    there = s["parents"] >= 0
    up = s["parents"].clamp(min=0).long()
    lens = torch.where(there, s["lens"][up], 0).long()
    grow = torch.where(there, s["grow"], 0).long()
    j = torch.arange(P, device="cuda")[None]
    had = (lens + ps - 1) // ps
    table = torch.where(j < had[:, None], s["table"][up], NONE).long()
    held = torch.zeros(pages + 1, dtype=torch.int64, device="cuda")  # one behind the last: no page
    held.scatter_add_(0, torch.where(table < 0, pages, table).flatten(), torch.ones(N * P, dtype=torch.int64, device="cuda"))
    # part-filled last pages that grow: the first of their holders stays if all of them grow from there
    last = (had - 1).clamp(min=0)[:, None]
    tail = table.gather(1, last)[:, 0]
    writes = (grow > 0) & (lens % ps > 0)
    mine = torch.where(writes, tail, pages)
    writers = torch.zeros_like(held).scatter_add_(0, mine, torch.ones_like(mine))
    first = torch.full_like(held, N).scatter_reduce_(0, mine, torch.arange(N, device="cuda"), "amin")
    at = tail.clamp(min=0)
    copies = writes & ~((writers[at] == held[at]) & (first[at] == torch.arange(N, device="cuda")))
    # free pages in order: each sequence's copy, then its room
    need = (lens + grow + ps - 1) // ps - had
    start = (copies + need).cumsum(0) - need - copies.long()
    free = (held[:pages] > 0).to(torch.int32).sort(stable=True)[1]
    fresh = free[start.clamp(max=pages - 1)]
    table.scatter_(1, last, torch.where(copies, fresh, tail)[:, None])
    new = (j >= had[:, None]) & (j < (had + need)[:, None])
    table = torch.where(new, free[(start[:, None] + copies[:, None] + j - had[:, None]).clamp(0, pages - 1)], table)
    copies = copies.nonzero()[:, 0]
    src, to = tail[copies], fresh[copies]
    row = (torch.arange(ps, device="cuda")[None] < (lens % ps)[copies][:, None])[None, :, None, :, None]
    for x in (s["k"], s["v"]):
        x[:, to] = torch.where(row, x[:, src], x[:, to])
    s["table_out"].copy_(table)
    s["lens_out"].copy_(lens)
    return dict(table=s["table_out"], lens=s["lens_out"], k=s["k"], v=s["v"])


def _beams(s):
    c = s["case"]
    B, R, V, K = c["batch"], c["beams"], c["vocab"], c["keep"]
    x, done = s["logits"], (s["done"] != 0)[..., None]
    m = x.amax(2, keepdim=True)
    total = s["scores"][..., None] + (x - m - torch.log(torch.exp(x - m).sum(2, keepdim=True)))
    ended = torch.where(torch.arange(V, device="cuda") == 0, s["scores"][..., None], -math.inf)  # one continuation: none
    total = torch.where(done, ended, total)
    rank, at = (total * s["scale"][..., None]).view(B, R * V).topk(K, dim=1)  # equal ranks do not occur above -inf
    best = total.view(B, R * V).gather(1, at)
    none = rank == -math.inf
    row = at // V
    tokens = torch.where(none | done[..., 0].gather(1, row), NONE, at % V)
    parents = torch.where(none, NONE, row + R * torch.arange(B, device="cuda")[:, None])
    return dict(parents=parents.to(torch.int32), tokens=tokens.to(torch.int32), scores=best)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "beams":
        rows = c["batch"] * (1 if c["first"] else 0.87 * c["beams"])  # rows that live: an ended one's logits are not read
        return dict(bytes=8.0 * rows * c["vocab"] + 20.0 * c["batch"] * c["beams"] + 16.0 * c["batch"] * c["keep"],
                    flops=3.0 * rows * c["vocab"])
    mean = (c["lo"] + c["hi"]) / 2
    if c["kind"] == "attention":
        n = c["rows"] if c["rows"] == 1 else 0.625 * c["rows"]  # ragged
        groups = c["batch"] / c["beams"]
        shared = c["prompt"] // c["page"] * c["page"]
        cached = groups * (shared + c["beams"] * (mean - shared))  # rows, a shared one once
        seen = mean + (n + 1) / 2
        bias = c["batch"] * n * seen if c["by_row"] else c["hi"] + c["rows"]
        return dict(bytes=c["heads"] * (32.0 * c["dh"] * (cached + c["batch"] * 3 * n) + 8.0 * bias),
                    flops=float(c["batch"] * c["heads"] * n * seen * 8 * c["dh"]))
    N = c["groups"] * c["beams"]
    # about six of ten take a parent that an earlier one keeps; tails are half full
    copied = 0.6 * N * (c["page"] / 2) if c["grow"] and c["beams"] > 1 else 0.0
    tables = 8.0 * N * mean / c["page"]
    return dict(bytes=64.0 * c["layers"] * c["heads"] * c["dh"] * copied + tables + 20.0 * N, flops=float(N))


# ---------------------------------------------------------------------------
# the same results from the definitions, one sequence or row at a time
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "fork": _exact_fork, "beams": _exact_beams}[case["kind"]](case, s)


def _exact_attention(c, s):
    H, dh, ps = c["heads"], c["dh"], c["page"]
    k, v, out = s["k"].clone(), s["v"].clone(), torch.zeros_like(s["q"])
    table = s["table"].cpu().numpy()
    for b in range(c["batch"]):
        L, n = int(s["lens"][b]), int(s["counts"][b])
        pages = torch.from_numpy(table[b, :-(-(L + n) // ps)].astype(np.int64)).cuda()
        for h in range(H):
            cols = slice(h * dh, (h + 1) * dh)
            rows = []
            for pool, new in ((k, s["k_new"]), (v, s["v_new"])):
                x = pool[pages, h].reshape(-1, dh)
                x[L:L + n] = new[b, :n, cols]
                pool[pages, h] = x.view(-1, ps, dh)
                rows.append(x[:L + n])
            q = s["q"][b, :n, cols]
            kt = rows[0].t().contiguous()
            x = (q.real.contiguous() @ kt.real.contiguous() - q.imag.contiguous() @ kt.imag.contiguous()) / (EPS + math.sqrt(dh))
            x += s["bias"][h, L:L + n, :L + n] if c["by_row"] else s["bias"][h, :L + n]
            x.masked_fill_(torch.ones(n, L + n, dtype=torch.bool, device="cuda").triu(L + 1), -math.inf)
            w = torch.exp(x - x.amax(1, keepdim=True))
            w = w / w.sum(1, keepdim=True)
            out[b, :n, cols] = torch.complex(w @ rows[1].real.contiguous(), w @ rows[1].imag.contiguous())
    return dict(out=out, k=k, v=v)


def _exact_fork(c, s):
    ps, N = c["page"], c["groups"] * c["beams"]
    had, lens, parents = s["table"].cpu().numpy(), s["lens"].cpu().numpy(), s["parents"].cpu().numpy()
    k, v = s["k"].clone(), s["v"].clone()
    new = [[] if p < 0 else had[p, :-(-lens[p] // ps)].tolist() for p in parents]
    n = [0 if p < 0 else int(lens[p]) for p in parents]
    holders, free = {}, set(range(s["pages"]))
    for i in range(N):
        for j, page in enumerate(new[i]):
            writes = c["grow"] > 0 and n[i] % ps and j == len(new[i]) - 1
            holders.setdefault(page, []).append((i, bool(writes)))
            free.discard(page)
    free = sorted(free, reverse=True)
    table = np.full((N, s["table_width"]), NONE, np.int32)
    for i in range(N):
        if parents[i] >= 0 and c["grow"] > 0:
            if n[i] % ps:
                those = holders[new[i][-1]]
                if not all(w for _, w in those) or those[0][0] != i:
                    to = free.pop()
                    for x in (k, v):
                        x[:, to, :, :n[i] % ps] = x[:, new[i][-1], :, :n[i] % ps]
                    new[i][-1] = to
            while len(new[i]) * ps < n[i] + c["grow"]:
                new[i].append(free.pop())
        table[i, :len(new[i])] = new[i]
    return dict(table=torch.from_numpy(table).cuda(), lens=torch.tensor(n, dtype=torch.int32, device="cuda"), k=k, v=v)


def _exact_beams(c, s):
    B, R, V, K = c["batch"], c["beams"], c["vocab"], c["keep"]
    x, scores = s["logits"].cpu().numpy().astype(np.longdouble), s["scores"].cpu().numpy()
    done, scale = s["done"].cpu().numpy(), s["scale"].cpu().numpy()
    parents, tokens, best = np.full((B, K), NONE, np.int32), np.full((B, K), NONE, np.int32), np.full((B, K), -np.inf)
    for b in range(B):
        all_of = []
        for r in range(R):
            if scores[b, r] == -np.inf:
                continue
            if done[b, r]:
                all_of.append((-scores[b, r] * scale[b, r], r, NONE, scores[b, r]))
                continue
            y = x[b, r]
            y = y - y.max()
            y = scores[b, r] + (y - np.log(np.exp(y).sum()))
            for t in np.argsort(-y, kind="stable")[:K]:
                if y[t] > -np.inf:
                    all_of.append((-y[t] * scale[b, r], r, int(t), float(y[t])))
        for j, (_, r, t, y) in enumerate(sorted(all_of, key=lambda a: a[:3])[:K]):
            parents[b, j], tokens[b, j], best[b, j] = b * R + r, t, y
    put = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    return dict(parents=put(parents), tokens=put(tokens), scores=put(best))

"""What is timed of the operators of a serving loop: several drafted tokens
checked in one pass over the KV cache, rows evicted from it by the attention
they received, and the rules that turn logits into a token.

Everything is complex double precision (logits and weights real double), the
model's own types; there are no others.  A case is one of

  tree    attention of `nodes` drafted tokens per sequence over `lo`..`hi`
          cached rows and their own ancestors among the drafted ones; the
          attention that the first `weigh` nodes pay is added to the weights.
  evict   of `lo`..`hi` cached rows `keep` stay, the first `sinks`, the last
          `recent` and those of largest weight, packed into a cache of `keep` rows.
  logits  repetition, presence and frequency penalties over a history, biases
          and a mask of allowed tokens on rows of logits, and the greedy id.

With `own` the framework's entry points run, otherwise elementary torch
operations.  Both read the same tensors.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-8  # the attention's scale is 1 / (EPS + sqrt(head width))


def listed():
    return [
        # one user, one token: the plain decode step as a tree of one node; launches and latency
        dict(name="tree one token b1", kind="tree", batch=1, nodes=1, heads=8, dh=64, ctx=512, lo=160, hi=160, weigh=1,
             shape="chain"),
        # a few users, a short drafted chain each, ragged lengths
        dict(name="tree chain b5 ragged", kind="tree", batch=5, nodes=7, heads=8, dh=64, ctx=512, lo=37, hi=171,
             weigh=1, shape="chain"),
        # the headline batch with a small tree of guesses each
        dict(name="tree 16 nodes b32", kind="tree", batch=32, nodes=16, heads=8, dh=64, ctx=512, lo=128, hi=496,
             weigh=1, shape="tree"),
        # the wide batch, one token each, over caches near their end: the cache is streamed once
        dict(name="tree one token b64", kind="tree", batch=64, nodes=1, heads=12, dh=64, ctx=512, lo=400, hi=511,
             weigh=1, shape="chain"),
        # long context, a large tree, every node's attention weighed
        dict(name="tree 64 nodes long b4", kind="tree", batch=4, nodes=64, heads=12, dh=64, ctx=2048, lo=1900, hi=1984,
             weigh=64, shape="tree"),
        # the smallest model's cache, one user
        dict(name="evict tiny b1", kind="evict", batch=1, heads=4, dh=16, ctx=512, lo=320, hi=320, keep=256, sinks=4,
             recent=32),
        # the headline batch at odd lengths, some not yet full
        dict(name="evict b32 ragged", kind="evict", batch=32, heads=8, dh=64, ctx=512, lo=201, hi=512, keep=256,
             sinks=4, recent=64),
        # long context halved
        dict(name="evict long b4", kind="evict", batch=4, heads=12, dh=64, ctx=2048, lo=2048, hi=2048, keep=1024,
             sinks=4, recent=256),
        # one user of the smallest model
        dict(name="logits b1", kind="logits", rows=1, vocab=4096, history=48, biases=3, mask=True),
        # the headline batch, half of it under a grammar
        dict(name="logits b32", kind="logits", rows=32, vocab=32000, history=256, biases=16, mask=True),
        # every node of the headline batch's trees on the default stack's odd vocabulary
        dict(name="logits tree b512", kind="logits", rows=512, vocab=50280, history=512, biases=16, mask=True),
        # penalties alone, an odd vocabulary, a long history
        dict(name="logits penalties b7", kind="logits", rows=7, vocab=31999, history=2000, biases=0, mask=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return w["bytes"] / 4e12 + w["flops"] / 40e12


def draw(rng):
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0.0), _cost(c))
    while True:
        kind = rng.choice(["tree", "tree", "evict", "logits"])
        if kind == "tree":
            nodes = _log(rng, 1, 64)
            ctx = rng.choice([512, 512, 2048])
            hi = _log(rng, 8, ctx - nodes)
            c = dict(kind=kind, batch=_log(rng, 1, 64), nodes=nodes, heads=rng.randint(1, 12),
                     dh=rng.choice([16, 24, 32, 64, 64, 128]), ctx=ctx, lo=rng.choice([hi, rng.randint(0, hi)]), hi=hi,
                     weigh=rng.choice([0, 1, nodes]), shape=rng.choice(["chain", "tree", "tree"]))
        elif kind == "evict":
            ctx = rng.choice([512, 512, 2048])
            hi = rng.randint(ctx // 4, ctx)
            keep = _log(rng, 8, hi)
            sinks = rng.randint(0, min(8, keep // 2))
            c = dict(kind=kind, batch=_log(rng, 1, 32), heads=rng.randint(1, 12), dh=rng.choice([16, 24, 32, 64, 64, 128]),
                     ctx=ctx, lo=rng.choice([hi, rng.randint(1, hi)]), hi=hi, keep=keep, sinks=sinks,
                     recent=rng.randint(0, (keep - sinks) // 2))
        else:
            c = dict(kind=kind, rows=_log(rng, 1, 512), vocab=_log(rng, 2000, 50280), history=_log(rng, 1, 2000),
                     biases=rng.choice([0, _log(rng, 1, 64)]), mask=rng.choice([True, False]))
        if _cost(c) <= most[kind]:
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _parents(case, r):
    """Each node's parent among the earlier ones of its sequence, -1 for the root."""
    B, n = case["batch"], case["nodes"]
    p = np.full((B, n), -1, np.int64)
    for i in range(1, n):
        p[:, i] = i - 1 if case["shape"] == "chain" else r.integers(max(0, i // 2 - 1), i, B)
    return p


def _closure(parents):
    """seen[b][i][j]: node j is node i or one of its ancestors; depth[b][i]."""
    B, n = parents.shape
    seen = np.zeros((B, n, n), bool)
    b = np.arange(B)
    for i in range(n):
        up = parents[:, i]
        seen[:, i] = seen[b, up] & (up >= 0)[:, None]
        seen[:, i, i] = True
    return seen, seen.sum(2) - 1


def _lens(case, r):
    n = r.integers(case["lo"], case["hi"] + 1, case["batch"])
    n[0] = case["hi"]  # one sequence is as long as declared
    return n.astype(np.uint32)


def prepare(case, seed):
    r = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    real = dict(dtype=torch.float64, device="cuda", generator=g)
    rows = lambda *s: torch.randn(*s, dtype=torch.complex128, device="cuda", generator=g) * math.sqrt(2.0)  # noqa: E731
    if case["kind"] == "logits":
        R, V, H, b = case["rows"], case["vocab"], case["history"], case["biases"]
        s = dict(case=case, logits=3.0 * torch.randn(R, V, **real), out=torch.empty(R, V, dtype=torch.float64, device="cuda"),
                 ids=torch.empty(R, dtype=torch.int32, device="cuda"))
        # a history repeats a few tokens often; shorter ones end in -1
        old = (V * torch.rand(R, H, **real) ** 3).to(torch.int32)
        n = torch.from_numpy(r.integers(1, H + 1, R)).cuda()
        s["history"] = torch.where(torch.arange(H, device="cuda")[None] < n[:, None], old, -1).to(torch.int32)
        s["penalties"] = torch.from_numpy(np.stack([r.uniform(1.0, 1.5, R), r.uniform(-0.5, 1.0, R),
                                                    r.uniform(0.0, 0.3, R)], 1)).cuda()
        s["bias_ids"] = s["bias"] = s["allowed"] = None
        if b:  # distinct tokens
            s["bias_ids"] = torch.rand(R, min(V, 4096), **real).argsort(1)[:, :b].to(torch.int32).contiguous()
            s["bias"] = 2.0 * torch.randn(R, b, **real)
        if case["mask"]:  # every second row allows all, the others about one token in 30
            w = -(-V // 32)
            bits = (torch.rand(R, w * 32, **real) < 0.03) | (torch.arange(R, device="cuda") % 2 == 0)[:, None]
            s["allowed"] = (bits.view(R, w, 32).long() << torch.arange(32, device="cuda")).sum(2).to(torch.int32)
        return s
    B, H, dh, ctx = case["batch"], case["heads"], case["dh"], case["ctx"]
    lens = _lens(case, r)
    k, v = rows(B, H, ctx, dh), rows(B, H, ctx, dh)
    # attention that earlier steps paid: most rows little, a few much
    weights = torch.rand(B, H, ctx, **real) ** 4
    s = dict(case=case, k=k, v=v, weights=weights, lens=lens, lens_d=torch.from_numpy(lens.astype(np.int64)).cuda())
    if case["kind"] == "tree":
        p = _parents(case, r)
        seen, depth = _closure(p)
        s.update(q=rows(B, case["nodes"], H * dh), bias=0.1 * torch.randn(H, ctx, **real),
                 parents=p.astype(np.uint32),  # -1 is 0xFFFFFFFF
                 seen=torch.from_numpy(seen).cuda(), depth=torch.from_numpy(depth).cuda())
        s["out"] = torch.empty_like(s["q"])
    else:
        K = case["keep"]
        new = dict(device="cuda")
        s.update(ko=torch.zeros(B, H, K, dh, dtype=torch.complex128, **new), vo=torch.zeros(B, H, K, dh, dtype=torch.complex128, **new),
                 wo=torch.zeros(B, H, K, dtype=torch.float64, **new), kept=torch.empty(B, H, K, dtype=torch.int32, **new))
    return s


_handle = None


def _network():
    """The handle that a program keeps for its whole life."""
    global _handle
    if _handle is None:
        import rustcrates_amd

        _handle = rustcrates_amd.Network(0)
    return _handle


def _at(t):
    return None if t is None else t.data_ptr()


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"tree": _tree, "evict": _evict, "logits": _logits}[c["kind"]](s)
    net = _network()
    if c["kind"] == "tree":
        net.tree_attention_device(_at(s["q"]), _at(s["k"]), _at(s["v"]), s["lens"], s["parents"], c["heads"], c["dh"],
                                  c["ctx"], _at(s["out"]), bias=_at(s["bias"]), bias_stride=c["ctx"],
                                  weights=_at(s["weights"]), weigh_nodes=c["weigh"])
        return dict(out=s["out"], weights=s["weights"])
    if c["kind"] == "evict":
        n = net.evict_rows_device(_at(s["k"]), _at(s["v"]), _at(s["weights"]), s["lens"], c["heads"], c["dh"], c["ctx"],
                                  c["keep"], c["sinks"], c["recent"], _at(s["ko"]), _at(s["vo"]), _at(s["wo"]),
                                  c["keep"], kept=_at(s["kept"]))
        return dict(k=s["ko"], v=s["vo"], weights=s["wo"], kept=s["kept"], lens=n.astype(np.int64))
    net.process_logits_device(_at(s["logits"]), c["rows"], c["vocab"], out=_at(s["out"]), ids=_at(s["ids"]),
                              history=_at(s["history"]), max_history=c["history"], penalties=_at(s["penalties"]),
                              bias_ids=_at(s["bias_ids"]), bias=_at(s["bias"]), max_bias=c["biases"],
                              allowed=_at(s["allowed"]))
    return dict(logits=s["out"], ids=s["ids"])


# ---------------------------------------------------------------------------
# the plain forms (64 bits throughout: the types are double)
# ---------------------------------------------------------------------------
def _tree(s):
    c = s["case"]
    B, n, H, dh = c["batch"], c["nodes"], c["heads"], c["dh"]
    T = c["hi"] + n
    L = s["lens_d"]
    t = torch.arange(T, device="cuda")
    j = (t[None] - L[:, None]).clamp(0, n - 1)  # the node whose row a slot may hold
    old, new = t[None] < L[:, None], (t[None] >= L[:, None]) & (t[None] < L[:, None] + n)
    b = torch.arange(B, device="cuda")[:, None]
    visible = old[:, None] | (new[:, None] & s["seen"].transpose(1, 2)[b, j].transpose(1, 2))  # [B][n][T]
    column = torch.where(new, L[:, None] + s["depth"][b, j], t[None])
    # Re(q k) is a real product of length 2 dh: (re, -im) with (re, im)
    u = torch.view_as_real(s["q"].conj().resolve_conj()).reshape(B, n, H, 2 * dh).permute(0, 2, 3, 1).reshape(B * H, 2 * dh, n)
    k = torch.view_as_real(s["k"]).view(B * H, c["ctx"], 2 * dh)[:, :T]
    v = torch.view_as_real(s["v"]).view(B * H, c["ctx"], 2 * dh)[:, :T]
    x = torch.bmm(k, u).view(B, H, T, n) / (EPS + math.sqrt(dh)) + s["bias"][:, column].transpose(0, 1)[..., None]
    x = x.masked_fill(~visible.transpose(1, 2)[:, None], -math.inf)
    e = torch.exp(x - x.amax(2, keepdim=True))
    w = e / e.sum(2, keepdim=True)
    o = torch.bmm(w.view(B * H, T, n).transpose(1, 2).contiguous(), v).view(B, H, n, dh, 2).transpose(1, 2)
    paid = w[..., :c["weigh"]].sum(3)
    if c["weigh"]:
        had = s["weights"][:, :, :T]
        s["weights"][:, :, :T] = torch.where(old[:, None], had + paid, torch.where(new[:, None], paid, had))
    return dict(out=torch.view_as_complex(o.contiguous()).reshape(B, n, H * dh), weights=s["weights"])


def _evict(s):
    c = s["case"]
    B, H, dh, K = c["batch"], c["heads"], c["dh"], c["keep"]
    T = c["hi"]
    t, L = torch.arange(T, device="cuda"), s["lens_d"][:, None]
    safe = (t < c["sinks"]) | (t >= L - c["recent"]) | (L <= K)
    x = torch.where(safe[:, None], math.inf, s["weights"][:, :, :T]).masked_fill((t >= L)[:, None], -math.inf)
    order = torch.sort(x, dim=2, descending=True, stable=True)[1][..., :K]  # equal weights: the lowest slot first
    order = torch.where((order < L[..., None]), order, T)
    order = torch.sort(order, dim=2)[0]
    there = order < T
    at = order.clamp(max=T - 1)
    rows = at[..., None].expand(B, H, K, dh)
    s["ko"].copy_(torch.where(there[..., None], s["k"].gather(2, rows), s["ko"]))
    s["vo"].copy_(torch.where(there[..., None], s["v"].gather(2, rows), s["vo"]))
    s["wo"].copy_(torch.where(there, s["weights"].gather(2, at), s["wo"]))
    kept = torch.where(there, at, -1).to(torch.int32)
    return dict(k=s["ko"], v=s["vo"], weights=s["wo"], kept=kept, lens=np.minimum(s["lens"], K).astype(np.int64))


def _logits(s):
    c = s["case"]
    R, V = c["rows"], c["vocab"]
    h = s["history"].long()
    spread = torch.arange(c["history"], device="cuda") % V  # an unused entry adds nothing, each at a place of its own
    count = torch.zeros(R, V, dtype=torch.int32, device="cuda")
    count.scatter_add_(1, torch.where(h < 0, spread, h), (h >= 0).to(torch.int32))
    theta, presence, frequency = (s["penalties"][:, i:i + 1] for i in range(3))
    x = s["logits"]
    x = torch.where(count > 0, torch.where(x > 0, x / theta, x * theta) - (frequency * count.double() + presence), x)
    if c["biases"]:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias"])
    if c["mask"]:
        bits = (s["allowed"][..., None] >> torch.arange(32, dtype=torch.int32, device="cuda")) & 1
        x = x.masked_fill(bits.view(R, -1)[:, :V] == 0, -math.inf)
    best = x.argmax(1)
    ids = torch.where(x.gather(1, best[:, None])[:, 0] > -math.inf, best, -1).to(torch.int32)
    return dict(logits=x, ids=ids)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "logits":
        a_row = 16.0 * c["vocab"] + 4.0 * c["history"] + 24 + 12.0 * c["biases"] + 4 + (c["vocab"] / 8 if c["mask"] else 0)
        return dict(bytes=c["rows"] * a_row, flops=float(c["rows"] * c["vocab"]))
    mean = (c["lo"] + c["hi"]) / 2
    lanes = c["batch"] * c["heads"]
    if c["kind"] == "tree":
        n, T = c["nodes"], mean + c["nodes"]
        weighed = 16.0 * T if c["weigh"] else 0.0
        seen = mean + (n / 2 if c["shape"] == "chain" else math.log2(n + 1))
        return dict(bytes=lanes * (32.0 * c["dh"] * (T + n) + weighed) + 8.0 * c["heads"] * c["hi"],
                    flops=float(lanes * n * seen * 8 * c["dh"]))
    kept = min(mean, c["keep"])
    return dict(bytes=lanes * (64.0 * c["dh"] * kept + 8.0 * mean + 12.0 * kept), flops=float(lanes * mean))


# ---------------------------------------------------------------------------
# the same results from the definitions, one sequence or row at a time
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "evict": _exact_evict, "logits": _exact_logits}[case["kind"]](case, s)


def _exact_tree(c, s):
    B, n, H, dh = c["batch"], c["nodes"], c["heads"], c["dh"]
    out, weights = torch.zeros_like(s["q"]), s["weights"].clone()
    parents = s["parents"].astype(np.int32)
    for b in range(B):
        L = int(s["lens"][b])
        hide = np.ones((n, n), bool)
        deep = np.zeros(n, np.int64)
        for i in range(n):
            j = i
            while j >= 0:
                hide[i, j] = False
                j = int(parents[b, j])
                deep[i] += j >= 0
        hide = torch.from_numpy(np.concatenate([np.zeros((n, L), bool), hide], 1)).cuda()
        col = torch.from_numpy(np.concatenate([np.arange(L), L + deep])).cuda()
        for h in range(H):
            q = s["q"][b, :, h * dh:(h + 1) * dh]
            k, v = s["k"][b, h, :L + n], s["v"][b, h, :L + n]
            kt = k.t().contiguous()
            x = (q.real.contiguous() @ kt.real.contiguous() - q.imag.contiguous() @ kt.imag.contiguous()) / (EPS + math.sqrt(dh))
            w = (x + s["bias"][h, col]).masked_fill(hide, -math.inf)
            w = torch.exp(w - w.amax(1, keepdim=True))  # torch.softmax of long rows is 1e-8 off here
            w = w / w.sum(1, keepdim=True)
            out[b, :, h * dh:(h + 1) * dh] = torch.complex(w @ v.real.contiguous(), w @ v.imag.contiguous())
            if c["weigh"]:
                weights[b, h, L:L + n] = 0
                weights[b, h, :L + n] += w[:c["weigh"]].sum(0)
    return dict(out=out, weights=weights)


def _exact_evict(c, s):
    B, H, K = c["batch"], c["heads"], c["keep"]
    k, v, w = torch.zeros_like(s["ko"]), torch.zeros_like(s["vo"]), torch.zeros_like(s["wo"])
    kept = np.full((B, H, K), -1, np.int32)
    host = s["weights"].cpu().numpy()
    for b in range(B):
        L = int(s["lens"][b])
        for h in range(H):
            stay = list(range(L))
            if L > K:
                middle = range(c["sinks"], L - c["recent"])
                best = sorted(middle, key=lambda t: (-host[b, h, t], t))[:K - c["sinks"] - c["recent"]]
                stay = sorted([*range(c["sinks"]), *best, *range(L - c["recent"], L)])
            at = torch.tensor(stay, device="cuda")
            k[b, h, :len(stay)], v[b, h, :len(stay)], w[b, h, :len(stay)] = s["k"][b, h, at], s["v"][b, h, at], s["weights"][b, h, at]
            kept[b, h, :len(stay)] = stay
    return dict(k=k, v=v, weights=w, kept=kept, lens=np.minimum(s["lens"], K).astype(np.int64))


def _exact_logits(c, s):
    R, V = c["rows"], c["vocab"]
    x, ids = s["logits"].clone(), torch.full((R,), -1, dtype=torch.int32, device="cuda")
    hist, pen = s["history"].cpu().numpy(), s["penalties"].cpu().numpy()
    words = None if s["allowed"] is None else s["allowed"].cpu().numpy().view(np.uint32)
    for r in range(R):
        tokens, times = np.unique(hist[r][hist[r] >= 0], return_counts=True)
        at = torch.from_numpy(tokens.astype(np.int64)).cuda()
        y, (theta, presence, frequency) = x[r, at], pen[r]
        y = torch.where(y > 0, y / theta, y * theta)
        x[r, at] = y - frequency * torch.from_numpy(times).double().cuda() - presence
        if c["biases"]:
            x[r, s["bias_ids"][r].long()] += s["bias"][r]
        if words is not None:
            bits = np.unpackbits(words[r].view(np.uint8), bitorder="little")[:V]
            x[r, torch.from_numpy(bits == 0).cuda()] = -math.inf
        top = x[r].max()
        if top > -math.inf:
            ids[r] = int((x[r] == top).nonzero().max())
    return dict(logits=x, ids=ids)

"""A layer stack of plain numpy products in 64 bits, one sequence at a time: what
the tests of trees, evictions and logit rules hold the library to.  Its cache is
a list of rows per attention layer and head, so a path through a tree is a run
of single steps and an eviction takes rows out of a list.
test_plain_stack.py holds it to the CPU checker."""
from __future__ import annotations

import copy
import math

import numpy as np


def norm(x, eps, gamma, beta):
    t = x - x.mean(-1, keepdims=True)
    s = np.sqrt((t * t).mean(-1, keepdims=True).astype(complex) + eps)
    return ((t / s) * gamma + beta).real.astype(complex)


def gelu(z):
    f = (z + 0.044715 * z * (z * z)) * math.sqrt(2.0 / math.pi)
    f = np.clip(f.real, -30, 30) + 1j * np.clip(f.imag, -30, 30)
    return 0.5 * z * (1.0 + np.tanh(f))


class Sequence:
    """One sequence through cfg's stack; `t` as conftest.seeded_tensors gives it.
    weights[layer][head]: the attention each cached row has received from steps
    called with weigh=True."""

    def __init__(self, cfg, t):
        self.cfg, self.t = cfg, t
        self.k = [[[] for _ in range(cfg.heads)] for _ in range(cfg.layers)]
        self.v = copy.deepcopy(self.k)
        self.weights = copy.deepcopy(self.k)
        self.pos = 0  # tokens seen

    def rotate(self, x, p):
        d, half = self.cfg.d, self.cfg.d // 2
        a = np.clip(p / self.cfg.rope_base ** (2 * np.arange(half) / d), -1, 1)
        c, s = np.cos(a), np.sin(a)
        out = np.empty_like(x)
        out[0::2], out[1::2] = x[0::2] * c - x[1::2] * s, x[0::2] * s + x[1::2] * c
        return out

    def prompt(self, ids):
        """Every prompt row; the last row's Re-logits."""
        cfg, t = self.cfg, self.t
        table = t[0]["table"].reshape(cfg.vocab, cfg.d)
        S, dh = len(ids), cfg.dh
        x = np.where((np.asarray(ids) == 1)[:, None], 0, table[np.asarray(ids, np.int64)])
        if cfg.rope:
            x = np.stack([self.rotate(x[i], i) for i in range(S)])
        mask = np.tril(np.ones((S, S), bool))
        for layer in range(cfg.layers):
            n, a, f = t[1 + 3 * layer: 4 + 3 * layer]
            x = norm(x, cfg.norm_eps, n["gamma"], n["beta"])
            heads = []
            for h in range(cfg.heads):
                q, k, v = (x @ a[w].reshape(cfg.heads, cfg.d, dh)[h] for w in ("wq", "wk", "wv"))
                bias = np.real(a["bias_pos"]).reshape(cfg.heads, cfg.max_ctx, cfg.max_ctx)[h, :S, :S]
                s = np.where(mask, (q @ k.T).real / (1e-8 + math.sqrt(dh)) + bias, -np.inf)
                w = np.exp(s - s.max(1, keepdims=True))
                heads.append((w / w.sum(1, keepdims=True)) @ v)
                self.k[layer][h], self.v[layer][h] = list(k), list(v)
                self.weights[layer][h] = [0.0] * S
            x = self.rest(x, np.concatenate(heads, 1), a, f)
        self.pos = S
        return self.logits(x[-1])

    def rest(self, x, cat, a, f):
        cfg = self.cfg
        x = norm((cat + x).real, cfg.attn_eps, a["gamma"], a["beta"])
        h = gelu(x @ f["w1"].reshape(cfg.d, cfg.ffn) + f["b1"])
        return h @ f["w2"].reshape(cfg.ffn, cfg.d) + f["b2"]

    def logits(self, x):
        w = self.t[-1]
        return (x @ w["w"].reshape(self.cfg.d, self.cfg.vocab) + w["b"]).real

    def step(self, token, weigh=False):
        """One more token; its Re-logits."""
        cfg, t, dh = self.cfg, self.t, self.cfg.dh
        x = np.zeros(cfg.d, complex) if token == 1 else t[0]["table"].reshape(cfg.vocab, cfg.d)[token]
        if cfg.rope:
            x = self.rotate(x, self.pos)
        for layer in range(cfg.layers):
            n, a, f = t[1 + 3 * layer: 4 + 3 * layer]
            x = norm(x, cfg.norm_eps, n["gamma"], n["beta"])
            heads = []
            for h in range(cfg.heads):
                q, k, v = (x @ a[w].reshape(cfg.heads, cfg.d, dh)[h] for w in ("wq", "wk", "wv"))
                self.k[layer][h].append(k)
                self.v[layer][h].append(v)
                self.weights[layer][h].append(0.0)
                K, V = np.array(self.k[layer][h]), np.array(self.v[layer][h])
                bias = np.real(a["bias_pos"]).reshape(cfg.heads, cfg.max_ctx, cfg.max_ctx)[h, 0, :len(K)]
                s = (K @ q).real / (1e-8 + math.sqrt(dh)) + bias
                w = np.exp(s - s.max())
                w /= w.sum()
                heads.append(w @ V)
                if weigh:
                    self.weights[layer][h] = list(np.array(self.weights[layer][h]) + w)
            x = self.rest(x, np.concatenate(heads), a, f)
        self.pos += 1
        return self.logits(x)

    def fork(self):
        other = copy.copy(self)
        other.k, other.v, other.weights = (copy.deepcopy(r) for r in (self.k, self.v, self.weights))
        return other

    def evict(self, keep, sinks, recent):
        for layer in range(self.cfg.layers):
            for h in range(self.cfg.heads):
                stay = kept_rows(self.weights[layer][h], keep, sinks, recent)
                for rows in (self.k, self.v, self.weights):
                    rows[layer][h] = [rows[layer][h][i] for i in stay]


def kept_rows(weights, keep, sinks, recent):
    """Slots that an eviction keeps, ascending."""
    L = len(weights)
    if L <= keep:
        return list(range(L))
    rank = [(-w if w == w else np.inf, w != w, t) for t, w in enumerate(weights)]  # NaN after every number
    best = sorted(range(sinks, L - recent), key=lambda t: rank[t])[: keep - sinks - recent]
    return sorted([*range(sinks), *best, *range(L - recent, L)])


def apply_rules(x, history=(), penalties=(1.0, 0.0, 0.0), bias=(), allowed=None):
    """One row of logits after the rules, and its greedy id (-1: none).  bias: (id, value) pairs, the last of equal ids counts."""
    x = np.array(x, np.float64)
    theta, presence, frequency = penalties
    ids, times = np.unique(np.asarray([t for t in history if t >= 0], np.int64), return_counts=True)
    for t, c in zip(ids, times):
        x[t] = x[t] / theta if x[t] > 0 else x[t] * theta
        x[t] -= frequency * c + presence
    for t, v in dict((t, v) for t, v in bias if t >= 0).items():
        x[t] += v
    if allowed is not None:
        x[~np.asarray(allowed, bool)] = -np.inf
    top = np.max(x)
    return x, (int(np.flatnonzero(x == top)[-1]) if top > -np.inf else -1)

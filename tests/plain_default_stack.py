"""create_transformer's default stack in plain numpy products, one sequence at a
time: Embedding, DiscreteWavelet on the prompt, Norm, RoPE at the uncompressed
positions, two attention layers of 2 and 4 heads with their FeedForwards,
Linear.  The wavelet's rows come from the oracle's layer.
test_plain_default_stack.py holds it to the oracle."""
from __future__ import annotations

import copy
import math

import numpy as np

import oracle
from plain_stack import gelu, kept_rows, norm
from rustcrates_amd import configs

D = configs.REFERENCE_DIM


def tensors(net, vocab, max_ctx):
    """The stack's weights, read from a network of it (either library's)."""
    get = net.get_tensor
    layers = []
    for i, (heads, ffn) in enumerate([(2, 512), (4, 1024)]):
        a, f, dh = 4 + 2 * i, 5 + 2 * i, D // heads
        layers.append(dict(heads=heads, dh=dh, **{w: get(a, s, D * D).reshape(heads, D, dh) for s, w in enumerate(["wq", "wk", "wv"])},
                           bias=np.real(get(a, 3, heads * max_ctx * max_ctx)).reshape(heads, max_ctx, max_ctx),
                           gamma=get(a, 6, D), beta=get(a, 7, D), w1=get(f, 0, D * ffn).reshape(D, ffn), b1=get(f, 4, ffn),
                           w2=get(f, 1, ffn * D).reshape(ffn, D), b2=get(f, 5, D)))
    return dict(table=get(0, 0, vocab * D).reshape(vocab, D), gamma=get(2, 6, D), beta=get(2, 7, D), layers=layers,
                w=get(8, 0, D * vocab).reshape(D, vocab), b=get(8, 4, vocab))


class Sequence:
    def __init__(self, t):
        self.t = t
        self.k = [[[] for _ in range(layer["heads"])] for layer in t["layers"]]
        self.v, self.weights = copy.deepcopy(self.k), copy.deepcopy(self.k)
        self.pos = 0

    def embed(self, ids):
        return np.where((np.asarray(ids) == 1)[:, None], 0, self.t["table"][np.asarray(ids, np.int64)])

    def rows(self, x, positions, first_rows, weigh):
        """x [n][D] behind the wavelet; first_rows: a prompt, row i under bias row i; the last row's Re-logits."""
        t = self.t
        x = norm(x, 1e-8, t["gamma"], t["beta"])
        a = np.clip(np.asarray(positions)[:, None] / 1250.0 ** (2 * np.arange(D // 2) / D), -1, 1)
        y = np.empty_like(x)
        y[:, 0::2], y[:, 1::2] = x[:, 0::2] * np.cos(a) - x[:, 1::2] * np.sin(a), x[:, 0::2] * np.sin(a) + x[:, 1::2] * np.cos(a)
        x = y
        for i, p in enumerate(t["layers"]):
            out = []
            for h in range(p["heads"]):
                q, k, v = (x @ p[w][h] for w in ("wq", "wk", "wv"))
                had = len(self.k[i][h])
                self.k[i][h] += list(k)
                self.v[i][h] += list(v)
                self.weights[i][h] += [0.0] * len(x)
                K, V = np.array(self.k[i][h]), np.array(self.v[i][h])
                n = len(K)
                s = (q @ K.T).real / (1e-8 + math.sqrt(p["dh"])) + (p["bias"][h, :n, :n] if first_rows else p["bias"][h, :1, :n])
                s = np.where(np.arange(n)[None] <= had + np.arange(len(x))[:, None], s, -np.inf)
                w = np.exp(s - s.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                out.append(w @ V)
                if weigh:
                    self.weights[i][h] = list(np.array(self.weights[i][h]) + w.sum(0))
            x = norm((np.concatenate(out, 1) + x).real, 1e-12, p["gamma"], p["beta"])
            x = gelu(x @ p["w1"] + p["b1"]) @ p["w2"] + p["b2"]
        return (x[-1] @ t["w"] + t["b"]).real

    def prompt(self, ids):
        o = oracle.Network()
        o.add_discrete_wavelet(D, configs.WAVELET_DB2, configs.WAVELET_MODE_SYMMETRIC)
        x = o.forward_layers(0, 1, self.embed(ids)[None], mask=np.ones((1, len(ids)), np.uint32), forward_only=False)[0]
        o.close()
        self.pos = len(ids)
        return self.rows(x, range(len(x)), True, False)

    def step(self, token, weigh=False):
        self.pos += 1
        return self.rows(self.embed([token]), [self.pos - 1], False, weigh)

    def fork(self):
        other = copy.copy(self)
        other.k, other.v, other.weights = (copy.deepcopy(r) for r in (self.k, self.v, self.weights))
        return other

    def evict(self, keep, sinks, recent):
        for i, p in enumerate(self.t["layers"]):
            for h in range(p["heads"]):
                stay = kept_rows(self.weights[i][h], keep, sinks, recent)
                for r in (self.k, self.v, self.weights):
                    r[i][h] = [r[i][h][j] for j in stay]

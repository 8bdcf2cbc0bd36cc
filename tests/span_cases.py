"""A paged cache with poison wherever no call may look, and 64-bit attention over it.

Every slot that holds no token, and every page that a table names outside of what its rows see,
is NaN: one read of it that reaches an output shows. (A page id that no call may read is the
poison page's, a valid one, so that such a read would be wrong and not out of range.)
"""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE = 16


class Cache:
    """fp16 pools of `layers` layers for requests of `lens` tokens, on `dev`; K and V of layer
    `layer` as f64 [tokens][kv head][head_dim] lists."""

    def __init__(self, dev, seed, lens, n_kv, hd, layers=2, layer=1, keep_pages=None):
        rng = np.random.default_rng(seed)
        self.lens, self.n_kv, self.hd, self.layers, self.layer = list(lens), n_kv, hd, layers, layer
        self.kv_dim, self.batch = n_kv * hd, len(lens)
        need = [-(-n // PAGE) for n in lens]
        self.stride = max(1, max(need)) + 1
        self.n_pages = sum(need) + 3
        ids = 1 + rng.permutation(self.n_pages - 1)  # page 0 is the poison page
        self.tables = np.zeros((self.batch, self.stride), np.int32)
        k = np.full((self.n_pages, layers, PAGE, self.kv_dim), np.nan, np.float16)
        v = np.full((self.n_pages, layers, self.kv_dim, PAGE), np.nan, np.float16)
        self.k, self.v = [], []
        at = 0
        for b, n in enumerate(lens):
            x = rng.standard_normal((2, n, self.kv_dim)).astype(np.float16)
            self.k.append(x[0].astype(np.float64).reshape(n, n_kv, hd))
            self.v.append(x[1].astype(np.float64).reshape(n, n_kv, hd))
            for i in range(need[b]):
                page, m = ids[at], min(PAGE, n - i * PAGE)
                at += 1
                if keep_pages is None or keep_pages(b, i):
                    self.tables[b, i] = page
                k[page, layer, :m] = x[0, i * PAGE:i * PAGE + m]
                v[page, layer, :, :m] = x[1, i * PAGE:i * PAGE + m].T
        self.host_k, self.host_v = k, v
        self.k_pool = torch.from_numpy(k.reshape(-1)).to(dev)
        self.v_pool = torch.from_numpy(v.reshape(-1)).to(dev)
        self.d_tables = torch.from_numpy(self.tables).to(dev)

    def shape(self, n_head):
        return n_head, self.n_kv, self.hd


def attention(q, k, v, positions, sees):
    """(outputs [rows][heads][hd], weights [heads][rows][tokens]) in f64: row r at positions[r]
    sees token j where sees(p, j); rows that see nothing are 0."""
    rows, heads, hd = q.shape
    group = heads // k.shape[1]
    j = np.arange(k.shape[0])
    seen = np.array([[bool(sees(p, t)) for t in j] for p in positions]).reshape(rows, len(j))
    out, weights = np.zeros((rows, heads, hd)), np.zeros((heads, rows, len(j)))
    for h in range(heads):
        s = q[:, h] @ k[:, h // group].T / math.sqrt(hd)
        s = np.where(seen, s, -np.inf)
        top = s.max(1, initial=-np.inf)
        e = np.exp(s - np.where(np.isinf(top), 0.0, top)[:, None])
        total = e.sum(1)
        w = e / np.where(total == 0, 1.0, total)[:, None]
        weights[h] = w
        out[:, h] = w @ v[:, h // group]
    return out, weights


def window_sees(window, n_sink):
    return lambda p, j: j <= p and (j < n_sink or p - j < window)


def queries(rng, rows, heads, hd, dtype):
    q = rng.standard_normal((rows, heads, hd))
    return q.astype({torch.float16: np.float16, torch.float32: np.float32}[dtype])

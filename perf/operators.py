"""Operators for bounded key-value caches and for drafted tokens, as cases that can be timed and
compared.

A case is a dict of plain values. ``prepare`` makes what a caller has in hand before the call,
``run`` makes one pass, in plain torch (``own = False``) or through the framework's entry points
(``own = True``), ``exact`` gives the same outputs in 64-bit arithmetic straight from the
definitions, and ``work`` counts the bytes and operations that a pass cannot do without.

Operations (``case["op"]``):

* ``decode`` - attention of one new token a request over the paged cache, of which it sees the
  first ``sink`` tokens and the last ``window`` (``Gpu.attention_decode_window_paged``).
* ``chunk``  - the same for chunks of rows packed back to back: prompts, or drafted tokens behind
  a cached history (``Gpu.attention_prefill_window_tiled``).
* ``weigh``  - attention of one new token over the whole cache that also adds the weight each
  cached token received to a pool of running sums (``Gpu.attention_decode_weigh_paged``).
* ``observe`` - the sums that a prompt starts with: the weights that its last ``observe`` rows
  give to the cached tokens (``Gpu.cache_weigh_tiled``).
* ``evict``  - every request cut down to its ``keep`` heaviest tokens, first and newest ones
  kept, in every layer and KV head (``Gpu.cache_evict_paged``).
* ``verify`` - drafted tokens against the target's and the draft's probabilities from given
  random numbers (``Gpu.verify_drafts``).

Layouts are the library's: K pools [page][layer][16][kv_dim], V pools [page][layer][kv_dim][16],
both fp16; the pools of weights (f32) and positions (int32) [page][layer][kv head][16].
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16
VOCAB = 50257
_DTYPE = {"f16": torch.float16, "f32": torch.float32}
_DEV = "cuda"


# ------------------------------------------------------------------------------- the cases

def listed():
    return [
        # One user, one step, a short window: the smallest call, where latency counts.
        dict(name="decode_b1", op="decode", batch=1, n_head=12, n_kv=3, head_dim=64, lo=1024,
             hi=1024, window=256, sink=4, q="f32", out="f32"),
        # A loaded server with long histories behind a 4096-token window, fp16 throughout.
        dict(name="decode_b32_hd128", op="decode", batch=32, n_head=16, n_kv=4, head_dim=128,
             lo=2000, hi=32768, window=4096, sink=4, q="f16", out="f16"),
        # Drafted tokens behind cached histories: a few rows over many keys.
        dict(name="chunk_drafts", op="chunk", n_head=12, n_kv=3, head_dim=64,
             starts="300,9000,1711,16000,4096,640,12345,2047,77,5000,8191,15000,33,7000,1024,10001",
             lens="5,5,3,5,5,2,5,6,5,5,1,5,5,4,5,5", window=4096, sink=4, q="f32", out="f32"),
        # One long prompt.
        dict(name="chunk_8192", op="chunk", n_head=12, n_kv=3, head_dim=64, starts="0",
             lens="8192", window=1024, sink=4, q="f16", out="f32"),
        # Continuous batching, contexts 64..2048 (the benchmark's headline shape).
        dict(name="weigh_b16", op="weigh", batch=16, n_head=12, n_kv=3, head_dim=64, lo=64,
             hi=2048, q="f32", out="f32"),
        # Few requests, long caches.
        dict(name="weigh_b4_hd128", op="weigh", batch=4, n_head=16, n_kv=4, head_dim=128,
             lo=28000, hi=32768, q="f16", out="f32"),
        # Eight ragged prompts, every row observed (the packed benchmark's shape).
        dict(name="observe_packed", op="observe", n_head=16, n_kv=4, head_dim=64,
             starts="0,0,0,0,0,0,0,0", lens="137,420,46,311,98,275,402,190", observe=512,
             q="f32"),
        # The last rows of one long prompt: what is kept before it is cut down.
        dict(name="observe_16384", op="observe", n_head=12, n_kv=3, head_dim=64, starts="0",
             lens="16384", observe=64, q="f32"),
        # A serving loop's regular cut: up to 64 tokens over the budget, all 12 layers.
        dict(name="evict_b16", op="evict", batch=16, n_kv=3, head_dim=64, layers=12, lo=1025,
             hi=1088, keep=1024, sink=4, recent=256),
        # Long prompts cut to 2048 tokens.
        dict(name="evict_prompts", op="evict", batch=4, n_kv=3, head_dim=64, layers=12, lo=4000,
             hi=16384, keep=2048, sink=4, recent=512),
        # Four drafted tokens of one user.
        dict(name="verify_b1", op="verify", batch=1, drafts=4, vocab=VOCAB, ragged=False,
             draft_logits=True, temperature=1.0, dtype="f32"),
        # A batch of up to seven drafted tokens each.
        dict(name="verify_b32", op="verify", batch=32, drafts=7, vocab=VOCAB, ragged=True,
             draft_logits=True, temperature=0.8, dtype="f32"),
    ]


_HEADS = [(12, 3), (12, 12), (16, 4), (8, 1), (12, 4), (6, 6)]
_DIMS = [64, 64, 64, 128, 128, 96, 32, 80]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    """One more case of the ranges above."""
    op = rng.choice(["decode", "chunk", "weigh", "observe", "evict", "verify"])
    n_head, n_kv = rng.choice(_HEADS)
    hd = rng.choice(_DIMS)
    heads = dict(n_head=n_head, n_kv=n_kv, head_dim=hd)
    sink = rng.choice([0, 1, 4, 4, 16, 37])
    if op in ("decode", "weigh"):
        hi = _log_int(rng, 1, 32768)
        lo = rng.choice([0, rng.randint(1, hi), hi])
        window = _log_int(rng, 1, 8192) if op == "decode" else hi
        batch = _log_int(rng, 1, 64)
        while batch > 1 and batch * min(hi, window + sink) * n_kv * hd * 4 > 250e6:
            batch //= 2
        c = dict(op=op, batch=batch, **heads, lo=lo, hi=hi, q=rng.choice(["f16", "f32"]),
                 out=rng.choice(["f16", "f32", "f32"]))
        return dict(c, window=window, sink=sink) if op == "decode" else c
    if op in ("chunk", "observe"):
        n = _log_int(rng, 1, 16)
        short = rng.random() < 0.4  # drafted tokens behind long histories, or prompts
        starts = [_log_int(rng, 1, 16000) if short else rng.choice([0, 0, _log_int(rng, 1, 2000)])
                  for _ in range(n)]
        lens = [_log_int(rng, 1, 8) if short else _log_int(rng, 1, 6000) for _ in range(n)]
        ends = [a + b for a, b in zip(starts, lens)]
        while sum(lens) * max(ends) * n_head * hd > 1.2e10 or n * max(lens) * max(ends) * n_head > 1e9:
            lens = [max(1, x * 3 // 4) for x in lens]
            starts = [x * 3 // 4 for x in starts]
            ends = [a + b for a, b in zip(starts, lens)]
        c = dict(op=op, **heads, starts=",".join(map(str, starts)), lens=",".join(map(str, lens)),
                 q=rng.choice(["f16", "f32"]))
        if op == "observe":
            return dict(c, observe=rng.choice([0, 1, 32, 64, 100, 8192]))
        return dict(c, window=_log_int(rng, 1, 8192), sink=sink,
                    out=rng.choice(["f16", "f32", "f32"]))
    if op == "evict":
        hi = _log_int(rng, 2, 16384)
        lo = rng.randint(1, hi)
        keep = rng.randint(1, hi)
        sink = min(sink, keep)
        recent = rng.randint(0, keep - sink)
        layers = rng.choice([1, 2, 4, 12])
        batch = _log_int(rng, 1, 32)
        while batch > 1 and batch * hi * layers * n_kv * hd * 4 > 400e6:
            batch //= 2
        while layers > 1 and batch * hi * layers * n_kv * hd * 4 > 400e6:
            layers //= 2
        return dict(op=op, batch=batch, n_kv=n_kv, head_dim=hd, layers=layers, lo=lo, hi=hi,
                    keep=keep, sink=sink, recent=recent)
    return dict(op=op, batch=_log_int(rng, 1, 32), drafts=rng.randint(1, 7),
                vocab=rng.choice([_log_int(rng, 2, VOCAB), VOCAB]), ragged=rng.random() < 0.7,
                draft_logits=rng.random() < 0.7, temperature=rng.choice([1.0, 0.8, 0.3, 1.7]),
                dtype=rng.choice(["f32", "f32", "f16"]))


# ------------------------------------------------------------------------------- inputs

class _Seeded:
    """Values on the device and whole numbers on the host, from one seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device=_DEV)
        self.g.manual_seed(int(seed))
        self.host = np.random.default_rng(int(seed))

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return torch.empty(shape, dtype=dtype, device=_DEV).normal_(0.0, std, generator=self.g)

    def uniform(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device=_DEV).uniform_(0.0, 1.0,
                                                                             generator=self.g)

    def to(self, a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(_DEV)


def _ints(text):
    return np.array([int(x) for x in text.split(",")], np.int64)


def _tables(host, lens, freed=None, room=0):
    """Disjoint page tables over a shuffled pool of at least `room` pages. Entries of pages that hold no token, or that a
    windowed cache has given back (pages freed[b][0] up to freed[b][1]), are -1."""
    held = []
    for b, n in enumerate(lens):
        pages = np.arange(-(-int(n) // PAGE))
        held.append(pages if freed is None else pages[(pages < freed[b][0]) | (pages >= freed[b][1])])
    n_pages = max(room, 4 + sum(map(len, held)))
    perm = host.permutation(n_pages).astype(np.int32)
    tables = np.full((len(lens), max(1, -(-int(max(lens)) // PAGE))), -1, np.int32)
    at = 0
    for row, pages in zip(tables, held):
        row[pages] = perm[at:at + len(pages)]
        at += len(pages)
    return tables, n_pages


def _pools(r, s, case, layers, lens, freed=None, weights=None):
    """The pools of the cache, its tables, and where its tokens lie. What the first tokens of a
    request get of the attention is large, as it is in trained decoders. `weights`: about what
    one token's sum of weights has come to, in a pool that holds every request at its longest."""
    hd, n_kv = case["head_dim"], case["n_kv"]
    room = case["batch"] * -(-case["hi"] // PAGE) if weights and "hi" in case else 0
    tables, n_pages = _tables(r.host, lens, freed, room)
    s["n_layer"], s["layer"], s["stride"], s["kv_dim"] = layers, layers - 1, tables.shape[1], n_kv * hd
    s["k_pool"] = r.normal(n_pages * layers * PAGE * n_kv * hd, dtype=torch.float16)
    s["v_pool"] = r.normal(n_pages * layers * PAGE * n_kv * hd, dtype=torch.float16)
    first = torch.from_numpy(np.maximum(tables[:, 0], 0)).long().to(_DEV)
    s["k_pool"].view(n_pages, layers, PAGE, -1)[first, :, :4] *= 2.0
    s["tables"] = r.to(tables)
    if weights:  # sums over many queries: a few tokens hold most of them
        s["w_pool"] = weights * torch.exp(1.5 * r.normal(n_pages * layers * n_kv * PAGE))
        s["pos_pool"] = torch.zeros(n_pages * layers * n_kv * PAGE, dtype=torch.int32, device=_DEV)
        s["pos_pool"].view(n_pages, layers, n_kv, PAGE).copy_(_positions(tables, n_pages, r)[:, None, None])


def _positions(tables, n_pages, r):
    """[page][slot]: the position of the token in it, 0 where there is none."""
    at = np.zeros((n_pages, PAGE), np.int32)
    for row in tables:
        held = np.nonzero(row >= 0)[0]
        at[row[held]] = held[:, None] * PAGE + np.arange(PAGE)
    return r.to(at)


def _pairs(lens):
    """(request, slot) of every cached token, as two device tensors."""
    n = torch.from_numpy(np.asarray(lens, np.int64)).to(_DEV)
    total = int(np.sum(lens))
    who = torch.repeat_interleave(torch.arange(len(lens), device=_DEV), n, output_size=total)
    first = torch.cumsum(n, 0) - n
    return who, torch.arange(total, device=_DEV) - first[who]


def _decode_lens(case, host):
    lens = host.integers(case["lo"], case["hi"] + 1, size=case["batch"])
    if not lens.any():
        lens[0] = case["hi"]
    return lens


def _prepare_rows(case, seed):
    """One new token a request (its K and V are in the cache already)."""
    r, s = _Seeded(seed), {"case": case}
    lens = _decode_lens(case, r.host)
    width = case["n_head"] * case["head_dim"]
    weigh = case["op"] == "weigh"
    freed = None if weigh else [
        (-(-case["sink"] // PAGE), max(-(-case["sink"] // PAGE), (int(n) - case["window"]) // PAGE))
        for n in lens]
    _pools(r, s, case, 2, lens, freed, weights=1e-3 if weigh else None)
    s["q"] = r.normal(case["batch"], width, dtype=_DTYPE[case["q"]])
    s["out"] = torch.zeros((case["batch"], width), dtype=_DTYPE[case["out"]], device=_DEV)
    s["host_lens"], s["lens"] = lens, r.to(lens.astype(np.int32))
    s["positions"] = r.to((lens - 1).astype(np.int32))
    if weigh:
        s["who"], s["slot"] = _pairs(lens)
        s["active"] = r.to(np.nonzero(lens)[0])
    return s


def _prepare_chunk(case, seed):
    """Chunks of rows packed back to back, their K and V in the cache already."""
    r, s = _Seeded(seed), {"case": case}
    starts, lens = _ints(case["starts"]), _ints(case["lens"])
    width, rows = case["n_head"] * case["head_dim"], int(lens.sum())
    observe = case["op"] == "observe"
    freed = None if observe else [
        (-(-case["sink"] // PAGE), max(-(-case["sink"] // PAGE), (int(a) - case["window"] + 1) // PAGE))
        for a in starts]
    _pools(r, s, case, 2, starts + lens, freed, weights=1e-3 if observe else None)
    s["q"] = r.normal(rows, width, dtype=_DTYPE[case["q"]])
    if not observe:
        s["out"] = torch.zeros((rows, width), dtype=_DTYPE[case["out"]], device=_DEV)
    packed = np.concatenate([[0], np.cumsum(lens)[:-1]])
    seg = np.stack([packed, lens, starts, np.arange(len(lens))], 1).astype(np.int32)
    s["segments"], s["host_starts"], s["host_lens"] = r.to(seg), starts, lens
    s["who"], s["offset"] = _pairs(lens)
    s["positions"] = r.to(np.concatenate([a + np.arange(n) for a, n in zip(starts, lens)]).astype(np.int32))
    if observe:
        s["all_who"], s["all_slot"] = _pairs(starts + lens)
    return s


def _prepare_evict(case, seed):
    r, s = _Seeded(seed), {"case": case}
    lens = r.host.integers(case["lo"], case["hi"] + 1, size=case["batch"])
    _pools(r, s, case, case["layers"], lens, weights=1.0)
    s["host_lens"], s["lens"] = lens, r.to(lens.astype(np.int32))
    s["new_lens"] = torch.zeros_like(s["lens"])
    # A pass cuts the cache down; the sums and positions that decide about the next one are put
    # back first, so that every pass has the same work.
    s["w_start"], s["pos_start"] = s["w_pool"].clone(), s["pos_pool"].clone()
    return s


def _prepare_verify(case, seed):
    """The draft's logits are the target's with noise; the drafts are drawn from them."""
    r, s = _Seeded(seed), {"case": case}
    b, k, v = case["batch"], case["drafts"], case["vocab"]
    dtype = _DTYPE[case["dtype"]]
    target = r.normal(b, k + 1, v, std=3.0)
    draft = target[:, :k] + r.normal(b, k, v, std=0.7)
    s["target"], s["draft"] = target.to(dtype), draft.to(dtype) if case["draft_logits"] else None
    noise = -torch.log(-torch.log(r.uniform(b, k, v).clamp_(1e-30, 1 - 1e-7)))
    s["drafts"] = (draft / case["temperature"] + noise).argmax(-1).to(torch.int32)
    n = r.host.integers(0, k + 1, size=b) if case["ragged"] else np.full(b, k)
    s["n_draft"] = r.to(n.astype(np.int32))
    s["u_accept"], s["u_sample"] = r.uniform(b, k), r.uniform(b)
    s["tokens"] = torch.full((b, k + 1), -1, dtype=torch.int32, device=_DEV)
    s["accepted"] = torch.zeros(b, dtype=torch.int32, device=_DEV)
    return s


_PREPARE = {"decode": _prepare_rows, "weigh": _prepare_rows, "chunk": _prepare_chunk,
            "observe": _prepare_chunk, "evict": _prepare_evict, "verify": _prepare_verify}


def prepare(case, seed):
    return _PREPARE[case["op"]](case, seed)


# ------------------------------------------------------------------------------- plain torch

def _views(s):
    case = s["case"]
    kv, n_layer = s["kv_dim"], s["n_layer"]
    k = s["k_pool"].view(-1, n_layer, PAGE, kv)
    v = s["v_pool"].view(-1, n_layer, kv, PAGE)
    small = [s[x].view(-1, n_layer, case["n_kv"], PAGE) if x in s else None for x in ("w_pool", "pos_pool")]
    return k, v, *small


def _page_of(s, who, slot):
    """Page of cached token `slot` of request `who` (any page where none is held)."""
    at = (slot // PAGE).clamp(0, s["stride"] - 1)
    return s["tables"].long()[who, at].clamp(min=0)


def _keys(s, who, j):
    """K and V of tokens j [requests, n] as f32 [requests, kv heads, n, head_dim]."""
    k, v, _, _ = _views(s)
    page, hd = _page_of(s, who[:, None], j), s["case"]["head_dim"]
    shape = (*j.shape, -1, hd)
    kd = k[page, s["layer"], j % PAGE].float().view(shape).transpose(1, 2)
    vd = v[page, s["layer"], :, j % PAGE].float().view(shape).transpose(1, 2)
    return kd, vd


def _softmax(q, k, seen):
    """Weights [requests, kv heads, rows, group, n] of rows q [requests, rows, heads, head_dim];
    seen [requests, rows, n]. A row that sees nothing has weights 0."""
    n, rows, heads, hd = q.shape
    kv = k.shape[1]
    qg = q.float().view(n, rows, kv, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd)
    sc = torch.matmul(qg, k.transpose(2, 3).contiguous()).view(n, kv, rows, heads // kv, -1)
    sc = (sc * (1.0 / math.sqrt(hd))).masked_fill(~seen[:, None, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _weighted(p, v):
    """[requests, rows, heads * head_dim] of weights p over values v."""
    n, kv, rows, group, keys = p.shape
    o = torch.matmul(p.reshape(n, kv, rows * group, keys), v.contiguous())
    return o.view(n, kv, rows, group, -1).permute(0, 2, 1, 3, 4).reshape(n, rows, -1)


def _plain_window(s, q, first, n_rows, longest):
    """Rows q [requests, rows, heads, head_dim] of requests whose first row is at position
    first[r]; n_rows[r] of them count. `longest`: the most tokens that a request holds."""
    case, rows = s["case"], q.shape[1]
    sink, window = case["sink"], case["window"]
    who = torch.arange(q.shape[0], device=_DEV)
    width = max(0, min(longest - sink, window + rows - 1))
    base = (first - window + 1).clamp(min=sink)
    head = torch.arange(sink, device=_DEV).expand(len(who), sink)
    j = torch.cat([head, base[:, None] + torch.arange(width, device=_DEV)], 1)
    k, v = _keys(s, who, j)
    at = (first[:, None] + torch.arange(rows, device=_DEV))[:, :, None]
    j = j[:, None]
    seen = (j <= at) & ((j < sink) | (j > at - window)) & (at < (first + n_rows)[:, None, None])
    return _weighted(_softmax(q, k, seen), v)


def _plain_decode(s):
    case, lens = s["case"], s["lens"].long()
    q = s["q"].view(case["batch"], 1, case["n_head"], -1)
    o = _plain_window(s, q, lens - 1, (lens > 0).long(), int(s["host_lens"].max()))[:, 0]
    s["out"].copy_(torch.where((lens > 0)[:, None], o.to(s["out"].dtype), s["out"]))
    return {"out": s["out"]}


def _padded(s, x, lens, rows):
    """Rows of packed x as [requests, rows, heads, head_dim], the last rows[r] of each."""
    at = s["segments"][:, 0].long() + lens
    i = (at[:, None] - rows + torch.arange(rows, device=_DEV)).clamp(min=0)
    return x.view(x.shape[0], s["case"]["n_head"], -1)[i]


def _plain_chunk(s):
    starts, lens = s["segments"][:, 2].long(), s["segments"][:, 1].long()
    rows = int(s["host_lens"].max())
    i = s["segments"][:, 0].long()[:, None] + torch.arange(rows, device=_DEV)
    q = s["q"].view(s["q"].shape[0], s["case"]["n_head"], -1)[i.clamp(max=s["q"].shape[0] - 1)]
    o = _plain_window(s, q, starts, lens, int((s["host_starts"] + s["host_lens"]).max()))
    s["out"].copy_(o[s["who"], s["offset"]].to(s["out"].dtype))
    return {"out": s["out"]}


def _plain_weigh(s):
    case, lens = s["case"], s["lens"].long()
    _, _, w, pos = _views(s)
    longest = int(s["host_lens"].max())
    who = torch.arange(case["batch"], device=_DEV)
    j = torch.arange(longest, device=_DEV).expand(case["batch"], longest)
    k, v = _keys(s, who, j)
    p = _softmax(s["q"].view(case["batch"], 1, case["n_head"], -1), k, (j < lens[:, None])[:, None])
    o = _weighted(p, v)[:, 0].to(s["out"].dtype)
    s["out"].copy_(torch.where((lens > 0)[:, None], o, s["out"]))
    got = p.sum((2, 3))[s["who"], :, s["slot"]]
    page, slot = _page_of(s, s["who"], s["slot"]), s["slot"] % PAGE
    newest = (s["slot"] == lens[s["who"]] - 1)[:, None]
    w[page, s["layer"], :, slot] = torch.where(newest, got, w[page, s["layer"], :, slot] + got)
    last = (lens - 1)[s["active"]]
    pos[_page_of(s, s["active"], last), s["layer"], :, last % PAGE] = s["positions"][s["active"]][:, None]
    return {"out": s["out"], "w_pool": s["w_pool"], "pos_pool": s["pos_pool"]}


def _plain_observe(s):
    case = s["case"]
    _, _, w, pos = _views(s)
    starts, lens = s["segments"][:, 2].long(), s["segments"][:, 1].long()
    longest = int((s["host_starts"] + s["host_lens"]).max())
    rows = min(case["observe"], int(s["host_lens"].max()))
    n = len(lens)
    j = torch.arange(longest, device=_DEV).expand(n, longest)
    got = torch.zeros((n, case["n_kv"], longest), device=_DEV)
    if rows:
        k, _ = _keys(s, torch.arange(n, device=_DEV), j)
        at = (starts + lens)[:, None] - rows + torch.arange(rows, device=_DEV)
        seen = (j[:, None] <= at[:, :, None]) & (at >= starts[:, None])[:, :, None]
        got = _softmax(_padded(s, s["q"], lens, rows), k, seen).sum((2, 3))
    who, slot = s["all_who"], s["all_slot"]
    page, new = _page_of(s, who, slot), (slot >= starts[who])[:, None]
    got, old = got[who, :, slot], w[page, s["layer"], :, slot % PAGE]
    w[page, s["layer"], :, slot % PAGE] = torch.where(new, got, old + got)
    slot = starts[s["who"]] + s["offset"]
    pos[_page_of(s, s["who"], slot), s["layer"], :, slot % PAGE] = s["positions"][:, None]
    return {"w_pool": s["w_pool"], "pos_pool": s["pos_pool"]}


def _plain_evict(s):
    case, lens = s["case"], s["lens"].long()
    keep, hd, n_kv, layers = case["keep"], case["head_dim"], case["n_kv"], case["layers"]
    k, v, w, pos = _views(s)
    b, longest = case["batch"], int(s["host_lens"].max())
    j = torch.arange(longest, device=_DEV)
    page = _page_of(s, torch.arange(b, device=_DEV)[:, None], j[None])
    wd = w[page, :, :, j % PAGE].permute(0, 2, 3, 1)       # [request, layer, head, token]
    pd = pos[page, :, :, j % PAGE].permute(0, 2, 3, 1)
    held = (j < lens[:, None])[:, None, None]
    newest = torch.where(held, pd, torch.full_like(pd, -1)).amax(-1, keepdim=True)
    safe = (pd < case["sink"]) | (pd > newest - case["recent"])
    rank = torch.where(held, torch.where(safe, torch.full_like(wd, math.inf), wd),
                       torch.full_like(wd, -math.inf))
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(held.expand_as(rank)).scatter_(-1, order[..., :keep], True)
    new = torch.minimum(lens, torch.full_like(lens, keep))
    s["new_lens"].copy_(new)
    most = max(0, longest - keep)
    if not most:
        return {x: s[x] for x in ("k_pool", "v_pool", "w_pool", "pos_pool", "new_lens")}
    # The i-th free place below `keep` takes the i-th kept token at or past it. Pairs past the
    # last one move a token onto itself.
    over = (lens > keep)[:, None, None, None]
    hole, mover = ~kept & (j < keep) & over, kept & (j >= keep) & over
    own_slot = (lens - 1).clamp(min=0)[:, None, None, None].expand(b, layers, n_kv, most + 1)
    src, dst = own_slot.clone(), own_slot.clone()
    for_all = j.expand_as(kept)
    spare = torch.full_like(for_all, most)
    dst.scatter_(-1, torch.where(hole, (hole.cumsum(-1) - 1).clamp(max=most), spare), for_all)
    src.scatter_(-1, torch.where(mover, (mover.cumsum(-1) - 1).clamp(max=most), spare), for_all)
    src, dst = src[..., :most], dst[..., :most]
    idle = torch.arange(most, device=_DEV) >= mover.sum(-1, keepdim=True)
    src = torch.where(idle, own_slot[..., :most], src)
    dst = torch.where(idle, own_slot[..., :most], dst)
    who = torch.arange(b, device=_DEV)[:, None, None, None]
    layer = torch.arange(layers, device=_DEV)[None, :, None, None]
    head = torch.arange(n_kv, device=_DEV)[None, None, :, None]
    sp, dp, ss, ds = _page_of(s, who, src), _page_of(s, who, dst), src % PAGE, dst % PAGE
    kh, vh = k.view(-1, layers, PAGE, n_kv, hd), v.view(-1, layers, n_kv, hd, PAGE)
    kh[dp, layer, ds, head] = kh[sp, layer, ss, head]
    vh[dp, layer, head, :, ds] = vh[sp, layer, head, :, ss]
    w[dp, layer, head, ds] = w[sp, layer, head, ss]
    pos[dp, layer, head, ds] = pos[sp, layer, head, ss]
    return {x: s[x] for x in ("k_pool", "v_pool", "w_pool", "pos_pool", "new_lens")}


def _probabilities(x, temperature):
    x = x.double()
    e = torch.exp((x - x.amax(-1, keepdim=True)) / temperature)
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    """In 64 bits: a sum that 32 would round moves the border between two tokens."""
    case = s["case"]
    k, v = case["drafts"], case["vocab"]
    p = _probabilities(s["target"], case["temperature"])
    t = s["drafts"].long()
    if s["draft"] is None:
        q = torch.zeros_like(p[:, :k]).scatter_(2, t[:, :, None], 1.0)
    else:
        q = _probabilities(s["draft"], case["temperature"])
    pt, qt = (x.gather(2, t[:, :, None])[:, :, 0] for x in (p[:, :k], q))
    count = torch.arange(k, device=_DEV) < s["n_draft"].long()[:, None]
    taken = ((s["u_accept"].double() * qt < pt) & count).long().cumprod(1)
    n = taken.sum(1)
    row = n[:, None, None].expand(-1, 1, v)
    mass = p.gather(1, row)[:, 0]
    less = (mass - q.gather(1, row.clamp(max=k - 1))[:, 0]).clamp(min=0)
    rejected = (n < s["n_draft"].long())[:, None] & (less.sum(1, keepdim=True) > 0)
    mass = torch.where(rejected, less, mass)
    run_sum = mass.cumsum(1)
    border = s["u_sample"].double()[:, None] * run_sum[:, -1:]
    last = torch.where(mass > 0, torch.arange(v, device=_DEV), torch.zeros_like(row[:, 0])).amax(1)
    token = torch.minimum((run_sum <= border).sum(1), last)
    i = torch.arange(k + 1, device=_DEV)
    known = torch.cat([t, torch.full_like(t[:, :1], -1)], 1)
    got = torch.where(i < n[:, None], known, torch.where(i == n[:, None], token[:, None], -1))
    s["tokens"].copy_(got)
    s["accepted"].copy_(n)
    return {"tokens": s["tokens"], "accepted": s["accepted"]}


_PLAIN = {"decode": _plain_decode, "chunk": _plain_chunk, "weigh": _plain_weigh,
          "observe": _plain_observe, "evict": _plain_evict, "verify": _plain_verify}


# ------------------------------------------------------------------------------- the framework

def _gpu():
    from crucible_amd.gpu import Gpu

    if "gpu" not in _HELD:
        _HELD["gpu"] = Gpu(0)
    return _HELD["gpu"]


_HELD = {}  # the library handle, as a program holds one


def _heads(s):
    c = s["case"]
    return c["n_head"], c["n_kv"], c["head_dim"]


def _own_decode(s):
    c = s["case"]
    _gpu().attention_decode_window_paged(
        s["q"], s["k_pool"], s["v_pool"], s["out"], s["tables"], s["lens"], c["batch"], *_heads(s),
        s["stride"], s["n_layer"], s["layer"], s["kv_dim"], s["stride"] * PAGE, c["window"],
        c["sink"])
    return {"out": s["out"]}


def _own_chunk(s):
    c = s["case"]
    _gpu().attention_prefill_window_tiled(
        s["q"], s["k_pool"], s["v_pool"], s["out"], s["tables"], s["segments"],
        len(s["host_lens"]), int(s["host_lens"].max()), s["stride"], *_heads(s), s["n_layer"],
        s["layer"], s["kv_dim"], c["window"], c["sink"])
    return {"out": s["out"]}


def _own_weigh(s):
    c = s["case"]
    _gpu().attention_decode_weigh_paged(
        s["q"], s["k_pool"], s["v_pool"], s["w_pool"], s["pos_pool"], s["out"], s["tables"],
        s["positions"], s["lens"], c["batch"], *_heads(s), s["stride"], s["n_layer"], s["layer"],
        s["kv_dim"], s["stride"] * PAGE)
    return {"out": s["out"], "w_pool": s["w_pool"], "pos_pool": s["pos_pool"]}


def _own_observe(s):
    c = s["case"]
    _gpu().cache_weigh_tiled(
        s["q"], s["k_pool"], s["w_pool"], s["pos_pool"], s["tables"], s["segments"],
        s["positions"], len(s["host_lens"]), int(s["host_lens"].max()), s["stride"], *_heads(s),
        s["n_layer"], s["layer"], s["kv_dim"], c["observe"])
    return {"w_pool": s["w_pool"], "pos_pool": s["pos_pool"]}


def _own_evict(s):
    c = s["case"]
    _gpu().cache_evict_paged(
        s["k_pool"], s["v_pool"], s["w_pool"], s["pos_pool"], s["tables"], s["lens"],
        s["new_lens"], c["batch"], c["n_kv"], c["head_dim"], s["stride"], s["n_layer"],
        s["kv_dim"], s["stride"] * PAGE, c["keep"], c["sink"], c["recent"])
    return {x: s[x] for x in ("k_pool", "v_pool", "w_pool", "pos_pool", "new_lens")}


def _own_verify(s):
    c = s["case"]
    _gpu().verify_drafts(s["target"], s["draft"], s["drafts"], s["n_draft"], s["u_accept"],
                         s["u_sample"], s["tokens"], s["accepted"], c["batch"], c["drafts"],
                         c["vocab"], c["temperature"])
    return {"tokens": s["tokens"], "accepted": s["accepted"]}


_OWN = {"decode": _own_decode, "chunk": _own_chunk, "weigh": _own_weigh, "observe": _own_observe,
        "evict": _own_evict, "verify": _own_verify}


def run(state):
    op = state["case"]["op"]
    if op == "evict":
        state["w_pool"].copy_(state["w_start"])
        state["pos_pool"].copy_(state["pos_start"])
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


# ------------------------------------------------------------------------------- work

def _mean_len(case, f):
    """Mean of f over the lengths that a request may have."""
    lens = np.arange(case["lo"], case["hi"] + 1, dtype=np.float64)
    return float(np.mean(f(lens)))


def work(case):
    op = case["op"]
    if op == "verify":
        b, k, v = case["batch"], case["drafts"], case["vocab"]
        rows = b * (k + 1 + (k if case["draft_logits"] else 0))
        size = 2 if case["dtype"] == "f16" else 4
        return {"bytes": rows * v * size + b * (12 * k + 16), "flops": rows * v * 4.0}
    hd, n_kv = case["head_dim"], case["n_kv"]
    if op == "evict":
        keep, sink, recent = case["keep"], case["sink"], case["recent"]

        def moved(n):  # kept tokens at or past `keep`, for weights in no order
            tail = np.maximum(n - keep, 0)
            new = np.minimum(tail, recent)
            others = np.maximum(n - sink - recent, 1)
            return new + (tail - new) * np.clip((keep - sink - recent) / others, 0, 1)

        each = case["batch"] * case["layers"] * n_kv
        bytes_ = each * (8 * _mean_len(case, lambda n: n) + 2 * (4 * hd + 8) * _mean_len(case, moved))
        return {"bytes": bytes_, "flops": each * 2 * _mean_len(case, lambda n: n)}
    heads = case["n_head"]
    qb = 2 if case["q"] == "f16" else 4
    ob = 2 if case.get("out") == "f16" else 4
    if op in ("decode", "weigh"):
        see = (lambda n: np.minimum(n, case["window"] + np.minimum(case["sink"], np.maximum(
            n - case["window"], 0)))) if op == "decode" else (lambda n: n)
        keys = case["batch"] * _mean_len(case, see)
        bytes_ = keys * n_kv * hd * 4 + case["batch"] * heads * hd * (qb + ob)
        if op == "weigh":
            bytes_ += keys * n_kv * 8
        return {"bytes": bytes_, "flops": 4.0 * keys * heads * hd}
    starts, lens = _ints(case["starts"]), _ints(case["lens"])
    keys = pairs = rows = 0
    for a, n in zip(starts.tolist(), lens.tolist()):
        if op == "observe":
            o = min(case["observe"], n)
            p = np.arange(a + n - o, a + n, dtype=np.int64)
            pairs += int((p + 1).sum())
            keys += a + n if o else 0
            rows += o
        else:
            p = np.arange(a, a + n, dtype=np.int64)
            near = np.maximum(0, p - case["window"] + 1)
            pairs += int((p + 1 - near + np.minimum(case["sink"], near)).sum())
            lo = max(0, a - case["window"] + 1)
            keys += a + n - lo + min(case["sink"], lo)
            rows += n
    if op == "observe":
        new = int((starts + lens).sum()) * n_kv
        return {"bytes": keys * n_kv * hd * 2 + rows * heads * hd * qb + 8 * new
                + 4 * int(starts.sum()) * n_kv, "flops": 2.0 * pairs * heads * hd + 2.0 * pairs * heads}
    return {"bytes": keys * n_kv * hd * 4 + rows * heads * hd * (qb + ob),
            "flops": 4.0 * pairs * heads * hd}


# ------------------------------------------------------------------------------- 64 bits

def _exact_cache(s, b, n):
    """K and V [kv heads, n, head_dim] of request b in f64, zeros where no page is held."""
    hd, n_kv = s["case"]["head_dim"], s["case"]["n_kv"]
    pages = s["tables"][b, : -(-n // PAGE)].long()
    k = s["k_pool"].view(-1, s["n_layer"], PAGE, n_kv * hd)[pages.clamp(min=0), s["layer"]]
    v = s["v_pool"].view(-1, s["n_layer"], n_kv * hd, PAGE)[pages.clamp(min=0), s["layer"]]
    gone = (pages < 0)[:, None, None]
    k = k.double().masked_fill(gone, 0.0).reshape(-1, n_kv, hd)[:n]
    v = v.double().masked_fill(gone, 0.0).transpose(1, 2).reshape(-1, n_kv, hd)[:n]
    return k.transpose(0, 1), v.transpose(0, 1)


def _exact_rows(q, k, v, hidden):
    """(outputs [rows, heads, head_dim], weights [kv heads, rows, keys]) of f64 rows
    q [rows, heads, head_dim]; hidden [rows, keys]."""
    group = q.shape[1] // k.shape[0]
    outs, sums = [], []
    for g in range(k.shape[0]):
        total = 0
        for h in range(g * group, (g + 1) * group):
            z = torch.mm(q[:, h], k[g].t()) / math.sqrt(q.shape[2])
            z[hidden] = -math.inf
            w = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
            outs.append(torch.mm(w, v[g]))
            total = total + w
        sums.append(total)
    return torch.stack(outs, 1), torch.stack(sums)


def _exact_attention(s):
    case = s["case"]
    decode = case["op"] in ("decode", "weigh")
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_DEV)
    w = s["w_pool"].double() if "w_pool" in s else None
    pos = s["pos_pool"].clone() if "w_pool" in s else None
    packed = 0
    for b, n in enumerate(s["host_lens"].tolist()):
        first, rows = (n - 1, 1) if decode else (int(s["host_starts"][b]), n)
        if n == 0:
            continue
        at, j = torch.arange(first, first + rows, device=_DEV), torch.arange(first + rows, device=_DEV)
        row0 = b if decode else packed
        packed += rows
        if case["op"] == "observe":
            seen_rows = min(case["observe"], rows)
            at, row0 = at[rows - seen_rows:], row0 + rows - seen_rows
        hidden = j[None] > at[:, None]
        if "window" in case:
            hidden |= (j[None] >= case["sink"]) & (at[:, None] - j[None] >= case["window"])
        q = s["q"][row0:row0 + len(at)].double().view(len(at), case["n_head"], case["head_dim"])
        k, v = _exact_cache(s, b, first + rows)
        o, sums = _exact_rows(q, k, v, hidden)
        out[row0:row0 + len(at)] = o.flatten(1)
        if w is not None:
            page = s["tables"][b, j // PAGE].long()
            idx = (page * s["n_layer"] + s["layer"]) * case["n_kv"] * PAGE + j % PAGE
            idx = idx[None] + PAGE * torch.arange(case["n_kv"], device=_DEV)[:, None]
            old = w[idx]
            old[:, first:] = 0.0
            w[idx] = old + sums.sum(1)
            true = s["positions"][b:b + 1] if decode else s["positions"][packed - rows:packed]
            pos[idx[:, first:]] = true.expand(case["n_kv"], rows)
    if case["op"] == "observe":
        return {"w_pool": w, "pos_pool": pos}
    return {"out": out} if w is None else {"out": out, "w_pool": w, "pos_pool": pos}


def _exact_evict(s):
    case = s["case"]
    n_kv, hd, layers, keep = case["n_kv"], case["head_dim"], case["layers"], case["keep"]
    w = s["w_start"].cpu().numpy().reshape(-1, layers, n_kv, PAGE)
    pos = s["pos_start"].cpu().numpy().reshape(-1, layers, n_kv, PAGE)
    k = s["k_pool"].cpu().numpy().reshape(-1, layers, PAGE, n_kv, hd)
    v = s["v_pool"].cpu().numpy().reshape(-1, layers, n_kv, hd, PAGE)
    tables = s["tables"].cpu().numpy()
    w2, pos2, k2, v2 = w.copy(), pos.copy(), k.copy(), v.copy()
    for b, n in enumerate(s["host_lens"].tolist()):
        if n <= keep:
            continue
        j = np.arange(n)
        page, slot = tables[b, j // PAGE], j % PAGE
        for la in range(layers):
            for h in range(n_kv):
                wj, pj = w[page, la, h, slot].astype(np.float64), pos[page, la, h, slot]
                wj[(pj < case["sink"]) | (pj > pj.max() - case["recent"])] = np.inf
                best = np.lexsort((j, -wj))[:keep]
                kept = np.zeros(n, bool)
                kept[best] = True
                to, src = np.nonzero(~kept[:keep])[0], keep + np.nonzero(kept[keep:])[0]
                a, z = (page[to], la, h, slot[to]), (page[src], la, h, slot[src])
                w2[a], pos2[a] = w[z], pos[z]
                k2[page[to], la, slot[to], h] = k[page[src], la, slot[src], h]
                v2[page[to], la, h, :, slot[to]] = v[page[src], la, h, :, slot[src]]
    flat = lambda x: torch.from_numpy(x.reshape(-1))  # noqa: E731
    return {"k_pool": flat(k2).double(), "v_pool": flat(v2).double(), "w_pool": flat(w2).double(),
            "pos_pool": flat(pos2),
            "new_lens": torch.from_numpy(np.minimum(s["host_lens"], keep).astype(np.int32))}


def _exact_verify(s):
    case = s["case"]
    k, v = case["drafts"], case["vocab"]
    host = {x: s[x].cpu().numpy() for x in ("target", "drafts", "n_draft", "u_accept", "u_sample")}
    draft = None if s["draft"] is None else s["draft"].cpu().numpy()
    tokens, accepted = np.full((case["batch"], k + 1), -1, np.int32), np.zeros(case["batch"], np.int32)

    def share(x):
        x = x.astype(np.float64) / case["temperature"]
        e = np.exp(x - x.max())
        return e / e.sum()

    for b in range(case["batch"]):
        n = 0
        while True:
            mass = share(host["target"][b, n])
            if n == host["n_draft"][b]:
                break
            t = host["drafts"][b, n]
            if draft is None:
                q = np.zeros(v)
                q[t] = 1.0
            else:
                q = share(draft[b, n])
            if not np.float64(host["u_accept"][b, n]) * q[t] < mass[t]:
                less = np.maximum(mass - q, 0.0)
                mass = less if less.sum() > 0 else mass
                break
            tokens[b, n] = t
            n += 1
        border = np.float64(host["u_sample"][b]) * mass.sum()
        past = np.nonzero(np.cumsum(mass) > border)[0]
        tokens[b, n] = past[0] if len(past) else np.nonzero(mass)[0][-1]
        accepted[b] = n
    return {"tokens": torch.from_numpy(tokens), "accepted": torch.from_numpy(accepted)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(s)
    if case["op"] == "verify":
        return _exact_verify(s)
    return _exact_attention(s)

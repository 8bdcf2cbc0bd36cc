"""The operators for bounded caches and drafted tokens as they are used together, and pools whose
offsets pass 32 bits.

Every step is checked against 64-bit or plain arithmetic on what the step was given (the pools as
they were before it), with the tolerances of test_gpu_cache_weights.py; moves are bit for bit.
"""
import numpy as np
import pytest
import torch

from crucible_amd.paged import PagePool, SequencePages
from gates import element_gate
from span_cases import PAGE, attention, window_sees
from test_gpu_cache_weights import plain_evict
from test_gpu_verify import plain as plain_verify

pytestmark = pytest.mark.gpu
F32 = torch.float32


class Pools:
    """Empty pools over the library's allocator, and host copies of them."""

    def __init__(self, dev, n_pages, layers, n_kv, hd, stride):
        self.dev, self.layers, self.n_kv, self.hd, self.stride = dev, layers, n_kv, hd, stride
        self.kv_dim, self.n_pages = n_kv * hd, n_pages
        self.pool = PagePool(n_pages, layers, self.kv_dim)
        n = n_pages * layers * PAGE
        self.k = torch.full((n * self.kv_dim,), float("nan"), dtype=torch.float16, device=dev)
        self.v = torch.full((n * self.kv_dim,), float("nan"), dtype=torch.float16, device=dev)
        self.w = torch.full((n * n_kv,), float("nan"), device=dev)
        self.pos = torch.full((n * n_kv,), -1, dtype=torch.int32, device=dev)

    def host(self):
        shape = (self.n_pages, self.layers)
        return (self.w.cpu().numpy().reshape(*shape, self.n_kv, PAGE).copy(),
                self.pos.cpu().numpy().reshape(*shape, self.n_kv, PAGE).copy(),
                self.k.cpu().numpy().reshape(*shape, PAGE, self.kv_dim).copy(),
                self.v.cpu().numpy().reshape(*shape, self.kv_dim, PAGE).copy())

    def cached(self, host, tables, b, layer, n):
        """K and V [n][kv head][hd] of request b in f64."""
        j = np.arange(n)
        page, slot = tables[b, j // PAGE], j % PAGE
        return (host[2][page, layer, slot].astype(np.float64).reshape(n, self.n_kv, self.hd),
                host[3][page, layer, :, slot].astype(np.float64).reshape(n, self.n_kv, self.hd))


def append(gpu, p, tables, owners, positions, rng, layer):
    rows = len(owners)
    own = torch.tensor(owners, dtype=torch.int32, device=p.dev)
    pos = torch.tensor(positions, dtype=torch.int32, device=p.dev)
    for pool, kind in ((p.k, "k"), (p.v, "v")):
        src = torch.from_numpy(rng.standard_normal((rows, p.kv_dim)).astype(np.float32)).to(p.dev)
        gpu.cache_store_packed_paged(src, pool, tables, own, pos, rows, p.kv_dim, p.stride,
                                     p.layers, layer, kind=kind)


def test_serving_with_a_cache_cut_by_weight(gpu, dev):
    """Prompts observed, cut to a budget and their pages given back; then steps of append, weighing
    decode and, whenever a request is 16 over the budget, a cut, with pages for 16 more tokens."""
    rng = np.random.default_rng(91)
    layers, n_kv, heads, hd, keep, n_sink, n_recent, slack = 2, 2, 6, 64, 48, 3, 12, 16
    prompts = [150, 31, 64, 90]
    p = Pools(dev, 40, layers, n_kv, hd, 12)
    seqs = [SequencePages() for _ in prompts]
    for s, n in zip(seqs, prompts):
        s.grow(p.pool, n)
    tables = np.stack([s.table_padded(p.stride) for s in seqs])
    d_tables = torch.from_numpy(tables).to(dev)
    owners = np.repeat(np.arange(len(prompts)), prompts)
    positions = np.concatenate([np.arange(n) for n in prompts])
    start = np.concatenate([[0], np.cumsum(prompts)[:-1]])
    seg = torch.from_numpy(np.stack([start, prompts, 0 * start, np.arange(4)], 1).astype(np.int32)).to(dev)
    d_pos = torch.from_numpy(positions.astype(np.int32)).to(dev)
    for layer in range(layers):
        append(gpu, p, d_tables, owners, positions, rng, layer)
        q = rng.standard_normal((len(owners), heads, hd)).astype(np.float32)
        gpu.cache_weigh_tiled(torch.from_numpy(q).to(dev), p.k, p.w, p.pos, d_tables, seg, d_pos, 4,
                              max(prompts), p.stride, heads, n_kv, hd, layers, layer, p.kv_dim, 20)
        host = p.host()
        for b, n in enumerate(prompts):
            k, v = p.cached(host, tables, b, layer, n)
            at = np.arange(n - 20, n)
            _, w = attention(q[start[b] + at].astype(np.float64), k, v, at, lambda x, j: j <= x)
            j = np.arange(n)
            got = host[0][tables[b, j // PAGE], layer, :, j % PAGE]
            element_gate(got, w.sum(1).reshape(n_kv, heads // n_kv, n).sum(1).T, "prompt sums")
            assert (host[1][tables[b, j // PAGE], layer, :, j % PAGE] == j[:, None]).all()

    lens = np.array(prompts)
    d_lens = torch.from_numpy(lens.astype(np.int32)).to(dev)
    at = np.array(prompts)  # positions of the next tokens

    def cut():
        nonlocal lens
        before = p.host()
        gpu.cache_evict_paged(p.k, p.v, p.w, p.pos, d_tables, d_lens, d_lens, 4, n_kv, hd, p.stride,
                              layers, p.kv_dim, p.stride * PAGE, keep, n_sink, n_recent)

        class C:
            pass
        c = C()
        c.stride, c.tables, c.layers, c.n_kv, c.hd = p.stride, tables, layers, n_kv, hd
        new = plain_evict(c, *before, lens.tolist(), keep, n_sink, n_recent)
        assert d_lens.cpu().tolist() == new
        after = p.host()
        for x, y in zip(after, before):
            assert np.array_equal(x.view(np.uint16 if x.itemsize == 2 else np.uint32),
                                  y.view(np.uint16 if y.itemsize == 2 else np.uint32))
        lens = np.array(new)

    cut()
    used = p.pool.used_pages()
    for b, s in enumerate(seqs):
        s.shrink(p.pool, int(lens[b]))
        s.grow(p.pool, keep + slack - int(lens[b]))
    assert p.pool.used_pages() < used
    tables = np.stack([s.table_padded(p.stride) for s in seqs])
    d_tables.copy_(torch.from_numpy(tables))
    for step in range(40):
        d_lens.add_(1)
        lens = lens + 1
        for layer in range(layers):
            append(gpu, p, d_tables, range(4), lens - 1, rng, layer)
            q = rng.standard_normal((4, heads, hd)).astype(np.float32)
            out = torch.zeros((4, heads, hd), device=dev)
            before = p.host()
            gpu.attention_decode_weigh_paged(
                torch.from_numpy(q).to(dev), p.k, p.v, p.w, p.pos, out, d_tables,
                torch.from_numpy(at.astype(np.int32)).to(dev), d_lens, 4, heads, n_kv, hd, p.stride,
                layers, layer, p.kv_dim, p.stride * PAGE)
            after = p.host()
            for b, n in enumerate(lens):
                k, v = p.cached(before, tables, b, layer, n)
                want, w = attention(q[b:b + 1].astype(np.float64), k, v, [n - 1], lambda x, j: True)
                element_gate(out[b:b + 1].cpu().numpy(), want, f"step {step}")
                j = np.arange(n)
                page, slot = tables[b, j // PAGE], j % PAGE
                old = before[0][page, layer, :, slot].astype(np.float64)
                old[-1] = 0.0
                element_gate(after[0][page, layer, :, slot],
                             old + w[:, 0].reshape(n_kv, -1, n).sum(1).T, "sums")
                assert (after[1][page[-1], layer, :, slot[-1]] == at[b]).all()
        at = at + 1
        if lens.max() == keep + slack:
            cut()
    assert lens.max() <= keep + slack
    for s in seqs:
        s.release(p.pool)
    assert p.pool.free_pages() == p.n_pages


def test_drafted_tokens_behind_windows(gpu, dev):
    """Rounds of drafts: their rows appended and attended as one chunk, the target's logits
    verified, and what was refused written over; the pages behind the window given back. Each row
    of a chunk is also what a single-token call gives at its length."""
    rng = np.random.default_rng(92)
    n_kv, heads, hd, window, n_sink, k, vocab = 2, 8, 64, 70, 5, 4, 500
    p = Pools(dev, 60, 1, n_kv, hd, 24)
    lens = np.array([200, 7, 130])
    seqs = [SequencePages() for _ in lens]
    for s in seqs:
        s.grow(p.pool, p.stride * PAGE // 2)
    tables = np.stack([s.table_padded(p.stride) for s in seqs])
    d_tables = torch.from_numpy(tables).to(dev)
    append(gpu, p, d_tables, np.repeat(np.arange(3), lens), np.concatenate([np.arange(n) for n in lens]),
           rng, 0)
    sees = window_sees(window, n_sink)
    for step in range(6):
        drafted = rng.integers(0, k + 1, size=3)
        chunk = drafted + 1  # the last token taken, then the drafts
        owners = np.repeat(np.arange(3), chunk)
        at = np.concatenate([lens[b] + np.arange(chunk[b]) for b in range(3)])
        append(gpu, p, d_tables, owners, at, rng, 0)
        host = p.host()
        # behind every window: given back, and the table may say anything that is a page
        gone = d_tables.clone()
        for b in range(3):
            first, last = -(-n_sink // PAGE), max(0, (lens[b] - window + 1) // PAGE)
            gone[b, first:max(first, last)] = 59
        p.k.view(60, -1)[59] = float("nan")
        p.v.view(60, -1)[59] = float("nan")
        start = np.concatenate([[0], np.cumsum(chunk)[:-1]])
        seg = torch.from_numpy(np.stack([start, chunk, lens, np.arange(3)], 1).astype(np.int32)).to(dev)
        rows = len(owners)
        q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
        out = torch.zeros((rows, heads, hd), device=dev)
        gpu.attention_prefill_window_tiled(torch.from_numpy(q).to(dev), p.k, p.v, out, gone, seg, 3,
                                           int(chunk.max()), p.stride, heads, n_kv, hd, 1, 0,
                                           p.kv_dim, window, n_sink)
        one = torch.zeros((3, heads, hd), device=dev)
        gpu.attention_decode_window_paged(
            torch.from_numpy(q[start + chunk - 1]).to(dev), p.k, p.v, one, gone,
            torch.from_numpy((lens + chunk).astype(np.int32)).to(dev), 3, heads, n_kv, hd, p.stride,
            1, 0, p.kv_dim, p.stride * PAGE, window, n_sink)
        got = out.cpu().numpy()
        for b in range(3):
            kb, vb = p.cached(host, tables, b, 0, lens[b] + chunk[b])
            r = np.arange(start[b], start[b] + chunk[b])
            want, _ = attention(q[r].astype(np.float64), kb, vb, lens[b] + np.arange(chunk[b]), sees)
            element_gate(got[r], want, f"round {step}")
            element_gate(one[b:b + 1].cpu().numpy(), want[-1:], f"round {step}, one token")
        target = rng.normal(0, 3, (3, k + 1, vocab)).astype(np.float32)
        draft = (target[:, :k] + rng.normal(0, 0.5, (3, k, vocab))).astype(np.float32)
        drafts = (draft + rng.gumbel(size=draft.shape)).argmax(-1).astype(np.int32)
        ua, us = rng.random((3, k)).astype(np.float32), rng.random(3).astype(np.float32)
        tokens = torch.zeros((3, k + 1), dtype=torch.int32, device=dev)
        taken = torch.zeros(3, dtype=torch.int32, device=dev)
        to = lambda x: torch.from_numpy(x).to(dev)  # noqa: E731
        gpu.verify_drafts(to(target), to(draft), to(drafts), to(drafted.astype(np.int32)), to(ua),
                          to(us), tokens, taken, 3, k, vocab, 0.9)
        want = plain_verify(target, draft, drafts, drafted, ua, us, 0.9)
        assert np.array_equal(tokens.cpu().numpy(), want[0])
        assert np.array_equal(taken.cpu().numpy(), want[1])
        lens = lens + 1 + want[1]


def test_offsets_past_32_bits(gpu, dev):
    """The last pages of pools of 4.4 billion elements: every operator gives the bits that it
    gives in a small pool."""
    n_kv, hd, layers, layer = 12, 64, 12, 11
    kv_dim, page = n_kv * hd, 12 * PAGE * 12 * 64
    many = 2 ** 32 // page + 700
    free, _ = torch.cuda.mem_get_info()
    if free < 3 * 2 * many * page:
        pytest.skip("the device's memory is taken")
    rng = np.random.default_rng(93)
    lens, few = [600, 37], 50
    stride = 40

    def make(n_pages):
        k = torch.zeros(n_pages * page, dtype=torch.float16, device=dev)
        v = torch.zeros(n_pages * page, dtype=torch.float16, device=dev)
        w = torch.zeros(n_pages * layers * n_kv * PAGE, device=dev)
        return [k, v, w, torch.zeros_like(w, dtype=torch.int32)]

    small, big = make(few), make(many)
    g = torch.Generator(device=dev).manual_seed(94)
    for x in small[:2]:
        x.normal_(generator=g)
    small[2].exponential_(generator=g)
    pos = torch.arange(PAGE, device=dev, dtype=torch.int32).repeat(few * layers * n_kv)
    small[3].copy_(pos + 16 * (torch.arange(len(pos), device=dev, dtype=torch.int32) // (layers * n_kv * PAGE)))
    for x, y in zip(small, big):
        y[-len(x):] = x  # the small pool's pages are the big one's last
    tab = torch.zeros((2, stride), dtype=torch.int32)
    tab[0, :38] = torch.arange(38)
    tab[1, :3] = torch.arange(40, 43)
    tab = tab.to(dev)
    d_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    q = torch.from_numpy(rng.standard_normal((2, 24, hd)).astype(np.float32)).to(dev)
    qc = torch.from_numpy(rng.standard_normal((150, 24, hd)).astype(np.float32)).to(dev)
    seg = torch.tensor([[0, 140, 460, 0], [140, 10, 27, 1]], dtype=torch.int32, device=dev)
    p_rows = torch.arange(150, dtype=torch.int32, device=dev)
    outs = []
    for (k, v, w, pos), t in ((small, tab), (big, tab + (many - few))):
        shape = (24, n_kv, hd)
        a, b, c = torch.zeros_like(q), torch.zeros_like(qc), torch.zeros_like(q)
        gpu.attention_decode_window_paged(q, k, v, a, t, d_lens, 2, *shape, stride, layers, layer,
                                          kv_dim, stride * PAGE, 300, 4)
        gpu.attention_prefill_window_tiled(qc, k, v, b, t, seg, 2, 140, stride, *shape, layers,
                                           layer, kv_dim, 300, 4)
        gpu.attention_decode_weigh_paged(q, k, v, w, pos, c, t, d_lens, d_lens, 2, *shape, stride,
                                         layers, layer, kv_dim, stride * PAGE)
        gpu.cache_weigh_tiled(qc, k, w, pos, t, seg, p_rows, 2, 140, stride, *shape, layers, layer,
                              kv_dim, 64)
        new = torch.zeros_like(d_lens)
        gpu.cache_evict_paged(k, v, w, pos, t, d_lens, new, 2, n_kv, hd, stride, layers, kv_dim,
                              stride * PAGE, 500, 4, 32)
        outs.append((a, b, c, new, *(x[-len(y):] for x, y in zip((k, v, w, pos), small))))
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    assert outs[0][3].tolist() == [500, 37] and float(outs[0][0].abs().sum()) > 0

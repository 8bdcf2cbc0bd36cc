"""Running sums of attention weights, a prompt's first sums, and the cut of a cache by them,
against 64-bit and plain implementations.

Outputs meet the reference validator's element gate (tests/gates.py). So do sums of weights: a
weight is 2^x with x a score of at most some 20 in log2 units, known to about 22 bits (fp16 hi + lo)
and so to 5e-6 absolutely, 4e-6 of the weight; its f32 additions (at most a few hundred here, 6e-8
each) stay below that, and 2e-5 of the sum holds both. What a cut moves, it moves bit for bit.
"""
import numpy as np
import pytest
import torch

from gates import element_gate
from span_cases import PAGE, Cache, attention, queries

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
CAUSAL = lambda p, j: j <= p  # noqa: E731


class Sums:
    """Pools of sums and positions beside a Cache, with values everywhere."""

    def __init__(self, dev, c, seed, values=None):
        rng = np.random.default_rng(seed)
        shape = (c.n_pages, c.layers, c.n_kv, PAGE)
        self.w = rng.exponential(size=shape).astype(np.float32) if values is None else values(shape)
        self.pos = rng.integers(-5, 5, size=shape).astype(np.int32)
        self.w_pool = torch.from_numpy(self.w.reshape(-1)).to(dev)
        self.pos_pool = torch.from_numpy(self.pos.reshape(-1)).to(dev)

    def read(self):
        return (self.w_pool.cpu().numpy().reshape(self.w.shape),
                self.pos_pool.cpu().numpy().reshape(self.pos.shape))


def weigh(gpu, dev, c, s, q, out, positions, lens=None, workspace=None):
    gpu.attention_decode_weigh_paged(
        torch.from_numpy(q).to(dev), c.k_pool, c.v_pool, s.w_pool, s.pos_pool, out, c.d_tables,
        torch.from_numpy(positions.astype(np.int32)).to(dev),
        torch.tensor(c.lens if lens is None else lens, dtype=torch.int32, device=dev), c.batch,
        q.shape[1], c.n_kv, c.hd, c.stride, c.layers, c.layer, c.kv_dim, c.stride * PAGE,
        workspace=workspace)


LENS = [1, 0, 15, 16, 17, 33, 64, 257, 300, 31]


@pytest.mark.parametrize("n_head,n_kv,hd", [(12, 3, 64), (12, 12, 64), (16, 4, 128), (8, 1, 96),
                                            (4, 2, 32), (6, 3, 80), (40, 1, 64), (160, 2, 8),
                                            (4, 1, 160), (4, 2, 192), (2, 1, 224), (3, 1, 256)])
@pytest.mark.parametrize("qt,ot", [(F32, F32), (F16, F16)])
def test_weighing_decode_matches_f64(gpu, dev, n_head, n_kv, hd, qt, ot):
    c = Cache(dev, 31, LENS, n_kv, hd)
    s = Sums(dev, c, 32)
    q = queries(np.random.default_rng(33), c.batch, n_head, hd, qt)
    out = torch.full((c.batch, n_head, hd), -7.0, dtype=ot, device=dev)
    positions = 1000 + np.arange(c.batch)
    weigh(gpu, dev, c, s, q, out, positions)
    got = out.cpu().numpy().astype(np.float64)
    want_w, want_pos = s.w.astype(np.float64), s.pos.copy()
    for b, n in enumerate(LENS):
        if n == 0:
            assert (got[b] == -7.0).all()
            continue
        o, p = attention(q[b:b + 1].astype(np.float64), c.k[b], c.v[b], [n - 1], CAUSAL)
        element_gate(got[b:b + 1], o, f"request {b}", out_f16=ot == F16)
        p = p[:, 0].reshape(n_kv, n_head // n_kv, n).sum(1)
        for j in range(n):
            at = (c.tables[b, j // PAGE], c.layer, slice(None), j % PAGE)
            want_w[at] = p[:, j] + (want_w[at] if j < n - 1 else 0.0)
        want_pos[at] = positions[b]
    w, pos = s.read()
    element_gate(w, want_w, "sums")
    assert np.array_equal(pos, want_pos)


@pytest.mark.parametrize("hd", [64, 128])
def test_long_caches_split(gpu, dev, hd):
    lens = [5000, 1, 2049, 777]
    c = Cache(dev, 34, lens, 2, hd)
    s = Sums(dev, c, 35)
    q = queries(np.random.default_rng(36), 4, 6, hd, F32)
    out = torch.zeros((4, 6, hd), dtype=F32, device=dev)
    weigh(gpu, dev, c, s, q, out, np.array(lens) - 1)
    w, _ = s.read()
    for b, n in enumerate(lens):
        o, p = attention(q[b:b + 1].astype(np.float64), c.k[b], c.v[b], [n - 1], CAUSAL)
        element_gate(out[b:b + 1].cpu().numpy(), o)
        p = p[:, 0].reshape(2, 3, n).sum(1)
        j = np.arange(n)
        page, slot = c.tables[b, j // PAGE], j % PAGE
        old = s.w[page, c.layer, :, slot].astype(np.float64)
        old[-1] = 0.0
        element_gate(w[page, c.layer, :, slot], old + p.T, f"sums {b}")


def test_infinities_are_as_in_f32_sums(gpu, dev):
    """A key whose score is -inf weighs nothing, an infinite value leaves the sums alone and is
    infinite in its output."""
    n, hd = 50, 64
    c = Cache(dev, 37, [n], 1, hd)
    k = c.k_pool.view(c.n_pages, c.layers, PAGE, hd)
    q = np.ones((1, 2, hd), np.float32)
    k[c.tables[0, 1], c.layer, 4, 7] = -float("inf")   # token 20
    c.v_pool.view(c.n_pages, c.layers, hd, PAGE)[c.tables[0, 2], c.layer, 5, 3] = float("inf")
    s = Sums(dev, c, 38, lambda shape: np.zeros(shape, np.float32))
    out = torch.zeros((1, 2, hd), dtype=F32, device=dev)
    weigh(gpu, dev, c, s, q, out, np.array([n - 1]))
    o, p = attention(q.astype(np.float64), c.k[0], c.v[0], [n - 1], lambda p, j: j != 20)
    got = out.cpu().numpy().astype(np.float64)
    assert np.isposinf(got[:, :, 5]).all()
    got[:, :, 5] = o[:, :, 5]
    element_gate(got, o)
    w, _ = s.read()
    j = np.arange(n)
    element_gate(w[c.tables[0, j // PAGE], c.layer, 0, j % PAGE], p[:, 0].sum(0))


def observe(gpu, dev, c, s, q, starts, lens, packed, positions, n_observe):
    seg = np.stack([packed, lens, starts, np.arange(len(lens))], 1).astype(np.int32)
    gpu.cache_weigh_tiled(
        torch.from_numpy(q).to(dev), c.k_pool, s.w_pool, s.pos_pool, c.d_tables,
        torch.from_numpy(seg).to(dev), torch.from_numpy(positions).to(dev), len(lens),
        int(max(lens)), c.stride, q.shape[1], c.n_kv, c.hd, c.layers, c.layer, c.kv_dim,
        n_observe)


@pytest.mark.parametrize("starts,lens", [([0], [1]), ([0, 0, 0], [17, 1, 16]),
                                         ([63, 0, 255, 5], [17, 64, 129, 3]),
                                         ([1500, 900, 17], [5, 2, 7]), ([0, 40], [300, 33])])
@pytest.mark.parametrize("n_head,n_kv,hd", [(12, 3, 64), (4, 4, 64), (16, 4, 128), (8, 1, 96),
                                            (4, 2, 32), (6, 3, 80), (5, 1, 256), (36, 1, 160)])
@pytest.mark.parametrize("n_observe", [0, 1, 7, 64, 1000])
def test_prompt_sums_match_f64(gpu, dev, starts, lens, n_head, n_kv, hd, n_observe):
    ends = [a + n for a, n in zip(starts, lens)]
    for qt in (F32, F16):
        c = Cache(dev, 41, ends, n_kv, hd)
        s = Sums(dev, c, 42)
        packed = 2 + np.concatenate([[0], np.cumsum(lens)[:-1]])
        rows = 2 + sum(lens)
        q = queries(np.random.default_rng(43), rows, n_head, hd, qt)
        positions = (7 * np.arange(rows)).astype(np.int32)
        observe(gpu, dev, c, s, q, starts, lens, packed, positions, n_observe)
        want_w, want_pos = s.w.astype(np.float64), s.pos.copy()
        for b, (a, n) in enumerate(zip(starts, lens)):
            o = min(n_observe, n)
            at = np.arange(packed[b] + n - o, packed[b] + n)
            _, p = attention(q[at].astype(np.float64), c.k[b], c.v[b], range(a + n - o, a + n),
                             CAUSAL)
            p = p.sum(1).reshape(n_kv, n_head // n_kv, a + n).sum(1)
            j = np.arange(a + n)
            page, slot = c.tables[b, j // PAGE], j % PAGE
            old = want_w[page, c.layer, :, slot]
            old[a:] = 0.0
            want_w[page, c.layer, :, slot] = old + p.T
            want_pos[page[a:], c.layer, :, slot[a:]] = positions[packed[b]:packed[b] + n, None]
        w, pos = s.read()
        element_gate(w, want_w, "sums")
        assert np.array_equal(pos, want_pos)


def plain_evict(c, w, pos, k, v, lens, keep, n_sink, n_recent):
    """The cut on host copies, in place; returns the new lengths."""
    old = [x.copy() for x in (w, pos, k, v)]
    for b, n in enumerate(lens):
        if n <= keep or n > c.stride * PAGE:
            continue
        j = np.arange(n)
        page, slot = c.tables[b, j // PAGE], j % PAGE
        for layer in range(c.layers):
            for g in range(c.n_kv):
                wj = old[0][page, layer, g, slot].astype(np.float64)
                pj = old[1][page, layer, g, slot]
                wj = np.where(np.isnan(wj), -np.inf, wj)
                rank = np.where((pj < n_sink) | (pj > pj.max() - n_recent), np.inf, wj)
                order = sorted(range(n), key=lambda i: (-rank[i], i))
                kept = np.zeros(n, bool)
                kept[order[:keep]] = True
                to, src = np.nonzero(~kept[:keep])[0], keep + np.nonzero(kept[keep:])[0]
                assert len(to) == len(src)
                ch = slice(g * c.hd, (g + 1) * c.hd)
                for x, y in zip(to, src):
                    a, z = (page[x], layer, g, slot[x]), (page[y], layer, g, slot[y])
                    w[a], pos[a] = old[0][z], old[1][z]
                    k[page[x], layer, slot[x], ch] = old[2][page[y], layer, slot[y], ch]
                    v[page[x], layer, ch, slot[x]] = old[3][page[y], layer, ch, slot[y]]
    return [keep if keep < n <= c.stride * PAGE else n for n in lens]


def evict_and_compare(gpu, dev, lens, n_kv, hd, keep, n_sink, n_recent, values=None, seed=51,
                      layers=3, in_place=True, order=None):
    c = Cache(dev, seed, lens, n_kv, hd, layers=layers, layer=0)
    rng = np.random.default_rng(seed)
    k = rng.integers(0, 2 ** 16, size=c.host_k.shape, dtype=np.uint16)  # any bits, NaN too
    v = rng.integers(0, 2 ** 16, size=c.host_v.shape, dtype=np.uint16)
    k_pool = torch.from_numpy(k.reshape(-1).view(np.float16)).to(dev)
    v_pool = torch.from_numpy(v.reshape(-1).view(np.float16)).to(dev)
    s = Sums(dev, c, seed + 1, values)
    for b, n in enumerate(lens):  # positions as a cache holds them, or shuffled by an earlier cut
        for layer in range(layers):
            for g in range(n_kv):
                p = np.arange(n) + 3 * b if order is None else rng.permutation(n)
                s.pos[c.tables[b, np.arange(n) // PAGE], layer, g, np.arange(n) % PAGE] = p
    s.pos_pool.copy_(torch.from_numpy(s.pos.reshape(-1)))
    d_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    new = d_lens if in_place else torch.full_like(d_lens, -9)
    gpu.cache_evict_paged(k_pool, v_pool, s.w_pool, s.pos_pool, c.d_tables, d_lens, new, c.batch,
                          n_kv, hd, c.stride, layers, c.kv_dim, c.stride * PAGE, keep, n_sink,
                          n_recent)
    w, pos = s.w.copy(), s.pos.copy()
    want = plain_evict(c, w, pos, k, v, lens, keep, n_sink, n_recent)
    assert new.cpu().tolist() == want
    got_w, got_pos = s.read()
    assert np.array_equal(got_w.view(np.uint32), w.view(np.uint32))
    assert np.array_equal(got_pos, pos)
    assert np.array_equal(k_pool.cpu().numpy().view(np.uint16).reshape(k.shape), k)
    assert np.array_equal(v_pool.cpu().numpy().view(np.uint16).reshape(v.shape), v)


@pytest.mark.parametrize("keep,n_sink,n_recent", [(40, 4, 16), (1, 0, 0), (1, 1, 0), (16, 0, 16),
                                                  (33, 33, 0), (64, 0, 0), (299, 4, 100),
                                                  (1000, 4, 16)])
@pytest.mark.parametrize("n_kv,hd", [(3, 64), (1, 128), (2, 8), (4, 80)])
def test_cut_matches_plain(gpu, dev, keep, n_sink, n_recent, n_kv, hd):
    evict_and_compare(gpu, dev, [0, 1, 17, 40, 41, 64, 65, 300], n_kv, hd, keep, n_sink, n_recent)


@pytest.mark.parametrize("kind", ["equal", "few", "nan", "negative", "zeros"])
def test_equal_and_odd_sums(gpu, dev, kind):
    """Equal sums go by slot, -0 equals 0, NaN ranks last, negative sums in order."""
    def values(shape):
        rng = np.random.default_rng(52)
        x = rng.standard_normal(shape).astype(np.float32)
        if kind == "equal":
            return np.ones(shape, np.float32)
        if kind == "few":
            return rng.integers(0, 3, size=shape).astype(np.float32)
        if kind == "nan":
            return np.where(rng.random(shape) < 0.7, np.float32(np.nan), np.abs(x))
        if kind == "zeros":
            return np.where(rng.random(shape) < 0.5, np.float32(0.0), np.float32(-0.0))
        return x
    evict_and_compare(gpu, dev, [300, 129, 90], 2, 32, 70, 3, 20, values)


def test_a_cache_that_was_cut_before(gpu, dev):
    evict_and_compare(gpu, dev, [200, 100], 2, 64, 60, 5, 30, order="shuffled", in_place=False)


@pytest.mark.parametrize("n", [13000, 20011])
def test_long_caches_are_cut(gpu, dev, n):
    """Past the tokens whose keys fit in LDS, too."""
    evict_and_compare(gpu, dev, [n, 2000], 1, 8, 1500, 4, 256, layers=1)


def test_cut_is_captured_and_repeats(gpu, dev):
    """A step of a serving loop as a graph: weigh, then cut, with the lengths on the device."""
    lens, keep = [70, 64, 33], 64
    c = Cache(dev, 61, [80, 80, 80], 2, 64)
    k0, v0 = torch.nan_to_num(c.k_pool), torch.nan_to_num(c.v_pool)
    s = Sums(dev, c, 62)
    q = torch.from_numpy(queries(np.random.default_rng(63), 3, 4, 64, F32)).to(dev)
    start = torch.tensor(lens, dtype=torch.int32, device=dev)
    state = {"k": k0.clone(), "v": v0.clone(), "w": s.w_pool.clone(), "pos": s.pos_pool.clone(),
             "lens": start.clone(), "out": torch.zeros((3, 4, 64), device=dev)}

    def step():
        for layer in range(c.layers):
            gpu.attention_decode_weigh_paged(q, state["k"], state["v"], state["w"], state["pos"],
                                             state["out"], c.d_tables, state["lens"],
                                             state["lens"], 3, 4, 2, 64, c.stride, c.layers,
                                             layer, c.kv_dim, c.stride * PAGE)
        gpu.cache_evict_paged(state["k"], state["v"], state["w"], state["pos"], c.d_tables,
                              state["lens"], state["lens"], 3, 2, 64, c.stride, c.layers,
                              c.kv_dim, c.stride * PAGE, keep, 4, 16)
        state["lens"].add_(3)

    def reset():
        for x, y in (("k", k0), ("v", v0), ("w", s.w_pool), ("pos", s.pos_pool), ("lens", start)):
            state[x].copy_(y)

    eager = []
    for _ in range(4):
        step()
        eager.append({x: y.clone() for x, y in state.items()})
    reset()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for want in eager:
        g.replay()
        torch.cuda.synchronize()
        for x, y in want.items():
            assert torch.equal(state[x], y), x
        torch.zeros(1000, device=dev).sum().item()


@pytest.mark.parametrize("n", [255, 256, 257, 511, 513, 769, 1025, 1281, 1537, 2049, 4097, 8191,
                               12289, 16383])
@pytest.mark.parametrize("over", [5, 1000])
def test_cuts_at_the_sizes_where_the_selection_changes(gpu, dev, n, over):
    """Few moves, made by the selecting workgroup, and many, at the edges of its sizes."""
    keep = max(1, n - over)
    sink = min(2, keep)
    evict_and_compare(gpu, dev, [n, n - 1, 3], 1, 8, keep, sink, min(20, keep - sink), layers=1,
                      seed=n)


@pytest.mark.parametrize("n", [24577, 33000])
def test_cuts_past_what_registers_hold(gpu, dev, n):
    """The largest selection in registers, and the one that forms its keys again; with equal
    sums, too."""
    evict_and_compare(gpu, dev, [n], 1, 8, n - 400, 2, 20, layers=1, in_place=False)
    evict_and_compare(gpu, dev, [n], 1, 8, 300, 2, 20, layers=1,
                      values=lambda s: np.random.default_rng(1).integers(0, 3, size=s).astype(np.float32))


@pytest.mark.parametrize("n_head,n_kv,hd", [(70, 1, 64), (160, 2, 8), (48, 3, 96)])
def test_groups_of_many_heads(gpu, dev, n_head, n_kv, hd):
    """More query heads a KV head than a tile of 16 (and, windowed, of 64) columns holds."""
    from span_cases import window_sees
    lens = [1, 0, 300, 33]
    c = Cache(dev, 55, lens, n_kv, hd)
    q = queries(np.random.default_rng(56), 4, n_head, hd, F32)
    s = Sums(dev, c, 57)
    out, win = (torch.zeros((4, n_head, hd), device=dev) for _ in range(2))
    weigh(gpu, dev, c, s, q, out, np.arange(4))
    gpu.attention_decode_window_paged(
        torch.from_numpy(q).to(dev), c.k_pool, c.v_pool, win, c.d_tables,
        torch.tensor(lens, dtype=torch.int32, device=dev), 4, n_head, n_kv, hd, c.stride, c.layers,
        c.layer, c.kv_dim, c.stride * PAGE, 40, 3)
    w, _ = s.read()
    for b, n in enumerate(lens):
        if n == 0:
            continue
        o, p = attention(q[b:b + 1].astype(np.float64), c.k[b], c.v[b], [n - 1], CAUSAL)
        element_gate(out[b:b + 1].cpu().numpy(), o)
        j = np.arange(n)
        page, slot = c.tables[b, j // PAGE], j % PAGE
        old = s.w[page, c.layer, :, slot].astype(np.float64)
        old[-1] = 0.0
        element_gate(w[page, c.layer, :, slot], old + p[:, 0].reshape(n_kv, -1, n).sum(1).T)
        o, _ = attention(q[b:b + 1].astype(np.float64), c.k[b], c.v[b], [n - 1], window_sees(40, 3))
        element_gate(win[b:b + 1].cpu().numpy(), o)


def test_weighing_and_prompt_sums_are_captured(gpu, dev):
    """Replays, with other lengths each and eager work between them, give the eager bits; sums
    go on from where the last replay left them."""
    lens = [900, 17, 350, 1]
    c = Cache(dev, 61, lens, 3, 64)
    a, b = Sums(dev, c, 62), Sums(dev, c, 62)
    q = torch.from_numpy(queries(np.random.default_rng(63), 4, 12, 64, F32)).to(dev)
    rows = torch.from_numpy(queries(np.random.default_rng(64), 200, 12, 64, F32)).to(dev)
    d_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    at = torch.arange(200, dtype=torch.int32, device=dev)
    segments = torch.tensor([[0, 150, 700, 0], [150, 17, 0, 1]], dtype=torch.int32, device=dev)
    shape = (12, 3, 64)

    def run(s, out):
        gpu.attention_decode_weigh_paged(q, c.k_pool, c.v_pool, s.w_pool, s.pos_pool, out,
                                         c.d_tables, at, d_lens, 4, *shape, c.stride, c.layers,
                                         c.layer, c.kv_dim, c.stride * PAGE)
        gpu.cache_weigh_tiled(rows, c.k_pool, s.w_pool, s.pos_pool, c.d_tables, segments, at, 2,
                              150, c.stride, *shape, c.layers, c.layer, c.kv_dim, 70)

    outs = [torch.zeros((4, 12, 64), dtype=F32, device=dev) for _ in range(2)]
    run(a, outs[0])  # loads the kernels
    run(b, outs[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(a, outs[0])
    for step in range(3):
        d_lens[0] = 900 - 400 * step
        segments[0, 1] = 150 - 60 * step
        graph.replay()
        run(b, outs[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        assert np.array_equal(a.read()[0].view(np.uint32), b.read()[0].view(np.uint32))
        assert np.array_equal(a.read()[1], b.read()[1])


def test_two_streams_weigh_at_once(gpu, dev):
    """Calls on two streams, each with scratch of its own, on pools of their own."""
    c = Cache(dev, 65, [3000, 41, 800], 3, 64)
    q = torch.from_numpy(queries(np.random.default_rng(66), 3, 12, 64, F32)).to(dev)
    at = torch.arange(3, dtype=torch.int32, device=dev)
    d_lens = torch.tensor(c.lens, dtype=torch.int32, device=dev)
    sums = [Sums(dev, c, 67) for _ in range(3)]
    outs = [torch.zeros((3, 12, 64), dtype=F32, device=dev) for _ in range(3)]

    def run(i):
        for _ in range(6):
            gpu.attention_decode_weigh_paged(q, c.k_pool, c.v_pool, sums[i].w_pool,
                                             sums[i].pos_pool, outs[i], c.d_tables, at, d_lens, 3,
                                             12, 3, 64, c.stride, c.layers, c.layer, c.kv_dim,
                                             c.stride * PAGE)

    run(0)
    torch.cuda.synchronize()
    for i in (1, 2):
        with torch.cuda.stream(torch.cuda.Stream()):
            run(i)
    torch.cuda.synchronize()
    for i in (1, 2):
        assert torch.equal(outs[0], outs[i])
        assert np.array_equal(sums[0].read()[0].view(np.uint32), sums[i].read()[0].view(np.uint32))

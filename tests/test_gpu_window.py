"""Windowed attention with first tokens that stay visible, against 64-bit attention.

f32 outputs meet the reference validator's element gate (2e-5 + 2e-5 |ref|, tests/gates.py): with
values of order 1, f32 sums and fp16 hi + lo operands (22 bits) are off by 1e-6. fp16 outputs add
their rounding, 2^-11 |ref|.
"""
import numpy as np
import pytest
import torch

from gates import element_gate
from span_cases import PAGE, Cache, attention, queries, window_sees

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def decode(gpu, dev, c, q, out, window, n_sink, max_seq=None, workspace=None):
    gpu.attention_decode_window_paged(
        torch.from_numpy(q).to(dev), c.k_pool, c.v_pool, out, c.d_tables,
        torch.tensor(c.lens, dtype=torch.int32, device=dev), c.batch, q.shape[1], c.n_kv, c.hd,
        c.stride, c.layers, c.layer, c.kv_dim, max_seq or c.stride * PAGE, window, n_sink,
        workspace=workspace)


def held_pages(lens, window, n_sink, chunk=None):
    """Which pages a windowed cache keeps: those that any row sees."""
    def keep(b, i):
        first = lens[b] - (1 if chunk is None else chunk[b])
        return i * PAGE < n_sink or (i + 1) * PAGE > first - window + 1
    return keep


LENS = [1, 0, 15, 16, 17, 33, 64, 100, 257, 300, 31]


@pytest.mark.parametrize("n_head,n_kv,hd", [(12, 3, 64), (12, 12, 64), (16, 4, 128), (8, 1, 96),
                                            (4, 2, 32), (6, 3, 80), (20, 1, 64), (4, 1, 160),
                                            (4, 2, 192), (2, 1, 224), (3, 1, 256), (2, 2, 8)])
@pytest.mark.parametrize("window,n_sink", [(20, 4), (1, 0), (64, 33), (1000, 0), (0, 3)])
def test_decode_matches_f64(gpu, dev, n_head, n_kv, hd, window, n_sink):
    for qt, ot in ((F32, F32), (F16, F16)):
        c = Cache(dev, 3, LENS, n_kv, hd, keep_pages=held_pages(LENS, window, n_sink))
        q = queries(np.random.default_rng(5), c.batch, n_head, hd, qt)
        out = torch.full((c.batch, n_head, hd), -7.0, dtype=ot, device=dev)
        decode(gpu, dev, c, q, out, window, n_sink)
        got = out.cpu().numpy().astype(np.float64)
        for b, n in enumerate(LENS):
            if n == 0:
                assert (got[b] == -7.0).all()
                continue
            want, _ = attention(q[b:b + 1].astype(np.float64), c.k[b], c.v[b], [n - 1],
                                window_sees(window, n_sink))
            element_gate(got[b:b + 1], want, f"request {b}", out_f16=ot == F16)


@pytest.mark.parametrize("window,n_sink", [(700, 5), (5000, 0), (2048, 300), (16, 2000)])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_decode_splits_and_joins(gpu, dev, window, n_sink, hd):
    lens = [4100, 1, 2049, 700, 2999]
    c = Cache(dev, 4, lens, 3, hd, keep_pages=held_pages(lens, window, n_sink))
    q = queries(np.random.default_rng(6), c.batch, 12, hd, F32)
    out = torch.zeros((c.batch, 12, hd), dtype=F32, device=dev)
    decode(gpu, dev, c, q, out, window, n_sink)
    got = out.cpu().numpy()
    for b, n in enumerate(lens):
        want, _ = attention(q[b:b + 1].astype(np.float64), c.k[b], c.v[b], [n - 1],
                            window_sees(window, n_sink))
        element_gate(got[b:b + 1], want, f"request {b}")


def prefill(gpu, dev, c, q, out, starts, lens, window, n_sink, packed, tables=None):
    seg = np.stack([packed, lens, starts, np.arange(len(lens)) if tables is None else tables], 1)
    gpu.attention_prefill_window_tiled(
        torch.from_numpy(q).to(dev), c.k_pool, c.v_pool, out, c.d_tables,
        torch.from_numpy(np.ascontiguousarray(seg, dtype=np.int32)).to(dev), len(lens),
        int(max(lens)), c.stride, q.shape[1], c.n_kv, c.hd, c.layers, c.layer, c.kv_dim, window,
        n_sink)


CHUNKS = [  # starts, lens
    ([0], [1]), ([0, 0, 0], [17, 1, 16]), ([63, 0, 255, 5], [17, 64, 129, 3]),
    ([1500, 900, 17], [5, 2, 7]), ([0, 40], [300, 33])]


@pytest.mark.parametrize("starts,lens", CHUNKS)
@pytest.mark.parametrize("n_head,n_kv,hd", [(12, 3, 64), (4, 4, 64), (16, 4, 128), (8, 1, 96),
                                            (4, 2, 32), (6, 3, 80), (5, 1, 256)])
@pytest.mark.parametrize("window,n_sink", [(20, 4), (1, 0), (128, 37), (4096, 0), (0, 0), (0, 2)])
def test_chunks_match_f64(gpu, dev, starts, lens, n_head, n_kv, hd, window, n_sink):
    ends = [a + n for a, n in zip(starts, lens)]
    for qt, ot in ((F32, F32), (F16, F16)):
        c = Cache(dev, 7, ends, n_kv, hd, keep_pages=held_pages(ends, window, n_sink, lens))
        packed = 3 + np.concatenate([[0], np.cumsum(lens)[:-1]])  # rows that no segment names
        rows = 3 + sum(lens) + 2
        q = queries(np.random.default_rng(8), rows, n_head, hd, qt)
        out = torch.full((rows, n_head, hd), -7.0, dtype=ot, device=dev)
        prefill(gpu, dev, c, q, out, starts, lens, window, n_sink, packed)
        got = out.cpu().numpy().astype(np.float64)
        assert (got[:3] == -7.0).all() and (got[-2:] == -7.0).all()
        for b, (a, n) in enumerate(zip(starts, lens)):
            at = slice(packed[b], packed[b] + n)
            want, _ = attention(q[at].astype(np.float64), c.k[b], c.v[b], range(a, a + n),
                                window_sees(window, n_sink))
            element_gate(got[at], want, f"segment {b}", out_f16=ot == F16)
            if window == 0 and n_sink == 0:
                assert (got[at] == 0).all()


@pytest.mark.parametrize("window,n_sink", [(257, 4), (100000, 0)])
def test_long_chunk_behind_a_long_history(gpu, dev, window, n_sink):
    starts, lens = [3000, 1, 2047], [200, 1000, 33]
    ends = [a + n for a, n in zip(starts, lens)]
    c = Cache(dev, 9, ends, 2, 64, keep_pages=held_pages(ends, window, n_sink, lens))
    packed = np.concatenate([[0], np.cumsum(lens)[:-1]])
    q = queries(np.random.default_rng(10), sum(lens), 4, 64, F32)
    out = torch.zeros((sum(lens), 4, 64), dtype=F32, device=dev)
    prefill(gpu, dev, c, q, out, starts, lens, window, n_sink, packed)
    got = out.cpu().numpy()
    for b, (a, n) in enumerate(zip(starts, lens)):
        at = slice(packed[b], packed[b] + n)
        want, _ = attention(q[at].astype(np.float64), c.k[b], c.v[b], range(a, a + n),
                            window_sees(window, n_sink))
        element_gate(got[at], want, f"segment {b}")


@pytest.mark.parametrize("hd", [64, 128, 80])
def test_infinite_values_reach_only_the_rows_that_see_them(gpu, dev, hd):
    """An infinity in V of one token: rows that see it are infinite in that dimension, and rows
    of the same tile that do not are as if it were anything else."""
    n, window, n_sink, at = 40, 8, 2, 20
    c = Cache(dev, 11, [n], 1, hd)
    page = c.tables[0, at // PAGE]
    v = c.v_pool.view(c.n_pages, c.layers, c.kv_dim, PAGE)
    v[page, c.layer, 3, at % PAGE] = float("inf")
    q = queries(np.random.default_rng(12), n, 4, hd, F32)
    out = torch.zeros((n, 4, hd), dtype=F32, device=dev)
    prefill(gpu, dev, c, q, out, [0], [n], window, n_sink, [0])
    got = out.cpu().numpy().astype(np.float64)
    sees = window_sees(window, n_sink)
    want, _ = attention(q.astype(np.float64), c.k[0], c.v[0], range(n), sees)
    hit = np.array([sees(p, at) for p in range(n)])
    assert hit.sum() == window and np.isposinf(got[hit][:, :, 3]).all()
    got[hit, :, 3] = want[hit, :, 3]
    element_gate(got, want, "finite outputs")


def test_infinite_keys_and_queries_of_large_range(gpu, dev):
    """Queries of very different sizes keep their 22 bits; a NaN key makes the rows that see it
    NaN and no others."""
    n, hd = 50, 64
    c = Cache(dev, 13, [n], 1, hd)
    q = queries(np.random.default_rng(14), n, 2, hd, F32)
    q *= (10.0 ** np.random.default_rng(15).integers(-30, 1, size=(n, 2, 1))).astype(np.float32)
    c.k_pool.view(c.n_pages, c.layers, PAGE, c.kv_dim)[c.tables[0, 1], c.layer, 3, 5] = float("nan")
    out = torch.zeros((n, 2, hd), dtype=F32, device=dev)
    prefill(gpu, dev, c, q, out, [0], [n], 6, 1, [0])
    got = out.cpu().numpy().astype(np.float64)
    sees = window_sees(6, 1)
    hit = np.array([sees(p, 19) for p in range(n)])
    assert np.isnan(got[hit]).all()
    want, _ = attention(q.astype(np.float64), c.k[0], c.v[0], range(n), sees)
    element_gate(got[~hit], want[~hit], "rows that do not see it")


def test_unaligned_buffers_take_the_plain_rows(gpu, dev):
    lens = [70, 5]
    c = Cache(dev, 16, lens, 2, 64)
    q = queries(np.random.default_rng(17), 2, 4, 64, F32)
    room = torch.zeros(2 * 4 * 64 + 1, dtype=F32, device=dev)
    out = room[1:].view(2, 4, 64)
    decode(gpu, dev, c, q, out, 30, 4)
    for b, n in enumerate(lens):
        want, _ = attention(q[b:b + 1].astype(np.float64), c.k[b], c.v[b], [n - 1],
                            window_sees(30, 4))
        element_gate(out[b:b + 1].cpu().numpy(), want)


def test_a_window_past_every_length_is_causal_attention(gpu, dev):
    lens = [777, 16, 1]
    c = Cache(dev, 18, lens, 3, 64)
    q = queries(np.random.default_rng(19), 3, 12, 64, F32)
    a, b = (torch.zeros((3, 12, 64), dtype=F32, device=dev) for _ in range(2))
    decode(gpu, dev, c, q, a, 2 ** 31 - 1, 0)
    gpu.attention_decode_paged(torch.from_numpy(q).to(dev), c.k_pool, c.v_pool, b, c.d_tables,
                               torch.tensor(lens, dtype=torch.int32, device=dev), 3, 12, 3, 64,
                               c.stride, c.layers, c.layer, c.kv_dim, c.stride * PAGE)
    element_gate(a.cpu().numpy(), b.cpu().numpy())


def test_calls_are_the_same_bits_and_capture(gpu, dev):
    """Two streams at once, a caller's workspace, and replays of a graph give the eager bits."""
    lens = [4000, 2500, 16, 3001]
    c = Cache(dev, 20, lens, 3, 64)
    q = queries(np.random.default_rng(21), 4, 12, 64, F32)
    d_q, d_lens = torch.from_numpy(q).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)

    def call(out, ws=None):
        gpu.attention_decode_window_paged(d_q, c.k_pool, c.v_pool, out, c.d_tables, d_lens, 4, 12,
                                          3, 64, c.stride, c.layers, c.layer, c.kv_dim,
                                          c.stride * PAGE, 3500, 4, workspace=ws)

    outs = [torch.zeros((4, 12, 64), dtype=F32, device=dev) for _ in range(4)]
    call(outs[0])
    need = gpu.lib.crucible_attention_decode_window_workspace_bytes(4, 12, 3, 64, c.stride * PAGE,
                                                                    3500, 4)
    assert need > 0
    call(outs[1], torch.full((need,), 0xff, dtype=torch.uint8, device=dev))
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    for s, o in zip(sides, outs[2:]):
        with torch.cuda.stream(s):
            for _ in range(5):
                call(o)
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert torch.equal(outs[0], o)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(outs[3])
    for step in range(3):
        outs[3].zero_()
        d_lens[0] = lens[0] - 700 * step
        g.replay()
        call(outs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[2], outs[3])


@pytest.mark.parametrize("n_head,n_kv,hd", [(12, 3, 64), (4, 4, 128), (10, 2, 96), (8, 1, 32),
                                            (6, 3, 80), (4, 4, 24)])
@pytest.mark.parametrize("window,n_sink", [(100, 4), (1, 0), (3000, 0), (0, 5), (0, 0), (33, 130)])
def test_many_rows_in_wide_tiles(gpu, dev, n_head, n_kv, hd, window, n_sink):
    """Chunks enough for the kernel that stages keys for 128 columns, ragged, behind histories."""
    rng = np.random.default_rng(22)
    starts = [0, 0, 7, 300, 64, 0, 1, 1000] + [3] * 72
    lens = [129, 1, 64, 33, 200, 16, 2, 70] + rng.integers(1, 120, size=72).tolist()
    ends = [a + n for a, n in zip(starts, lens)]
    assert len(lens) * n_kv * -(-max(lens) * (n_head // n_kv) // 128) >= 256
    for qt, ot in ((F32, F32), (F16, F16)):
        c = Cache(dev, 23, ends, n_kv, hd, keep_pages=held_pages(ends, window, n_sink, lens))
        packed = np.concatenate([[0], np.cumsum(lens)[:-1]])
        q = queries(rng, sum(lens), n_head, hd, qt)
        out = torch.full((sum(lens) + 1, n_head, hd), -7.0, dtype=ot, device=dev)
        prefill(gpu, dev, c, q, out, starts, lens, window, n_sink, packed)
        got = out.cpu().numpy().astype(np.float64)
        assert (got[-1] == -7.0).all()
        for b in [0, 1, 2, 3, 4, 5, 6, 7, 30, 79]:
            a, n = starts[b], lens[b]
            at = slice(packed[b], packed[b] + n)
            want, _ = attention(q[at].astype(np.float64), c.k[b], c.v[b], range(a, a + n),
                                window_sees(window, n_sink))
            element_gate(got[at], want, f"segment {b}", out_f16=ot == F16)


def test_wide_tiles_infinities_and_growing_scores(gpu, dev):
    """An infinite value and a NaN key inside other rows' windows, and scores that grow by more
    than the maximum may lag behind, to hundreds of powers of two."""
    n, hd, window, n_sink = 800, 64, 50, 3
    starts, lens = [0] * 16, [n] * 16
    c = Cache(dev, 24, lens, 1, hd)
    q = queries(np.random.default_rng(25), n * 16, 4, hd, F32)
    grow = np.linspace(0.0, 60.0, n)
    for b in range(16):  # along dimension 0, which the queries see as 8: up to 60 a score
        k = c.k_pool.view(c.n_pages, c.layers, PAGE, hd)
        j = np.arange(n)
        k[c.tables[b, j // PAGE], c.layer, j % PAGE, 0] = torch.from_numpy(grow).to(dev).half()
        c.k[b][:, 0, 0] = grow.astype(np.float16)
    q[:, :, 0] = 8.0
    v = c.v_pool.view(c.n_pages, c.layers, hd, PAGE)
    v[c.tables[2, 100 // PAGE], c.layer, 9, 100 % PAGE] = float("inf")
    c.k_pool.view(c.n_pages, c.layers, PAGE, hd)[c.tables[3, 200 // PAGE], c.layer, 200 % PAGE, 7] = float("nan")
    out = torch.zeros((n * 16, 4, hd), dtype=F32, device=dev)
    packed = n * np.arange(16)
    prefill(gpu, dev, c, q, out, starts, lens, window, n_sink, packed)
    got = out.cpu().numpy().astype(np.float64).reshape(16, n, 4, hd)
    sees = window_sees(window, n_sink)
    for b in (0, 2, 3, 15):
        want, _ = attention(q[b * n:(b + 1) * n].astype(np.float64), c.k[b], c.v[b], range(n), sees)
        if b == 2:
            hit = np.array([sees(p, 100) for p in range(n)])
            assert hit.sum() == window and np.isposinf(got[2][hit][:, :, 9]).all()
            got[2][hit, :, 9] = want[hit, :, 9]
        if b == 3:
            hit = np.array([sees(p, 200) for p in range(n)])
            assert np.isnan(got[3][hit]).all()
            got[3][hit] = want[hit]
        element_gate(got[b], want, f"segment {b}")


def test_many_requests(gpu, dev):
    """2,000 requests of up to 40 tokens, inactive ones between them: one new token each, then
    chunks of one to three rows."""
    rng = np.random.default_rng(81)
    lens = rng.integers(3, 41, size=2000)
    c = Cache(dev, 82, lens, 1, 32)
    q = queries(rng, 2000, 2, 32, F32)
    live = np.arange(2000) % 7 != 3
    d_lens = torch.from_numpy(np.where(live, lens, 0).astype(np.int32)).to(dev)
    out = torch.full((2000, 2, 32), -7.0, dtype=F32, device=dev)
    gpu.attention_decode_window_paged(torch.from_numpy(q).to(dev), c.k_pool, c.v_pool, out,
                                      c.d_tables, d_lens, 2000, 2, 1, 32, c.stride, c.layers,
                                      c.layer, c.kv_dim, c.stride * PAGE, 9, 2)
    got = out.cpu().numpy().astype(np.float64)
    assert (got[~live] == -7.0).all()
    sees = window_sees(9, 2)
    want = np.stack([attention(q[b:b + 1].astype(np.float64), c.k[b], c.v[b], [n - 1], sees)[0][0]
                     for b, n in enumerate(lens)])
    element_gate(got[live], want[live])

    rows = rng.integers(1, 4, size=2000)
    packed = np.concatenate([[0], np.cumsum(rows)[:-1]])
    q = queries(rng, int(rows.sum()), 2, 32, F32)
    starts = lens - rows
    seg = np.stack([packed, np.where(live, rows, 0), starts, np.arange(2000)], 1).astype(np.int32)
    out = torch.full((int(rows.sum()), 2, 32), -7.0, dtype=F32, device=dev)
    gpu.attention_prefill_window_tiled(torch.from_numpy(q).to(dev), c.k_pool, c.v_pool, out,
                                       c.d_tables, torch.from_numpy(seg).to(dev), 2000, 3,
                                       c.stride, 2, 1, 32, c.layers, c.layer, c.kv_dim, 9, 2)
    got = out.cpu().numpy().astype(np.float64)
    for b in range(2000):
        at = slice(packed[b], packed[b] + rows[b])
        if not live[b]:
            assert (got[at] == -7.0).all()
            continue
        o, _ = attention(q[at].astype(np.float64), c.k[b], c.v[b], range(starts[b], lens[b]), sees)
        element_gate(got[at], o, f"request {b}")

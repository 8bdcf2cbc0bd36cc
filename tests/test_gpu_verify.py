"""Verification of drafted tokens against a plain implementation in 64 bits.

Tokens and counts are whole numbers and have to be equal. A draw's token changes where a random
number times the total lies within rounding of a running sum: f64 sums of 50,257 terms in another
order differ by some 1e-14 of the total, borders are 2e-5 apart on average, so one draw in 10^9
could: none of the few thousand here.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def plain(target, draft, drafts, n_draft, u_accept, u_sample, t):
    k = drafts.shape[1]
    tokens, accepted = np.full((len(drafts), k + 1), -1, np.int32), np.zeros(len(drafts), np.int32)

    def share(x):
        x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
        top = x.max()
        if top == -np.inf:
            return np.zeros(len(x))
        with np.errstate(invalid="ignore"):
            e = np.where(x == top, 1.0, np.exp((x - top) / t))
        return e / e.sum()

    for b in range(len(drafts)):
        last, n = min(n_draft[b], k), 0
        if last < 0:  # inactive
            continue
        while True:
            mass = share(target[b, n])
            if n == last:
                break
            d = drafts[b, n]
            inside = 0 <= d < len(mass)
            q = share(draft[b, n]) if draft is not None else np.eye(1, len(mass), d)[0] if inside else 0 * mass
            if not (inside and np.float64(u_accept[b, n]) * q[d] < mass[d]):
                left = np.maximum(mass - q, 0.0)
                mass = left if left.sum() > 0 else mass
                break
            tokens[b, n] = d
            n += 1
        # a token without mass is never drawn (also for numbers below 0)
        past = np.nonzero((np.cumsum(mass) > np.float64(u_sample[b]) * mass.sum()) & (mass > 0))[0]
        some = np.nonzero(mass)[0]
        tokens[b, n] = past[0] if len(past) else some[-1] if len(some) else 0
        accepted[b] = n
    return tokens, accepted


def check(gpu, dev, target, draft, drafts, n_draft, u_accept, u_sample, t, dtype=F32):
    batch, rows, vocab = target.shape
    tokens = torch.full((batch, rows), -5, dtype=torch.int32, device=dev)
    accepted = torch.full((batch,), -5, dtype=torch.int32, device=dev)
    to = lambda x, ty: torch.from_numpy(np.ascontiguousarray(x)).to(dev).to(ty)  # noqa: E731
    d_target = to(target, dtype)
    d_draft = None if draft is None else to(draft, dtype)
    gpu.verify_drafts(d_target, d_draft, to(drafts, torch.int32), to(n_draft, torch.int32),
                      to(u_accept, F32), to(u_sample, F32), tokens, accepted, batch, rows - 1,
                      vocab, t)
    got = tokens.cpu().numpy(), accepted.cpu().numpy()
    want = plain(d_target.cpu().float().numpy(), None if draft is None else d_draft.cpu().float().numpy(),
                 drafts, n_draft, u_accept.astype(np.float32), u_sample.astype(np.float32), t)
    live = n_draft >= 0
    assert np.array_equal(got[0][live], want[0][live])
    assert np.array_equal(got[1][live], want[1][live])
    assert (got[0][~live] == -5).all() and (got[1][~live] == -5).all()
    return got


def inputs(seed, batch, k, vocab, noise=0.7, scale=3.0):
    rng = np.random.default_rng(seed)
    target = rng.normal(0, scale, (batch, k + 1, vocab)).astype(np.float32)
    draft = (target[:, :k] + rng.normal(0, noise, (batch, k, vocab))).astype(np.float32)
    drafts = (draft + rng.gumbel(size=draft.shape)).argmax(-1).astype(np.int32).reshape(batch, k)
    return (target, draft, drafts, rng.integers(-1, k + 1, size=batch).astype(np.int32),
            rng.random((batch, k)).astype(np.float32), rng.random(batch).astype(np.float32))


@pytest.mark.parametrize("batch,k,vocab", [(1, 1, 2), (3, 4, 7), (40, 7, 100), (5, 3, 2047),
                                           (5, 3, 2048), (5, 3, 2049), (17, 5, 6000),
                                           (4, 4, 50257), (2, 64, 300), (6, 0, 999), (3, 2, 1)])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("t,dtype", [(1.0, F32), (0.3, F16), (1.7, F32)])
def test_matches_plain(gpu, dev, batch, k, vocab, with_draft, t, dtype):
    target, draft, drafts, n, ua, us = inputs(71, batch, k, vocab)
    check(gpu, dev, target, draft if with_draft else None, drafts, n, ua, us, t, dtype)


def test_counts_past_the_drafts_and_tokens_outside(gpu, dev):
    target, draft, drafts, n, ua, us = inputs(72, 12, 4, 50, noise=0.1)
    n[:] = [4, 9, 100, 4, 4, 4, -1, -100, 0, 1, 2, 3]
    drafts[3, 0], drafts[4, 2], drafts[5, 1] = -1, 50, 2 ** 31 - 1
    ua[:6] = 0.0  # taken wherever the target gives the draft anything
    got = check(gpu, dev, target, draft, drafts, n, ua, us, 1.0)
    assert got[1][:6].tolist() == [4, 4, 4, 0, 2, 1]
    check(gpu, dev, target, None, drafts, n, ua, us, 1.0)


def test_random_numbers_at_the_ends(gpu, dev):
    target, draft, drafts, n, ua, us = inputs(73, 8, 3, 500)
    us[:] = [0.0, 0.0, 1.0, 1.0, 1.0 - 2.0 ** -24, 2.0, -1.0, 0.5]
    ua[:] = np.array([0.0, 1.0, 0.5] * 8).reshape(8, 3)
    n[:] = 3
    check(gpu, dev, target, draft, drafts, n, ua, us, 1.0)


def test_the_same_draft_and_target(gpu, dev):
    """p = q: u < 1 takes every draft; u = 1 refuses with nothing left over, and p decides."""
    target, _, drafts, n, ua, us = inputs(74, 16, 3, 300)
    n[:] = 3
    ua[8:, 1] = 1.0
    got = check(gpu, dev, target, target[:, :3].copy(), drafts, n, ua, us, 1.0)
    assert (got[1][:8] == 3).all() and (got[1][8:] == 1).all()


def test_infinite_and_nan_logits(gpu, dev):
    inf = np.float32(np.inf)
    target, draft, drafts, n, ua, us = inputs(75, 10, 2, 40)
    n[:] = 2
    target[0, 0, :] = -inf            # no probability at all
    target[1, 0, 1:] = -inf           # one token
    target[2, 0, :20] = np.nan
    target[3, 0, [5, 30]] = inf       # share everything
    draft[4, 0, :] = -inf
    draft[5, 0, 7] = inf
    draft[6, 0, :] = np.nan
    target[7, 1, :] = np.nan
    target[8, 0, drafts[8, 0]] = -inf
    target[9, 2, :39] = -inf
    for t in (1.0, 0.25):
        check(gpu, dev, target, draft, drafts, n, ua, us, t)
        check(gpu, dev, target, None, drafts, n, ua, us, t)


def test_graph_replays_and_streams(gpu, dev):
    target, draft, drafts, n, ua, us = inputs(76, 6, 4, 5000)
    n[:] = 4
    d = [torch.from_numpy(x).to(dev) for x in (target, draft, drafts, n, ua, us)]
    outs = [(torch.zeros((6, 5), dtype=torch.int32, device=dev),
             torch.zeros(6, dtype=torch.int32, device=dev)) for _ in range(3)]

    def call(o):
        gpu.verify_drafts(*d, *o, 6, 4, 5000, 0.9)

    call(outs[0])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(outs[1])
    side = torch.cuda.Stream()
    for step in range(4):
        d[5].copy_(torch.rand(6, generator=torch.Generator().manual_seed(step)))
        d[4].mul_(0.7)
        g.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            call(outs[2])
        torch.cuda.synchronize()
        for x, y in zip(outs[1], outs[2]):
            assert torch.equal(x, y)
    want = plain(target, draft, drafts, n, d[4].cpu().numpy(), d[5].cpu().numpy(), 0.9)
    assert np.array_equal(outs[1][0].cpu().numpy(), want[0])


@pytest.mark.parametrize("vocab", [65537, 70001, 262145])
@pytest.mark.parametrize("with_draft", [True, False])
def test_many_chunks_of_columns(gpu, dev, vocab, with_draft):
    """More chunks than half a wave, or a wave, takes at once; borders in the last ones too."""
    target, draft, drafts, n, ua, us = inputs(78, 7, 2, vocab, noise=0.5)
    n[:] = [2, 1, 0, 2, 2, 0, 2]
    us[:] = [0.999999, 0.5, 0.97, 1.0, 0.0, 1.0, 0.75]
    ua[:4] = 1.0  # refused wherever the target likes the draft less
    target[5, 0, 1000:] = -np.inf
    check(gpu, dev, target, draft if with_draft else None, drafts, n, ua, us, 1.0)

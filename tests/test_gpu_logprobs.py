"""Log probabilities, ranks, entropies and alternatives on the GPU against 64 bits.

Bounds (u = 2^-24): a log probability is x - m - L.  L = log1p(rest): an exponential is off by 4 u and by u times its
argument, which its own size outweighs (e^-d d <= 0.4), a sum of n by u for each of at most n / 256 + 32 steps; the two
subtractions and the logarithm round once each.  The entropy is L plus a mean of |d| <= ln n + a few, off by the same
steps times its size.
"""
import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
U = 2.0**-24


def on(dev, a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def plain(x, t, k):
    """One row in 64 bits: (log probability, rank, entropy, top values, top indices, m, L)."""
    x64 = x.astype(np.float64)
    m = x64.max()
    if m == -np.inf:
        return -np.inf, 1 + np.count_nonzero(np.arange(len(x)) < t), 0.0, np.full(k, -np.inf), np.arange(k), 0.0, 0.0
    d = x64 - m
    e = np.exp(d)
    top = int(np.argmax(x64))
    rest = e[:top].sum() + e[top + 1:].sum()
    L = np.log1p(rest)
    with np.errstate(invalid="ignore"):
        H = L - np.where(e > 0, e * d, 0.0).sum() / (1 + rest)
    order = np.lexsort((np.arange(len(x)), -(x + np.float32(0))))[:k]
    rank = 1 + np.count_nonzero((x > x[t]) | ((x == x[t]) & (np.arange(len(x)) < t)))
    return d[t] - L, rank, H, d[order] - L, order, m, L


def check(ie, dev, x, t, k, n=None):
    n = x.shape[1] if n is None else n
    out = ie.token_logprobs(on(dev, x)[:, :n], on(dev, t), k)
    lp, rank, ent, top, idx = (o.cpu().numpy() for o in out)
    steps = n / 256 + 32
    for r in range(len(x)):
        w_lp, w_rank, w_ent, w_top, w_idx, m, L = plain(x[r, :n], t[r], k)
        assert rank[r] == w_rank, r
        assert np.array_equal(idx[r], w_idx), r

        def near(got, want):
            if want < -np.finfo(np.float32).max:  # below the type's range (-3.4e38 under 3e38 is -6.4e38): its nearest is -inf
                return got == -np.inf
            # |x - m| and L each round; a difference that cancels (a token that is nearly certain) has only L's error
            return abs(got - want) <= U * (2 * abs(want + L) + steps * min(1.0, 2 * L) + 4 * L)

        assert near(lp[r], w_lp), (r, lp[r], w_lp)
        assert all(near(a, b) for a, b in zip(top[r], w_top)), r
        assert abs(ent[r] - w_ent) <= U * 4 * steps * (w_ent + L), (r, ent[r], w_ent)
    return out


def logits(r, rows, n, spread=1.0):
    x = (r.standard_normal((rows, n)) * spread).astype(np.float32)
    for i in range(rows):
        j = r.integers(0, n, 4)
        x[i, j] += r.uniform(0, 12, 4).astype(np.float32)
    return x


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (3, 2, 1), (2, 5, 5), (4, 63, 7), (1, 64, 64), (2, 65, 0), (5, 257, 20),
                                      (3, 1000, 128), (2, 4099, 3), (1, 50257, 0), (8, 50257, 5), (2, 50257, 128),
                                      (1, 32768, 1), (1, 65536, 20), (2, 131072, 4), (1, 200001, 20), (1, 1 << 19, 2),
                                      (300, 1009, 3)])
def test_rows(ie, dev, rows, n, k):
    r = rng(n + k)
    x = logits(r, rows, n)
    t = r.integers(0, n, rows).astype(np.int32)
    t[::2] = x[::2].argmax(axis=1)
    a = check(ie, dev, x, t, k)
    b = ie.token_logprobs(on(dev, x), on(dev, t), k)
    assert all(np.array_equal(p.cpu().numpy(), q.cpu().numpy()) for p, q in zip(a, b))


@pytest.mark.parametrize("offset,pad", [(0, 47), (1, 3), (2, 1), (3, 0)])
def test_strides_and_alignment(ie, dev, offset, pad):
    """Rows that lie apart or begin off a 16-byte boundary; what lies between is NaN and does not count."""
    import torch

    r = rng(offset + pad)
    rows, n = 5, 3001
    x = logits(r, rows, n)
    buf = torch.full((offset + rows * (n + pad) + 8,), float("nan"), device=dev)
    view = buf[offset:offset + rows * (n + pad)].view(rows, n + pad)[:, :n]
    view.copy_(on(dev, x))
    t = r.integers(0, n, rows).astype(np.int32)
    want = check(ie, dev, x, t, 9)
    got = ie.token_logprobs(view, on(dev, t), 9)
    for i, (a, b) in enumerate(zip(got, want)):
        if a.dtype == torch.int32:
            assert torch.equal(a, b), i
        else:
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6), i


@pytest.mark.parametrize("n", [300, 50257, 140000])
def test_ties(ie, dev, n):
    """Equal logits everywhere, in part, and both zeros: the lowest index first, ranks to match."""
    r = rng(n)
    x = np.zeros((4, n), np.float32)
    x[1] = r.integers(0, 3, n)
    x[2] = np.where(r.random(n) < 0.5, np.float32(0.0), np.float32(-0.0))
    x[3, ::7] = 5.0
    check(ie, dev, x, np.array([n - 1, n // 2, 17, n - 2], np.int32), 100)


@pytest.mark.parametrize("n", [40, 50257, 70001])
def test_masks(ie, dev, n):
    """Tokens masked by -inf and by the type's lowest value, rows with one token left and with none."""
    r = rng(n)
    x = logits(r, 6, n)
    low = np.finfo(np.float32).min
    x[0, r.random(n) < 0.9] = -np.inf
    x[1, r.random(n) < 0.9] = low
    x[2] = -np.inf
    x[2, n // 3] = -3.0
    x[3] = -np.inf
    x[4] = low
    x[5] = low
    x[5, n - 1] = 3e38
    t = np.array([np.argmin(x[0]), 3, n // 3, 5, 6, n - 1], np.int32)
    check(ie, dev, x, t, 20)


def test_nearly_certain(ie, dev):
    """-log p of a token that has all but 1e-3 .. 1e-12 of the probability keeps its leading bits."""
    r = rng(7)
    n = 50257
    x = r.standard_normal((10, n)).astype(np.float32)
    for i in range(10):
        x[i, 100 * i] = 18 + 2 * i
    t = (100 * np.arange(10)).astype(np.int32)
    lp, _, ent, _, _ = (o.cpu().numpy().astype(np.float64) for o in ie.token_logprobs(on(dev, x), on(dev, t), 2))
    for i in range(10):
        want, _, w_ent, _, _, _, _ = plain(x[i], t[i], 1)
        assert abs(lp[i] - want) <= U * (n / 256 + 40) * abs(want)
        assert abs(ent[i] - w_ent) <= 4 * U * (n / 256 + 40) * w_ent


def test_targets_outside_and_none(ie, dev):
    r = rng(1)
    x = logits(r, 4, 50)
    lp, rank, ent, _, _ = (o.cpu().numpy() for o in ie.token_logprobs(on(dev, x), on(dev, np.array([-1, 50, -5, 7], np.int32)), 2))
    assert lp[0] == 0 and np.isnan(lp[1]) and np.isnan(lp[2]) and lp[3] < 0
    assert list(rank[:3]) == [0, 0, 0] and rank[3] >= 1
    out = ie.token_logprobs(on(dev, x), None, 0)
    assert not out[0].any() and not out[1].any() and np.array_equal(out[2].cpu().numpy(), ent)
    assert ie.token_logprobs(on(dev, x)[:0], None, 3)[3].shape == (0, 3)


@pytest.mark.parametrize("n", [100, 50257, 140000])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_not_finite(ie, dev, n, bad):
    """NaN or +inf in a row shows in that row alone, its indices stay in range."""
    r = rng(n)
    x = logits(r, 3, n)
    x[1, n // 2] = bad
    t = np.array([1, 2, 3], np.int32)
    out = [o.cpu().numpy() for o in ie.token_logprobs(on(dev, x), on(dev, t), 6)]
    assert np.isnan(out[0][1]) and np.isnan(out[2][1]) and np.isnan(out[3][1]).all()
    assert (out[4][1] >= 0).all() and (out[4][1] < n).all()
    keep = [0, 2]
    rest = [o.cpu().numpy() for o in ie.token_logprobs(on(dev, x[keep]), on(dev, t[keep]), 6)]
    for a, b in zip(out, rest):
        assert np.allclose(a[keep], b, rtol=1e-6, atol=1e-6)


def test_graph_and_stream(ie, dev):
    """Captured once and replayed on other logits, and on a side stream: the eager bits."""
    import torch

    r = rng(3)
    xs = [on(dev, logits(r, 4, 50257)) for _ in range(4)]
    t = on(dev, np.array([5, 6, 7, 8], np.int32))
    want = [ie.token_logprobs(x, t, 5) for x in xs]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = ie.token_logprobs(xs[1], t, 5, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    x = xs[0].clone()
    need = ie.call("ie_token_logprobs_workspace_bytes", 4, 50257, 5)
    ws = torch.empty(max(need // 4, 2), device=dev)
    out = tuple(torch.empty_like(a) for a in want[0])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ie.token_logprobs(x, t, 5, out=out, workspace=ws)
    for i in range(4):
        x.copy_(xs[i])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i


def test_binding_refusals(ie, dev):
    import torch

    x = torch.zeros(3, 40, device=dev)
    t = torch.zeros(3, dtype=torch.int32, device=dev)
    for f in (lambda: ie.token_logprobs(x.half(), t), lambda: ie.token_logprobs(x.cpu(), t),
              lambda: ie.token_logprobs(x.t(), t), lambda: ie.token_logprobs(x, t.long()),
              lambda: ie.token_logprobs(x, t[:2]), lambda: ie.token_logprobs(x.expand(3, 40)[:, ::2], t)):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(ie.IeError):
        ie.token_logprobs(x, t, 41)


@pytest.mark.parametrize("n", [3000, 50257])
def test_no_error_of_one_sign(ie, dev, n):
    """-log p of a token under which n others lie by 78 to 82: the sum of their exponentials, whose errors average out.
    Each exponent (up to 119 in base 2) rounds once, by at most 82 u of the exponential with no preferred sign: over n >=
    2999 elements 82 / sqrt(3 n) u, at six times that 5.2 u; the exponential is off by 1 in its last place, 2 u; of at most
    n / 256 + 32 additions, half a step each at random in 256 chains of their own, (n / 256 + 32)^0.5 / (3^0.5 16) u, at six
    times that 3.3 u; log1p keeps it.  So an exponential that many elements share (a thread's sums against the row's
    maximum) has to be exact to its last places: one that is rounded as an element's is would put up to 82 u into all of
    them, and a factor of the exponent that is off by 1.3e-8 adds 80 * 1.3e-8 = 18 u in every row."""
    r = rng(n)
    x = r.uniform(-82, -78, (32, n)).astype(np.float32)
    t = r.integers(0, n, 32).astype(np.int32)
    x[np.arange(32), t] = 0
    lp = ie.token_logprobs(on(dev, x), on(dev, t), 0)[0].cpu().numpy().astype(np.float64)
    want = np.array([plain(x[i], t[i], 0)[0] for i in range(32)])
    assert (want < 0).all()
    assert np.abs(lp / want - 1).max() <= (82 * 6 / (3 * n) ** 0.5 + 2 + 6 * (n / 256 + 32) ** 0.5 / (3**0.5 * 16)) * U

"""include/ie_paged.h on the GPU against 64 bits (paged_oracle has the tolerances)."""
import math

import numpy as np
import pytest
import torch

import paged_oracle as po
from conftest import rng
from paged_forms import FORMS

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(np.asarray(x, dtype=np.int32), device=dev)


def normal(r, dev, *shape, scale=1.0):
    return torch.from_numpy((r.standard_normal(shape) * scale).astype(np.float32)).to(dev)


def near(got, want):
    o, tol, live = want
    off = (got.double() - o).abs() - tol
    assert bool((off[live] <= 0).all()), f"off by {float(off[live].max()):.3g} more than {float(tol[live].max()):.3g}"


def case(r, dev, B, P, H_kv, G, d, block, half, starts, lens=None, q_scale=1.0, fill=float("nan")):
    held = [s + (P if lens is None else max(0, min(lens[b], P))) for b, s in enumerate(starts)]
    table, pages = po.tables(r, held, block)
    caches = po.cache_of(r, table, pages, held, block, H_kv, d, half, dev, fill)
    return table, caches, normal(r, dev, B, P, H_kv * G, d, scale=q_scale), max(held)


def check_ranges(ie, dev, r, B, P, H_kv, G, d, block, half, starts, lens=None, first=None, end=None, window=0, scale=None,
                 cap=0.0, slopes=False, splits=0, q_scale=1.0):
    table, caches, q, top = case(r, dev, B, P, H_kv, G, d, block, half, starts, lens, q_scale)
    sl = normal(r, dev, H_kv * G).abs() if slopes else None
    kw = dict(window=window, scale=scale, cap=cap, slopes=sl)
    want = po.ranges(q, caches, table, block, starts, lens, top, first, end, **kw)
    out = torch.full_like(q, 7.0)
    got = ie.paged_attn(q, *caches, i32(table, dev), i32(starts, dev), top, lens=None if lens is None else i32(lens, dev),
                        first=None if first is None else i32(first, dev), end=None if end is None else i32(end, dev),
                        splits=splits, out=out, **kw)
    near(got, want)
    assert bool((got[~want[2]] == 7.0).all())  # rows left out stay as they were
    return table, caches, q, top, got


# ------------------------------------------------------------------ attention over ranges
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("d,H_kv,G,block", [(64, 3, 1, 16), (128, 2, 4, 16), (64, 2, 3, 24), (128, 1, 16, 1), (64, 1, 40, 256),
                                            (128, 4, 2, 7)])
@pytest.mark.parametrize("P,starts,lens", [(1, [0, 1, 63, 500], None), (1, [31, 32, 33, 700], [1, 0, 1, 1]),
                                           (5, [0, 3, 60, 300], [5, 1, 4, 0]), (33, [0, 130], None), (70, [0, 57], [70, 69])])
def test_causal(ie, dev, half, d, H_kv, G, block, P, starts, lens):
    r = rng(P * 100 + block + d + G)
    check_ranges(ie, dev, r, len(starts), P, H_kv, G, d, block, half, starts, lens)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("d,G", [(64, 1), (128, 4)])
@pytest.mark.parametrize("P", [1, 3, 50, 150])
@pytest.mark.parametrize("cap,slopes,window", [(30.0, False, 0), (0.5, False, 40), (0.0, True, 0), (20.0, True, 33), (0.0, False, 1),
                                               (1e30, False, 100)])
def test_scores(ie, dev, half, d, G, P, cap, slopes, window):
    r = rng(P + d + int(min(cap, 99) * 10) + window)
    check_ranges(ie, dev, r, 3, P, 2, G, d, 16, half, [0, 90, 333], [P, max(1, P - 1), P], cap=cap, slopes=slopes, window=window,
                 scale=None if P != 3 else 0.37, q_scale=6.0 if cap > 1 else 1.0)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("d,G,P", [(64, 1, 40), (128, 2, 200), (64, 8, 130), (128, 1, 4)])
def test_ranges(ie, dev, half, d, G, P):
    """Documents, a prefix, both ways, empty ranges, ranges past either end."""
    r = rng(P + d)
    starts = [0, 17, 250]
    n = [s + P for s in starts]
    first = np.zeros((3, P), np.int32)
    end = np.zeros((3, P), np.int32)
    for t in range(P):
        first[0, t], end[0, t] = t // 13 * 13, t // 13 * 13 + 13  # documents that see themselves whole
        first[1, t], end[1, t] = -5, max(60, 17 + t + 1)  # a prefix
        a, b = sorted(r.integers(-20, n[2] + 40, 2))
        first[2, t], end[2, t] = (a, b) if t % 3 else (b, a)  # any, every third empty
    for kw in (dict(first=first, end=end), dict(first=first), dict(end=end), dict(first=first, end=end, window=25, slopes=True)):
        check_ranges(ie, dev, r, 3, P, 2, G, d, 16, half, starts, **kw)
    none = np.full((3, P), n[2] + 3, np.int32)
    assert not check_ranges(ie, dev, r, 3, P, 2, G, d, 16, half, starts, first=none)[-1].any()
    assert not check_ranges(ie, dev, r, 3, P, 2, G, d, 16, half, starts, end=np.zeros_like(none))[-1].any()


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("B,P,H_kv,G,d,starts", [(1, 1, 2, 4, 128, [9000]), (2, 1, 1, 1, 64, [20000, 4097]), (1, 40, 2, 2, 64, [3001]),
                                                 (2, 130, 1, 4, 128, [1500, 0]), (1, 600, 2, 2, 128, [0]), (1, 300, 1, 3, 64, [77])])
@pytest.mark.parametrize("splits", [0, 1, 2, 7, 64])
def test_long_and_split(ie, dev, half, B, P, H_kv, G, d, starts, splits):
    r = rng(B + P + d + splits)
    table, caches, q, top, got = check_ranges(ie, dev, r, B, P, H_kv, G, d, 32, half, starts, splits=splits)
    again = ie.paged_attn(q, *caches, i32(table, dev), i32(starts, dev), top, splits=splits)
    assert torch.equal(again, got)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("P,splits", [(1, 1), (1, 5), (40, 1), (40, 3), (200, 1)])
def test_values_that_are_not_seen_never_arrive(ie, dev, half, P, splits):
    """Infinite and NaN K and V outside a query's range, in the same pages and blocks as what it sees; a query that sees one
    has what fp32 makes of it."""
    r = rng(P + splits)
    d, H, starts = 64, 1, [400, 300]
    table, caches, q, top = case(r, dev, 2, P, H, 2, d, 16, half, starts)
    first = np.array([[100 + 2 * t for t in range(P)], [0] * P], np.int32)
    end = first + 90
    want = po.ranges(q, caches, table, 16, starts, None, top, first, end)
    for b in range(2):
        lo, hi = first[b].min(), end[b].max()
        for j in [*range(max(0, lo - 40), lo), *range(hi, min(hi + 40, starts[b] + P))]:
            for c, x in zip(caches, ((float("nan"), float("inf")) if j % 2 else (float("-inf"), float("nan")))):
                c[table[b, j // 16], j % 16] = x
    args = (i32(table, dev), i32(starts, dev), top)
    kw = dict(first=i32(first, dev), end=i32(end, dev), splits=splits)
    near(ie.paged_attn(q, *caches, *args, **kw), want)
    # keys that some queries see and others do not: only the first are touched
    j = int(first[0, 0]) + 1
    caches[1][table[0, j // 16], j % 16, :, 5] = float("inf")
    caches[0][table[0, (j + 1) // 16], (j + 1) % 16] = float("nan")
    got = ie.paged_attn(q, *caches, *args, **kw)
    sees_v = torch.from_numpy((first[0] <= j) & (j < end[0])).to(dev)
    sees_k = torch.from_numpy((first[0] <= j + 1) & (j + 1 < end[0])).to(dev)
    assert bool(torch.isnan(got[0, sees_k]).all())
    only_v = sees_v & ~sees_k
    assert bool((~torch.isfinite(got[0, only_v][..., 5])).all()) or not bool(only_v.any())
    clean = ~(sees_v | sees_k)
    off = (got.double() - want[0]).abs() - want[1]
    assert bool((off[0, clean] <= 0).all()) and bool((off[1] <= 0).all())


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("P", [1, 40])
@pytest.mark.parametrize("size_q,size_k,size_v", [(1e-30, 1e30, 1.0), (1e30, 1e-30, 1e-30), (1e-36, 1e36, 1e30), (1e-3, 1e3, 1e37),
                                                  (0.0, 1.0, 1.0)])
def test_extreme_sizes(ie, dev, half, P, size_q, size_k, size_v):
    r = rng(int(P + 10 * size_v % 97))
    table, caches, q, top = case(r, dev, 1, P, 2, 2, 64, 16, half, [70], fill=0.0)
    q *= size_q
    caches[0].mul_(size_k)
    caches[1].mul_(size_v)
    want = po.ranges(q, caches, table, 16, [70], None, top)
    near(ie.paged_attn(q, *caches, i32(table, dev), i32([70], dev), top), want)


def test_large_scores(ie, dev):
    """Scores of thousands: one key takes all, without overflow."""
    for half in (True, False):
        check_ranges(ie, dev, rng(8), 2, 20, 2, 2, 128, 16, half, [0, 333], q_scale=3000.0)


def test_starts_and_lens_outside_their_range(ie, dev):
    """A negative start counts as 0, lens past P as P, below 0 as none; keys end at max_ctx."""
    r = rng(12)
    table, caches, q, top = case(r, dev, 3, 6, 2, 1, 64, 16, True, [0, 40, 40])
    want = po.ranges(q, caches, table, 16, [0, 40, 40], [6, 6, 0], 43)
    out = torch.full_like(q, 7.0)
    got = ie.paged_attn(q, *caches, i32(table, dev), i32([-3, 40, 40], dev), 43, lens=i32([6, 99, -1], dev), out=out)
    near(got, want)
    assert bool((got[2] == 7.0).all())


def test_no_context(ie, dev):
    """max_ctx 0 and a table without pages: zeros."""
    q = torch.randn(2, 3, 2, 64, device=dev)
    k = torch.zeros(1, 16, 2, 64, device=dev)
    assert not ie.paged_attn(q, k, k, torch.zeros(2, 0, dtype=torch.int32, device=dev), i32([0, 0], dev), 0).any()


# ------------------------------------------------------------------ trees
def shapes(r, T):
    return {"chain": [t - 1 for t in range(T)], "star": [-1] * T, "random": [int(r.integers(-1, t)) if t else -1 for t in range(T)],
            "recent": [int(r.integers(max(-1, t - 4), t)) if t else -1 for t in range(T)],
            "wrong": [int(r.choice([t, t + 1, -7, 2**31 - 1, t - 1 if t else -1])) for t in range(T)]}


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("T", [1, 2, 8, 33, 64, 65, 256])
@pytest.mark.parametrize("d,H_kv,G,block,ctx", [(64, 2, 1, 16, [0, 1, 100]), (128, 1, 4, 24, [31, 1000, 33])])
def test_tree(ie, dev, half, T, d, H_kv, G, block, ctx):
    r = rng(T + d)
    table, caches, q, _ = case(r, dev, 3, T, H_kv, G, d, block, half, ctx)
    kinds = list(shapes(r, T).values())
    lens = [T, max(1, T - 3), 0]
    for i, (kw, ln) in enumerate([({}, None), ({}, lens), (dict(cap=5.0, slopes=normal(r, dev, H_kv * G).abs()), None),
                                  (dict(window=3), None), (dict(window=40, slopes=normal(r, dev, H_kv * G).abs()), lens),
                                  (dict(window=1, scale=0.2), None)]):
        parents = [kinds[(i + b) % len(kinds)] for b in range(3)]
        want = po.tree(q, caches, table, block, ctx, parents, ln, **kw)
        out = torch.full_like(q, 7.0)
        got = ie.tree_attn(q, *caches, i32(table, dev), i32(ctx, dev), i32(parents, dev), max(ctx),
                           lens=None if ln is None else i32(ln, dev), out=out, **kw)
        near(got, want)
        assert bool((got[~want[2]] == 7.0).all())


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("T,G,d,splits", [(8, 1, 64, 0), (63, 4, 128, 0), (255, 2, 64, 0), (16, 8, 128, 5), (200, 1, 128, 64)])
def test_tree_behind_a_long_context(ie, dev, half, T, G, d, splits):
    r = rng(T + G)
    ctx = [5000, 123]
    table, caches, q, _ = case(r, dev, 2, T, 2, G, d, 16, half, ctx)
    parents = [shapes(r, T)["recent"], shapes(r, T)["random"]]
    want = po.tree(q, caches, table, 16, ctx, parents)
    got = ie.tree_attn(q, *caches, i32(table, dev), i32(ctx, dev), i32(parents, dev), 5000, splits=splits)
    near(got, want)
    assert torch.equal(got, ie.tree_attn(q, *caches, i32(table, dev), i32(ctx, dev), i32(parents, dev), 5000, splits=splits))


@pytest.mark.parametrize("half", [True, False])
def test_other_branches_never_arrive(ie, dev, half):
    """Rows of nodes that are no ancestors may hold anything."""
    r = rng(9)
    T, ctx = 40, [90]
    table, caches, q, _ = case(r, dev, 1, T, 1, 3, 64, 16, half, ctx)
    parents = [[-1, 0, 0] + [1 if t % 2 else 2 for t in range(3, T)]]
    want = po.tree(q, caches, table, 16, ctx, parents)
    for t in (2, 5, 20):
        for c in caches:
            c[table[0, (90 + t) // 16], (90 + t) % 16] = float("nan")
    got = ie.tree_attn(q, *caches, i32(table, dev), i32(ctx, dev), i32(parents, dev), 90)
    clean = torch.tensor([not ({2, 5, 20} & set(line)) for line in po.lines(parents[0])], device=dev)
    off = (got.double() - want[0]).abs() - want[1]
    assert bool((off[0, clean] <= 0).all()) and bool(torch.isnan(got[0, ~clean]).all())


# ------------------------------------------------------------------ every form of the kernels
def ragged(r, B, top):
    """Positions before the queries: one sequence at `top`, the others anywhere, one at 0."""
    starts = [int(x) for x in r.integers(0, top + 1, B)]
    starts[0] = top
    if B > 2:
        starts[B // 2] = 0
    return starts


@pytest.mark.parametrize("kv,d,rows,groups,splits,call", FORMS)
def test_every_form_ranges(ie, dev, kv, d, rows, groups, splits, call):
    B, P, H, G, keys = call
    r = rng(rows + d + kv + splits)
    starts = ragged(r, B, keys - P)
    lens = [P] + [int(x) for x in r.integers(0, P + 1, B - 1)]
    check_ranges(ie, dev, r, B, P, H, G, d, 16, bool(kv), starts, cap=4.0, q_scale=3.0)
    check_ranges(ie, dev, r, B, P, H, G, d, 24, bool(kv), starts, lens, slopes=True, scale=0.1)
    check_ranges(ie, dev, r, B, P, H, G, d, 16, bool(kv), starts, lens, q_scale=400.0)  # (weights far apart)
    first = r.integers(-5, keys, (B, P)).astype(np.int32)
    end = (first + r.integers(-30, keys, (B, P))).astype(np.int32)
    check_ranges(ie, dev, r, B, P, H, G, d, 32, bool(kv), starts, lens, first=first, end=end, cap=30.0, slopes=True)
    table, caches, q, top = case(r, dev, B, P, H, G, d, 16, bool(kv), starts)
    # one key that every other query sees is not finite
    x = starts[0] // 2
    first = np.zeros((B, P), np.int32)
    first[0, ::2] = x + 1
    want = po.ranges(q, caches, table, 16, starts, None, top, first)
    caches[0][table[0, x // 16], x % 16] = float("nan")
    caches[1][table[0, x // 16], x % 16] = float("inf")
    got = ie.paged_attn(q, *caches, i32(table, dev), i32(starts, dev), top, first=i32(first, dev))
    off = (got.double() - want[0]).abs() - want[1]
    assert bool((off[1:] <= 0).all()) and bool((off[0, ::2] <= 0).all()) and bool(torch.isnan(got[0, 1::2]).all())
    # and again in other splits: the same answers, the same bits again
    if splits > 1:
        for s in (1, 2, splits + 1):
            again = [ie.paged_attn(q, *caches, i32(table, dev), i32(starts, dev), top, first=i32(first, dev), splits=s) for _ in range(2)]
            off = (again[0].double() - want[0]).abs() - want[1]
            assert bool((off[1:] <= 0).all()) and torch.equal(again[0].view(torch.int32), again[1].view(torch.int32))


@pytest.mark.parametrize("kv,d,rows,groups,splits,call", [f for f in FORMS if f[5][1] <= 256])
def test_every_form_tree(ie, dev, kv, d, rows, groups, splits, call):
    B, T, H, G, keys = call
    r = rng(rows + d + kv + splits)
    ctx = ragged(r, B, keys - T)
    table, caches, q, _ = case(r, dev, B, T, H, G, d, 16, bool(kv), ctx)
    parents = [list(shapes(r, T).values())[b % 5] for b in range(B)]
    lens = [T] + [int(x) for x in r.integers(0, T + 1, B - 1)]
    for kw in ({}, dict(window=max(2, T // 3), cap=20.0, slopes=normal(r, dev, H * G).abs())):
        want = po.tree(q, caches, table, 16, ctx, parents, lens, **kw)
        got = ie.tree_attn(q, *caches, i32(table, dev), i32(ctx, dev), i32(parents, dev), max(ctx), lens=i32(lens, dev),
                           out=torch.full_like(q, 7.0), **kw)
        near(got, want)
        assert bool((got[~want[2]] == 7.0).all())


# ------------------------------------------------------------------ rotated writes
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("H_q,H_kv,d,rot", [(4, 2, 64, 64), (32, 8, 128, 128), (1, 1, 64, 32), (0, 3, 128, 128), (5, 1, 128, 0),
                                            (3, 2, 64, 62), (2, 2, 128, 36), (12, 12, 64, 8), (40, 40, 128, 2)])
@pytest.mark.parametrize("P,starts,lens", [(1, [0, 17, 300], None), (7, [0, 5, 30], [7, 0, 3]), (300, [2, 0, 1], [300, 299, 1])])
def test_rope(ie, dev, half, pairs, H_q, H_kv, d, rot, P, starts, lens):
    r = rng(P + rot + H_q)
    B, block = 3, 24
    qkv = normal(r, dev, B, P, (H_q + 2 * H_kv) * d + 4)  # rows with something behind them
    q, k, v = (x.unflatten(-1, (-1, d)) if x.shape[-1] else None for x in
               (qkv[..., :H_q * d], qkv[..., H_q * d:(H_q + H_kv) * d], qkv[..., (H_q + H_kv) * d:(H_q + 2 * H_kv) * d]))
    table, pages = po.tables(r, [s + P for s in starts], block)
    t = torch.bfloat16 if half else torch.float32
    kc, vc = (torch.full((pages, block, H_kv, d), 3.0, dtype=t, device=dev) for _ in range(2))
    want_k, want_v, tol_k = kc.double(), vc.double(), torch.zeros(kc.shape, dtype=torch.float64, device=dev)
    freq = torch.from_numpy((10000.0 ** (-np.arange(rot // 2) / max(1, rot // 2))).astype(np.float32)).to(dev)
    places = np.array([[10 * s + 3 * t for t in range(P)] for s in starts], np.int32)
    for positions in (None, places):
        out = torch.full((B, P, H_q, d), 7.0, device=dev)
        got = ie.rope_kv_write(q, k, v, freq, i32(starts, dev), kc, vc, i32(table, dev), lens=None if lens is None else i32(lens, dev),
                               positions=None if positions is None else i32(positions, dev), interleaved=pairs, out=out)
        for b in range(B):
            n = P if lens is None else lens[b]
            at = starts[b] + torch.arange(n, device=dev)
            pos = at if positions is None else i32(positions[b, :n], dev)
            page = i32(table[b], dev).long()[at // block]
            if q is not None:
                y, tol = po.rotated(q[b, :n], pos, freq, pairs)
                assert bool(((got[b, :n].double() - y).abs() <= tol).all()) and bool((got[b, n:] == 7.0).all())
            y, tol = po.rotated(k[b, :n], pos, freq, pairs)
            want_k[page, at % block], tol_k[page, at % block] = y, tol
            want_v[page, at % block] = v[b, :n].to(t).double()
        # rounded to the cache's type once
        step = 2.0**-8 if half else 0.0
        assert bool(((kc.double() - want_k).abs() <= tol_k + step * (want_k.abs() + tol_k)).all())
        assert torch.equal(vc.double(), want_v)


@pytest.mark.parametrize("pos", [1, 4095, 10**6, 2**24 + 1, 2**30 - 5, -2**30, 2**31 - 1, -2**31])
def test_rope_far_positions(ie, dev, pos):
    """Angles of far positions are those of 64 bits; separate tensors of Q and of K and V; a row that has no place in the
    cache has its Q all the same."""
    r = rng(4)
    q, k = normal(r, dev, 2, 1, 3, 128), normal(r, dev, 2, 1, 2, 128)
    kc, vc = (torch.full((4, 16, 2, 128), 3.0, device=dev) for _ in range(2))
    freq = torch.from_numpy((10000.0 ** (-np.arange(64) / 64)).astype(np.float32)).to(dev)
    table = i32([[0, 1], [2, 3]], dev)
    got = ie.rope_kv_write(q, k, k, freq, i32([31, -1], dev), kc, vc, table, positions=i32([pos, pos], dev))
    at = torch.tensor([pos], device=dev)
    for b in range(2):
        y, tol = po.rotated(q[b], at, freq, False)
        assert bool(((got[b].double() - y).abs() <= tol).all())
    y, tol = po.rotated(k[0], at, freq, False)
    assert bool(((kc[1, 15].double() - y[0]).abs() <= tol[0]).all()) and torch.equal(vc[1, 15], k[0, 0])
    kc[1, 15] = vc[1, 15] = 3.0
    assert bool((kc == 3.0).all()) and bool((vc == 3.0).all())
    for start in (32, 2**31 - 1, -2**31):  # past the table's row, and as far as a start can be
        got = ie.rope_kv_write(q, k, k, freq, i32([start, start], dev), kc, vc, table, positions=i32([5, 5], dev))
        y, tol = po.rotated(q[0], torch.tensor([5], device=dev), freq, False)
        assert bool(((got[0].double() - y).abs() <= tol).all()) and bool((kc == 3.0).all())


# ------------------------------------------------------------------ accepted paths
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("layers", [1, 3, 64, 65, 130])
@pytest.mark.parametrize("H,d,block", [(1, 64, 16), (12, 64, 7), (20, 128, 32)])
def test_keep(ie, dev, half, layers, H, d, block):
    r = rng(layers + H)
    ctx = [0, 5, 31, 10, 12, 3]
    paths = [[0, 1, 2, 3, 4, 5, 6, 7, 8, 9], [1, 2, 3, 4, 5, 6, 7, 8, 9, 40], [3, 9, 10, 11, 30, 31, 32, 38, 39, 40], [4, 5, 5, 6, 7, 0, 0, 0, 0, 0],
             [-1, 1, 2, 3, 4, 5, 6, 7, 8, 9], [2, 7, 2**31 - 1, 9, 10, 11, 12, 13, 14, 15]]
    counts = [10, 10, 99, 10, 10, 10]
    moves = [paths[0], paths[1], paths[2], [4, 5], [], [2, 7]]
    table, pages = po.tables(r, [c + 41 for c in ctx], block)
    t = torch.bfloat16 if half else torch.float32
    k, v = (normal(r, dev, layers, pages, block, H, d).to(t) for _ in range(2))
    want = [k.clone(), v.clone()]
    for w, c in zip(want, (k, v)):
        for b, move in enumerate(moves):
            for j, p in enumerate(move):
                x, y = ctx[b] + j, ctx[b] + p
                w[:, table[b, x // block], x % block] = c[:, table[b, y // block], y % block]
    ie.kv_cache_keep(list(k), list(v), i32(table, dev), i32(ctx, dev), i32(paths, dev), i32(counts, dev))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_keep_ends_at_the_table(ie, dev):
    k = torch.arange(2 * 4, device=dev, dtype=torch.float32).reshape(2, 4, 1, 1).expand(2, 4, 1, 64).contiguous()
    v = k.clone()
    table, paths = i32([[0, 1]], dev), i32([[1, 2, 3]], dev)
    for ctx, counts in ((6, 3), (-1, 3), (0, 0), (0, -4), (2**31 - 1, 3)):
        kc, vc = k.clone(), v.clone()
        ie.kv_cache_keep([kc], [vc], table, i32([ctx], dev), paths, i32([counts], dev))
        want = k.clone()
        if ctx == 6:
            want[1, 2] = k[1, 3]  # 6 + 1 goes to 6; 6 + 2 is past the table
        assert torch.equal(kc, want) and torch.equal(vc, want)


# ------------------------------------------------------------------ streams, graphs, and all of them together
def test_two_streams_and_a_graph(ie, dev):
    """Calls on two streams at once with a workspace each, and a captured call replayed between eager ones."""
    r = rng(21)
    table, caches, q, top = case(r, dev, 2, 1, 2, 4, 128, 16, True, [6000, 5000])
    args = (*caches, i32(table, dev), i32([6000, 5000], dev), top)
    q2 = normal(r, dev, 2, 1, 8, 128)
    want, want2 = ie.paged_attn(q, *args), ie.paged_attn(q2, *args)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = [(ie.paged_attn(q, *args, stream=a), ie.paged_attn(q2, *args, stream=b)) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) and torch.equal(y, want2) for x, y in got)
    out = torch.empty_like(q)
    S = ie.paged_attn_num_splits(2, 1, 8, 2, 128, ie.KV_BF16, top)
    ws = torch.empty(max(1, 2 * 8 * S * 130), device=dev)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ie.paged_attn(q, *args, out=out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ie.paged_attn(q, *args, out=out, workspace=ws)
    for x, y in ((q2.clone(), want2), (q.clone(), want), (q2.clone(), want2)):
        q.copy_(x)
        out.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y)
        assert torch.equal(ie.paged_attn(q2, *args), want2)


@pytest.mark.parametrize("half", [True, False])
def test_a_drafted_step(ie, dev, half):
    """Prompt rows rotated and written, a tree drafted behind them and attended to, its accepted path kept, the next token's
    attention: the same as the accepted tokens written one after another."""
    r = rng(33)
    B, H, G, d, block, layers = 2, 2, 2, 64, 16, 3
    ctx, T = [45, 70], 12
    table, pages = po.tables(r, [c + T + 1 for c in ctx], block)
    t = torch.bfloat16 if half else torch.float32
    freq = torch.from_numpy((10000.0 ** (-np.arange(d // 2) / (d // 2))).astype(np.float32)).to(dev)
    tb, starts = i32(table, dev), i32(ctx, dev)
    parents = [[-1, -1, 0, 0, 1, 2, 3, 3, 5, 6, 7, 8], [-1, 0, 0, 1, 1, 2, 4, 4, 6, 7, 7, 10]]
    paths = [[0, 3, 7, 10], [0, 1, 4, 6]]
    deep = np.array([[len(x) - 1 for x in po.lines(p)] for p in parents])
    prompt = [normal(r, dev, B, max(ctx), (H * G + 2 * H), d) for _ in range(layers)]
    draft = [normal(r, dev, B, T, (H * G + 2 * H), d) for _ in range(layers)]
    last = [normal(r, dev, B, 1, (H * G + 2 * H), d) for _ in range(layers)]

    def part(x):
        return x[:, :, :H * G], x[:, :, H * G:H * (G + 1)], x[:, :, H * (G + 1):]

    def fresh():
        return [[torch.zeros(pages, block, H, d, dtype=t, device=dev) for _ in range(layers)] for _ in range(2)]

    k, v = fresh()
    k2, v2 = fresh()
    zero = i32([0, 0], dev)
    place = i32([[c + x for x in row] for c, row in zip(ctx, deep)], dev)
    for l in range(layers):
        for kk, vv in ((k, v), (k2, v2)):
            ie.rope_kv_write(*part(prompt[l]), freq, zero, kk[l], vv[l], tb, lens=starts)
        q = ie.rope_kv_write(*part(draft[l]), freq, starts, k[l], v[l], tb, positions=place)
        o = ie.tree_attn(q, k[l], v[l], tb, starts, i32(parents, dev), max(ctx))
        # the path's tokens one after another, in the second caches
        for j in range(4):
            x = torch.stack([draft[l][b, paths[b][j]] for b in range(B)])[:, None]
            at = i32([c + j for c in ctx], dev)
            q1 = ie.rope_kv_write(*part(x), freq, at, k2[l], v2[l], tb)
            o1 = ie.paged_attn(q1, k2[l], v2[l], tb, at, max(ctx) + j + 1)
            want = po.ranges(q1, (k2[l], v2[l]), table, block, [c + j for c in ctx], None, max(ctx) + j + 1)
            near(o1, want)
            near(torch.stack([o[b, paths[b][j]] for b in range(B)])[:, None], want)
    ie.kv_cache_keep(k, v, tb, starts, i32(paths, dev), i32([4, 4], dev))
    at = i32([c + 4 for c in ctx], dev)
    for l in range(layers):
        outs = []
        for kk, vv in ((k, v), (k2, v2)):
            q = ie.rope_kv_write(*part(last[l]), freq, at, kk[l], vv[l], tb)
            outs.append(ie.paged_attn(q, kk[l], vv[l], tb, at, max(ctx) + 5))
        assert torch.equal(outs[0], outs[1])


def test_binding_refuses(ie, dev):
    q = torch.randn(1, 2, 4, 64, device=dev)
    k = torch.zeros(4, 16, 2, 64, device=dev)
    table, s = i32([[0, 1, 2, 3]], dev), i32([0], dev)
    ok = dict(Q=q, k_cache=k, v_cache=k, block_table=table, starts=s, max_ctx=2)
    ie.paged_attn(**ok)
    for bad in (dict(Q=q.half()), dict(Q=q.cpu()), dict(Q=q.transpose(1, 2)), dict(k_cache=k.half()), dict(v_cache=k.bfloat16()),
                dict(v_cache=k[:3]), dict(block_table=table.long()), dict(block_table=table[:, ::2]), dict(starts=s.long()),
                dict(starts=i32([0, 0], dev)), dict(lens=i32([1, 2], dev)), dict(first=s), dict(end=s), dict(slopes=q[0, 0, 0]),
                dict(out=q.double()), dict(max_ctx=2**31), dict(window=-2**40), dict(workspace=q.double())):
        with pytest.raises(ValueError):
            ie.paged_attn(**(ok | bad))
    for bad in (dict(max_ctx=65), dict(window=-1), dict(cap=-1.0), dict(scale=math.inf), dict(out=q)):
        with pytest.raises(ie.IeError):
            ie.paged_attn(**(ok | bad))
    ok = dict(Q=q, k_cache=k, v_cache=k, block_table=table, context_lens=s, parents=i32([[-1, 0]], dev), max_ctx=2)
    ie.tree_attn(**ok)
    for bad in (dict(parents=s), dict(parents=i32([[-1, 0]], dev).long()), dict(lens=i32([1, 1], dev))):
        with pytest.raises(ValueError):
            ie.tree_attn(**(ok | bad))
    with pytest.raises(ie.IeError):
        ie.tree_attn(**(ok | dict(max_ctx=63)))
    f = torch.ones(32, device=dev)
    kv = torch.randn(1, 2, 2, 64, device=dev)
    ok = dict(Q=q, K=kv, V=kv, inv_freq=f, starts=s, k_cache=k, v_cache=k.clone(), block_table=table)
    ie.rope_kv_write(**ok)
    for bad in (dict(K=kv[:, :, :1]), dict(V=kv.double()), dict(inv_freq=f.double()), dict(Q=q[..., :32]), dict(positions=s),
                dict(out=q.half()), dict(K=kv.transpose(1, 2))):
        with pytest.raises(ValueError):
            ie.rope_kv_write(**(ok | bad))
    for bad in (dict(inv_freq=torch.ones(33, device=dev)), dict(out=q)):
        with pytest.raises(ie.IeError):
            ie.rope_kv_write(**(ok | bad))
    paths = i32([[0, 1]], dev)
    ie.kv_cache_keep([k], [k.clone()], table, s, paths, i32([2], dev))
    for bad in (([k], []), ([k], [k.half()]), ([k, k[:2]], [k, k])):
        with pytest.raises(ValueError):
            ie.kv_cache_keep(*bad, table, s, paths, i32([2], dev))
    with pytest.raises(ValueError):
        ie.kv_cache_keep([k], [k], table, s, s, i32([2], dev))

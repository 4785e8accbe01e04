"""include/ie_paged.h on the GPU at the edges of what it takes (paged_oracle has the tolerances)."""
import math

import numpy as np
import pytest
import torch

import paged_oracle as po
from conftest import rng
from paged_forms import ASKED, FORMS
from test_gpu_paged import case, check_ranges, i32, near, normal, ragged

pytestmark = pytest.mark.gpu
LARGEST = float(np.finfo(np.float32).max)


# ------------------------------------------------------------------ caps and slopes near the largest fp32
@pytest.mark.parametrize("kv,d,rows,groups,splits,call", FORMS)
def test_a_cap_that_no_score_feels(ie, dev, kv, d, rows, groups, splits, call):
    """The largest fp32 as a cap, which times log2(e) is no fp32 any more, is no cap; so is any that is as far off."""
    B, P, H, G, keys = call
    starts = ragged(rng(d + rows), B, keys - P)
    for cap in (LARGEST, 1e37, 1e26):
        check_ranges(ie, dev, rng(d + rows), B, P, H, G, d, 16, bool(kv), starts, cap=cap)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("P,G", [(1, 1), (2, 1), (3, 2), (100, 4)])
def test_slopes_of_the_largest_size(ie, dev, half, P, G):
    """A query sees itself alone, at distance 0."""
    r = rng(P)
    table, caches, q, top = case(r, dev, 2, P, 2, G, 64, 16, half, [0, 70])
    slopes = torch.full((2 * G,), LARGEST, device=dev)
    want = po.ranges(q, caches, table, 16, [0, 70], None, top, slopes=slopes)
    got = ie.paged_attn(q, *caches, i32(table, dev), i32([0, 70], dev), top, slopes=slopes)
    near(got, want)
    for b, s in enumerate((0, 70)):
        for h in range(2 * G):
            own = po.rows(caches[1], table[b], s + P, h // G)[s:]
            assert bool(((got[b, :, h].double() - own).abs() <= 2.0**-22 * own.abs()).all())


@pytest.mark.parametrize("kv,d,rows,groups,splits,call", FORMS)
def test_small_scales_of_large_queries(ie, dev, kv, d, rows, groups, splits, call):
    """A scale of 1e-28 for queries of 1e28: scores that the cap bends."""
    B, P, H, G, keys = call
    starts = ragged(rng(d + rows), B, keys - P)
    check_ranges(ie, dev, rng(d + rows), B, P, H, G, d, 16, bool(kv), starts, cap=5.0, scale=1e-28, q_scale=1e28)


# ------------------------------------------------------------------ ranges far apart
@pytest.mark.parametrize("kv,d,rows,groups,splits,call", [f for f in FORMS if f[5][1] > 1])
def test_pages_between_ranges_are_not_read(ie, dev, kv, d, rows, groups, splits, call):
    """Queries of a tile on separate passages: a table's entries between them are not looked up, so that what
    they lead to changes no bit."""
    B, P, H, G, keys = call
    r = rng(rows + d + splits)
    starts = [keys - P] * B
    block = 4
    table, caches, q, top = case(r, dev, B, P, H, G, d, block, bool(kv), starts)
    wide = max(1, keys // 9)
    begin = np.array([0, keys // 2 - wide // 2, keys - wide])
    which = r.integers(0, 3, (B, P))
    which[:, :2] = 0, 2
    first = begin[which]
    end = first + r.integers(1, wide + 1, (B, P))
    end[:, 5::7] = first[:, 5::7]  # some see nothing
    want = po.ranges(q, caches, table, block, starts, None, top, first, end)
    outs = []
    spare = caches[0].shape[0] - 1  # (no sequence's)
    seen = np.zeros((B, keys + block), bool)
    for b in range(B):
        for x, y in zip(first[b], end[b]):
            seen[b, x:y] = True
    used = np.stack([[seen[b, p * block:(p + 1) * block].any() for p in range(table.shape[1])] for b in range(B)])
    assert not used.all()
    table = np.where(used, table, spare)
    for fill in (0.0, float("nan")):
        for c in caches:
            c[spare] = fill
        outs.append(ie.paged_attn(q, *caches, i32(table, dev), i32(starts, dev), top, first=i32(first, dev), end=i32(end, dev)))
        near(outs[-1], want)
    assert torch.equal(*outs)


# ------------------------------------------------------------------ values near the largest fp32
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("P,G,d", [(1, 1, 64), (1, 1, 128), (2, 1, 64), (1, 2, 128), (1, 4, 64), (30, 1, 128), (100, 2, 64)])
@pytest.mark.parametrize("splits", [1, 3])
def test_weights_of_large_values(ie, dev, half, P, G, d, splits):
    """100 keys whose score is 5.3 above the 500 before them, values of 5e35: no 600 of them pass fp32's largest, four
    times the weight that the later keys have in the earlier ones' unit, 200, do."""
    r = rng(P + d)
    keys = 600
    table, caches, q, top = case(r, dev, 1, P, 1, G, d, 16, half, [keys - P])
    k = torch.zeros(keys, d)
    k[500:, 0] = 5.3
    place = i32(table[0], dev).long()[torch.arange(keys, device=dev) // 16], torch.arange(keys, device=dev) % 16
    caches[0][place] = k.to(dev)[:, None].to(caches[0].dtype)
    caches[1][place] = torch.full((keys, 1, d), 5e35, device=dev).to(caches[1].dtype)
    q.zero_()
    q[..., 0] = 1.0
    want = po.ranges(q, caches, table, 16, [keys - P], None, top, scale=1.0)
    near(ie.paged_attn(q, *caches, i32(table, dev), i32([keys - P], dev), top, scale=1.0, splits=splits), want)


@pytest.mark.parametrize("kv,d,rows,groups,splits,call", FORMS)
def test_sums_of_large_values(ie, dev, kv, d, rows, groups, splits, call):
    """Values up to 3e38, whose weighted sum before its division passes fp32's largest; the answer does not."""
    B, P, H, G, keys = call
    r = rng(rows + d)
    starts = ragged(r, B, keys - P)
    table, caches, q, top = case(r, dev, B, P, H, G, d, 16, bool(kv), starts, fill=0.0)
    caches[1].copy_(torch.rand(caches[1].shape, device=dev) * 2e38 + 1e38)
    want = po.ranges(q, caches, table, 16, starts, None, top)
    for s in {1, splits}:
        near(ie.paged_attn(q, *caches, i32(table, dev), i32(starts, dev), top, splits=s), want)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("P,G", [(1, 1), (2, 1), (3, 2), (100, 4)])
def test_an_infinite_value_that_is_seen(ie, dev, half, P, G):
    """It makes its channel infinite, with a weight of 2^-50 and with one of 2^-110 (an fp32 number all the same), and no other."""
    table, caches, q, top = case(rng(P), dev, 1, P, 1, G, 64, 16, half, [70])
    k, v = caches
    q.zero_()
    q[..., 0] = 1.0
    k[table[0, 0], :, :, 0] = 1.0
    for gap in (50, 110):
        k[..., 0] = 1.0
        k[table[0, 0], 3, :, 0] = 1.0 - gap / 2
        v[table[0, 0], 3, :, 7] = math.inf
        got = ie.paged_attn(q, k, v, i32(table, dev), i32([70], dev), top, scale=2 * math.log(2))
        assert bool((got[..., 7] == math.inf).all()) and bool(torch.isfinite(got[..., :7]).all()) and bool(torch.isfinite(got[..., 8:]).all())


# ------------------------------------------------------------------ far positions
def turns(pos, freq):
    """pos * freq / 2 pi less its whole turns, from 300 bits of pi."""
    one = 1 << 300

    def atan_inverse(x):
        term, total, n, sign = one // x, 0, 1, 1
        while term:
            total += sign * (term // n)
            term //= x * x
            n += 2
            sign = -sign
        return total

    two_pi = 8 * (4 * atan_inverse(5) - atan_inverse(239))
    out = []
    for f in freq:
        num, den = float(f).as_integer_ratio()
        rest = (pos * num * one // den) * one // two_pi % one
        out.append((rest - one if rest > one // 2 else rest) / one)
    return np.array(out)


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("pos", [0, 1, -1, 77, 10**5, 2**24 - 1, 2**30 + 12345, -2**31, 2**31 - 1])
def test_rope_angles(ie, dev, pairs, pos):
    """Cosines and sines of far positions and of frequencies above 1 against angles whose whole turns are taken off
    in integers.  A unit vector's rotation is its cosine and sine, each off by 4 U at most."""
    r = rng(5)
    freq = np.concatenate([10000.0 ** (-np.arange(24) / 24), r.random(20) * 3, r.random(10) * 100, [1.0, 0.0, 2.0, 64.0, 1e-30, 1e4, 1e6, 3.5, 0.1, 99.0]])
    freq = freq.astype(np.float32)
    x = torch.zeros(1, 1, 1, 128, device=dev)
    x[..., 0::2 if pairs else 1] = 1.0
    if not pairs:
        x[..., 64:] = 0.0
    kc = torch.zeros(1, 16, 1, 128, device=dev)
    got = ie.rope_kv_write(x, x, x, torch.from_numpy(freq).to(dev), i32([3], dev), kc, kc.clone(), i32([[0]], dev),
                           positions=i32([[pos]], dev), interleaved=pairs)[0, 0, 0].cpu().double().numpy()
    angle = 2 * math.pi * turns(pos, freq)
    cos, sin = (got[0::2], got[1::2]) if pairs else (got[:64], got[64:])
    assert np.abs(cos - np.cos(angle)).max() <= 4 * po.U and np.abs(sin - np.sin(angle)).max() <= 4 * po.U
    assert np.array_equal(kc[0, 3, 0].cpu().double().numpy(), got)


# ------------------------------------------------------------------ many sequences, long paths, many rows
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("B", [63, 64, 65, 100])
@pytest.mark.parametrize("P,G", [(1, 1), (2, 3), (20, 2)])
def test_many_sequences(ie, dev, half, B, P, G):
    """Up to 64 sequences come by length, more as they are."""
    r = rng(B + P)
    starts = ragged(r, B, 300)
    lens = [P] + [int(x) for x in r.integers(0, P + 1, B - 1)]
    check_ranges(ie, dev, r, B, P, 1, G, 64, 16, half, starts, lens)
    check_ranges(ie, dev, r, B, P, 1, G, 64, 16, half, starts, lens, splits=2)


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("n", [63, 64, 65, 128, 200])
def test_keep_long_paths(ie, dev, half, n):
    """Paths of more entries than a wave looks up at once: whole, cut at 64 and 65, ending at entry 64 by themselves."""
    r = rng(n)
    ctx = [0, 9, 40, 100]
    paths = [sorted(int(x) for x in r.choice(300, n, replace=False)) for _ in ctx]
    if n > 64:
        paths[2][64] = paths[2][63]  # ends there
    paths[3] = list(range(n))  # stays
    counts = [n, min(n, 64), n, n]
    moves = [paths[0], paths[1][:64], paths[2][:64], paths[3]]
    table, pages = po.tables(r, [c + 300 for c in ctx], 16)
    t = torch.bfloat16 if half else torch.float32
    k, v = (normal(r, dev, 2, pages, 16, 3, 64).to(t) for _ in range(2))
    want = [k.clone(), v.clone()]
    for w, c in zip(want, (k, v)):
        for b, move in enumerate(moves):
            for j, p in enumerate(move):
                x, y = ctx[b] + j, ctx[b] + p
                w[:, table[b, x // 16], x % 16] = c[:, table[b, y // 16], y % 16]
    ie.kv_cache_keep(list(k), list(v), i32(table, dev), i32(ctx, dev), i32(paths, dev), i32(counts, dev))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_a_join_of_many_rows(ie, dev):
    """More than 2^20 rows in six parts each."""
    r = rng(1)
    B, G, d = 70, 16384, 64
    starts = ragged(r, B, 700)
    table, caches, q, top = case(r, dev, B, 1, 1, 1, d, 16, True, starts)
    q = torch.randn(B, 1, G, d, device=dev, generator=torch.Generator(dev).manual_seed(2))
    got = ie.paged_attn(q, *caches, i32(table, dev), i32(starts, dev), top, splits=6)
    for h in ([0, 1, 2, 3], [G // 2 + 1], [G - 2, G - 1]):
        near(got[:, :, h], po.ranges(q[:, :, h].contiguous(), caches, table, 16, starts, None, top))


@pytest.mark.parametrize("kv,d,rows,groups,splits,call", ASKED)
def test_forms_in_asked_splits(ie, dev, kv, d, rows, groups, splits, call):
    """Forms that the plan splits only when asked, with ranges and as trees."""
    B, P, H, G, keys = call
    r = rng(rows + d)
    starts = ragged(r, B, keys - P)
    lens = [P] + [int(x) for x in r.integers(0, P + 1, B - 1)]
    check_ranges(ie, dev, r, B, P, H, G, d, 24, bool(kv), starts, lens, slopes=True, cap=20.0, splits=splits)
    first = r.integers(-5, keys, (B, P)).astype(np.int32)
    end = (first + r.integers(-30, keys, (B, P))).astype(np.int32)
    check_ranges(ie, dev, r, B, P, H, G, d, 16, bool(kv), starts, lens, first=first, end=end, splits=splits)
    table, caches, q, _ = case(r, dev, B, P, H, G, d, 16, bool(kv), starts)
    parents = [[int(r.integers(max(-1, t - 4), t)) if t else -1 for t in range(P)] for _ in range(B)]
    want = po.tree(q, caches, table, 16, starts, parents, lens, window=12)
    got = ie.tree_attn(q, *caches, i32(table, dev), i32(starts, dev), i32(parents, dev), max(starts), lens=i32(lens, dev), window=12,
                       splits=splits)
    near(got, want)


# ------------------------------------------------------------------ many workgroups of many stages, again and again
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("d,H,G,P,splits,kind", [(128, 8, 4, 4096, 1, "docs"), (64, 8, 4, 4096, 1, "docs"), (128, 8, 2, 2048, 1, "causal"),
                                                 (64, 4, 1, 2500, 1, "causal"), (128, 2, 8, 1000, 3, "causal"), (128, 4, 8, 255, 1, "tree"),
                                                 (64, 4, 8, 255, 3, "tree")])
def test_large_calls_repeat_their_bits(ie, dev, half, d, H, G, P, splits, kind):
    """150 calls of many workgroups at once, their waves at different speeds: each has the same bits, and they are right."""
    r = rng(P + d)
    B, starts = (2, [1500, 900]) if kind == "tree" else (1, [0])
    table, caches, q, top = case(r, dev, B, P, H, G, d, 32, half, starts)
    tb, at = i32(table, dev), i32(starts, dev)
    if kind == "tree":
        parents = [[int(r.integers(max(-1, t - 6), t)) if t else -1 for t in range(P)] for _ in range(B)]
        want = po.tree(q, caches, table, 32, starts, parents)
        pa = i32(parents, dev)
        call = lambda: ie.tree_attn(q, *caches, tb, at, pa, max(starts), splits=splits)
    else:
        cuts = np.sort(r.integers(0, P, P // 500))
        first = np.concatenate([[0], cuts])[np.searchsorted(cuts, np.arange(P), side="right")].astype(np.int32)[None] if kind == "docs" else None
        want = po.ranges(q, caches, table, 32, starts, None, top, first)
        fi = None if first is None else i32(first, dev)
        call = lambda: ie.paged_attn(q, *caches, tb, at, top, first=fi, splits=splits)
    got = call()
    near(got, want)
    different = sum((call() != got).any().long() for _ in range(150))
    assert int(different) == 0

"""The 8-bit KV cache on the GPU: its bytes against the rule in fp32 steps,
attention over it against 64 bits."""
import numpy as np
import pytest

import kv8_launch as kl
import kv8_oracle as ko
from conftest import rng

pytestmark = pytest.mark.gpu


def on(dev, *arrays):
    import torch

    out = [torch.from_numpy(np.ascontiguousarray(a)).to(dev) for a in arrays]
    return out if len(out) > 1 else out[0]


def same_bytes(want, got):
    k, v, ks, vs = got
    assert np.array_equal(want.ks, ks, equal_nan=True) and np.array_equal(want.vs, vs, equal_nan=True)
    assert np.array_equal(want.k, k)
    assert np.array_equal(want.v, v)


def rows(r, *shape, spread=0.5):
    """Values whose sizes differ from row to row and head to head."""
    return (r.standard_normal(shape) * np.exp(spread * r.standard_normal((*shape[:-1], 1)))).astype(np.float32)


# ------------------------------------------------------------------ writes and reads
@pytest.mark.parametrize("H,d,block", [(3, 64, 16), (2, 128, 16), (1, 64, 32), (2, 128, 64), (5, 64, 128), (2, 128, 128),
                                       (1, 64, 256), (2, 128, 256)])
@pytest.mark.parametrize("start,P", [(0, 1), (0, 16), (0, 300), (5, 7), (15, 2), (13, 290), (255, 2)])
def test_write(ie, dev, H, d, block, start, P):
    """Every byte after a prompt's write behind earlier rows; nothing else moves."""
    r = rng(H * 1000 + block + start + P)
    B = 2
    table, pages = ko.tables(r, [start + P] * B, block)
    want = ko.Cache(pages, H, d, block, r)
    for b in range(B):
        if start:
            want.write(rows(r, start, H, d), rows(r, start, H, d), table[b], 0)
    cache = want.tensors(ie, dev)
    K, V = rows(r, B, P, H, d), rows(r, B, P, H, d)
    for b in range(B):
        want.write(K[b], V[b], table[b], start)
    ie.kv8_cache_write(*on(dev, K, V), cache, on(dev, table), start)
    same_bytes(want, want.take(cache))
    # and back as values: code * scale rounds once
    n = start + P + 3
    starts, lens = np.array([0, start], np.int32), np.array([start + P, start + P], np.int32)
    gk, gv = ie.kv8_cache_read(cache, on(dev, table), *on(dev, starts, lens), n)
    for b in range(B):
        for h in range(H):
            k, v = want.rows(table[b], start + P, h)
            for got, ref in ((gk, k), (gv, v)):
                got = got[b, :, h].cpu().numpy()
                m = start + P - starts[b]
                assert np.array_equal(got[:m], ref[starts[b]:].astype(np.float32))
                assert not got[m:].any()


def test_write_takes_a_projections_columns(ie, dev):
    r = rng(5)
    B, P, H, d, block = 2, 21, 3, 64, 16
    table, pages = ko.tables(r, [P] * B, block)
    want = ko.Cache(pages, H, d, block, r)
    cache = want.tensors(ie, dev)
    qkv = rows(r, B, P, 3, H, d)
    for b in range(B):
        want.write(qkv[b, :, 1], qkv[b, :, 2], table[b], 0)
    t = on(dev, qkv)
    ie.kv8_cache_write(t[:, :, 1], t[:, :, 2], cache, on(dev, table), 0)
    same_bytes(want, want.take(cache))


@pytest.mark.parametrize("H,d,block", [(12, 64, 16), (2, 128, 16), (3, 64, 64), (2, 128, 256)])
def test_append(ie, dev, H, d, block):
    """Token by token from empty, each sequence at its own place; left-out ones stay as they were."""
    r = rng(H + d)
    n, B = 2 * block + 3, 4
    table, pages = ko.tables(r, [n + 3] * B, block)
    want = ko.Cache(pages, H, d, block, r)
    cache, tab = want.tensors(ie, dev), on(dev, table)
    for i in range(n if block < 256 else 40):
        K, V = rows(r, B, H, d, spread=1.0), rows(r, B, H, d, spread=1.0)
        at = np.array([i, i + 3 if i else 0, -1, table.shape[1] * block], np.int32)
        if i == 1:  # sequence 1 jumps ahead: its page's rows between are written first
            for j in (1, 2, 3):
                k1, v1 = rows(r, 1, H, d), rows(r, 1, H, d)
                want.write(k1, v1, table[1], j)
                ie.kv8_cache_append_batch(*on(dev, k1, v1), cache, tab[1:2], on(dev, np.array([j], np.int32)))
        for b in (0, 1):
            want.write(K[b:b + 1], V[b:b + 1], table[b], at[b])
        ie.kv8_cache_append_batch(*on(dev, K, V), cache, tab, on(dev, at))
    same_bytes(want, want.take(cache))


def test_error_of_grown_pages(ie, dev):
    """Rows that grow by a little each time: a value stays within 2.5 scales of what was appended (and a rounding's
    error of the products), within half a scale where the page came at once."""
    H, d, block = 2, 64, 64
    r = rng(9)
    table = np.arange(2, dtype=np.int32).reshape(2, 1)
    cache = ie.Kv8Cache.empty(2, H, d, block, dev)
    K = rows(r, block, H, d, spread=0.0) * (1.03 ** np.arange(block, dtype=np.float32))[:, None, None]
    tab, k = on(dev, table, K)
    for i in range(block):
        ie.kv8_cache_append_batch(k[i:i + 1], k[i:i + 1], cache, tab[:1], on(dev, np.array([i], np.int32)))
    ie.kv8_cache_write(k[None], k[None], cache, tab[1:], 0)
    zero, full = on(dev, np.zeros(2, np.int32), np.full(2, block, np.int32))
    got, _ = ie.kv8_cache_read(cache, tab, zero, full, block)
    scale = cache.k_scale.cpu().numpy().astype(np.float64)
    err = np.abs(got.cpu().numpy().astype(np.float64) - K)
    assert (err[0] <= (2.5 + 1e-4) * scale[0][None, :, None]).all()
    assert (err[1] <= (0.5 + 1e-4) * scale[1][None, :, None]).all()


def test_extreme_values(ie, dev):
    """Zeros, the smallest and largest numbers, infinities and NaN: the rule's bytes, and reads that show them."""
    H, d, block = 6, 64, 16
    r = rng(2)
    table, pages = ko.tables(r, [20], block)
    K = rows(r, 20, H, d)
    K[:, 0] = 0.0
    K[:, 1] *= np.float32(1e-42)
    K[:, 2] = np.where(K[:, 2] > 0, np.float32(3.4e38), np.float32(-3.4e38))
    K[3, 3, 5] = np.inf
    K[17, 4, 9] = np.nan
    want = ko.Cache(pages, H, d, block, r)
    cache = want.tensors(ie, dev)
    tab, k = on(dev, table, K)
    want.write(K[:18], K[:18], table[0], 0)
    ie.kv8_cache_write(k[None, :18], k[None, :18], cache, tab, 0)
    for i in (18, 19):
        want.write(K[i:i + 1], K[i:i + 1], table[0], i)
        ie.kv8_cache_append_batch(k[i:i + 1], k[i:i + 1], cache, tab, on(dev, np.array([i], np.int32)))
    same_bytes(want, want.take(cache))
    Q = rows(r, 1, H, d)
    o = ie.decode_attn_kv8(on(dev, Q), cache, tab, on(dev, np.array([20], np.int32)), 20).cpu().numpy()[0]
    assert not o[0].any() and np.isnan(o[3]).all() and np.isnan(o[4]).all() and np.isfinite(o[5]).all()


# ------------------------------------------------------------------ attention
def filled(r, lens, H, d, block, sizes=1.0):
    table, pages = ko.tables(r, lens, block)
    c = ko.Cache(pages, H, d, block, r)
    for b, n in enumerate(lens):
        if n:
            c.write(rows(r, n, H, d) * np.float32(sizes), rows(r, n, H, d), table[b], 0)
    return c, table


def check_decode(ie, dev, c, table, lens, Q, max_ctx, splits=0):
    cache, tab = c.tensors(ie, dev), on(dev, table)
    got = ie.decode_attn_kv8(on(dev, Q), cache, tab, on(dev, np.array(lens, np.int32)), max_ctx, splits=splits)
    got = got.cpu().numpy()
    G = Q.shape[1] // c.heads
    for b, n in enumerate(lens):
        for hq in range(Q.shape[1]):
            if n == 0:
                assert not got[b, hq].any()
                continue
            ref, tol = ko.attend(Q[b, hq], *c.rows(table[b], n, hq // G))
            assert np.abs(got[b, hq] - ref).max() <= tol, (b, hq, n)
    return got


@pytest.mark.parametrize("H,G,d,block", [(3, 1, 64, 16), (2, 3, 64, 32), (2, 4, 128, 16), (1, 8, 128, 64), (2, 2, 128, 128),
                                         (1, 12, 64, 16), (1, 5, 128, 256), (2, 17, 64, 16)])
@pytest.mark.parametrize("lens", [[1], [0, 1, 2, 15, 16, 17], [63, 64, 65, 0], [127, 129, 700, 5], [1030]])
def test_decode(ie, dev, H, G, d, block, lens):
    r = rng(H + 10 * G + d + len(lens))
    c, table = filled(r, lens, H, d, block)
    Q = rows(r, len(lens), H * G, d)
    first = check_decode(ie, dev, c, table, lens, Q, max(lens))
    for splits in (1, 2, 5, 64):
        check_decode(ie, dev, c, table, lens, Q, max(lens), splits)
    assert np.array_equal(first, check_decode(ie, dev, c, table, lens, Q, max(lens)))


def test_decode_all_empty(ie, dev):
    r = rng(3)
    c, table = filled(r, [0, 0], 2, 64, 16)
    check_decode(ie, dev, c, table, [0, 0], rows(r, 2, 4, 64), 0)
    check_decode(ie, dev, c, np.zeros((2, 9), np.int32), [0, 0], rows(r, 2, 4, 64), 140)


def test_decode_takes_lens_as_at_most_the_limit(ie, dev):
    """A device length past max_context_len, and a negative one, read nothing out of range."""
    r = rng(4)
    c, table = filled(r, [40, 40], 2, 64, 16)
    Q = rows(r, 2, 4, 64)
    got = ie.decode_attn_kv8(on(dev, Q), c.tensors(ie, dev), on(dev, table), on(dev, np.array([10**9, -7], np.int32)), 40)
    got = got.cpu().numpy()
    for hq in range(4):
        ref, tol = ko.attend(Q[0, hq], *c.rows(table[0], 40, hq // 2))
        assert np.abs(got[0, hq] - ref).max() <= tol
    assert not got[1].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["rising", "falling", "one", "far", "tiny", "huge"])
def test_decode_uneven_scores(ie, dev, d, kind):
    """Scores whose maximum moves all along, one key that outweighs all, pages of very different sizes, queries at the
    ends of the range."""
    r = rng(d + len(kind))
    n, H = 900, 2
    table, pages = ko.tables(r, [n], 16)
    c = ko.Cache(pages, H, d, 16, r)
    K, V = rows(r, n, H, d, spread=0.2), rows(r, n, H, d, spread=0.2)
    Q = rows(r, 1, H, d, spread=0.2)
    if kind in ("rising", "falling"):
        ramp = np.linspace(0, 6, n) * (1 if kind == "rising" else -1)
        K = (K + ramp[:, None, None] * Q[0][None] / np.linalg.norm(Q[0], axis=-1)[None, :, None]).astype(np.float32)
    if kind == "one":
        K[513] = 4 * Q[0]
    if kind == "far":
        V *= np.exp(4 * r.standard_normal((n // 15, 1, 1)).repeat(15, 0)).astype(np.float32)
        K *= np.exp(1.5 * r.standard_normal((n // 30, 1, 1)).repeat(30, 0)).astype(np.float32)
    if kind == "tiny":
        Q *= np.float32(1e-41)
    if kind == "huge":
        Q, K = Q * np.float32(1e30), K * np.float32(1e-30)
    c.write(K, V, table[0], 0)
    check_decode(ie, dev, c, table, [n], Q, n)
    check_prompt(ie, dev, c, table, n - 33, np.repeat(Q[:, None], 33, 1))


def check_prompt(ie, dev, c, table, start, Q):
    B, P, H_q, d = Q.shape
    cache, tab = c.tensors(ie, dev), on(dev, table)
    got = ie.prefill_attn_kv8(on(dev, Q), cache, tab, start).cpu().numpy()
    G = H_q // c.heads
    for b in range(B):
        for h in range(c.heads):
            k, v = c.rows(table[b], start + P, h)
            for t in range(P):
                for g in range(G):
                    ref, tol = ko.attend(Q[b, t, h * G + g], k[:start + t + 1], v[:start + t + 1])
                    assert np.abs(got[b, t, h * G + g] - ref).max() <= tol, (b, t, h, g)
    return got


@pytest.mark.parametrize("H,G,d,block", [(3, 1, 64, 16), (2, 3, 64, 32), (1, 4, 128, 16), (1, 2, 128, 128), (1, 9, 64, 256)])
@pytest.mark.parametrize("start,P", [(0, 1), (0, 15), (0, 16), (0, 65), (0, 200), (1, 1), (17, 3), (63, 2), (100, 140),
                                     (600, 33)])
def test_prompt(ie, dev, H, G, d, block, start, P):
    r = rng(H + 10 * G + d + start + P)
    B = 2
    c, table = filled(r, [start + P] * B, H, d, block)
    Q = rows(r, B, P, H * G, d)
    got = check_prompt(ie, dev, c, table, start, Q)
    assert np.array_equal(got, check_prompt(ie, dev, c, table, start, Q))


# ------------------------------------------------------------------ the prompt's forms
# By workgroups of 64 rows (row: token x query head of a KV head): for up to 32 rows a head, below 128 and, behind a
# context of many tiles, below 256 the split form, the contexts behind few rows cut; else two teams a block, from 1024
# one, with 32 rows a wave where d = 128.
FORMS = [(2, 3, 2, 64, 16, 300, 9), (1, 2, 3, 128, 64, 4100, 5), (8, 32, 1, 64, 16, 40, 20), (3, 16, 4, 128, 32, 60, 13),
         (2, 16, 1, 128, 16, 700, 200),
         # cut contexts: two teams (two and five parts), one team, 32 rows a wave in ten and four parts, two rounds
         (1, 8, 4, 128, 16, 1300, 77), (1, 12, 1, 64, 32, 1400, 200), (1, 12, 4, 64, 16, 3200, 120), (2, 12, 2, 64, 64, 1700, 400),
         (1, 16, 4, 128, 16, 5300, 80), (1, 8, 4, 128, 32, 2200, 500), (2, 16, 2, 128, 16, 1000, 600),
         (2, 12, 1, 128, 32, 0, 1536),  # (its first blocks have fewer tiles than parts)
         (4, 16, 1, 64, 16, 0, 250), (4, 16, 1, 128, 32, 37, 251), (2, 16, 3, 128, 64, 5, 177), (16, 16, 4, 64, 256, 0, 13),
         (8, 32, 1, 64, 16, 0, 250), (8, 32, 1, 128, 16, 100, 249), (4, 32, 5, 128, 64, 3, 103), (16, 64, 2, 64, 128, 0, 1)]


def prompt_in_64_bits(dev, c, table, start, Q):
    """(outputs, tolerances a row) as ko.attend, for all rows at once."""
    import torch

    B, P, H_q, d = Q.shape
    G, n = H_q // c.heads, start + P
    seen = torch.arange(n, device=dev) <= start + torch.arange(P, device=dev)[:, None]
    out, tol = torch.empty((B, P, H_q, d), dtype=torch.float64), torch.empty((B, P, H_q), dtype=torch.float64)
    for b in range(B):
        for h in range(c.heads):
            k, v = on(dev, *c.rows(table[b], n, h))
            kt, ka = k.T.contiguous(), k.abs().T.contiguous()
            for hq in range(h * G, (h + 1) * G):
                q = on(dev, Q[b, :, hq]).double()
                s = (q @ kt / d**0.5).masked_fill(~seen, -float("inf"))
                S = (q.abs() @ ka / d**0.5).masked_fill(~seen, 0).amax(1)
                most = torch.cummax(v.abs().amax(1), 0).values[start:]
                out[b, :, hq] = (torch.softmax(s, 1) @ v).cpu()
                tol[b, :, hq] = ((46 * S + 24 + seen.sum(1) / 16) * ko.U * most).cpu()
    return out.numpy(), tol.numpy()


@pytest.mark.parametrize("B,H,G,d,block,start,P", FORMS)
def test_prompt_forms(ie, dev, B, H, G, d, block, start, P):
    r = rng(B + H + G + d + start + P)
    c, table = filled(r, [start + P] * B, H, d, block)
    Q = rows(r, B, P, H * G, d)
    want, tol = prompt_in_64_bits(dev, c, table, start, Q)
    cache, tab, q = c.tensors(ie, dev), on(dev, table), on(dev, Q)
    got = ie.prefill_attn_kv8(q, cache, tab, start)
    assert (np.abs(got.cpu().numpy() - want).max(-1) <= tol).all()
    assert np.array_equal(got.cpu().numpy(), ie.prefill_attn_kv8(q, cache, tab, start).cpu().numpy())
    # without a workspace: the context in one piece
    whole = got.clone().fill_(7)
    ie.check("ie_prefill_attn_kv8", B, P, H * G, H, d, q.data_ptr(), *(t.data_ptr() for t in cache), tab.data_ptr(),
             tab.shape[1], block, start, whole.data_ptr(), None, 0, ie._stream())
    assert (np.abs(whole.cpu().numpy() - want).max(-1) <= tol).all()
    need = ie.call("ie_prefill_kv8_workspace_bytes", B, P, H * G, H, d, start)
    if need:
        import torch

        with pytest.raises(ie.IeError):
            ie.prefill_attn_kv8(q, cache, tab, start, workspace=torch.empty(need // 4 - 1, device=dev))


@pytest.mark.parametrize("bad", ["k", "v"])
@pytest.mark.parametrize("B,H,G,d,block,start,P", FORMS)
def test_prompt_rows_before_a_bad_page(ie, dev, B, H, G, d, block, start, P, bad):
    """A page whose scale is not finite: NaN for the rows that see a token of it, for the others the bits they had."""
    r = rng(B + H + G + d + start + P)
    c, table = filled(r, [start + P] * B, H, d, block)
    q, tab = on(dev, rows(r, B, P, H * G, d)), on(dev, table)
    good = ie.prefill_attn_kv8(q, c.tensors(ie, dev), tab, start).cpu().numpy()
    pages = range(start // block, (start + P - 1) // block + 1)
    at = pages[(len(pages) + 1) // 2 if len(pages) > 2 else -1]
    scales = c.ks if bad == "k" else c.vs
    scales[table[0, at], 0] = np.inf if bad == "k" else np.nan
    got = ie.prefill_attn_kv8(q, c.tensors(ie, dev), tab, start).cpu().numpy()
    hit = np.zeros(good.shape[:3], bool)
    hit[0, max(0, at * block - start):, :G] = True
    assert np.isnan(got[hit]).all()
    assert np.array_equal(got[~hit], good[~hit])


def test_nothing_behind_the_context_counts(ie, dev):
    """Pages past the end (their table entries out of range) and rows behind it, whatever they hold: the bits of the
    answer do not move."""
    r = rng(8)
    H, G, d, block, n = 2, 2, 64, 32, 70
    c, table = filled(r, [n], H, d, block)
    Q = rows(r, 1, H * G, d)
    a = check_decode(ie, dev, c, table, [n], Q, n)
    c.k[table[0, 2], :, 6:], c.v[table[0, 2], :, 6:] = 127, -128
    wide = np.full((1, 40), 2**30, np.int32)
    wide[0, :3] = table[0, :3]
    assert np.array_equal(a, check_decode(ie, dev, c, wide, [n], Q, n))
    p = check_prompt(ie, dev, c, wide, n - 5, np.repeat(Q[:, None], 5, 1))
    c.k[table[0, 2], :, 6:], c.v[table[0, 2], :, 6:] = -128, 127
    assert np.array_equal(p, check_prompt(ie, dev, c, wide, n - 5, np.repeat(Q[:, None], 5, 1)))


def test_past_4_gib(ie, dev):
    """Page offsets that 32 bits do not hold."""
    import torch

    H, d, block = 8, 128, 64
    pages = (5 << 30) // (H * d * block)
    cache = ie.Kv8Cache.empty(pages, H, d, block, dev)
    r = rng(11)
    n = 150
    far = np.array([[pages - 1, pages - 7, pages - 3]], np.int32)
    c = ko.Cache(3, H, d, block)
    c.write(K := rows(r, n, H, d), V := rows(r, n, H, d), np.arange(3), 0)
    tab = on(dev, far)
    ie.kv8_cache_write(on(dev, K)[None], on(dev, V)[None], cache, tab, 0)
    Q = rows(r, 1, H, d)
    got = ie.decode_attn_kv8(on(dev, Q), cache, tab, on(dev, np.array([n], np.int32)), n).cpu().numpy()
    pre = ie.prefill_attn_kv8(on(dev, Q)[None], cache, tab, n - 1).cpu().numpy()[0]
    back, _ = ie.kv8_cache_read(cache, tab, *on(dev, np.zeros(1, np.int32), np.array([n], np.int32)), n)
    for h in range(H):
        k, v = c.rows(np.arange(3), n, h)
        ref, tol = ko.attend(Q[0, h], k, v)
        assert np.abs(got[0, h] - ref).max() <= tol and np.abs(pre[0, h] - ref).max() <= tol
        assert np.array_equal(back[0, :, h].cpu().numpy(), k.astype(np.float32))
    del cache
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ together, streams, graphs, refusals
def test_a_prompt_then_tokens(ie, dev):
    """A batch's prompt chunks, then decode steps, all over one cache as a serving loop runs them."""
    r = rng(21)
    B, H, G, d, block = 3, 2, 2, 64, 16
    chunks, steps = (37, 20), 20
    total = sum(chunks) + steps
    table, pages = ko.tables(r, [total] * B, block)
    c = ko.Cache(pages, H, d, block, r)
    cache, tab = c.tensors(ie, dev), on(dev, table)
    at = 0
    for P in chunks:
        qkv = rows(r, B, P, H * (G + 2), d)
        t = on(dev, qkv)
        for b in range(B):
            c.write(qkv[b, :, H * G:H * G + H], qkv[b, :, H * G + H:], table[b], at)
        ie.kv8_cache_write(t[:, :, H * G:H * G + H], t[:, :, H * G + H:], cache, tab, at)
        got = ie.prefill_attn_kv8(t[:, :, :H * G].contiguous(), cache, tab, at).cpu().numpy()
        assert np.array_equal(got, check_prompt(ie, dev, c, table, at, qkv[:, :, :H * G]))
        at += P
    for _ in range(steps):
        K, V, Q = rows(r, B, H, d), rows(r, B, H, d), rows(r, B, H * G, d)
        for b in range(B):
            c.write(K[b:b + 1], V[b:b + 1], table[b], at)
        ie.kv8_cache_append_batch(*on(dev, K, V), cache, tab, on(dev, np.full(B, at, np.int32)))
        at += 1
        got = ie.decode_attn_kv8(on(dev, Q), cache, tab, on(dev, np.full(B, at, np.int32)), total).cpu().numpy()
        for b in range(B):
            for hq in range(H * G):
                ref, tol = ko.attend(Q[b, hq], *c.rows(table[b], at, hq // G))
                assert np.abs(got[b, hq] - ref).max() <= tol
    same_bytes(c, c.take(cache))


def test_graph_and_stream(ie, dev):
    """A captured append + attention step replayed as positions move, with eager work between, and the same on a side
    stream: the eager bits each time."""
    import torch

    r = rng(31)
    B, H, d, block, n0, steps = 2, 3, 64, 16, 600, 5
    table, pages = ko.tables(r, [n0 + steps] * B, block)
    c = ko.Cache(pages, H, d, block, r)
    for b in range(B):
        c.write(rows(r, n0, H, d), rows(r, n0, H, d), table[b], 0)
    tab = on(dev, table)
    K, V, Q = (on(dev, rows(r, steps, B, H, d)) for _ in range(3))

    def fresh():
        return c.tensors(ie, dev), torch.full((B,), n0, dtype=torch.int32, device=dev)

    cache, pos = fresh()
    want = []
    for i in range(steps):
        ie.kv8_cache_append_batch(K[i], V[i], cache, tab, pos)
        want.append(ie.decode_attn_kv8(Q[i], cache, tab, pos + 1, n0 + steps, splits=4))
        pos += 1
    side = torch.cuda.Stream()
    cache, pos = fresh()
    lens = pos + 1
    torch.cuda.synchronize()  # what the side stream reads is written
    ie.kv8_cache_append_batch(K[0], V[0], cache, tab, pos, stream=side)
    got = ie.decode_attn_kv8(Q[0], cache, tab, lens, n0 + steps, splits=4, stream=side)
    side.synchronize()
    assert torch.equal(got, want[0])

    cache, pos = fresh()
    k, v, q, lens = K[0].clone(), V[0].clone(), Q[0].clone(), torch.empty_like(pos)
    out = torch.empty_like(q)
    ws = torch.empty(B * H * 4 * (d + 2), device=dev)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ie.kv8_cache_append_batch(k, v, cache, tab, pos)
        torch.add(pos, 1, out=lens)
        ie.decode_attn_kv8(q, cache, tab, lens, n0 + steps, splits=4, out=out, workspace=ws)
    for i in range(steps):
        for a, x in ((k, K[i]), (v, V[i]), (q, Q[i])):
            a.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        pos += 1
        (Q[i] * 2).sum().item()


def test_results_made_for_another_stream(ie, dev):
    """What a call on a given stream allocates comes from that stream's memory: work of the current stream that is still
    under way on memory freed there cannot meet it."""
    import torch

    cache, tab = ie.Kv8Cache.empty(4, 2, 64, 16, dev), torch.arange(4, dtype=torch.int32, device=dev)[None]
    K = torch.ones(1, 40, 2, 64, device=dev)
    ie.kv8_cache_write(K, K, cache, tab, 0)
    lens, x = torch.full((1,), 40, dtype=torch.int32, device=dev), torch.ones(64, 2 * 64, device=dev)
    side = torch.cuda.Stream()
    calls = [lambda s: ie.decode_attn_kv8(K[:, 0], cache, tab, lens, 64, stream=s),
             lambda s: ie.prefill_attn_kv8(K, cache, tab, 0, stream=s),
             lambda s: ie.kv8_cache_read(cache, tab, lens * 0, lens, 40, stream=s)[1],
             lambda s: ie.token_logprobs(x, None, 3, stream=s).top_logprobs]
    torch.cuda.synchronize()
    for call in calls:
        used = {call(None).data_ptr() for _ in range(4)}  # freed at once, ready for the current stream's next
        got = call(side)
        side.synchronize()
        assert got.data_ptr() not in used
        assert torch.equal(got, call(None))


def test_two_streams_at_once(ie, dev):
    """Calls under way on two streams, each with its cache and what the binding makes for it: the bits of one alone."""
    import torch

    r = rng(41)
    H, G, d, block, n, P = 2, 4, 128, 16, 2000, 40
    work = []
    for i in range(2):
        c, table = filled(r, [n], H, d, block)
        q = on(dev, rows(r, 1, P, H * G, d))
        work.append((q, q[:, 0].contiguous(), c.tensors(ie, dev), on(dev, table), on(dev, np.array([n], np.int32))))

    def both(w, stream=None):
        q, q1, cache, tab, lens = w
        return ie.prefill_attn_kv8(q, cache, tab, n - P, stream=stream), ie.decode_attn_kv8(q1, cache, tab, lens, n, splits=8, stream=stream)

    want = [both(w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = [[], []]
    for _ in range(20):
        for i, w in enumerate(work):
            got[i].append(both(w, streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


def test_binding_refusals(ie, dev):
    import torch

    cache = ie.Kv8Cache.empty(4, 2, 64, 16, dev)
    tab = torch.zeros(1, 4, dtype=torch.int32, device=dev)
    K = torch.zeros(1, 3, 2, 64, device=dev)
    lens = torch.ones(1, dtype=torch.int32, device=dev)
    bad = [
        lambda: ie.kv8_cache_write(K.half(), K.half(), cache, tab, 0),
        lambda: ie.kv8_cache_write(K.cpu(), K.cpu(), cache, tab, 0),
        lambda: ie.kv8_cache_write(K.transpose(2, 3), K.transpose(2, 3), cache, tab, 0),
        lambda: ie.kv8_cache_write(K, K, cache, tab.long(), 0),
        lambda: ie.kv8_cache_write(K, K, cache, tab.repeat(2, 1), 0),
        lambda: ie.kv8_cache_write(K, K, cache._replace(v=cache.v[:2]), tab, 0),
        lambda: ie.decode_attn_kv8(K[0], cache, tab, lens, 3),
        lambda: ie.decode_attn_kv8(K[:, 0, :, :32], cache, tab, lens, 3),
        lambda: ie.decode_attn_kv8(K[:, 0], cache, tab, lens.long(), 3),
        lambda: ie.prefill_attn_kv8(K.double(), cache, tab, 0),
        lambda: ie.kv8_cache_append_batch(K[:, 0], K[:, 0], cache, tab, lens.repeat(2)),
        lambda: ie.kv8_cache_read(cache, tab, lens.float(), None, 3),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(ie.IeError):
        ie.kv8_cache_write(K, K, cache, tab, 62)
    Q = K[:, 0].contiguous()
    with pytest.raises(ie.IeError):
        ie.decode_attn_kv8(Q, cache, tab, lens, 64, splits=1, out=Q)


@pytest.mark.parametrize("B,H,G,d,start,P", [(1, 1, 1, 64, 500, 1), (8, 32, 1, 64, 330, 20), (2, 12, 1, 64, 330, 300),
                                             (2, 16, 2, 128, 330, 100), (4, 32, 1, 64, 330, 510), (4, 32, 2, 128, 330, 260)])
def test_large_values_behind_a_page_of_zeros(ie, dev, B, H, G, d, start, P):
    """Values of 1e20 at keys of score 0, zeros (whose page has the least scale) at one of score about 70: the large ones
    are all that the output has, e^-70 of them.  Values are positive, so the output is off by twice its weights' relative
    error (kv8_oracle.attend), whatever its size; before and behind the jump, in each of the prompt's forms and for one
    token."""
    r = rng(d + P)
    n, high = start + P, 4 * 64 + 5
    table, pages = ko.tables(r, [n] * B, 16)
    c = ko.Cache(pages, H, d, 16, r)
    q = rows(r, 1, H, 1, d, spread=0.0).repeat(G, 2)  # one query a KV head
    K, V = np.zeros((n, H, d), np.float32), np.zeros((n, H, d), np.float32)
    K[high] = 70 * d**0.5 * q[0, :, 0] / (q[0, :, 0] ** 2).sum(-1, keepdims=True)
    V[:64] = (1e20 * np.abs(1 + 0.1 * r.standard_normal((64, H, d)))).astype(np.float32)
    for b in range(B):
        c.write(K, V, table[b], 0)
    Q = np.broadcast_to(q.reshape(1, 1, H * G, d), (B, P, H * G, d)).copy()
    want, _ = prompt_in_64_bits(dev, c, table, start, Q)
    tol = (46 * 71 + 24 + n / 16) * ko.U
    cache, tab = c.tensors(ie, dev), on(dev, table)
    got = ie.prefill_attn_kv8(on(dev, Q), cache, tab, start).cpu().numpy()
    assert (np.abs(got - want) <= tol * want).all(), (got / want).min()
    lens = on(dev, np.full(B, n, np.int32))
    for splits in (1, 2):
        got = ie.decode_attn_kv8(on(dev, Q[:, 0]), cache, tab, lens, n, splits=splits).cpu().numpy()
        assert (np.abs(got - want[:, -1]) <= tol * want[:, -1]).all()


@pytest.mark.parametrize("value", [1e5, 1e9, 1e20, 1e33])
@pytest.mark.parametrize("B,H,G,d,start,P", [(1, 1, 1, 64, 100, 1), (8, 32, 1, 64, 130, 20), (2, 12, 1, 64, 130, 300),
                                             (2, 16, 2, 128, 130, 100), (4, 32, 2, 128, 130, 260)])
def test_large_values_beside_a_page_of_zeros(ie, dev, B, H, G, d, start, P, value):
    """The same within a tile, at a distance of 81: a weight is e^-81, the large values' scale is more than 2^127 units of
    the weights, their product is a number like any other."""
    r = rng(d + P)
    n, high = start + P, 20
    table, pages = ko.tables(r, [n] * B, 16)
    c = ko.Cache(pages, H, d, 16, r)
    q = rows(r, 1, H, 1, d, spread=0.0).repeat(G, 2)
    K, V = np.zeros((n, H, d), np.float32), np.zeros((n, H, d), np.float32)
    K[high] = 81 * d**0.5 * q[0, :, 0] / (q[0, :, 0] ** 2).sum(-1, keepdims=True)
    V[:16] = (value * np.abs(1 + 0.1 * r.standard_normal((16, H, d)))).astype(np.float32)
    for b in range(B):
        c.write(K, V, table[b], 0)
    Q = np.broadcast_to(q.reshape(1, 1, H * G, d), (B, P, H * G, d)).copy()
    want, _ = prompt_in_64_bits(dev, c, table, start, Q)
    tol = (46 * 82 + 24 + n / 16) * ko.U
    cache, tab = c.tensors(ie, dev), on(dev, table)
    got = ie.prefill_attn_kv8(on(dev, Q), cache, tab, start).cpu().numpy()
    assert (np.abs(got - want) <= tol * want).all(), (got / want).min()
    lens = on(dev, np.full(B, n, np.int32))
    for splits in (1, 2):
        got = ie.decode_attn_kv8(on(dev, Q[:, 0]), cache, tab, lens, n, splits=splits).cpu().numpy()
        assert (np.abs(got - want[:, -1]) <= tol * want[:, -1]).all(), (got / want[:, -1]).max()


# ------------------------------------------------------------------ append and attention in one launch
@pytest.mark.parametrize("H,G,d,block", [(12, 1, 64, 16), (2, 4, 128, 16), (3, 2, 64, 64)])
def test_append_and_attention_in_one_launch(ie, dev, H, G, d, block):
    """The launch of the engine's fused step against the two entry points: rows within the limit, at it and past it, past
    the table's end and at no position (the sequence is left out, its output zero)."""
    import torch

    r = rng(H + G + block)
    max_ctx, room = 90, 128
    pos = [0, 1, block - 1, block, 40, max_ctx - 1, max_ctx, max_ctx + 20, room - 1, room, 2**31 - 1, -1, -(2**31)]
    B = len(pos)
    table, pages = ko.tables(r, [room] * B, block)
    c = ko.Cache(pages, H, d, block, r)
    for b, p in enumerate(pos):
        n = min(max(p, 0), room)
        c.write(rows(r, n, H, d), rows(r, n, H, d), table[b], 0)
    K, V, Q = (on(dev, rows(r, B, n, d)) for n in (H, H, H * G))
    tab, p = on(dev, table), on(dev, np.array(pos, np.int32))
    two, one = c.tensors(ie, dev), c.tensors(ie, dev)
    ie.kv8_cache_append_batch(K, V, two, tab, p)
    lens = on(dev, np.array([q + 1 if 0 <= q < room else 0 for q in pos], np.int32))
    want = ie.decode_attn_kv8(Q, two, tab, lens, max_ctx, splits=1)
    got = torch.full_like(want, 7)
    a = kl.AttnArgs(B=B, P=1, H_q=H * G, Q=Q.data_ptr(), q_ld=H * G * d, max_ctx=max_ctx, O=got.data_ptr(), splits=1,
                    K=K.data_ptr(), V=V.data_ptr(), kv_ld=H * d, positions=p.data_ptr(),
                    c=kl.CacheArgs(*(t.data_ptr() for t in one), tab.data_ptr(), tab.shape[1], H, d, block.bit_length() - 1))
    assert kl.launch(ie, "decode", a, ie._stream()) == 0
    torch.cuda.synchronize()
    for x, y in zip(one, two):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert torch.equal(got, want)
    assert not got[-4:].any()


def test_rows_farther_apart_than_the_entry_points_take(ie, dev):
    """Distances between rows past 32 bits, and positions past them, are refused, not taken modulo 2^32."""
    import torch

    far = 2**32 + 512
    buf = torch.zeros(far + 512, device=dev)
    cache, tab = ie.Kv8Cache.empty(4, 2, 64, 16, dev), torch.arange(4, dtype=torch.int32, device=dev)[None]
    K = buf.as_strided((1, 2, 2, 64), (2 * far, far, 64, 1))
    with pytest.raises(ValueError):
        ie.kv8_cache_write(K, K, cache, tab, 0)
    with pytest.raises(ValueError):
        ie.kv8_cache_append_batch(K[0], K[0], cache, tab.expand(2, 4).contiguous(), torch.zeros(2, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        ie.token_logprobs(buf.as_strided((2, 500), (far, 1)), None, 3)
    x, lens = torch.zeros(1, 2, 2, 64, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    for f in (lambda: ie.kv8_cache_write(x, x, cache, tab, 2**32), lambda: ie.prefill_attn_kv8(x, cache, tab, 2**32),
              lambda: ie.decode_attn_kv8(x[:, 0].contiguous(), cache, tab, lens, 2**32 + 1)):
        with pytest.raises(ValueError):
            f()
    # (a single row's distance to the next one counts for nothing)
    ie.kv8_cache_write(K[:, :1], K[:, :1], cache, tab, 0)
    assert ie.token_logprobs(buf.as_strided((1, 500), (far, 1)), None, 3).top_indices.tolist() == [[0, 1, 2]]

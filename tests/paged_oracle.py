"""include/ie_paged.h restated in 64 bits (torch, any device): a rotation, an
attention row by row over gathered keys, trees by walking them."""
import math

import numpy as np
import torch

U = 2.0**-24  # half a step of fp32, relative


def tables(r, lens, block, spare=2, least=1):
    """A table of scattered pages for sequences of `lens` positions, entries past them at the last page; number of pages."""
    nb = [-(-n // block) for n in lens]
    pages = sum(nb) + spare
    perm = r.permutation(pages - 1)
    table, at = np.full((len(lens), max(least, max(nb))), pages - 1, np.int32), 0
    for b, n in enumerate(nb):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, pages


def cache_of(r, table, pages, lens, block, H, d, half, dev, fill=float("nan")):
    """K and V caches: normal values at the sequences' positions, `fill` elsewhere."""
    g = torch.Generator().manual_seed(int(r.integers(1 << 31)))
    out = []
    for _ in range(2):
        x = torch.full((pages, block, H, d), fill)
        for b, n in enumerate(lens):
            for p in range(-(-n // block)):
                m = min(block, n - p * block)
                x[table[b, p], :m] = torch.randn(m, H, d, generator=g) * math.exp(0.3 * float(torch.randn((), generator=g)))
        out.append(x.to(torch.bfloat16 if half else torch.float32).to(dev))
    return out


def rows(cache, table_row, n, h):
    pages = torch.as_tensor(table_row, device=cache.device).long()
    block, d = cache.shape[1], cache.shape[3]
    return cache[pages[:-(-n // block) if n else 0]][:, :, h].reshape(-1, d)[:n].double()


def attend(q, k, v, seen, gap, scale, cap=0.0, slope=0.0):
    """Outputs of query rows q [m, d] over keys k, v [n, d] in 64 bits, and how far fp32 arithmetic may be off, element
    by element.  With p the weights and s the scores: a score's error is
      e = U (16 a + 4 |s0| + 2 |s|), a = scale sum |q k|, s0 the product before its cap and s what the softmax sees:
    a sum of d products rounds like the root of their number, 16 covers d <= 128 with more than 1.4 to spare, scaling, the
    cap's tanh and the factor to base 2 round a few times each; what a cap does to e only shrinks it.  A weight is off by e
    and by the exponential's 2 U + U |s - max|, sums by their length's root and 16 roundings of the blocks' scaling."""
    n = k.shape[0]
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    if n == 0:
        return o, tol
    k, v = (torch.where(seen.any(0)[:, None], x, 0.0) for x in (k, v))
    s0 = scale * (q @ k.t())
    a = abs(scale) * (q.abs() @ k.abs().t())
    s = cap * torch.tanh(s0 / cap) if cap else s0
    s = s - slope * gap
    e = U * (16 * a + 4 * s0.abs().clamp(max=cap or math.inf) + 2 * s.abs())
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    w = torch.where(seen, torch.exp(s - top), 0.0)
    l = w.sum(-1, keepdim=True)
    p = w / torch.where(l > 0, l, 1.0)
    o = p @ v
    e = torch.where(seen, e + U * (2 + 2 * (s - top).abs()), 0.0)
    pe = p * e
    tol = pe @ v.abs() + pe.sum(-1, keepdim=True) * o.abs() + U * (16 + math.sqrt(n)) * (p @ v.abs() + o.abs())
    return o, tol + 2.0**-126


def ranges(q, caches, table, block, starts, lens, max_ctx, first=None, end=None, window=0, scale=None, cap=0.0, slopes=None):
    """(O, tolerance, live) of ie_paged_attn; q [B, P, H_q, d] (live: rows that are written)."""
    B, P, H, d = q.shape
    G = H // caches[0].shape[2]
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    live = torch.zeros(B, P, dtype=torch.bool, device=q.device)
    scale = scale or 1 / math.sqrt(d)
    for b in range(B):
        m = P if lens is None else min(lens[b], P)
        if m <= 0:
            continue
        start = max(starts[b], 0)
        n = min(start + m, max_ctx)
        live[b, :m] = True
        j, pos = torch.arange(n, device=q.device), start + torch.arange(m, device=q.device)[:, None]
        lo = torch.zeros_like(pos) if first is None else torch.as_tensor(first[b][:m], device=q.device)[:, None].clamp(min=0)
        hi = pos + 1 if end is None else torch.as_tensor(end[b][:m], device=q.device)[:, None]
        seen = (j >= lo) & (j < hi)
        if window:
            seen &= j > pos - window
        for h in range(H):
            k, v = (rows(c, table[b], n, h // G) for c in caches)
            out[b, :m, h], tol[b, :m, h] = attend(q[b, :m, h].double(), k, v, seen, (pos - j).abs().double(), scale, cap,
                                                  0.0 if slopes is None else float(slopes[h]))
    return out, tol, live


def lines(parents):
    """Each node's ancestors and itself; a parent that is no earlier node is none."""
    found = []
    for t, p in enumerate(parents):
        found.append((found[p] if 0 <= p < t else []) + [t])
    return found


def tree(q, caches, table, block, ctx, parents, lens=None, window=0, scale=None, cap=0.0, slopes=None):
    B, T, H, d = q.shape
    G = H // caches[0].shape[2]
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    live = torch.zeros(B, T, dtype=torch.bool, device=q.device)
    scale = scale or 1 / math.sqrt(d)
    for b in range(B):
        m = T if lens is None else min(lens[b], T)
        if m <= 0:
            continue
        live[b, :m] = True
        n, line = ctx[b] + m, lines(parents[b])[:m]
        deep = np.array([len(x) - 1 for x in line])
        place = np.concatenate([np.arange(ctx[b]), ctx[b] + deep])
        seen = np.zeros((m, n), bool)
        seen[:, :ctx[b]] = True
        for t in range(m):
            seen[t, [ctx[b] + u for u in line[t]]] = True
        gap = (ctx[b] + deep)[:, None] - place
        if window:
            seen &= gap < window
        seen, gap = torch.as_tensor(seen, device=q.device), torch.as_tensor(np.abs(gap), device=q.device).double()
        for h in range(H):
            k, v = (rows(c, table[b], n, h // G) for c in caches)
            out[b, :m, h], tol[b, :m, h] = attend(q[b, :m, h].double(), k, v, seen, gap, scale, cap,
                                                  0.0 if slopes is None else float(slopes[h]))
    return out, tol, live


def rotated(x, pos, freq, interleaved):
    """x [m, heads, d] at positions pos [m] in 64 bits, and how far fp32 may be off: a rotated value is two products, each
    of a value and a cos or sin that is off by 4 U at most, and one sum."""
    n = freq.shape[0]
    angle = (pos.double()[:, None] * freq.double())[:, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    i = torch.arange(n, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    y = x.double().clone()
    tol = torch.zeros_like(y)
    y[..., a] = x[..., a].double() * cos - x[..., b].double() * sin
    y[..., b] = x[..., b].double() * cos + x[..., a].double() * sin
    tol[..., a] = tol[..., b] = 7 * U * (x[..., a].double().abs() + x[..., b].double().abs())
    return y, tol

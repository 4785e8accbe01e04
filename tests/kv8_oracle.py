"""The 8-bit KV cache (include/ie_kv8.h) and attention over it, restated in
numpy: the cache's rule in the fp32 steps that define it, attention in 64 bits."""
import numpy as np

FLOOR = np.float32(2.0**-100)
F = np.float32
U = 2.0**-24  # half a step of fp32, relative


class Cache:
    """Pages in a plain layout: codes [pages, heads, block, d] int8, scales [pages, heads]."""

    def __init__(self, pages, heads, d, block, rng=None):
        self.block, self.d, self.heads = block, d, heads
        shape = (pages, heads, block, d)
        if rng is None:
            self.k, self.v = np.zeros(shape, np.int8), np.zeros(shape, np.int8)
        else:  # what a cache holds before its first write
            self.k, self.v = (rng.integers(-128, 128, shape, dtype=np.int8) for _ in range(2))
        self.ks, self.vs = (np.full((pages, heads), np.nan, F) for _ in range(2))

    def write(self, K, V, row, start):
        """K, V [P, heads, d] fp32 at positions start .. of the sequence with table row `row`."""
        P = K.shape[0]
        for codes, scales, X in ((self.k, self.ks, K), (self.v, self.vs, V)):
            pos = start
            while pos < start + P:
                page, r0 = row[pos // self.block], pos % self.block
                n = min(self.block - r0, start + P - pos)
                x = X[pos - start:pos - start + n].transpose(1, 0, 2)  # [heads, n, d]
                with np.errstate(all="ignore"):
                    need = np.maximum(np.abs(x).max(axis=(1, 2)) / F(127), FLOOR)
                    had = scales[page].copy()
                    scale = need if r0 == 0 else np.where(need <= had, had, np.maximum(need, F(1.25) * had))
                    inv = F(1) / scale
                    if r0:
                        grew = ~(scale == had)
                        moved = np.rint(codes[page, :, :r0].astype(F) * (had * inv)[:, None, None])
                        moved = np.nan_to_num(moved, nan=0.0).astype(np.int8)
                        codes[page, :, :r0] = np.where(grew[:, None, None], moved, codes[page, :, :r0])
                    q = np.rint(x * inv[:, None, None])
                codes[page, :, r0:r0 + n] = np.nan_to_num(q, nan=0.0).astype(np.int8)
                scales[page] = scale
                pos += n

    def rows(self, row, n, h):
        """K and V of the first n positions, head h, in 64 bits."""
        nb = -(-n // self.block)
        out = []
        for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
            pages = row[:nb]
            with np.errstate(all="ignore"):
                out.append((codes[pages, h].astype(np.float64) * scales[pages, h].astype(np.float64)[:, None, None])
                           .reshape(-1, self.d)[:n])
        return out

    def tensors(self, ie, dev):
        """The same cache as the library lays it out."""
        import torch

        n, h, block, d = self.v.shape
        v = self.v.reshape(n, h, block // 16, 16, d).swapaxes(3, 4)
        return ie.Kv8Cache(*(torch.from_numpy(np.ascontiguousarray(t)).to(dev) for t in (self.k, v, self.ks, self.vs)))

    def take(self, cache):
        """The library's tensors back in the plain layout."""
        k, v, ks, vs = (t.cpu().numpy() for t in cache)
        return k, v.swapaxes(3, 4).reshape(k.shape), ks, vs


def tables(rng, lens, block, spare=2):
    """A block table whose pages lie scattered; entries past a sequence's end are far out of range."""
    nb = [-(-n // block) for n in lens]
    order = rng.permutation(sum(nb) + spare).astype(np.int32)
    table = np.full((len(lens), max(1, max(nb, default=1))), 2**30, np.int32)
    at = 0
    for b, n in enumerate(nb):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(nb) + spare


def attend(q, K, V):
    """softmax(q K^T / sqrt(d)) V in 64 bits and how far fp32 arithmetic may be from it.

    The score of a key is off by at most 23 u S, S = sum |q_i k_i| / sqrt(d) at its largest (u = 2^-24): the query's two
    half-precision parts 4 u, up to 16 accumulation steps u each, 3 products; a weight by that and 12 u of its own (the
    exponent's argument and the exponential 4, two half-precision parts 8); the output is a weighted mean, so by twice
    the weights' error times max|v|, and u max|v| for each accumulation step, at most one in 16 keys."""
    q = np.asarray(q, np.float64)
    s = K @ q / np.sqrt(len(q))
    p = np.exp(s - s.max())
    S = (np.abs(K) @ np.abs(q)).max() / np.sqrt(len(q))
    return (p / p.sum()) @ V, (46 * S + 24 + len(K) / 16) * U * np.abs(V).max()

"""include/ie_paged.h on the GPU at the edges of what it takes (paged_oracle has the tolerances)."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from conftest import rng
from paged_forms import FORMS
from test_gpu_paged import case, i32, near

pytestmark = pytest.mark.gpu


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

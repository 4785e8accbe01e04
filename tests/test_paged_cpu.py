"""include/ie_paged.h without a GPU: exported as declared, refusals on the host
before any HIP call, the division behind its pages, and the oracle against closed forms."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import paged_oracle as po
from conftest import ROOT, rng
from paged_forms import ASKED, FORMS

P = 4096  # stands for a device pointer: no call below reaches HIP
OUT = 1 << 40
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3


def test_exported_as_declared(ie):
    text = open(os.path.join(ROOT, "include", "ie_paged.h")).read()
    declared = sorted(set(re.findall(r"^\s*(?:int|size_t)\s+(ie_\w+)\s*\(", text, re.M)))
    assert declared == sorted(ie.PAGED_SIGNATURES)
    lib = ctypes.CDLL(ie.LIB_PATH)
    for n in declared:
        assert hasattr(lib, n), n
    assert f"IE_TREE_MAX {ie.TREE_MAX}" in text and f"IE_PAGED_MAX_SPLITS {ie.PAGED_MAX_SPLITS}" in text


def rope(ie, B=1, n=4, Q=P, K=P, V=P, qld=256, ld=256, Hq=4, H=2, d=64, rot=64, pairs=0, freq=P, starts=P, lens=None,
         pos=None, out=OUT, k=P, v=P, kv=0, table=P, nbps=4, bs=16):
    return ie.call("ie_rope_kv_write", B, n, Q, K, V, qld, ld, Hq, H, d, rot, pairs, freq, starts, lens, pos, out, k, v, kv,
                   table, nbps, bs, None)


def attn(ie, B=1, n=4, Hq=4, H=2, d=64, Q=P, k=P, v=P, kv=0, table=P, nbps=4, bs=16, starts=P, lens=None, mx=64, first=None,
         end=None, window=0, scale=0.0, cap=0.0, slopes=None, O=OUT, ws=None, wsb=0, splits=0):
    return ie.call("ie_paged_attn", B, n, Hq, H, d, Q, k, v, kv, table, nbps, bs, starts, lens, mx, first, end, window, scale,
                   cap, slopes, O, ws, wsb, splits, None)


def tree(ie, B=1, n=4, Hq=4, H=2, d=64, Q=P, k=P, v=P, kv=0, table=P, nbps=4, bs=16, ctx=P, lens=None, parents=P, mx=60,
         window=0, scale=0.0, cap=0.0, slopes=None, O=OUT, ws=None, wsb=0, splits=0):
    return ie.call("ie_tree_attn", B, n, Hq, H, d, Q, k, v, kv, table, nbps, bs, ctx, lens, parents, mx, window, scale, cap,
                   slopes, O, ws, wsb, splits, None)


def keep(ie, B=1, most=4, layers=2, k=(P, P), v=(P, P), kv=0, table=P, nbps=4, bs=16, H=2, d=64, ctx=P, paths=P, counts=P):
    def arr(c):
        return None if c is None else (ctypes.c_void_p * max(1, len(c)))(*c)
    return ie.call("ie_kv_cache_keep", B, most, layers, arr(k), arr(v), kv, table, nbps, bs, H, d, ctx, paths, counts, None)


LAYOUT = [(dict(d=96), UNSUPPORTED), (dict(d=0), INVALID), (dict(H=0), INVALID), (dict(B=-1), INVALID), (dict(bs=0), INVALID),
          (dict(bs=-16), INVALID), (dict(nbps=-1), INVALID), (dict(kv=2), INVALID), (dict(kv=-1), INVALID)]
CACHE = [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(table=None), INVALID), (dict(k=P + 8), INVALID),
         (dict(v=P + 4), INVALID), (dict(table=P + 2), INVALID)]
SCORES = [(dict(Hq=3), INVALID), (dict(Hq=0), INVALID), (dict(n=-1), INVALID), (dict(mx=-1), INVALID), (dict(mx=65), INVALID),
          (dict(window=-1), INVALID), (dict(scale=-1.0), INVALID), (dict(scale=float("nan")), INVALID),
          (dict(scale=float("inf")), INVALID), (dict(cap=-1.0), INVALID), (dict(cap=float("nan")), INVALID),
          (dict(cap=1e-39, scale=1.0), INVALID), (dict(Q=None), INVALID), (dict(O=None), INVALID), (dict(Q=P + 4), INVALID),
          (dict(O=OUT + 4), INVALID), (dict(O=P + 1024), INVALID), (dict(mx=2**30 + 1, nbps=2**27, bs=256), UNSUPPORTED),
          (dict(B=2**21), UNSUPPORTED), (dict(splits=4, ws=None, nbps=256, mx=2048), INVALID),
          (dict(splits=4, nbps=256, mx=2048, ws=1 << 50, wsb=4 * 4 * 4 * 66 * 4 - 1), WORKSPACE),
          (dict(splits=4, nbps=256, mx=2048, ws=(1 << 50) + 4, wsb=1 << 30), INVALID),
          (dict(splits=4, nbps=256, mx=2048, ws=P, wsb=1 << 30), INVALID)]
CASES = [(rope, LAYOUT + CACHE + [(dict(n=-1), INVALID), (dict(Hq=-1), INVALID), (dict(rot=63), INVALID), (dict(rot=66), INVALID),
                                  (dict(rot=-2), INVALID), (dict(qld=252), INVALID), (dict(qld=258), INVALID),
                                  (dict(ld=124), INVALID), (dict(ld=130), INVALID), (dict(Q=None), INVALID),
                                  (dict(K=None), INVALID), (dict(V=None), INVALID), (dict(out=None), INVALID),
                                  (dict(freq=None), INVALID), (dict(starts=None), INVALID), (dict(Q=P + 4), INVALID),
                                  (dict(K=P + 8), INVALID), (dict(V=P + 4), INVALID), (dict(out=OUT + 8), INVALID),
                                  (dict(out=P), INVALID), (dict(out=P + 16), INVALID), (dict(K=OUT - 16), INVALID),
                                  (dict(freq=P + 2), INVALID), (dict(starts=P + 1), INVALID), (dict(lens=P + 2), INVALID),
                                  (dict(pos=P + 3), INVALID), (dict(nbps=2**27), UNSUPPORTED), (dict(n=2**21 + 1), UNSUPPORTED)]),
         (attn, LAYOUT + CACHE + SCORES + [(dict(starts=None), INVALID), (dict(starts=P + 2), INVALID), (dict(first=P + 1), INVALID),
                                           (dict(end=P + 2), INVALID), (dict(slopes=P + 2), INVALID)]),
         (tree, LAYOUT + CACHE + [(a | ({"mx": a["mx"] - 4} if a.get("mx") == 65 else {}), s) for a, s in SCORES]
          + [(dict(ctx=None), INVALID), (dict(parents=None), INVALID), (dict(parents=P + 2), INVALID), (dict(lens=P + 2), INVALID), (dict(n=257, nbps=99), UNSUPPORTED),
             (dict(mx=2**31 - 1), INVALID)]),
         (keep, LAYOUT + [(dict(most=-1), INVALID), (dict(layers=-1), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
                          (dict(k=(P, None)), INVALID), (dict(v=(P, P + 4)), INVALID), (dict(table=None), INVALID),
                          (dict(ctx=None), INVALID), (dict(paths=None), INVALID), (dict(counts=None), INVALID),
                          (dict(paths=P + 2), INVALID), (dict(counts=P + 1), INVALID),
                          (dict(B=65536), UNSUPPORTED), (dict(nbps=2**27), UNSUPPORTED)])]


@pytest.mark.parametrize("f,args,status", [(f, a, s) for f, cases in CASES for a, s in cases])
def test_refusals(ie, f, args, status):
    assert f(ie, **args) == status
    assert ie.last_error()


@pytest.mark.parametrize("f", [attn, tree])
@pytest.mark.parametrize("args", [dict(scale=3e38), dict(cap=3e38, scale=2.4e38), dict(cap=1e10, scale=1e-30)])
def test_refuses_scores_past_fp32(ie, f, args):
    """A scale that passes fp32 once times log2(e), a scale / cap below fp32's least normal."""
    assert f(ie, **args) == INVALID and "fp32" in ie.last_error()


def test_nothing_to_do(ie):
    """Empty calls succeed whatever their pointers."""
    assert rope(ie, B=0, K=None, k=None) == 0 and rope(ie, n=0, K=None, k=None) == 0
    assert attn(ie, B=0, Q=None, k=None) == 0 and attn(ie, n=0, Q=None, k=None) == 0
    assert tree(ie, B=0, Q=None, k=None) == 0 and tree(ie, n=0, Q=None, k=None) == 0
    assert keep(ie, B=0, k=None) == 0 and keep(ie, most=0, k=None) == 0 and keep(ie, layers=0, k=None) == 0


def test_num_splits(ie):
    f = ie.paged_attn_num_splits
    assert f(1, 1, 12, 12, 64, 0, 0) == 1 and f(0, 1, 12, 12, 64, 0, 100) == 1 and f(1, 1, 12, 8, 64, 0, 1000) == 1
    assert f(1, 1, 12, 12, 96, 0, 1000) == 1 and f(1, 1, 12, 12, 64, 7, 1000) == 1
    big = 2**31 - 1
    assert f(big, big, big, big, 128, 1, 2**30, 0, 64) == 1 and f(big, big, big, 1, 128, 1, 2**30, 0, 64) == 1
    for kv in (0, 1):
        for ctx in (1, 64, 1000, 8192, 1 << 20):
            for B in (1, 8, 64):
                for n in (1, 7, 300):
                    for asked in (0, 1, 3, 64, 1000):
                        s = f(B, n, 32, 8, 128, kv, ctx, 0, asked)
                        assert 1 <= s <= ie.PAGED_MAX_SPLITS and s <= max(1, -(-ctx // 32))
                        assert asked <= 0 or s <= asked
                        assert ie.call("ie_paged_attn_workspace_bytes", B, n, 32, 128, s) == (B * n * 32 * s * 130 * 4 if s > 1 else 0)


def test_page_division(tmp_path):
    """page_map's multiplication against division, at and around multiples, for every block up to 4096 and some others."""
    src = tmp_path / "pages.cpp"
    src.write_text('''
#include "paged.h"
#include <cstdio>
static bool fine(long long n, int block, const ie::PageMap& m) {
    if (n < 0 || n >= 1ll << 31) return true;
    const uint32_t q = m.mul ? (uint32_t)(((uint64_t)(uint32_t)n * m.mul) >> 32) >> m.shift : (uint32_t)n;
    return q == n / block;
}
int main() {
    long long bad = 0;
    auto all = [&](int block) {
        const ie::PageMap m = ie::page_map(nullptr, 1, block);
        for (long long base : {0ll, 1ll << 10, 1ll << 20, 1ll << 29, 1ll << 30, (1ll << 31) - 1})
            for (long long k = -3; k <= 3; ++k)
                for (long long e = -1; e <= 1; ++e) bad += !fine((base / block + k) * block + e, block, m);
    };
    for (int b = 1; b <= 4096; ++b) all(b);
    for (int b : {4097, 65535, 65536, 65537, 1 << 20, (1 << 20) + 1, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, 0x7fffffff}) all(b);
    printf("%lld", bad);
}
''')
    subprocess.run(["g++", "-std=c++17", "-O1", *INCLUDES, "-I/opt/rocm/include", "-D__HIP_PLATFORM_AMD__", str(src), "-o", str(tmp_path / "pages")], check=True)
    assert subprocess.run([str(tmp_path / "pages")], capture_output=True, text=True, check=True).stdout == "0"


INCLUDES = [f"-I{ROOT}/include", f"-I{ROOT}/cuda-llm-inference-engine_amd/csrc"]


def test_plans(ie, tmp_path):
    """paged_plan: the GPU tests' calls reach every form; splits stay within their limits and are those of the C ABI; an
    asked number is kept."""
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-std=c++17", "-O1", *INCLUDES, os.path.join(ROOT, "tests", "paged_plan.cpp"), "-o", exe], check=True)

    def plans(calls):
        out = subprocess.run([exe], input="\n".join(" ".join(map(str, c)) for c in calls), capture_output=True, text=True, check=True)
        return [tuple(map(int, line.split())) for line in out.stdout.splitlines()]

    calls = [(B, P, H * G, H, d, kv, keys, 0, 0) for kv, d, _, _, _, (B, P, H, G, keys) in FORMS]
    assert plans(calls) == [(rows, groups, splits) for _, _, rows, groups, splits, _ in FORMS]
    forms = {(kv, d, rows, groups) for kv, d, rows, groups, _, _ in FORMS}
    assert forms == {(kv, d, rows, groups) for kv in (0, 1) for d in (64, 128)
                     for rows, groups in ((1, 1), (2, 1), (16, 1), (32, 1), (64, 1), (128, 1), (128, 2))
                     if not (kv and rows == 2) and not (not kv and groups == 2)}
    calls = [(B, P, H * G, H, d, kv, keys, window, asked) for B in (1, 3, 70, 5000) for P in (1, 2, 20, 513, 9000) for H, G in ((1, 1), (8, 4))
             for d in (64, 128) for kv in (0, 1) for keys in (1, 127, 128, 129, 70000, 2**30) for window in (0, 1, 500, 2**31 - 1)
             for asked in (0, 1, 5, 64, 2**31 - 1)]
    for (B, P, Hq, H, d, kv, keys, window, asked), (rows, groups, splits) in zip(calls, plans(calls), strict=True):
        walked = min(keys, window + P) if window else keys
        most = min(64, -(-walked // 128))
        assert splits == min(asked, most) if asked else 1 <= splits <= most
        assert rows in (1, 2, 16, 32, 64, 128) and (rows <= 16 or rows < 2 * P * (Hq // H)) and (groups == 1 or rows == 128)
        if B * P * Hq * 64 < 2**21:  # (past it the C ABI may cut the splits)
            assert ie.paged_attn_num_splits(B, P, Hq, H, d, kv, keys, window, asked) == splits


def test_oracle_closed_forms():
    """The oracle against torch's own attention, and where the answer is known."""
    r = rng(3)
    lens, block, H, d = [37, 5], 7, 2, 64
    table, pages = po.tables(r, lens, block)
    caches = po.cache_of(r, table, pages, lens, block, H, d, False, "cpu")
    q = torch.randn(2, 5, 4, d, generator=torch.Generator().manual_seed(1))
    o, tol, live = po.ranges(q, caches, table, block, [32, 0], [5, 5], 64)
    for b in range(2):
        for h in range(4):
            k, v = (po.rows(c, table[b], lens[b], h // 2) for c in caches)
            mask = torch.ones(5, lens[b], dtype=torch.bool).tril(lens[b] - 5)
            want = torch.nn.functional.scaled_dot_product_attention(q[b, :, h].double()[None], k[None], v[None], mask[None])[0]
            assert (o[b, :, h] - want).abs().max() < 1e-12
    assert torch.allclose(o[1, 0, 0], po.rows(caches[1], table[1], 1, 0)[0])  # one key: its value
    assert bool(live.all()) and 0 < float(tol.max()) < 1e-4
    # a tree that is a chain is a prompt
    chain = [[-1, 0, 1, 2, 3]] * 2
    t, _, _ = po.tree(q, caches, table, block, [32, 0], chain)
    assert (t - o).abs().max() < 1e-12
    # a rotation keeps lengths, and by the same angle on both sides products
    x = torch.randn(3, 2, d)
    f = 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    for pairs in (False, True):
        y, _ = po.rotated(x, torch.tensor([0, 5, 1000]), f, pairs)
        assert torch.equal(y[0], x[0].double()) and (y.norm(dim=-1) - x.double().norm(dim=-1)).abs().max() < 1e-12


def test_walk_between_ranges(tmp_path):
    """paged_walk.h: what a walk over rows' ranges looks up is seen by a row, a key that is seen is looked up as itself, and
    parts are found once each; ranges that touch, repeat, nest, are empty or have gaps of one key among them."""
    src = tmp_path / "walk.cpp"
    src.write_text('''
#include "paged_walk.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
int main() {
    long long wrong = 0, gaps = 0;
    srand(1);
    for (int round = 0; round < 20000; ++round) {
        const int n = 1 + rand() % (round % 3 ? 6 : 128), span = 2 + rand() % (round % 2 ? 40 : 2000), wide = 1 + rand() % (1 + span / 3);
        std::vector<ie::KeyRange> rows;
        for (int i = 0; i < n; ++i) {
            const int lo = rand() % span;
            rows.push_back(rand() % 8 ? ie::KeyRange{lo, lo + rand() % wide} : ie::KeyRange{lo + 3, lo});
            if (rand() % 4 == 0) rows.back() = rows[rand() % (i + 1)];
        }
        std::vector<char> seen(2 * span + 2, 0);
        int least = 1 << 30, most = 0;
        for (auto r : rows)
            for (int j = r.lo; j < r.hi; ++j) seen[j] = 1, least = j < least ? j : least, most = j + 1 > most ? j + 1 : most;
        std::vector<int> begin, end;
        for (int i = 0; i < n; ++i) {
            if (rows[i].lo >= rows[i].hi) continue;
            bool b = true, e = true;
            for (int j = 0; j < n; ++j) b &= !ie::hides_begin(rows[i], rows[j], j < i), e &= !ie::hides_end(rows[i], rows[j], j < i);
            if (b) begin.push_back(rows[i].lo);
            if (e) end.push_back(rows[i].hi);
        }
        size_t parts = 0;
        for (int j = 0; j < most; ++j) parts += seen[j] && !(j && seen[j - 1]);
        wrong += begin.size() != parts || end.size() != parts;
        gaps += parts > 1;
        for (int p = least, last = least; p < most; ++p) {
            if (seen[p]) last = p;
            int b = -1, e = -1;
            for (int x : begin) b = x <= p && x > b ? x : b;
            for (int x : end) e = x <= p && x > e ? x : e;
            wrong += ie::stand_in(p, b, e) != last;
        }
    }
    printf("%lld %d", wrong, gaps > 1000);
}
''')
    exe = str(tmp_path / "walk")
    subprocess.run(["g++", "-std=c++17", "-O1", *INCLUDES, str(src), "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True, check=True).stdout == "0 1"


def test_forms_in_asked_splits(tmp_path):
    """The calls of ASKED reach their forms, so that every form is tested in several splits."""
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-std=c++17", "-O1", *INCLUDES, os.path.join(ROOT, "tests", "paged_plan.cpp"), "-o", exe], check=True)
    calls = "\n".join(f"{B} {P} {H * G} {H} {d} {kv} {keys} 0 {splits}" for kv, d, _, _, splits, (B, P, H, G, keys) in ASKED)
    out = subprocess.run([exe], input=calls, capture_output=True, text=True, check=True).stdout.split("\n")
    assert out[:-1] == [f"{rows} {groups} {splits}" for _, _, rows, groups, splits, _ in ASKED]
    assert {f[:4] for f in FORMS} == {f[:4] for f in FORMS + ASKED if f[4] > 1}

"""The 8-bit KV cache's C ABI without a GPU: exported as declared, refusals on
the host before any HIP call; and the oracle's cache rule against its bounds."""
import ctypes
import os
import re

import numpy as np
import pytest

import kv8_launch as kl
import kv8_oracle as ko
from conftest import ROOT, rng


def declared(header):
    text = open(os.path.join(ROOT, "include", header)).read()
    return sorted(set(re.findall(r"^\s*(?:int|size_t)\s+(ie_\w+)\s*\(", text, re.M)))


def test_exported_as_declared(ie):
    assert declared("ie_kv8.h") == sorted(ie.KV8_SIGNATURES)
    lib = ctypes.CDLL(ie.LIB_PATH)
    for n in ie.KV8_SIGNATURES:
        assert hasattr(lib, n), n


P = 4096  # stands for a device pointer: no call below reaches HIP


def write(ie, B=1, n=4, K=P, V=P, ld=128, k=P, v=P, ks=P, vs=P, table=P, nbps=4, start=0, H=2, d=64, bs=16):
    return ie.call("ie_kv8_cache_write", B, n, K, V, ld, k, v, ks, vs, table, nbps, start, H, d, bs, None)


def append(ie, B=1, K=P, V=P, ld=128, k=P, v=P, ks=P, vs=P, table=P, nbps=4, pos=P, H=2, d=64, bs=16):
    return ie.call("ie_kv8_cache_append_batch", B, K, V, ld, k, v, ks, vs, table, nbps, pos, H, d, bs, None)


def read(ie, B=1, n=4, starts=P, lens=P, k=P, v=P, ks=P, vs=P, table=P, nbps=4, H=2, d=64, bs=16, K=P, V=P):
    return ie.call("ie_kv8_cache_read", B, n, starts, lens, k, v, ks, vs, table, nbps, H, d, bs, K, V, None)


def decode(ie, B=1, Hq=4, H=2, d=64, Q=P, k=P, v=P, ks=P, vs=P, table=P, lens=P, mx=64, bs=16, nbps=4, O=1 << 20, ws=P,
           wsb=1 << 20, splits=1):
    return ie.call("ie_decode_attn_kv8", B, Hq, H, d, Q, k, v, ks, vs, table, lens, mx, bs, nbps, O, ws, wsb, splits, None)


def prompt(ie, B=1, n=4, Hq=4, H=2, d=64, Q=P, k=P, v=P, ks=P, vs=P, table=P, nbps=4, bs=16, start=0, O=1 << 20,
           ws=None, wsb=0):
    return ie.call("ie_prefill_attn_kv8", B, n, Hq, H, d, Q, k, v, ks, vs, table, nbps, bs, start, O, ws, wsb, None)


INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
LAYOUT = [(dict(d=96), UNSUPPORTED), (dict(d=0), INVALID), (dict(H=0), INVALID), (dict(B=-1), INVALID),
          (dict(bs=0), INVALID), (dict(bs=8), UNSUPPORTED), (dict(bs=48), UNSUPPORTED), (dict(bs=512), UNSUPPORTED),
          (dict(nbps=-1), INVALID)]
CACHE = [(dict(k=None), INVALID), (dict(v=None), INVALID), (dict(ks=None), INVALID), (dict(vs=None), INVALID),
         (dict(table=None), INVALID), (dict(k=P + 8), INVALID), (dict(v=P + 4), INVALID)]
SOURCE = [(dict(K=None), INVALID), (dict(V=None), INVALID), (dict(K=P + 4), INVALID), (dict(ld=124), INVALID),
          (dict(ld=130), INVALID)]
CASES = [(write, LAYOUT + CACHE + SOURCE + [(dict(start=-1), INVALID), (dict(n=-1), INVALID), (dict(start=61), INVALID),
                                            (dict(n=65), INVALID), (dict(start=2**31 - 1), INVALID),
                                            (dict(start=2**30, nbps=2**27, bs=256), UNSUPPORTED),
                                            (dict(B=2**20 + 1), UNSUPPORTED), (dict(B=2**20 + 1, H=1), UNSUPPORTED)]),
         (append, LAYOUT + CACHE + SOURCE + [(dict(pos=None), INVALID), (dict(B=2**20 + 1), UNSUPPORTED),
                                             (dict(B=2**20 + 1, H=1), UNSUPPORTED)]),
         (read, LAYOUT + CACHE + [(dict(n=-1), INVALID), (dict(starts=None), INVALID), (dict(K=None), INVALID),
                                  (dict(V=P + 8), INVALID), (dict(n=2**31 - 1), UNSUPPORTED)]),
         (decode, LAYOUT + CACHE + [(dict(Hq=3), INVALID), (dict(Hq=0), INVALID), (dict(mx=-1), INVALID),
                                    (dict(mx=65), INVALID), (dict(Q=None), INVALID), (dict(O=None), INVALID),
                                    (dict(Q=P + 4), INVALID), (dict(lens=None), INVALID), (dict(O=P + 256), INVALID),
                                    (dict(mx=2**30 + 1, nbps=2**27, bs=256), UNSUPPORTED),
                                    (dict(mx=1024, nbps=64, splits=8, ws=None), INVALID),
                                    (dict(mx=1024, nbps=64, splits=8, wsb=8 * 4 * 66 * 4 - 1), WORKSPACE),
                                    (dict(B=2**21, O=1 << 60), UNSUPPORTED)]),
         (prompt, LAYOUT + CACHE + [(dict(Hq=3), INVALID), (dict(n=-1), INVALID), (dict(start=-1), INVALID),
                                    (dict(start=61), INVALID), (dict(Q=None), INVALID), (dict(O=None), INVALID),
                                    (dict(O=P + 512), INVALID), (dict(O=(1 << 20) + 4), INVALID),
                                    (dict(start=2**30, nbps=2**27, bs=256), UNSUPPORTED),
                                    (dict(B=2**21, O=1 << 60), UNSUPPORTED)])]


@pytest.mark.parametrize("f,args,status", [(f, a, s) for f, cases in CASES for a, s in cases])
def test_refusals(ie, f, args, status):
    assert f(ie, **args) == status
    assert ie.last_error()


def test_nothing_to_do(ie):
    """Empty calls succeed whatever their pointers."""
    assert write(ie, B=0, K=None, k=None) == 0 and write(ie, n=0, K=None, k=None) == 0
    assert append(ie, B=0, K=None, k=None) == 0
    assert read(ie, B=0, k=None) == 0 and read(ie, n=0, k=None) == 0
    assert decode(ie, B=0, Q=None, k=None) == 0
    assert prompt(ie, B=0, Q=None, k=None) == 0 and prompt(ie, n=0, Q=None, k=None) == 0


def test_num_splits(ie):
    f = ie.decode_kv8_num_splits
    assert f(1, 12, 12, 64, 0) == 1 and f(0, 12, 12, 64, 100) == 1
    assert f(1, 12, 12, 64, 64, 9) == 1 and f(1, 12, 12, 64, 65, 9) == 2
    assert f(1, 12, 12, 64, 1 << 20, 1000) == ie.KV8_MAX_SPLITS
    for ctx in (1, 64, 1000, 8192, 1 << 20):
        for B in (1, 8, 64):
            assert 1 <= f(B, 32, 8, 128, ctx) <= min(ie.KV8_MAX_SPLITS, -(-ctx // 64))


BIG = 2**31 - 1


def test_sizes_whose_products_pass_64_bits(ie):
    """Refused like any other that is too large; head counts that do not divide choose nothing."""
    assert ie.decode_kv8_num_splits(1, 1, 2, 64, 1000) == 1 and ie.decode_kv8_num_splits(1, 12, 8, 64, 1000) == 1
    assert ie.decode_kv8_num_splits(BIG, BIG, BIG, 128, BIG) >= 1
    assert ie.call("ie_prefill_kv8_workspace_bytes", BIG, 2**30, BIG, 1, 64, 0) == 0
    far = dict(nbps=2**22, bs=256, O=1 << 63)
    for B, n, Hq in ((BIG, 2**29, BIG - 1), (2**26, 2**16, 2**26), (2**31 - 16, 2**30, 2**29)):
        assert prompt(ie, B=B, n=n, Hq=Hq, **far) == UNSUPPORTED
    for B, Hq in ((BIG, BIG - 1), (2**30, 2**30), (2**29, 2**30)):
        assert decode(ie, B=B, Hq=Hq, mx=2**30, splits=64, **far) == UNSUPPORTED


def test_prompt_workspace(ie):
    """Few rows behind a long context can be split, and then the workspace has to hold it."""
    f = ie.call
    need = f("ie_prefill_kv8_workspace_bytes", 1, 4, 8, 2, 64, 8000)
    assert need > 0 and need % (4 * 8 * 66 * 4) == 0
    assert prompt(ie, n=4, Hq=8, start=8000, nbps=1000, ws=P, wsb=need - 1) == WORKSPACE
    assert prompt(ie, n=4, Hq=8, start=8000, nbps=1000, ws=P + 4, wsb=need) == INVALID
    assert f("ie_prefill_kv8_workspace_bytes", 4, 2048, 32, 8, 128, 0) == 0
    for bad in ((0, 4, 8, 2, 64, 0), (1, 0, 8, 2, 64, 0), (1, 4, 7, 2, 64, 0), (1, 4, 8, 2, 64, -1), (1, 4, 8, 2, 64, 2**30)):
        assert f("ie_prefill_kv8_workspace_bytes", *bad) == 0


def test_oracle_rule_bounds():
    """The rule itself: half a scale for rows written with their page, 2.5 scales for ones it grew under, a scale that
    is at least need and grows by a quarter or not at all."""
    r = rng(1)
    H, d, block = 2, 64, 32
    c = ko.Cache(1, H, d, block, r)
    X = (r.standard_normal((block, H, d)) * (1.07 ** np.arange(block))[:, None, None]).astype(np.float32)
    before = None
    for i in range(block):
        c.write(X[i:i + 1], X[i:i + 1], [0], i)
        s = c.ks[0].copy()
        assert (s * 127 * (1 + 1e-6) >= np.abs(X[:i + 1]).max(axis=(0, 2))).all()
        assert before is None or ((s == before) | (s >= 1.2499 * before)).all()
        before = s
    err = np.abs(c.k[0].transpose(1, 0, 2) * c.ks[0].astype(np.float64)[None, :, None] - X)
    assert (err <= 2.5001 * c.ks[0][None, :, None]).all()
    c.write(X, X, [0], 0)
    err = np.abs(c.k[0].transpose(1, 0, 2) * c.ks[0].astype(np.float64)[None, :, None] - X)
    assert (err <= 0.50001 * c.ks[0][None, :, None]).all()


def launcher_args(**kw):
    a = dict(B=1, P=1, H_q=4, Q=P, q_ld=256, lens=P, max_ctx=64, O=1 << 20, ws=P, splits=1, c=kl.CacheArgs(P, P, P, P, P, 4, 4, 64, 4))
    return kl.AttnArgs(**{**a, **kw})


@pytest.mark.parametrize("which,args", [
    ("decode", dict(splits=2, ws=None)), ("decode", dict(splits=0)), ("decode", dict(splits=65)),
    ("decode", dict(positions=P, K=P, V=P, kv_ld=256, splits=2)),
    ("decode", dict(positions=P, K=P, V=P, kv_ld=256, H_q=20, q_ld=1280)),
    ("prefill", dict(splits=2, ws=None)), ("prefill", dict(splits=0)), ("prefill", dict(splits=65))])
def test_launchers_refuse_what_no_kernel_is_there_for(ie, which, args):
    """Parts without a place for them, and an append with parts or with more heads a KV head than one workgroup has."""
    ie.call("ie_kv8_cache_write", 1, -1, *[None] * 2, 0, *[None] * 5, 0, 0, 0, 0, 0, None)  # (an older message)
    before = ie.last_error()
    assert kl.launch(ie, which, launcher_args(**args)) == INVALID
    assert ie.last_error() != before

"""The log-probability entry points without a GPU: exported as declared, refusals on the host before any HIP call."""
import ctypes
import os
import re

import pytest

from conftest import ROOT

P = 4096  # stands for a device pointer: no call below reaches HIP


def call(ie, rows=2, x=P, ld=100, n=100, t=P, k=3, lp=P, rk=P, en=P, tv=P, ti=P, ws=P, wsb=1 << 20):
    return ie.call("ie_token_logprobs", rows, x, ld, n, t, k, lp, rk, en, tv, ti, ws, wsb, None)


def test_exported_as_declared(ie):
    text = open(os.path.join(ROOT, "include", "ie_logprobs.h")).read()
    assert sorted(set(re.findall(r"^\s*(?:int|size_t)\s+(ie_\w+)\s*\(", text, re.M))) == sorted(ie.LOGPROBS_SIGNATURES)
    lib = ctypes.CDLL(ie.LIB_PATH)
    for n in ie.LOGPROBS_SIGNATURES:
        assert hasattr(lib, n), n


@pytest.mark.parametrize("args,status", [
    (dict(rows=-1), 1), (dict(n=0), 1), (dict(n=-4), 1), (dict(ld=99), 1), (dict(k=-1), 1), (dict(k=101), 1),
    (dict(k=129, n=1000, ld=1000), 1), (dict(n=(1 << 19) + 1, ld=1 << 20), 2), (dict(rows=(1 << 20) + 1), 2),
    (dict(x=None), 1), (dict(x=P + 2), 1), (dict(tv=None), 1), (dict(ti=None), 1), (dict(t=P + 1), 1)])
def test_refusals(ie, args, status):
    assert call(ie, **args) == status
    assert ie.last_error()


def test_workspace(ie):
    """A call that needs one is refused without it; sizes that no call takes need none."""
    f = ie.call
    need = f("ie_token_logprobs_workspace_bytes", 1, 1 << 19, 5)
    if need:
        assert call(ie, rows=1, n=1 << 19, ld=1 << 19, k=5, ws=None) == 1
        assert call(ie, rows=1, n=1 << 19, ld=1 << 19, k=5, ws=P + 4) == 1
        assert call(ie, rows=1, n=1 << 19, ld=1 << 19, k=5, wsb=need - 1) == 3
    assert f("ie_token_logprobs_workspace_bytes", -1, 100, 5) == 0
    assert f("ie_token_logprobs_workspace_bytes", 1, (1 << 19) + 1, 5) == 0
    for rows in (1, 8, 300, 2048):
        for n in (50, 50257, 131072, 1 << 19):
            for k in (0, 5, 128 if n > 128 else 40):
                assert f("ie_token_logprobs_workspace_bytes", rows, n, k) <= rows * 16 * (8 + 2 * k) * 4


def test_nothing_to_do(ie):
    assert call(ie, rows=0, x=None, t=None, lp=None) == 0


def test_score_refuses_a_null_engine(ie):
    tokens = (ctypes.c_int * 4)()
    assert ie.call("ie_engine_score", None, 1, 4, ctypes.addressof(tokens), 0, None, None, None, None, None) == 1


@pytest.mark.parametrize("rows,n,k", [(1, 1 << 19, 5), (8, 50257, 5), (16, 50257, 80), (300, 32001, 1)])
def test_cut_rows_need_a_workspace(ie, rows, n, k):
    need = ie.call("ie_token_logprobs_workspace_bytes", rows, n, k)
    assert need > 0
    assert call(ie, rows=rows, n=n, ld=n, k=k, ws=None) == 1
    assert call(ie, rows=rows, n=n, ld=n, k=k, ws=P + 4, wsb=need) == 1
    assert call(ie, rows=rows, n=n, ld=n, k=k, wsb=need - 1) == 3

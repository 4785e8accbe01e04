"""The GPT-2 engine over the 8-bit KV cache, and its score of given tokens.

Parity with the CPU decode-step oracle whose cache follows the same rule (kv8_oracle): the bar of the other engine tests
for free runs, 3e-2 of the logits' scale, which comes from activations at an int8 rounding boundary; a key or value at a
boundary of its own moves by one code of 127.
"""
import numpy as np
import pytest

import kv8_oracle as ko

pytestmark = pytest.mark.gpu

TINY = dict(n_layers=2, n_heads=2, d_model=128, d_ff=512, vocab_size=1000, max_seq_len=64)
SMALL = dict(n_layers=2, vocab_size=1000, max_seq_len=256)  # GPT-2 Small's widths: the fused step


@pytest.fixture(scope="module")
def tiny_dir(tmp_path_factory, ie):
    d = tmp_path_factory.mktemp("gpt2_tiny_kv8")
    ie.write_random_model(d, seed=21, **TINY)
    return d


@pytest.fixture(scope="module")
def small_dir(tmp_path_factory, ie):
    d = tmp_path_factory.mktemp("gpt2_small_kv8")
    ie.write_random_model(d, seed=22, **SMALL)
    return d


def oracle(model_dir, B):
    """OracleGPT2 with the 8-bit rule between what the layers give and what attention reads."""
    from oracle import gpt2_step, orc

    class Kv8(gpt2_step.OracleGPT2):
        def __init__(self):
            super().__init__(str(model_dir), batch=B)
            self.q8 = [ko.Cache(B * self.nbps, self.H, self.dh, gpt2_step.BLOCK) for _ in self.layers]

        def layer(self, x, li, P):
            """x [B * P, d], row b * P + t at position pos + t, through layer li."""
            Lw, d, H, dh = self.layers[li], self.d, self.H, self.dh

            def linear(rows, name, epi, res=None):
                ap, asc = orc.quantize(rows)
                w, s, bias = Lw[name]
                return orc.gemm(ap, w, asc, s, epi, bias, *(() if res is None else (res,)))

            qkv = linear(orc.layernorm(x, *Lw["ln1"]), "qkv", 1)
            c = self.q8[li]
            for b in range(B):
                rows = qkv[b * P:(b + 1) * P]
                c.write(rows[:, d:2 * d].reshape(P, H, dh), rows[:, 2 * d:].reshape(P, H, dh), self.table[b], self.pos)
            K, V = (np.ascontiguousarray((q.astype(np.float32) * np.nan_to_num(s)[:, :, None, None]).swapaxes(1, 2))
                    for q, s in ((c.k, c.ks), (c.v, c.vs)))
            attn = np.empty((B * P, d), np.float32)
            for t in range(P):
                lens = np.full(B, self.pos + t + 1, np.int32)
                q = np.ascontiguousarray(qkv[t::P, :d]).reshape(B, H, dh)
                attn[t::P] = orc.decode_attn(q, K, V, self.table, lens, self.c["max_seq_len"], gpt2_step.BLOCK, H).reshape(B, d)
            x = linear(attn, "out", 3, x)
            h = linear(orc.layernorm(x, *Lw["ln2"]), "up", 2)
            return linear(h, "down", 3, x)

        def prompt(self, tokens):
            """tokens [B, P] at once; the last ones' logits [B, V]."""
            tokens = np.asarray(tokens, np.int32)
            P = tokens.shape[1]
            x = np.concatenate([orc.embedding(tokens[b], self.pos, self.wte, self.wpe) for b in range(B)])
            for li in range(len(self.layers)):
                x = self.layer(x, li, P)
            self.pos += P
            xf = orc.layernorm(np.ascontiguousarray(x[P - 1::P]), *self.lnf)
            return np.stack([orc.vocab_proj(r, self.wte) for r in xf])

        def step(self, tokens):
            return self.prompt(np.asarray(tokens)[:, None])

    return Kv8()


def near(got, want):
    scale = np.abs(want).max()
    assert np.abs(got - want).max() <= 3e-2 * scale, np.abs(got - want).max() / scale


@pytest.mark.parametrize("which", ["tiny_dir", "small_dir"])
@pytest.mark.parametrize("B", [1, 3])
def test_steps_match_oracle(ie, request, which, B):
    """Token by token from empty: pages grow under their scales."""
    d = request.getfixturevalue(which)
    r = np.random.default_rng(B)
    eng, om = ie.Engine(d, max_batch=B, kv_dtype=ie.KV_I8), oracle(d, B)
    for t in r.integers(0, 1000, (35, B)):
        near(eng.step(t), om.step(t))
    eng.close()


@pytest.mark.parametrize("which", ["tiny_dir", "small_dir"])
@pytest.mark.parametrize("P,chunk", [(1, 0), (37, 0), (37, 21)])
def test_prefill_then_steps_match_oracle(ie, request, which, P, chunk):
    d = request.getfixturevalue(which)
    B = 2
    r = np.random.default_rng(P + chunk)
    eng, om = ie.Engine(d, max_batch=B, kv_dtype=ie.KV_I8, prefill_chunk=chunk), oracle(d, B)
    prompt = r.integers(0, 1000, (B, P))
    got = eng.prefill(prompt)
    cut = chunk or P
    for at in range(0, P, cut):
        want = om.prompt(prompt[:, at:at + cut])
    near(got, want)
    for t in r.integers(0, 1000, (12, B)):
        near(eng.step(t), om.step(t))
    got, want = eng.prefill(prompt[:, :5]), om.prompt(prompt[:, :5])  # a continuation, mid-page
    near(got, want)
    eng.close()


def test_bits_hold_over_graphs_fusion_and_batch(ie, small_dir):
    """Replayed graphs, the unfused step and a sequence alone give the bits of the fused batch; so does a second session."""
    r = np.random.default_rng(5)
    toks = r.integers(0, 1000, (40, 3)).astype(np.int32)

    def run(t, **kw):
        eng = ie.Engine(small_dir, max_batch=t.shape[1], kv_dtype=ie.KV_I8, **kw)
        out = [eng.step(row) for row in t]
        eng.reset()
        again = [eng.step(row) for row in t]
        eng.close()
        assert all(np.array_equal(a, b) for a, b in zip(out, again))
        return out

    base = run(toks)
    for other in (run(toks, use_graph=False), run(toks, fuse=False)):
        assert all(np.array_equal(a, b) for a, b in zip(base, other))
    for b in range(3):
        alone = run(np.ascontiguousarray(toks[:, b:b + 1]))
        assert all(np.array_equal(a[b:b + 1], o) for a, o in zip(base, alone))


def test_heads_of_128(ie, tmp_path):
    """The same at 128 channels a head: against the oracle, and the fused step (append and attention in one launch)
    against the unfused one's two."""
    ie.write_random_model(tmp_path, seed=24, n_layers=1, n_heads=6, vocab_size=1000, max_seq_len=128)
    r = np.random.default_rng(8)
    a, b = (ie.Engine(tmp_path, max_batch=2, kv_dtype=ie.KV_I8, fuse=f) for f in (True, False))
    om = oracle(tmp_path, 2)
    prompt = r.integers(0, 1000, (2, 5))
    near(a.prefill(prompt), om.prompt(prompt))
    b.prefill(prompt)
    for t in r.integers(0, 1000, (30, 2)):
        got = a.step(t)
        assert np.array_equal(got, b.step(t))
        near(got, om.step(t))


def test_splits_past_1024_tokens(ie, tmp_path):
    """Contexts past 1024 take more than one split: on both sides of the change."""
    cfg = dict(TINY, n_layers=1, max_seq_len=1100)
    ie.write_random_model(tmp_path, seed=3, **cfg)
    r = np.random.default_rng(7)
    eng, om = ie.Engine(tmp_path, max_batch=1, kv_dtype=ie.KV_I8), oracle(tmp_path, 1)
    prompt = r.integers(0, 1000, (1, 1020))
    near(eng.prefill(prompt), om.prompt(prompt))
    for t in r.integers(0, 1000, (8, 1)):
        near(eng.step(t), om.step(t))
    eng.close()


@pytest.mark.parametrize("B", [1, 3])
def test_fused_step_past_1024_tokens(ie, tmp_path, B):
    """The same at GPT-2 Small's widths, where the fused step goes from one launch of append and attention to an append,
    split attention and a merge: against the oracle, and the same bits fused or not, replayed or not."""
    cfg = dict(n_layers=1, vocab_size=1000, max_seq_len=1100)
    ie.write_random_model(tmp_path, seed=31, **cfg)
    r = np.random.default_rng(17)
    engines = [ie.Engine(tmp_path, max_batch=B, kv_dtype=ie.KV_I8, **kw) for kw in (dict(), dict(fuse=False), dict(use_graph=False))]
    om = oracle(tmp_path, B)
    prompt = r.integers(0, 1000, (B, 1020))
    want = om.prompt(prompt)
    for e in engines:
        near(e.prefill(prompt), want)
    for t in r.integers(0, 1000, (9, B)):
        got = [e.step(t) for e in engines]
        assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
        near(got[0], om.step(t))
    for e in engines:
        e.close()


def test_sixteen_sequences(ie, small_dir):
    """The largest batch: a prompt and steps against the oracle, and each sequence's bits as in a batch of its own."""
    r = np.random.default_rng(18)
    eng, om, few = ie.Engine(small_dir, max_batch=16, kv_dtype=ie.KV_I8), oracle(small_dir, 16), ie.Engine(small_dir, max_batch=3, kv_dtype=ie.KV_I8)
    toks = r.integers(0, 1000, (20, 16))
    for t in toks:
        got = eng.step(t)
        near(got, om.step(t))
        assert np.array_equal(few.step(t[5:8]), got[5:8])
    prompt = r.integers(0, 1000, (16, 7))
    near(eng.prefill(prompt), om.prompt(prompt))
    near(eng.step(toks[0]), om.step(toks[0]))
    eng.close()
    few.close()


def test_generates_and_holds_a_quarter_of_the_bytes(ie):
    eng = ie.Engine(max_batch=2, kv_dtype=ie.KV_I8, n_layers=2, vocab_size=2000)
    out, m = eng.generate(np.arange(20).reshape(2, 10), 12, ignore_eos=True)
    assert out.shape == (2, 12) and (out >= 0).all() and m["tokens_generated"] == 12
    ids, _ = eng.generate_one(np.arange(9), 5, greedy=True)
    assert len(ids) == 5
    full = ie.Engine(max_batch=2, kv_dtype=ie.KV_F32, n_layers=2, vocab_size=2000)
    full.generate(np.arange(20).reshape(2, 10), 12, ignore_eos=True)
    weights = full.step_bytes(0)  # no sequence: no cache
    eng.generate(np.arange(20).reshape(2, 10), 12, ignore_eos=True)
    assert (eng.step_bytes(2) - weights) * 4 <= (full.step_bytes(2) - weights) * 1.05
    with pytest.raises(ie.IeError):
        ie.Engine(max_batch=1, kv_dtype=3, n_layers=1, vocab_size=100)


def test_fp32_backend(ie):
    """Over fp32 weights, against the fp32 cache: a code is off by half a step, and by another half after its page grew,
    of at most 1.25 / 127 of the page's largest value: under 1% of it."""
    r = np.random.default_rng(12)
    a, b = (ie.Engine(max_batch=2, kv_dtype=t, backend=ie.BACKEND_FP32, seed=4, **SMALL) for t in (ie.KV_I8, ie.KV_F32))
    prompt = r.integers(0, 1000, (2, 30))
    near(a.prefill(prompt), b.prefill(prompt))
    for t in r.integers(0, 1000, (10, 2)):
        near(a.step(t), b.step(t))


# ------------------------------------------------------------------ score
def log_softmax(x):
    x = x.astype(np.float64)
    d = x - x.max()
    return d - np.log(np.exp(d).sum())


@pytest.mark.parametrize("kw", [dict(), dict(prefill_chunk=7), dict(int8_lm_head=True)])
def test_score_matches_the_logits_of_every_prefix(ie, tiny_dir, kw):
    """Each entry against the logits that a prefill of the tokens before it gives.  Two fp32 dot products of 128 terms
    over |h| <= sqrt(128) (a LayerNorm row), |w| <= 0.025 sqrt(128) differ by at most 2 * 128 * 2^-24 * 3.2 = 5e-5, a log
    probability by twice that; with the int8 head the products are exact."""
    r = np.random.default_rng(9)
    B, P, k = 2, 23, 6
    toks = r.integers(0, 1000, (B, P)).astype(np.int32)
    eng = ie.Engine(tiny_dir, max_batch=B, **kw)
    s = eng.score(toks, k)
    assert eng.session_tokens() == P
    assert not s.logprobs[:, -1].any() and not s.ranks[:, -1].any()
    for t in range(P):
        eng.reset()
        logits = eng.prefill(toks[:, :t + 1])
        for b in range(B):
            lp = log_softmax(logits[b])
            H = -(np.exp(lp) * lp).sum()
            assert abs(s.entropy[b, t] - H) <= 1e-4 * (1 + H)
            assert np.abs(s.top_logprobs[b, t] - np.sort(lp)[::-1][:k]).max() <= 1.1e-4
            assert np.abs(s.top_logprobs[b, t] - lp[s.top_indices[b, t]]).max() <= 1.1e-4
            if t + 1 < P:
                y = toks[b, t + 1]
                assert abs(s.logprobs[b, t] - lp[y]) <= 1.1e-4
                assert (lp > lp[y] + 2.2e-4).sum() < s.ranks[b, t] <= (lp >= lp[y] - 2.2e-4).sum()
    eng.close()


def test_score_over_the_8_bit_cache(ie, small_dir):
    """The last row's prediction is the one whose logits a prefill of the same tokens leaves; the session goes on."""
    r = np.random.default_rng(10)
    toks = r.integers(0, 1000, (2, 50)).astype(np.int32)
    a, b = (ie.Engine(small_dir, max_batch=2, kv_dtype=ie.KV_I8) for _ in range(2))
    s = a.score(toks, 3)
    logits = b.prefill(toks)
    for i in range(2):
        lp = log_softmax(logits[i])
        # (768 terms: 2 * 768 * 2^-24 * 0.025 * 768 = 1.8e-3 at worst, twice that for a log probability)
        assert np.abs(s.top_logprobs[i, -1] - np.sort(lp)[::-1][:3]).max() <= 3.6e-3
    assert (s.logprobs[:, :-1] < 0).all() and (s.ranks[:, :-1] >= 1).all() and (s.entropy > 0).all()
    nxt = r.integers(0, 1000, 2)
    assert np.array_equal(a.step(nxt), b.step(nxt))


def test_score_in_any_order(ie, tiny_dir):
    """Calls of other sizes on one engine, in the middle of a session, and with arrays left out."""
    r = np.random.default_rng(11)
    toks = r.integers(0, 1000, (2, 40)).astype(np.int32)
    one, many = (ie.Engine(tiny_dir, max_batch=2, kv_dtype=ie.KV_I8) for _ in range(2))
    whole = one.score(toks, 8)
    at = 0
    for P, k in ((3, 0), (20, 8), (1, 2), (16, 8)):
        s = many.score(toks[:, at:at + P], k)
        for got, want in ((s.logprobs, whole.logprobs), (s.entropy, whole.entropy)):  # (a chunk's last token has no next one in it)
            assert np.abs(got[:, :P - 1] - want[:, at:at + P - 1]).max(initial=0) <= 3e-2 * np.abs(want).max()
        assert s.top_indices.shape == (2, P, k) and many.session_tokens() == at + P
        at += P
    lp = np.full((2, 40), 7, np.float32)
    one.reset()
    ie.check("ie_engine_score", one.h, 2, 40, toks.ctypes.data, 0, lp.ctypes.data, None, None, None, None)
    assert np.array_equal(lp, whole.logprobs)


def test_score_refusals(ie, tiny_dir):
    eng = ie.Engine(tiny_dir, max_batch=1)
    for toks, k in (([[1, 2]], -1), ([[1, 2]], ie.LOGPROBS_TOP_MAX + 1), ([[1, 1000]], 0), ([[1] * 65], 0), ([[1], [2]], 0)):
        with pytest.raises(ie.IeError):
            eng.score(np.array(toks), k)
    assert eng.session_tokens() == 0
    eng.close()


@pytest.mark.parametrize("kw", [dict(), dict(int8_lm_head=True)])
def test_score_with_fewer_alternatives_than_before(ie, kw):
    """At GPT-2's vocabulary, where rows are cut and fewer alternatives allow more parts (and a larger workspace): any
    order of k, and rows that grow between, give the bits of an engine that is asked once."""
    cfg = dict(TINY, n_layers=1, vocab_size=50257, seed=5, kv_dtype=ie.KV_I8, max_batch=2, **kw)
    r = np.random.default_rng(13)
    many = ie.Engine(**cfg)
    for P, k in ((8, 100), (8, 20), (8, 10), (8, 128), (8, 5), (8, 0), (3, 1), (30, 81), (30, 7), (60, 12)):
        toks = r.integers(0, 50257, (2, P)).astype(np.int32)
        many.reset()
        got = many.score(toks, k)
        once = ie.Engine(**cfg)
        assert all(np.array_equal(a, b) for a, b in zip(got, once.score(toks, k))), (P, k)
        once.close()
    many.close()


# ------------------------------------------------------------------ a step past the end of text
EOS = 50256
WIDE = dict(n_layers=2, vocab_size=EOS + 1, max_seq_len=1100)  # GPT-2 Small's widths: the fused step


@pytest.fixture(scope="module")
def wide_dir(tmp_path_factory, ie):
    d = tmp_path_factory.mktemp("gpt2_wide_kv8")
    ie.write_random_model(d, seed=23, **WIDE)
    return d


def end_after(ie, model_dir, prompts, scale):
    """Makes <|endoftext|> the token that follows each of the prompts: its embedding becomes scale times the sum of their
    last hidden rows (found from their logits by least squares), whose logits stand far above the others'.  Larger ones
    than the prompt's, they give the key and value rows of the step that is fed with it."""
    wte = np.fromfile(model_dir / "wte.bin", np.float32).reshape(EOS + 1, -1)
    eng = ie.Engine(model_dir, max_batch=len(prompts), kv_dtype=ie.KV_I8)
    logits = eng.prefill(prompts).astype(np.float64)
    eng.close()
    w = wte[:EOS].astype(np.float64)
    hidden = np.linalg.solve(w.T @ w, w.T @ logits[:, :EOS].T)  # [d, prompts]
    wte[EOS] = scale * hidden.sum(axis=1)
    wte.tofile(model_dir / "wte.bin")


@pytest.mark.parametrize("B,P,kw", [(1, 17, dict()), (1, 18, dict(fuse=False)), (1, 21, dict(use_graph=False)), (1, 16, dict()),
                                    (2, 31, dict()), (2, 19, dict(fuse=False)), (1, 1026, dict()), (2, 1035, dict()),
                                    (1, 1030, dict(fuse=False, use_graph=False))])
def test_a_step_past_the_end_leaves_no_trace(ie, wide_dir, B, P, kw):
    """Greedy decoding has the step behind <|endoftext|> under way before the host reads that token.  The session that goes
    on from there has the bits of one that was never fed it, where the step's rows made pages' scales grow too: in the
    middle of a page, at its first row, in one launch with the attention and in two, and past the change to split contexts."""
    r = np.random.default_rng(P)
    prompts = r.integers(0, EOS, (B, P)).astype(np.int32)
    end_after(ie, wide_dir, prompts, 0.02)
    a, b = (ie.Engine(wide_dir, max_batch=2, kv_dtype=ie.KV_I8, **kw) for _ in range(2))
    for _ in range(2):  # (the second time over pages that hold the first one's)
        if B == 1:
            ids, _ = a.generate_one(prompts[0], 9, greedy=True)
            assert ids == []
        else:
            out, _ = a.generate(prompts, 9)
            assert (out == -1).all()
        b.reset()
        b.prefill(prompts)
        assert a.session_tokens() == b.session_tokens() == P
        for t in r.integers(0, EOS, (4, B)).astype(np.int32):
            assert np.array_equal(a.step(t), b.step(t))
        more = r.integers(0, EOS, (B, 5)).astype(np.int32)
        assert np.array_equal(a.prefill(more), b.prefill(more))
    a.close()
    b.close()

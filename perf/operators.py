"""The operators around a KV cache held in 8 bits and around a model's log probabilities, as cases that can be timed and checked.

A case is one pass: rows into the cache (a prompt's, or one token a sequence) and back out of it as values, one token's
attention over it, a prompt's attention over it, or the log probabilities of given tokens with their ranks, the rows'
entropies and the top alternatives.  listed() holds fixed sizes, draw() others from the ranges that they stand for.  Where
`own` is false, run() computes the plain form: elementary torch operations in fp32.

The cache: pages of `block` tokens; K codes [pages, heads, block, d] int8, V codes [pages, heads, block / 16, d, 16] int8
(the 16 tokens of a group side by side for each channel), and a scale for each page and head, [pages, heads] fp32, of K
and of V.  A value is its code times its scale.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
FLOOR = 2.0**-100  # the least scale: a page of zeros has it
GROWTH = 1.25  # a scale that has to grow grows by this at least


def listed():
    return [
        # one decoded token's rows a sequence for a small batch at GPT-2 Small's heads: launches and latency
        _write("append-batch8", B=8, P=1, start=700, H=12, d=64, block=16),
        # a batch of prompts that go on behind a page's middle
        _write("write-prompts-2k", B=4, P=2000, start=21, H=8, d=128, block=16),
        # one GPT-2 Small sequence's decode attention at its full context: latency
        _decode("decode-one-1k", B=1, H_kv=12, G=1, d=64, ctx=1024, block=16, ragged=False),
        # three queries a head, odd ragged contexts, larger pages
        _decode("decode-odd", B=7, H_kv=4, G=3, d=64, ctx=1001, block=32, ragged=True),
        # grouped-query decode attention over long ragged contexts: the serving batch
        _decode("decode-gqa-8k", B=32, H_kv=8, G=4, d=128, ctx=8192, block=16, ragged=True),
        # two very long contexts, eight queries a head
        _decode("decode-long", B=2, H_kv=8, G=8, d=128, ctx=40000, block=64, ragged=False),
        # a batch of GPT-2-like prompts
        _prompt("prompt-512", B=4, P=512, start=0, H_kv=12, G=1, d=64, block=16),
        # a short chunk behind a long context, odd sizes
        _prompt("prompt-chunk", B=1, P=77, start=4001, H_kv=8, G=4, d=128, block=16),
        # a long prompt with grouped queries
        _prompt("prompt-4k", B=1, P=4096, start=0, H_kv=8, G=4, d=128, block=32),
        # a decode batch's log probabilities with five alternatives
        _logprobs("logprobs-step", rows=8, n=50257, k=5, pad=0, masked=False),
        # fewer tokens allowed than the vocabulary has (a grammar's mask), an odd width
        _logprobs("logprobs-masked", rows=300, n=32001, k=1, pad=0, masked=True),
        # a scored prompt with twenty alternatives, rows padded to a multiple of 64
        _logprobs("logprobs-prompt", rows=2048, n=50257, k=20, pad=47, masked=False),
    ]


def draw(rng):
    kind = rng.choice(("write", "decode", "decode", "prompt", "prompt", "logprobs"))
    d, block = rng.choice((64, 128)), rng.choice((16, 16, 32, 64, 128))
    while True:
        if kind == "write":
            c = _write(None, B=_log(rng, 1, 64), P=rng.choice((1, 1, _log(rng, 2, 2048))), start=_log(rng, 1, 2048) - 1,
                       H=rng.choice((2, 4, 8, 12, 16)), d=d, block=block)
            if c["B"] * c["P"] * c["H"] * d <= 8192 * 1024:
                return c
        elif kind == "decode":
            c = _decode(None, B=_log(rng, 1, 64), H_kv=rng.choice((1, 2, 4, 8, 12)), G=rng.choice((1, 1, 2, 3, 4, 6, 8, 12)),
                        d=d, ctx=_log(rng, 1, 16384), block=block, ragged=rng.random() < 0.5)
            if work(c)["bytes"] <= 300e6:
                return c
        elif kind == "prompt":
            c = _prompt(None, B=_log(rng, 1, 8), P=_log(rng, 1, 2048), start=rng.choice((0, _log(rng, 1, 4096))),
                        H_kv=rng.choice((1, 2, 4, 8, 12)), G=rng.choice((1, 1, 2, 3, 4, 8)), d=d, block=block)
            if work(c)["flops"] <= 6e10:
                return c
        else:
            c = _logprobs(None, rows=_log(rng, 1, 2048), n=_log(rng, 50, 131072), k=rng.choice((0, 1, _log(rng, 2, 40))),
                          pad=rng.choice((0, 0, rng.randint(1, 64))), masked=rng.random() < 0.3)
            if c["rows"] * c["n"] <= 60e6:
                return c


def prepare(case, seed):
    return _OPS[case["op"]]["prepare"](case, seed)


def run(state):
    if own:
        return _OPS[state["op"]]["own"](_package(), state)
    return _OPS[state["op"]]["plain"](state)


def work(case):
    return _OPS[case["op"]]["work"](case)


def exact(case, seed):
    return _OPS[case["op"]]["exact"](case, seed)


# ------------------------------------------------------------------ sizes and inputs
def _package():
    if "ie_amd" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "cuda-llm-inference-engine_amd"))
    import ie_amd

    return ie_amd


def _named(name, c):
    return dict(c, name=name) if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def _lens(case):
    """Context lengths: all ctx, or spread over its upper half with one sequence that holds nothing yet."""
    if not case["ragged"]:
        return [case["ctx"]] * case["B"]
    r = random.Random(case["ctx"])
    lens = [r.randint((case["ctx"] + 1) // 2, case["ctx"]) for _ in range(case["B"])]
    return lens[:-1] + [0] if len(lens) > 2 else lens


def _pages(n, block):
    return (n + block - 1) // block


def _codes(x):
    """Pages of values [pages, heads, block, d] as codes and scales."""
    scale = (x.abs().amax(dim=(2, 3)) / torch.full((), 127.0, device=DEV)).clamp_(min=FLOOR)
    inv = torch.ones_like(scale) / scale
    return (x * inv[:, :, None, None]).round_().clamp_(-127, 127).to(torch.int8), scale


def _grouped(v):
    """V codes [pages, heads, block, d] as the cache holds them."""
    n, h, block, d = v.shape
    return v.reshape(n, h, block // 16, 16, d).transpose(3, 4).contiguous()


def _cache(g, lens, H, d, block):
    """A cache whose sequences' pages lie scattered, rows as a model's keys and values have them, and the block table."""
    nb = [_pages(n, block) for n in lens]
    total = sum(nb) + 1
    size = torch.exp(0.3 * _normal(g, total, H, 1, 1))
    k, ks = _codes((_normal(g, total, H, block, d) + 0.5 * _normal(g, H, 1, d)) * size)
    v, vs = _codes(_normal(g, total, H, block, d) * size)
    order = torch.randperm(total, device=DEV, generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max(1, max(nb)), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(nb):
        table[b, :n] = order[at:at + n]
        at += n
    return {"k": k, "v": _grouped(v), "ks": ks, "vs": vs, "table": table}


def _values(codes, scales, table):
    """The rows behind table [B, nb] as [B, heads, nb * block, d]: codes [pages, heads, block, d] times their scales."""
    x = codes[table.long()].float() * scales[table.long()][..., None, None]
    B, nb, H, block, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, nb * block, d)


def _ungrouped(v):
    n, h, groups, d, _ = v.shape
    return v.transpose(3, 4).reshape(n, h, groups * 16, d)


# ------------------------------------------------------------------ rows into the cache and out of it
def _write(name, B, P, start, H, d, block):
    return _named(name, dict(op="write", B=B, P=P, start=start, H=H, d=d, block=block))


def _write_starts(case):
    """Where each sequence goes on: a prompt's chunk at one place, single tokens at places of their own."""
    if case["P"] > 1:
        return [case["start"]] * case["B"]
    r = random.Random(case["start"])
    return [r.randint(case["start"] // 2, case["start"]) for _ in range(case["B"])]


def _write_inputs(case, seed):
    g, B, P, H, d = _generator(seed), case["B"], case["P"], case["H"], case["d"]
    starts = _write_starts(case)
    s = _cache(g, [n + P for n in starts], H, d, case["block"])
    s["qkv"] = _normal(g, B, P, 3, H, d) * torch.exp(0.3 * _normal(g, B, P, 1, 1, 1))  # a projection's rows: K and V lie inside
    return s, starts


def _write_prepare(case, seed):
    s, starts = _write_inputs(case, seed)
    B, P, H, d, block = case["B"], case["P"], case["H"], case["d"], case["block"]
    n = P + case["start"] % block if P > 1 else block
    s |= {"op": "write", "P": P, "start": case["start"], "n": n, "block": block, "new_k": s["qkv"][:, :, 1], "new_v": s["qkv"][:, :, 2]}
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["first"] = s["starts"] // block * block  # the rows read back begin with the page
    s["ends"] = s["starts"] + P
    s["out_k"], s["out_v"] = (torch.empty(B, n, H, d, device=DEV) for _ in range(2))
    return s


def _write_own(ie, s):
    cache = ie.Kv8Cache(s["k"], s["v"], s["ks"], s["vs"])
    if s["P"] == 1:
        ie.kv8_cache_append_batch(s["new_k"][:, 0], s["new_v"][:, 0], cache, s["table"], s["starts"])
    else:
        ie.kv8_cache_write(s["new_k"], s["new_v"], cache, s["table"], s["start"])
    return ie.kv8_cache_read(cache, s["table"], s["first"], s["ends"], s["n"], out=(s["out_k"], s["out_v"]))


def _write_plain(s):
    block, P, n = s["block"], s["P"], s["n"]
    B, H, d = s["qkv"].shape[0], s["qkv"].shape[3], s["qkv"].shape[4]
    nb = _pages(n, block)
    page = s["first"][:, None] // block + torch.arange(nb, device=DEV)  # [B, nb], in each sequence's own order
    phys = torch.gather(s["table"], 1, page.clamp(max=s["table"].shape[1] - 1).long()).long()
    pos = page[:, :, None] * block + torch.arange(block, device=DEV)  # [B, nb, block]
    t = pos - s["starts"][:, None, None]
    fresh, old = ((t >= 0) & (t < P))[..., None, None], (t < 0)[..., None, None]
    begins = (pos[:, :, 0] >= s["starts"][:, None])[:, :, None]  # the page's first row is written, or one before it is none of ours
    out = []
    for name, scales, new in (("k", "ks", s["new_k"]), ("v", "vs", s["new_v"])):
        x = torch.gather(new, 1, t.clamp(0, P - 1).reshape(B, -1, 1, 1).expand(-1, -1, H, d)).reshape(B, nb, block, H, d)
        x = torch.where(fresh, x, 0.0)
        had = s[scales][phys]  # [B, nb, H]
        need = (x.abs().amax(dim=(2, 4)) / torch.full((), 127.0, device=DEV)).clamp_(min=FLOOR)
        grown = torch.where(need <= had, had, torch.maximum(need, GROWTH * had))
        scale = torch.where(begins, need, grown)
        inv = torch.ones_like(scale) / scale
        codes = (s["k"][phys] if name == "k" else _ungrouped(s["v"][phys.reshape(-1)]).reshape(B, nb, H, block, d)).permute(0, 1, 3, 2, 4)
        moved = (codes.float() * (had * inv)[:, :, None, :, None]).round().to(torch.int8)
        kept = torch.where((scale == had)[:, :, None, :, None], codes, moved)
        fine = (x * inv[:, :, None, :, None]).round_().clamp_(-127, 127).to(torch.int8)
        codes = torch.where(fresh, fine, torch.where(old, kept, codes))
        pages = codes.permute(0, 1, 3, 2, 4).reshape(B * nb, H, block, d)
        s[name][phys.reshape(-1)] = pages.contiguous() if name == "k" else _grouped(pages)
        s[scales][phys.reshape(-1)] = scale.reshape(B * nb, H)
        value = torch.where(pos[..., None, None] < s["ends"][:, None, None, None, None], codes.float() * scale[:, :, None, :, None], 0.0)
        out.append(value.reshape(B, nb * block, H, d)[:, :n])
    return out


def _write_work(case):
    values = case["B"] * case["P"] * case["H"] * case["d"]
    back = case["B"] * (case["P"] + case["start"] % case["block"] if case["P"] > 1 else case["block"]) * case["H"] * case["d"]
    return {"bytes": 2 * (4 * values + values + back + 4 * back), "flops": 6 * values}


def _write_exact(case, seed):
    """Page by page, from the cache's definition: its scales and its products are fp32 numbers, so these steps round as fp32 does."""
    s, starts = _write_inputs(case, seed)
    B, P, H, d, block = case["B"], case["P"], case["H"], case["d"], case["block"]
    if B * P // block > 2000:
        return None
    n, table, out = P + case["start"] % block if P > 1 else block, s["table"].tolist(), []
    for which, codes, scales in ((1, s["k"], s["ks"]), (2, _ungrouped(s["v"]), s["vs"])):
        got = torch.zeros(B, n, H, d, dtype=torch.float64, device=DEV)
        for b in range(B):
            first = starts[b] // block * block
            for page in range(first // block, _pages(starts[b] + P, block)):
                lo, hi = max(starts[b], page * block), min(starts[b] + P, (page + 1) * block)
                before, p = lo - page * block, table[b][page]
                x = s["qkv"][b, lo - starts[b]:hi - starts[b], which].double()  # [rows, H, d]
                need = (x.abs().amax(dim=(0, 2)) / 127).float().clamp(min=FLOOR)
                had = scales[p]
                bigger = torch.maximum(need.double(), (GROWTH * had.double()).float().double()).float()
                scale = need if before == 0 else torch.where(need > had, bigger, had)
                inv = (1 / scale.double()).float().double()
                q = (x * inv[None, :, None]).float().round().clamp(-127, 127).double()
                if before:
                    q0 = codes[p, :, :before].double().transpose(0, 1)  # [rows, H, d]
                    moved = (q0 * (had.double() * inv).float().double()[None, :, None]).float().round().double()
                    q = torch.cat([torch.where((scale == had)[None, :, None], q0, moved), q])
                at = page * block - first
                got[b, at:at + before + hi - lo] = (q * scale.double()[None, :, None])
        out.append(got)
    return out


# ------------------------------------------------------------------ one token's attention over the cache
def _decode(name, B, H_kv, G, d, ctx, block, ragged):
    return _named(name, dict(op="decode", B=B, H_kv=H_kv, G=G, d=d, ctx=ctx, block=block, ragged=ragged))


def _decode_inputs(case, seed):
    g, lens = _generator(seed), _lens(case)
    s = _cache(g, lens, case["H_kv"], case["d"], case["block"])
    s["q"] = _normal(g, case["B"], case["H_kv"] * case["G"], case["d"])
    return s, lens


def _decode_prepare(case, seed):
    s, lens = _decode_inputs(case, seed)
    B, H, d = s["q"].shape
    s |= {"op": "decode", "top": max(lens), "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "out": torch.empty_like(s["q"])}
    s["workspace"] = torch.empty(B * H * 64 * (d + 2), device=DEV)
    return s


def _decode_own(ie, s):
    cache = ie.Kv8Cache(s["k"], s["v"], s["ks"], s["vs"])
    return ie.decode_attn_kv8(s["q"], cache, s["table"], s["lens"], s["top"], out=s["out"], workspace=s["workspace"])


def _decode_plain(s):
    B, H, d = s["q"].shape
    k, v = _values(s["k"], s["ks"], s["table"]), _values(_ungrouped(s["v"]), s["vs"], s["table"])  # [B, H_kv, n, d]
    H_kv, n = k.shape[1], k.shape[2]
    score = torch.matmul(s["q"].reshape(B, H_kv, H // H_kv, d), k.transpose(2, 3).contiguous()) / math.sqrt(d)
    seen = (torch.arange(n, device=DEV) < s["lens"][:, None])[:, None, None, :]
    score = torch.where(seen, score, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = torch.where(seen, torch.exp(score - top), 0.0)
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return o.reshape(B, H, d)


def _decode_work(case):
    n, H = sum(_lens(case)), case["H_kv"] * case["G"]
    pages = sum(_pages(x, case["block"]) for x in _lens(case))
    return {"bytes": 2 * n * case["H_kv"] * case["d"] + pages * (8 * case["H_kv"] + 4) + 8 * case["B"] * H * case["d"],
            "flops": 4 * n * H * case["d"]}


def _attention64(q, k, v, mask=None):
    """softmax(q k^T / sqrt(d)) v in 64 bits: q [G, t, d], k and v [n, d]."""
    score = (q @ k.t()) / math.sqrt(q.shape[-1])
    if mask is not None:
        score = score.masked_fill(~mask, -math.inf)
    return torch.softmax(score, dim=-1) @ v


def _head64(s, b, h, n):
    """The first n rows of sequence b, head h in 64 bits: K and V [n, d]."""
    pages = s["table"][b].long()
    k = s["k"][pages, h].double() * s["ks"][pages, h].double()[:, None, None]  # [nb, block, d]
    v = s["v"][pages, h].double() * s["vs"][pages, h].double()[:, None, None, None]  # [nb, groups, d, 16]
    d = k.shape[-1]
    return k.reshape(-1, d)[:n], v.permute(0, 1, 3, 2).reshape(-1, d)[:n]


def _decode_exact(case, seed):
    s, lens = _decode_inputs(case, seed)
    G = case["G"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        for h in range(case["H_kv"] if n else 0):
            q = s["q"][b, h * G:(h + 1) * G].double()[:, None]
            out[b, h * G:(h + 1) * G] = _attention64(q, *_head64(s, b, h, n))[:, 0]
    return out


# ------------------------------------------------------------------ a prompt's attention over the cache
def _prompt(name, B, P, start, H_kv, G, d, block):
    return _named(name, dict(op="prompt", B=B, P=P, start=start, H_kv=H_kv, G=G, d=d, block=block))


def _prompt_inputs(case, seed):
    g, n = _generator(seed), case["start"] + case["P"]
    s = _cache(g, [n] * case["B"], case["H_kv"], case["d"], case["block"])
    s["q"] = _normal(g, case["B"], case["P"], case["H_kv"] * case["G"], case["d"])
    return s


def _prompt_prepare(case, seed):
    s = _prompt_inputs(case, seed)
    return s | {"op": "prompt", "start": case["start"], "out": torch.empty_like(s["q"])}


def _prompt_own(ie, s):
    return ie.prefill_attn_kv8(s["q"], ie.Kv8Cache(s["k"], s["v"], s["ks"], s["vs"]), s["table"], s["start"], out=s["out"])


def _prompt_plain(s):
    B, P, H, d = s["q"].shape
    k, v = _values(s["k"], s["ks"], s["table"]), _values(_ungrouped(s["v"]), s["vs"], s["table"])
    H_kv, n = k.shape[1], k.shape[2]
    q = s["q"].permute(0, 2, 1, 3).reshape(B, H_kv, H // H_kv * P, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d)
    seen = (torch.arange(n, device=DEV) <= s["start"] + torch.arange(P, device=DEV)[:, None]).repeat(H // H_kv, 1)
    score = torch.where(seen, score, -math.inf)
    p = torch.exp(score - score.amax(dim=-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)
    return o.reshape(B, H, P, d).permute(0, 2, 1, 3).contiguous()


def _prompt_work(case):
    B, P, start, d, H = case["B"], case["P"], case["start"], case["d"], case["H_kv"] * case["G"]
    pages = B * _pages(start + P, case["block"])
    return {"bytes": 8 * B * P * H * d + 2 * B * (start + P) * case["H_kv"] * d + pages * (8 * case["H_kv"] + 4),
            "flops": 4 * B * H * d * (P * start + P * (P + 1) // 2)}


def _prompt_exact(case, seed):
    s, B, P, G, n = _prompt_inputs(case, seed), case["B"], case["P"], case["G"], case["start"] + case["P"]
    mask = torch.arange(n, device=DEV)[None, :] <= case["start"] + torch.arange(P, device=DEV)[:, None]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for b in range(B):
        for h in range(case["H_kv"]):
            q = s["q"][b, :, h * G:(h + 1) * G].double().transpose(0, 1)
            out[b, :, h * G:(h + 1) * G] = _attention64(q, *_head64(s, b, h, n), mask).transpose(0, 1)
    return out


# ------------------------------------------------------------------ log probabilities
def _logprobs(name, rows, n, k, pad, masked):
    return _named(name, dict(op="logprobs", rows=rows, n=n, k=min(k, n), pad=pad, masked=masked))


def _logprobs_inputs(case, seed):
    """Rows as a model gives them: most near-normal with a few tokens well above the rest, some nearly certain; pads hold NaN."""
    g, rows, n = _generator(seed), case["rows"], case["n"]
    x = _normal(g, rows, n + case["pad"]) * torch.exp(0.7 * _normal(g, rows, 1))
    likely = torch.randint(n, (rows, 8), device=DEV, generator=g)
    x.scatter_add_(1, likely, 4.0 + 12.0 * torch.rand(rows, 8, device=DEV, generator=g))
    if case["masked"]:
        allowed = torch.rand(x.shape, device=DEV, generator=g) < 0.05
        x = torch.where(allowed.scatter(1, likely, True), x, -math.inf)
    x[:, n:] = math.nan
    pick = torch.randint(8, (rows, 1), device=DEV, generator=g)
    anywhere = torch.randint(n, (rows, 1), device=DEV, generator=g)
    likely = torch.gather(likely, 1, pick)
    targets = torch.where(torch.rand(rows, 1, device=DEV, generator=g) < 0.7, likely, anywhere)[:, 0]
    return x, targets.to(torch.int32)


def _logprobs_prepare(case, seed):
    x, targets = _logprobs_inputs(case, seed)
    rows, k = case["rows"], case["k"]
    whole, real = (dict(dtype=t, device=DEV) for t in (torch.int32, torch.float32))
    return {"op": "logprobs", "x": x[:, :case["n"]], "targets": targets, "k": k,
            "out": (torch.empty(rows, **real), torch.empty(rows, **whole), torch.empty(rows, **real),
                    torch.empty(rows, k, **real), torch.empty(rows, k, **whole)),
            "workspace": torch.empty(rows * 16 * (8 + 2 * k), **real)}


def _logprobs_own(ie, s):
    return ie.token_logprobs(s["x"], s["targets"], s["k"], out=s["out"], workspace=s["workspace"])


def _logprobs_plain(s):
    x, n = s["x"], s["x"].shape[1]
    t = s["targets"].long()[:, None]
    x_t = torch.gather(x, 1, t)
    index = torch.arange(n, device=DEV)
    rank = 1 + ((x > x_t) | ((x == x_t) & (index < t))).sum(dim=1)
    down = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(down)
    total = e.sum(dim=1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total - (e * torch.where(e > 0, down, 0.0)).sum(dim=1, keepdim=True) / total
    logprob = torch.gather(down, 1, t) - log_total
    first = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["k"]]
    return (logprob[:, 0], rank.to(torch.int32), entropy[:, 0], torch.gather(down, 1, first) - log_total, first.to(torch.int32))


def _logprobs_work(case):
    rows, n, k = case["rows"], case["n"], case["k"]
    return {"bytes": 4 * rows * n + rows * (16 + 8 * k), "flops": 6 * rows * n}


def _logprobs_exact(case, seed):
    x, targets = _logprobs_inputs(case, seed)
    x, rows = x[:, :case["n"]], torch.arange(case["rows"], device=DEV)
    logprob, entropy, first = [], [], []
    for lo in range(0, case["rows"], 256):
        y = torch.log_softmax(x[lo:lo + 256].double(), dim=1)
        entropy.append(-torch.where(torch.isinf(y), 0.0, torch.exp(y) * y).sum(dim=1))
        logprob.append(y[torch.arange(y.shape[0], device=DEV), targets[lo:lo + 256].long()])
        first.append(torch.sort(y, dim=1, descending=True).values[:, :case["k"]])
    x_t = x[rows, targets.long()][:, None]
    rank = 1 + (x > x_t).sum(dim=1) + ((x == x_t) & (torch.arange(case["n"], device=DEV)[None] < targets[:, None])).sum(dim=1)
    return torch.cat(logprob), rank, torch.cat(entropy), torch.cat(first), None


_OPS = {
    "write": dict(prepare=_write_prepare, own=_write_own, plain=_write_plain, work=_write_work, exact=_write_exact),
    "decode": dict(prepare=_decode_prepare, own=_decode_own, plain=_decode_plain, work=_decode_work, exact=_decode_exact),
    "prompt": dict(prepare=_prompt_prepare, own=_prompt_own, plain=_prompt_plain, work=_prompt_work, exact=_prompt_exact),
    "logprobs": dict(prepare=_logprobs_prepare, own=_logprobs_own, plain=_logprobs_plain, work=_logprobs_work, exact=_logprobs_exact),
}

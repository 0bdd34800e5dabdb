"""Cases of the paged serving operators: what is timed, in plain form and through the framework.

One step of a served model keeps its keys and values in pages: the new tokens'
rows are rotated and appended (``append``), the queries attend to the cached
ones through the page table, all of them or a window with a few first tokens
(``attend``), a batch that shares a long prefix reads it once for all
(``prefix``), and the next tokens are drawn from the logits (``sample``).

``run`` computes a case with elementary torch operations in 32 bits, or, where
``own`` is true, through ``nkipy_b200.runtime``.  ``exact`` restates the
definitions in 64 bits.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _append(name, seqs, new, past, hq, hkv, d, rot, page, dtype, ragged):
    return dict(name=name, op="append", seqs=seqs, new=new, past=past, hq=hq, hkv=hkv, d=d, rot=rot, page=page,
                dtype=dtype, ragged=ragged)


def _attend(name, seqs, new, past, window, sinks, hq, hkv, d, page, dtype, ragged):
    return dict(name=name, op="attend", seqs=seqs, new=new, past=past, window=window, sinks=sinks, hq=hq, hkv=hkv, d=d,
                page=page, dtype=dtype, ragged=ragged)


def _prefix(name, seqs, prefix, new, past, hq, hkv, d, page, dtype, ragged):
    return dict(name=name, op="prefix", seqs=seqs, prefix=prefix, new=new, past=past, hq=hq, hkv=hkv, d=d, page=page,
                dtype=dtype, ragged=ragged)


def _sample(name, rows, vocab, dtype, mix):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, dtype=dtype, mix=mix)


def listed():
    return [
        # one decode step's cache update: 8 sequences, one token each, the 32/8-head attention layer
        _append("append decode 8", 8, 1, 2047, 32, 8, 128, 128, 16, "bf16", False),
        # a ragged chunk of prompts in fp16, 64-wide heads of which the first 32 dimensions rotate
        _append("append chunk 1500", 5, 300, 700, 12, 4, 64, 32, 64, "f16", True),
        # prefill of 4 prompts of 2048 tokens: every row of q, k and v of one layer
        _append("append prefill 8192", 4, 2048, 0, 32, 8, 128, 128, 16, "bf16", False),
        # one user, one token, a short context: latency alone
        _attend("attend decode 1", 1, 1, 500, 0, 0, 32, 8, 128, 16, "bf16", False),
        # the batch of a decode step against 2048 cached tokens each, no window
        _attend("attend decode 8x2048", 8, 1, 2047, 0, 0, 32, 8, 128, 16, "bf16", False),
        # long ragged contexts (up to 32k tokens) read through a window of 4096 and 4 first tokens
        _attend("attend decode 64 window", 64, 1, 32000, 4096, 4, 32, 8, 128, 64, "bf16", True),
        # one 500-token chunk of a 16k-token prompt, no window, eight 64-wide query heads per key head
        _attend("attend chunk 500 of 16k", 1, 500, 15900, 0, 0, 32, 4, 64, 32, "f16", False),
        # prefill of 4 prompts of 2048 tokens with a window of 1024 and 4 first tokens
        _attend("attend prefill 8192 window", 4, 2048, 0, 1024, 4, 32, 8, 128, 16, "bf16", False),
        # few users of a system prompt of 1000 tokens
        _prefix("prefix 4x1000", 4, 1000, 1, 77, 32, 8, 128, 16, "bf16", True),
        # 64 decoding sequences that share 8192 tokens and own some hundreds each
        _prefix("prefix 64x8192", 64, 8192, 1, 400, 32, 8, 128, 64, "bf16", True),
        # one user's next token over a vocabulary of 32000, all filters on
        _sample("sample 1x32000", 1, 32000, "f32", "all"),
        # a batch of 128 over 151936 entries, each user with settings of their own
        _sample("sample 128x151936", 128, 151936, "bf16", "mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hkv = rng.choice([1, 2, 4, 8])
    return hkv * rng.choice([1, 2, 3, 4, 5, 7, 8]), hkv


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "prefix", "sample"])
    hq, hkv = _heads(rng)
    d, page, ragged = rng.choice([64, 64, 96, 128, 128]), rng.choice([16, 32, 64, 128]), rng.random() < 0.6
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(2, 8192 // seqs))
        rot = rng.choice([d, d, d // 2])
        return {k: v for k, v in _append("", seqs, new, _log(rng, 1, 4000), hq, hkv, d, rot, page,
                                         rng.choice([dtype, dtype, "f32"]), ragged).items() if k != "name"}
    if op == "attend":
        if rng.random() < 0.5:  # single tokens: at most the keys of 64 windows of 4096
            seqs = _log(rng, 1, 64)
            past = _log(rng, 1, max(2, 250000 // seqs))
            new = 1
        else:  # chunks and prompts: at most the products of 4 prompts of 2048
            seqs = _log(rng, 1, 8)
            new = _log(rng, 2, 2048 // max(1, seqs // 4))
            past = _log(rng, 1, max(2, 4000000 // (seqs * new))) if rng.random() < 0.5 else 0
            past = min(past, 16000)
        window, sinks = (0, 0) if rng.random() < 0.4 else (_log(rng, 1, 4096), rng.choice([0, 1, 4, 19]))
        return {k: v for k, v in _attend("", seqs, new, past, window, sinks, hq, hkv, d, page, dtype,
                                         ragged).items() if k != "name"}
    if op == "prefix":
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.7 else rng.randint(2, 5)
        return {k: v for k, v in _prefix("", seqs, _log(rng, 20, 8192), new, _log(rng, 1, 400), hq, hkv, d, page,
                                         dtype, ragged).items() if k != "name"}
    vocab = _log(rng, 1000, 151936)
    return {k: v for k, v in _sample("", _log(rng, 1, 128), vocab, rng.choice(["bf16", "f16", "f32"]),
                                     rng.choice(["plain", "all", "mixed"])).items() if k != "name"}


def _lengths(case):
    """New tokens and earlier tokens of each sequence: from the case alone."""
    n, new, past = case["seqs"], case["new"], case["past"]
    if not case["ragged"]:
        return [new] * n, [past] * n
    rng = random.Random(n * 1000003 + new * 1009 + past)
    news = [max(1, int(new * rng.uniform(0.2, 1.8))) if new > 1 else 1 for _ in range(n)]
    while sum(news) > n * new:  # the case's total is the most
        news[news.index(max(news))] -= 1
    return news, [int(past * rng.uniform(0.1, 1.0)) for _ in range(n)]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(gen, case, lengths, extra_pages=0):
    """Page table, and caches whose pages lie in any order, as after hours of serving."""
    page, hkv, d = case["page"], case["hkv"], case["d"]
    counts = [-(-n // page) for n in lengths]
    width, total = max(1, max(counts)), sum(counts) + extra_pages + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    at = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"))
    first = torch.tensor(np.cumsum([0] + counts[:-1]), device="cuda")
    used = torch.arange(sum(counts), device="cuda")
    table[at, used - first[at]] = order[: sum(counts)]
    dtype = DTYPES[case["dtype"]]
    k = _normal(gen, (total, page, hkv, d), dtype)
    v = _normal(gen, (total, page, hkv, d), dtype)
    return k, v, table, order[sum(counts) :]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "op": case["op"]}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # logits of a language model: a spread body and a few likely tokens
        x = torch.randn((rows, vocab), generator=gen, device="cuda") * 2.0
        top = torch.randint(vocab, (rows, 24), generator=gen, device="cuda")
        x.scatter_add_(1, top, torch.rand((rows, 24), generator=gen, device="cuda") * 9.0)
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["u"] = torch.rand((rows,), generator=gen, device="cuda")
        full = lambda v, t=torch.float32: torch.full((rows,), v, dtype=t, device="cuda")  # noqa: E731
        if case["mix"] == "plain":
            temperature, top_k, top_p, min_p = full(1.0), full(0, torch.int32), full(1.0), full(0.0)
        elif case["mix"] == "all":
            temperature, top_k, top_p, min_p = full(0.7), full(50, torch.int32), full(0.9), full(0.05)
        else:
            pick = lambda vals, t=torch.float32: torch.tensor(vals, dtype=t, device="cuda")[  # noqa: E731
                torch.randint(len(vals), (rows,), generator=gen, device="cuda")]
            temperature = pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3])
            top_k = pick([0, 0, 20, 50, 1000], torch.int32)
            top_p = pick([1.0, 1.0, 0.95, 0.8, 0.5])
            min_p = pick([0.0, 0.0, 0.05, 0.2])
        s.update(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        return s
    news, pasts = _lengths(case)
    lengths = [a + b for a, b in zip(news, pasts)]
    tokens, dtype = sum(news), DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    n_prefix = -(-case["prefix"] // case["page"]) if case["op"] == "prefix" else 0
    s["k_cache"], s["v_cache"], s["table"], free = _cache(gen, case, lengths, n_prefix)
    s["kv_len"], s["news"], s["pasts"] = _ints(lengths), news, pasts
    s["seq"] = torch.repeat_interleave(torch.arange(len(news), device="cuda"), torch.tensor(news, device="cuda"))
    s["local"] = torch.cat([torch.arange(n, device="cuda") for n in news])
    s["past"] = torch.tensor(pasts, device="cuda")
    s["q_start"] = None if case["new"] == 1 else _ints(np.cumsum([0] + news).tolist())
    if case["op"] == "append":
        # one projection's output holds q, k and v side by side
        qkv = _normal(gen, (tokens, hq + 2 * hkv, d), dtype)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
        ang = torch.arange(max(lengths), device="cuda", dtype=torch.float32)[:, None] * (
            500000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float32) / case["rot"]))
        s["cos"], s["sin"] = torch.cos(ang), torch.sin(ang)
        return s
    s["q"] = _normal(gen, (tokens, hq, d), dtype)
    if case["op"] == "prefix":
        s["prefix_pages"], s["prefix_len"] = free[:n_prefix].contiguous(), case["prefix"]
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from nkipy_b200 import runtime as nk

    if s["op"] == "sample":
        return {"tokens": nk.sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])}
    if s["op"] == "append":
        q = nk.paged_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["kv_len"], q_start=s["q_start"],
                            q=s["q"], cos=s["cos"], sin=s["sin"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if s["op"] == "prefix":
        return {"out": nk.prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"], s["prefix_len"],
                                           s["table"], s["kv_len"], q_start=s["q_start"])}
    return {"out": nk.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["kv_len"], q_start=s["q_start"],
                                      window=s["case"]["window"], sinks=s["case"]["sinks"])}


def _rotated(x, cos, sin, rot):
    """Half-split rotation of the first `rot` dimensions, in 32 bits, rounded once."""
    f = x.float()
    a, b, rest = f[..., : rot // 2], f[..., rot // 2 : rot], f[..., rot:]
    c, t = cos[:, None, :], sin[:, None, :]
    return torch.cat([a * c - b * t, a * t + b * c, rest], -1).to(x.dtype)


def _rows(cache, table, pos):
    """Cached rows of each sequence at positions (sequences, keys), in 32 bits."""
    page = cache.shape[1]
    pages = torch.gather(table.long(), 1, (pos // page).clamp(max=table.shape[1] - 1)).clamp(min=0)
    return cache[pages, pos % page].float()


def _softmax_product(parts, shape):
    """sum over parts of (scores, seen, values): the softmax over all parts' seen keys times their values."""
    scores = [torch.where(seen, x, float("-inf")) for x, seen, _ in parts]
    top = torch.cat([x.amax(-1, keepdim=True) for x in scores], -1).amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    e = [torch.exp(x - top) for x in scores]
    total = torch.cat([x.sum(-1, keepdim=True) for x in e], -1).sum(-1, keepdim=True)
    out = torch.stack([torch.matmul(x, v) for x, (_, _, v) in zip(e, parts)]).sum(0)
    return torch.where(total > 0, out / torch.where(total > 0, total, 1.0), 0.0).reshape(shape)


def _plain(s):
    case = s["case"]
    if s["op"] == "sample":
        return {"tokens": _plain_sample(s)}
    seq, local, past, page = s["seq"], s["local"], s["past"], case["page"]
    pos = past[seq] + local  # of each new token
    if s["op"] == "append":
        q, k = (_rotated(x, s["cos"][pos], s["sin"][pos], case["rot"]) for x in (s["q"], s["k"]))
        pages = s["table"][seq, pos // page].long()
        s["k_cache"][pages, pos % page] = k
        s["v_cache"][pages, pos % page] = s["v"]
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    n, most, g = case["seqs"], max(s["news"]), hq // hkv
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    # queries as (sequences, kv heads, new tokens * query heads of a group, d)
    q = torch.zeros((n, most, hq, d), device="cuda")
    q[seq, local] = s["q"].float()
    q = q.view(n, most, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, most * g, d) / math.sqrt(d)
    length = s["kv_len"].long()
    # the keys that any query of the sequence sees: the first ones and the windows'
    first = (past - window + 1).clamp(min=0) if window else torch.zeros_like(past)
    width = max(p + m - (max(0, p - window + 1) if window else 0) for p, m in zip(s["pasts"], s["news"]))
    at = torch.cat([torch.arange(sinks, device="cuda").expand(n, sinks),
                    first[:, None] + torch.arange(width, device="cuda")], 1)
    once = torch.ones_like(at, dtype=torch.bool)
    once[:, sinks:] = at[:, sinks:] >= sinks
    qpos = past[:, None] + torch.arange(most, device="cuda")
    seen = (once & (at < length[:, None]))[:, None, :] & (at[:, None, :] <= qpos[:, :, None])
    if window:
        seen &= (qpos[:, :, None] - at[:, None, :] < window) | (at < sinks)[:, None, :]
    seen = seen[:, None, :, None, :].expand(n, 1, most, g, at.shape[1]).reshape(n, 1, most * g, at.shape[1])
    k = _rows(s["k_cache"], s["table"], at).permute(0, 2, 3, 1)
    v = _rows(s["v_cache"], s["table"], at).permute(0, 2, 1, 3)
    parts = [(torch.matmul(q, k), seen, v)]
    if s["op"] == "prefix":
        where = torch.arange(s["prefix_len"], device="cuda")[None]
        pk = _rows(s["k_cache"], s["prefix_pages"][None], where).permute(0, 2, 3, 1)
        pv = _rows(s["v_cache"], s["prefix_pages"][None], where).permute(0, 2, 1, 3)
        scores = torch.matmul(q.transpose(0, 1).reshape(1, hkv, -1, d), pk)
        scores = scores.view(hkv, n, most * g, -1).transpose(0, 1)
        parts.append((scores, torch.ones((), dtype=torch.bool, device="cuda"), pv))
    out = _softmax_product(parts, (n, hkv, most, g, d))
    out = out.permute(0, 2, 1, 3, 4).reshape(n, most, hq, d)
    return {"out": out[seq, local].to(s["q"].dtype)}


def _plain_sample(s):
    """A token for each row.  Weights are exp in 32 bits, held as whole multiples of 2^-32 of the largest, so that
    sums do not depend on their order; ties in the logits go to the lowest index."""
    x = s["logits"].float()
    rows, vocab = x.shape
    greedy = s["temperature"] <= 0
    inv = torch.where(greedy, torch.ones_like(s["u"]), 1.0 / s["temperature"])[:, None]
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    top = x.gather(1, order[:, :1])
    e = torch.exp((x - top) * inv)
    w = (e * 4294967296.0).to(torch.int64)
    rank = torch.arange(vocab, device="cuda")
    k = torch.where((s["top_k"] <= 0) | (s["top_k"] > vocab), vocab, s["top_k"])
    ws = w.gather(1, order) * (rank < k[:, None])
    before = torch.cumsum(ws, 1) - ws
    total = ws.sum(1, keepdim=True)
    most = (s["top_p"].double()[:, None] * total.double()).to(torch.int64).clamp(min=1)
    ws = ws * ((s["top_p"] >= 1)[:, None] | (before < most))
    kept = torch.zeros_like(w).scatter_(1, order, ws) * (e >= s["min_p"][:, None])
    sums = torch.cumsum(kept, 1)
    at = (s["u"].double() * sums[:, -1].double()).to(torch.int64)
    token = (sums <= at[:, None]).sum(1)
    return torch.where(greedy, order[:, 0], token).to(torch.int32)


# ---------------------------------------------------------------------------
# work, and the definitions in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * size + 24), "flops": 4 * case["rows"] * case["vocab"]}
    news, pasts = _lengths(case)
    tokens, hq, hkv, d = sum(news), case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        spans = [(p, p + n) for p, n in zip(pasts, news)]
        spans.sort()
        rows, end = 0, 0
        for a, b in spans:  # rows of the tables that are read at least once
            rows += max(0, b - max(a, end))
            end = max(end, b)
        return {"bytes": 2 * tokens * (hq + 2 * hkv) * d * size + rows * case["rot"] * 4 + 4 * (tokens + 2 * len(news)),
                "flops": 3 * tokens * (hq + hkv) * case["rot"]}
    window, sinks, prefix = case.get("window", 0), case.get("sinks", 0), case.get("prefix", 0)
    keys = pairs = 0
    for n, p in zip(news, pasts):
        low = max(0, p - window + 1) if window else 0
        keys += p + n - low + min(sinks, low)
        for i in range(p, p + n):
            at = max(0, i - window + 1) if window else 0
            pairs += i + 1 - at + min(sinks, at) + prefix
    rows = keys + prefix
    return {"bytes": (2 * tokens * hq + 2 * rows * hkv) * d * size + 4 * (rows // case["page"] + 2 * len(news)),
            "flops": 4 * pairs * hq * d}


def exact(case, seed):
    if case["op"] == "sample":
        return None  # whole numbers
    s = prepare(case, seed)
    page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["d"]
    table = s["table"].cpu().numpy()
    starts = np.cumsum([0] + s["news"])
    if case["op"] == "append":
        half = case["rot"] // 2
        out = {"q": s["q"].double(), "k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
        for b, (n, p) in enumerate(zip(s["news"], s["pasts"])):
            at = np.arange(p, p + n)
            pages = torch.tensor(table[b][at // page], dtype=torch.long, device="cuda")
            slots = torch.tensor(at % page, device="cuda")
            t = slice(starts[b], starts[b + 1])
            z = torch.complex(s["cos"][p : p + n].double(), s["sin"][p : p + n].double())[:, None]
            turned = []
            for x in (s["q"][t].double(), s["k"][t].double()):
                y = torch.complex(x[..., :half], x[..., half : 2 * half]) * z
                turned.append(torch.cat([y.real, y.imag, x[..., 2 * half :]], -1))
            out["q"][t] = turned[0]
            out["k_cache"][pages, slots] = turned[1]
            out["v_cache"][pages, slots] = s["v"][t].double()
        return out
    if work(case)["flops"] > 4e12:
        return None
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    out = torch.zeros((starts[-1], hq, d), dtype=torch.float64, device="cuda")
    for b, (n, p) in enumerate(zip(s["news"], s["pasts"])):
        at = np.arange(p + n)
        pages = torch.tensor(table[b][at // page], dtype=torch.long, device="cuda")
        slots = torch.tensor(at % page, device="cuda")
        qpos, kpos = torch.arange(p, p + n, device="cuda")[:, None], torch.arange(p + n, device="cuda")[None]
        seen = kpos <= qpos
        if window:
            seen &= (kpos > qpos - window) | (kpos < sinks)
        if case["op"] == "prefix":
            pre = torch.arange(s["prefix_len"], device="cuda")
            pages = torch.cat([s["prefix_pages"].long()[pre // page], pages])
            slots = torch.cat([pre % page, slots])
            seen = torch.cat([torch.ones((n, s["prefix_len"]), dtype=torch.bool, device="cuda"), seen], 1)
        for h in range(hkv):
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            q = s["q"][starts[b] : starts[b + 1], heads].double().transpose(0, 1)
            k = s["k_cache"][pages, slots, h].double()
            v = s["v_cache"][pages, slots, h].double()
            a = (q @ k.T / math.sqrt(d)).masked_fill(~seen, float("-inf"))
            out[starts[b] : starts[b + 1], heads] = (torch.softmax(a, -1) @ v).transpose(0, 1)
    return {"out": out}

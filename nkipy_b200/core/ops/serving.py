"""Serving over a paged KV cache, as ops of a kernel body: ``paged_append``,
``paged_attention``, ``prefix_attention``, ``sample_tokens``.

The reference keeps one dense cache with one position for the whole batch
(``examples/models/qwen3/kernels/attention.py:95-140``) and samples greedily
(``examples/models/qwen3/kernels/sampling.py:113-147``); these ops are the paged,
ragged form and have no counterpart there.  Conventions (``include/nkb.h``): a
cache is (pages, page_size, kv_heads, head_dim); ``page_table`` (sequences,
width), ``kv_len`` (sequences,) and ``q_start`` (sequences + 1,) are int32; the
new tokens lie in sequence order, ``q_start=None`` means one per sequence, and
``kv_len`` counts a sequence's cached tokens with the new ones.

* "cpu": NumPy, statistics in float32, results rounded once.
* "hlo": one node per call (``paged-append`` returns the two caches and the
  rotated queries as a tuple; the caches are mutated parameters).
"""

import math

import numpy as np

from nkipy_b200.core.graph import get_trace_context
from nkipy_b200.core.ops._registry import Op
from nkipy_b200.core.tensor import NKIPyTensorRef


def _spans(page_table, kv_len, q_start, tokens):
    """(sequence, first token, tokens, position of the first) of each sequence that has new tokens."""
    seqs = page_table.shape[0]
    if q_start is None and tokens != seqs:
        raise ValueError(f"without q_start there is one token per sequence: {tokens} tokens, {seqs} sequences")
    first = np.arange(seqs + 1) if q_start is None else np.asarray(q_start).astype(np.int64)
    for b in range(seqs):
        n = int(first[b + 1] - first[b])
        if n > 0:
            yield b, int(first[b]), n, int(kv_len[b]) - n


def _rows(cache, pages, positions):
    """Cached rows at ``positions`` of a page list, in float32; zeros where the cache has no such page."""
    size = cache.shape[1]
    ids = np.asarray(pages)[positions // size].astype(np.int64)
    ok = (ids >= 0) & (ids < cache.shape[0])
    rows = cache[np.where(ok, ids, 0), positions % size].astype(np.float32)
    return np.where(ok[:, None, None], rows, np.float32(0))


def _rotate(x, cos, sin, rows):
    half = cos.shape[1]
    f = x.astype(np.float32)
    rows = np.clip(rows, 0, cos.shape[0] - 1)
    c, s = cos[rows].astype(np.float32)[:, None], sin[rows].astype(np.float32)[:, None]
    lo, hi = f[..., :half], f[..., half : 2 * half]
    return np.concatenate([lo * c - hi * s, lo * s + hi * c, f[..., 2 * half :]], -1).astype(x.dtype)


paged_append = Op("paged_append")


@paged_append.impl("cpu")
def _paged_append_cpu(k, v, k_cache, v_cache, page_table, kv_len, q_start=None, q=None, cos=None, sin=None, pos_offset=0):
    _check_append(k, v, k_cache, v_cache, page_table, kv_len, q_start, q, cos, sin)
    pages, size = k_cache.shape[:2]
    # rows that are read from the caches are those of before the call
    k, v, q, cos, sin = (x.copy() if x is not None and any(np.may_share_memory(x, c) for c in (k_cache, v_cache)) else x
                         for x in (k, v, q, cos, sin))
    out = None if q is None else np.zeros_like(q)
    for b, t, n, p in _spans(page_table, kv_len, q_start, k.shape[0]):
        pos = np.arange(p, p + n)
        kb = k[t : t + n] if cos is None else _rotate(k[t : t + n], cos, sin, pos + pos_offset)
        if q is not None:
            out[t : t + n] = q[t : t + n] if cos is None else _rotate(q[t : t + n], cos, sin, pos + pos_offset)
        inside = (pos >= 0) & (pos < page_table.shape[1] * size)
        ids = np.where(inside, np.asarray(page_table[b])[np.where(inside, pos, 0) // size], -1).astype(np.int64)
        ok = (ids >= 0) & (ids < pages)
        k_cache[ids[ok], pos[ok] % size] = kb[ok].astype(k_cache.dtype)
        v_cache[ids[ok], pos[ok] % size] = v[t : t + n][ok].astype(v_cache.dtype)
    return out


def _attend(q, k, v, seen, scale):
    """Rows of softmax(q k^T scale, over what is seen) v, in float32; zeros where nothing is seen."""
    n, hq, d = q.shape
    hkv = k.shape[1]
    some = seen.any(0)[:, None, None]
    k, v = np.where(some, k, np.float32(0)), np.where(some, v, np.float32(0))
    qf = q.astype(np.float32).reshape(n, hkv, hq // hkv, d)
    s = np.einsum("nhgd,khd->nhgk", qf, k) * np.float32(scale)
    s = np.where(seen[:, None, None, :], s, -np.inf)
    top = s.max(-1, initial=-np.inf, keepdims=True)
    e = np.where(seen[:, None, None, :], np.exp(s - np.where(np.isinf(top), np.float32(0), top)), np.float32(0))
    total = e.sum(-1, keepdims=True)
    out = np.einsum("nhgk,khd->nhgd", e, v) / np.where(total > 0, total, np.float32(1))
    return out.reshape(n, hq, d).astype(q.dtype)


def _attention_cpu(q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, prefix_pages, prefix_len):
    _check_attention(q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, prefix_pages, prefix_len)
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    out = np.zeros_like(q)
    before = np.arange(prefix_len)
    for b, t, n, p in _spans(page_table, kv_len, q_start, q.shape[0]):
        keys = np.arange(max(0, min(p + n, page_table.shape[1] * k_cache.shape[1])))
        pos = np.arange(p, p + n)[:, None]
        seen = keys <= pos
        if window:
            seen &= (keys > pos - window) | (keys < sinks)
        parts = [(_rows(k_cache, page_table[b], keys), _rows(v_cache, page_table[b], keys), seen)]
        if prefix_len:
            parts.insert(0, (_rows(k_cache, prefix_pages, before), _rows(v_cache, prefix_pages, before),
                             np.ones((n, prefix_len), bool)))
        k, v = (np.concatenate([x[i] for x in parts]) for i in (0, 1))
        out[t : t + n] = _attend(q[t : t + n], k, v, np.concatenate([x[2] for x in parts], 1), scale)
    return out


paged_attention = Op("paged_attention")
prefix_attention = Op("prefix_attention")


@paged_attention.impl("cpu")
def _paged_attention_cpu(q, k_cache, v_cache, page_table, kv_len, q_start=None, window=0, sinks=0, scale=None):
    return _attention_cpu(q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, None, 0)


@prefix_attention.impl("cpu")
def _prefix_attention_cpu(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, kv_len, q_start=None, scale=None):
    return _attention_cpu(q, k_cache, v_cache, page_table, kv_len, q_start, 0, 0, scale, prefix_pages, prefix_len)


sample_tokens = Op("sample_tokens")


@sample_tokens.impl("cpu")
def _sample_tokens_cpu(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    _check_sample(logits, u, temperature, top_k, top_p, min_p)
    rows, vocab = logits.shape
    out = np.full(rows, -1, np.int32)
    value = lambda a, r, default: default if a is None else np.asarray(a)[r]  # noqa: E731
    for r in range(rows):
        x = np.where(np.isnan(logits[r].astype(np.float32)), -np.inf, logits[r].astype(np.float32)).astype(np.float32)
        top = x.max()
        t = np.float32(value(temperature, r, 1.0))
        if top == -np.inf:
            continue
        if not t > 0:
            out[r] = np.argmax(x)
            continue
        with np.errstate(all="ignore"):
            e = np.exp((x - top) * (np.float32(1) / t), dtype=np.float32)
        # (a finite logit below an infinite one, at an infinite temperature, has a quotient of NaN)
        e = np.where(x == top, np.float32(1), np.where((x == -np.inf) | np.isnan(e), np.float32(0), e))
        w = (e.astype(np.float64) * 2.0**32).astype(np.int64)  # whole numbers: sums are exact
        order = np.argsort(-x, kind="stable")
        k, p = int(value(top_k, r, 0)), np.float32(value(top_p, r, 1.0))
        ws = np.where(np.arange(vocab) < (k if 0 < k < vocab else vocab), w[order], 0)
        if p < 1:
            most = max(1, int(np.float64(p) * np.float64(ws.sum())))
            ws = np.where(np.cumsum(ws) - ws < most, ws, 0)
        kept = np.zeros_like(w)
        kept[order] = ws
        kept = np.where(e < min(np.float32(value(min_p, r, 0.0)), np.float32(1)), 0, kept)
        sums = np.cumsum(kept)
        uu = np.float32(value(u, r, 0.0))
        at = min(int(np.float64(uu if uu > 0 else 0) * np.float64(sums[-1])), int(sums[-1]) - 1)
        out[r] = np.argmax(sums > at)
    return out


# ---------------------------------------------------------------------------
# arguments (arrays and traced tensors alike)
# ---------------------------------------------------------------------------
def _fail(message):
    raise ValueError(message)


def _floating(dtype):
    return np.dtype(dtype) in (np.dtype(np.float32), np.dtype(np.float16)) or np.dtype(dtype).name == "bfloat16"


def _vector(a, name, length, kinds="iu"):
    if a is not None and (len(a.shape) != 1 or a.shape[0] != length or (kinds == "iu") != (np.dtype(a.dtype).kind in "iu")):
        _fail(f"{name}: expected {length} {'integers' if kinds == 'iu' else 'float32 values'}, got {a.dtype} {tuple(a.shape)}")


def _check_tables(page_table, kv_len, q_start, tokens):
    if len(page_table.shape) != 2 or np.dtype(page_table.dtype).kind not in "iu":
        _fail(f"page_table: expected integers with 2 axes, got {page_table.dtype} {tuple(page_table.shape)}")
    _vector(kv_len, "kv_len", page_table.shape[0])
    _vector(q_start, "q_start", page_table.shape[0] + 1)
    if q_start is None and tokens != page_table.shape[0]:
        _fail(f"without q_start there is one token per sequence: {tokens} tokens, {page_table.shape[0]} sequences")


def _check_caches(k_cache, v_cache):
    if len(k_cache.shape) != 4 or tuple(k_cache.shape) != tuple(v_cache.shape) or k_cache.dtype != v_cache.dtype:
        _fail(f"k_cache {k_cache.dtype} {tuple(k_cache.shape)} and v_cache {v_cache.dtype} {tuple(v_cache.shape)}: "
              "expected two (pages, page_size, kv_heads, head_dim) caches of one type")
    if not _floating(k_cache.dtype):
        _fail(f"caches must be float32, bfloat16 or float16, got {k_cache.dtype}")


def _check_append(k, v, k_cache, v_cache, page_table, kv_len, q_start, q, cos, sin):
    _check_caches(k_cache, v_cache)
    if k_cache is v_cache:
        _fail("k_cache and v_cache are one tensor")
    if len(k.shape) != 3 or tuple(k.shape) != tuple(v.shape) or k.dtype != v.dtype or not _floating(k.dtype):
        _fail(f"k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)}: expected two (tokens, kv_heads, head_dim)")
    if tuple(k.shape[1:]) != tuple(k_cache.shape[2:]):
        _fail(f"k {tuple(k.shape)} does not go with caches {tuple(k_cache.shape)}")
    if q is not None and (len(q.shape) != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or q.dtype != k.dtype):
        _fail(f"q {q.dtype} {tuple(q.shape)} does not go with k {k.dtype} {tuple(k.shape)}")
    if (cos is None) != (sin is None):
        _fail("cos and sin go together")
    if cos is not None and (len(cos.shape) != 2 or tuple(cos.shape) != tuple(sin.shape) or cos.dtype != sin.dtype
                            or not _floating(cos.dtype) or cos.shape[0] < 1 or 2 * cos.shape[1] > k.shape[2]):
        _fail(f"cos {tuple(cos.shape)} and sin {tuple(sin.shape)}: expected (positions, at most head_dim / 2)")
    _check_tables(page_table, kv_len, q_start, k.shape[0])


def _check_attention(q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, prefix_pages, prefix_len):
    _check_caches(k_cache, v_cache)
    if len(q.shape) != 3 or q.shape[2] != k_cache.shape[3] or q.shape[1] % k_cache.shape[2] or q.dtype != k_cache.dtype:
        _fail(f"q {q.dtype} {tuple(q.shape)} does not go with caches {k_cache.dtype} {tuple(k_cache.shape)}")
    if window < 0 or sinks < 0 or prefix_len < 0:
        _fail("window, sinks and prefix_len must not be negative")
    if scale is not None and not math.isfinite(scale):
        _fail("scale must be finite")
    if prefix_len and (prefix_pages is None or len(prefix_pages.shape) != 1
                       or prefix_len > prefix_pages.shape[0] * k_cache.shape[1]):
        _fail(f"prefix of {prefix_len} tokens needs as many page ids as hold them")
    _check_tables(page_table, kv_len, q_start, q.shape[0])


def _check_sample(logits, u, temperature, top_k, top_p, min_p):
    if len(logits.shape) != 2 or not _floating(logits.dtype):
        _fail(f"logits: expected (rows, vocab) of a float type, got {logits.dtype} {tuple(logits.shape)}")
    for a, name in ((u, "u"), (temperature, "temperature"), (top_p, "top_p"), (min_p, "min_p")):
        _vector(a, name, logits.shape[0], "f")
    _vector(top_k, "top_k", logits.shape[0])


# ---------------------------------------------------------------------------
# traced form
# ---------------------------------------------------------------------------
def _trace(op, args, names, shape, dtype, attrs):
    """A node over the arguments that are given; ``operands`` names them in order."""
    ctx = get_trace_context()
    given = [(n, a) for n, a in zip(names, args) if a is not None]
    tensors = [_tensor(ctx, a) for _, a in given]
    for (n, _), t in zip(given, tensors):
        want = {"page_table": "int32", "kv_len": "int32", "q_start": "int32", "prefix_pages": "int32", "top_k": "int32",
                "u": "float32", "temperature": "float32", "top_p": "float32", "min_p": "float32"}.get(n)
        if want and np.dtype(t.dtype) != np.dtype(want):
            raise TypeError(f"{op}: {n} must be {want} in a traced kernel, got {t.dtype}")
    return ctx, ctx.build_op(op, tensors, shape, dtype, {"operands": [n for n, _ in given], **attrs})


def _tensor(ctx, a):
    if isinstance(a, NKIPyTensorRef):
        return a.backend_tensor
    if isinstance(a, np.ndarray):
        from nkipy_b200.core.ops.creation import constant

        return constant(a).backend_tensor
    return a


@paged_append.impl("hlo")
def _paged_append_hlo(k, v, k_cache, v_cache, page_table, kv_len, q_start=None, q=None, cos=None, sin=None, pos_offset=0):
    _check_append(k, v, k_cache, v_cache, page_table, kv_len, q_start, q, cos, sin)
    for c, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if not isinstance(c, NKIPyTensorRef):
            raise TypeError(f"paged_append: {name} must be a tensor of the traced kernel, it is written in place")
    names = ["k", "v", "k_cache", "v_cache", "page_table", "kv_len", "q_start", "q", "cos", "sin"]
    ctx, node = _trace("paged-append", [k, v, k_cache, v_cache, page_table, kv_len, q_start, q, cos, sin], names,
                       k_cache.shape, k_cache.dtype, {"pos_offset": int(pos_offset)})
    for i, c in enumerate((k_cache, v_cache)):
        c._rebind(NKIPyTensorRef(ctx.build_op("get-tuple-element", [node], c.shape, c.dtype, {"tuple_index": i})))
        c._is_mutated = True
    if q is None:
        return None
    return NKIPyTensorRef(ctx.build_op("get-tuple-element", [node], q.shape, q.dtype, {"tuple_index": 2}))


def _attention_hlo(q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, prefix_pages, prefix_len):
    _check_attention(q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, prefix_pages, prefix_len)
    if prefix_len == 0:
        prefix_pages = None
    names = ["q", "k_cache", "v_cache", "page_table", "kv_len", "q_start", "prefix_pages"]
    _, node = _trace("paged-attention", [q, k_cache, v_cache, page_table, kv_len, q_start, prefix_pages], names, q.shape,
                     q.dtype, {"window": int(window), "sinks": int(sinks), "prefix_len": int(prefix_len),
                               "scale": float(1 / math.sqrt(q.shape[2]) if scale is None else scale)})
    return NKIPyTensorRef(node)


@paged_attention.impl("hlo")
def _paged_attention_hlo(q, k_cache, v_cache, page_table, kv_len, q_start=None, window=0, sinks=0, scale=None):
    return _attention_hlo(q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, None, 0)


@prefix_attention.impl("hlo")
def _prefix_attention_hlo(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, kv_len, q_start=None, scale=None):
    return _attention_hlo(q, k_cache, v_cache, page_table, kv_len, q_start, 0, 0, scale, prefix_pages, prefix_len)


@sample_tokens.impl("hlo")
def _sample_tokens_hlo(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    _check_sample(logits, u, temperature, top_k, top_p, min_p)
    names = ["logits", "u", "temperature", "top_k", "top_p", "min_p"]
    _, node = _trace("sample-tokens", [logits, u, temperature, top_k, top_p, min_p], names, (logits.shape[0],), np.int32, {})
    return NKIPyTensorRef(node)

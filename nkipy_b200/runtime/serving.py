"""Serving over a paged KV cache: direct calls on device memory (torch tensors).

The calls of one decode step or one chunk of prompts: ``paged_append`` rotates
the new tokens' keys (and queries) and stores keys and values in their pages,
``paged_attention`` attends to them (all of them, or a sliding window with a
few first tokens), ``prefix_attention`` does so over a prefix that the whole
batch shares, and ``sample_tokens`` draws the next tokens.  Kernel bodies reach
the same kernels through ``nkipy_b200.core.tensor_apis``.

Conventions (``include/nkb.h``): a cache is (pages, page_size, kv_heads,
head_dim) with a contiguous last axis and any other strides; ``page_table``
(sequences, width), ``kv_len`` (sequences,) and ``q_start`` (sequences + 1,)
are int32; the new tokens lie in sequence order; ``kv_len`` counts a
sequence's cached tokens with the new ones; ``q_start=None`` means one new
token per sequence.  Lengths and tables are read on the device when the
kernels run, nothing is synchronised, and every launch goes to the current
torch stream, so a call can be captured into a CUDA graph.
"""

import ctypes
import functools
import math
import struct

from nkipy_b200.spike import _nkb, get_spike_singleton

try:
    import torch

    _CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    _FLOAT32, _INT32, _CONTIGUOUS = torch.float32, torch.int32, torch.contiguous_format
except ImportError:  # pragma: no cover
    torch = None

# nkb_paged_append_args, nkb_paged_attention_args, nkb_sample_args: 8-byte fields only
_APPEND = struct.Struct("=11Q3q6q3q8q8q2q")
_ATTENTION = struct.Struct("=9Q6q4q8q2q4qd")
_SAMPLE = struct.Struct("=7Q4q")


def _fail(message):
    raise ValueError(message)


def _on_device(*tensors):
    """The device index of all given tensors (None entries skipped): the runtime's device."""
    device = get_spike_singleton().device
    for t in tensors:
        if t is not None and t.get_device() != device:
            _fail(f"expected tensors on cuda:{device} (this process's device), got one on {t.device}")
    return device


def _rows(t, name, ndim):
    """Type code, shape and strides of a float tensor with ``ndim`` axes, the last one contiguous."""
    code, shape, strides = _CODES.get(t.dtype), t.shape, t.stride()
    if code is None:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    if len(strides) != ndim:
        _fail(f"{name}: expected {ndim} axes, got shape {tuple(shape)}")
    if strides[-1] != 1 and shape[-1] > 1:
        _fail(f"{name}: the last axis must be contiguous")
    return code, shape, strides


def _int32(t, name, length=None):
    """Checks a contiguous int32 vector of the given length (None: any length)."""
    if t.dtype is not _INT32:
        raise TypeError(f"{name}: expected int32, got {t.dtype}")
    if t.dim() != 1 or (length is not None and t.numel() != length) or not t.is_contiguous():
        of = "" if length is None else f" of {length}"
        _fail(f"{name}: expected a contiguous vector{of}, got shape {tuple(t.shape)}")


def _batch(page_table, kv_len, q_start, tokens):
    """Checks a call's page table and lengths; sequences, table width and row stride."""
    if page_table.dtype is not _INT32:
        raise TypeError(f"page_table: expected int32, got {page_table.dtype}")
    if page_table.dim() != 2:
        _fail(f"page_table: expected 2 axes, got shape {tuple(page_table.shape)}")
    seqs, width = page_table.shape
    stride, last = page_table.stride()
    if last != 1 and width > 1:
        _fail("page_table: the last axis must be contiguous")
    _int32(kv_len, "kv_len", seqs)
    if q_start is not None:
        _int32(q_start, "q_start", seqs + 1)
    elif tokens != seqs:
        _fail(f"without q_start there is one token per sequence: {tokens} tokens, {seqs} sequences")
    return seqs, width, stride


def _caches(k_cache, v_cache):
    """Type code and shape of the caches, and both strides up to the last axis."""
    code, shape, ks = _rows(k_cache, "k_cache", 4)
    vs = v_cache.stride()
    if v_cache.dtype is not k_cache.dtype or v_cache.shape != shape:
        _fail(f"k_cache and v_cache differ: {tuple(shape)} {k_cache.dtype}, {tuple(v_cache.shape)} {v_cache.dtype}")
    if vs[3] != 1 and shape[3] > 1:
        _fail("v_cache: the last axis must be contiguous")
    return code, shape, ks[:3] + vs[:3]


def _like(t, code, shape, out, name):
    """``out``, checked against ``t``, or a new tensor; and its first two strides."""
    if out is None:
        return torch.empty_like(t, memory_format=_CONTIGUOUS), (shape[1] * shape[2], shape[2])
    other, other_shape, strides = _rows(out, name, 3)
    if other != code or other_shape != shape:
        _fail(f"{name} {tuple(other_shape)} {out.dtype} differs from q {tuple(shape)} {t.dtype}")
    return out, strides[:2]


def _ptr(t):
    return 0 if t is None else t.data_ptr()


@functools.lru_cache(maxsize=4096)
def _workspace(tokens_by_start, *sizes):
    need = ctypes.c_size_t()
    _nkb.check(_nkb.lib().nkb_paged_attention_workspace(
        _ATTENTION.pack(*([0] * 6), int(tokens_by_start), 0, 0, *sizes, 0, 1.0), need))
    return need.value


def attention_workspace(sizes, tokens_by_start) -> int:
    """Workspace bytes of an attention call: ``sizes`` are the integers of
    ``nkb_paged_attention_args`` up to ``prefix_len``, ``tokens_by_start`` whether
    ``q_start`` is given."""
    return _workspace(bool(tokens_by_start), *(int(n) for n in sizes))


def _launch(fn, packed, device):
    """Issues a call on the current stream of ``device``."""
    if torch._C._cuda_getDevice() != device:
        with torch.cuda.device(device):
            return _launch(fn, packed, device)
    status = fn(packed, torch._C._cuda_getCurrentRawStream(device))
    if status:
        _nkb.check(status)


def paged_append(k, v, k_cache, v_cache, page_table, kv_len, q_start=None, q=None, cos=None, sin=None, pos_offset=0,
                 q_out=None):
    """Store the new tokens' ``k`` and ``v`` (tokens, kv_heads, head_dim) in their
    sequences' pages, in place.  With ``cos`` / ``sin`` (positions, rot_dim / 2) the
    first rot_dim dimensions of ``k``, and of ``q`` (tokens, q_heads, head_dim) when
    given, are rotated (half split) by the token's position + ``pos_offset`` on the
    way, in fp32.  Returns the rotated queries (``q_out``; may be ``q`` itself), or
    None without ``q``.  A row whose page is not in the cache, or whose position is
    outside the table, is not stored."""
    device = _on_device(k, v, k_cache, v_cache, page_table, kv_len, q_start, q, cos, sin, q_out)
    code, shape, ks = _rows(k, "k", 3)
    tokens, hkv, d = shape
    vs = v.stride()
    if v.shape != shape or v.dtype is not k.dtype or (vs[2] != 1 and d > 1):
        _fail(f"k and v differ: {tuple(shape)} {k.dtype}, {tuple(v.shape)} {v.dtype} (strides {ks}, {vs})")
    cache_code, (pages, page_size, heads, dim), cache_strides = _caches(k_cache, v_cache)
    if heads != hkv or dim != d:
        _fail(f"caches hold {heads} heads of {dim}, k has {hkv} of {d}")
    seqs, width, table_stride = _batch(page_table, kv_len, q_start, tokens)
    rot = rows = stride = rope_code = 0
    if (cos is None) != (sin is None):
        _fail("cos and sin go together")
    if cos is not None:
        rope_code, (rows, rot), rope_strides = _rows(cos, "cos", 2)
        if sin.shape != cos.shape or sin.dtype is not cos.dtype or sin.stride() != rope_strides:
            _fail("cos and sin differ in shape, type or strides")
        rot, stride = 2 * rot, rope_strides[0]
        if rot > d:
            _fail(f"cos and sin rotate {rot} dimensions, head_dim is {d}")
    hq, q_strides, out_strides = 0, (0, 0), (0, 0)
    if q is not None:
        q_code, q_shape, q_strides = _rows(q, "q", 3)
        hq = q_shape[1]
        if q_code != code or q_shape[0] != tokens or q_shape[2] != d:
            _fail(f"q {tuple(q_shape)} {q.dtype} does not go with k {tuple(shape)} {k.dtype}")
        q_out, out_strides = _like(q, code, q_shape, q_out, "q_out")
    elif q_out is not None:
        _fail("q_out without q")
    packed = _APPEND.pack(
        k.data_ptr(), v.data_ptr(), _ptr(q), _ptr(q_out), k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(),
        kv_len.data_ptr(), _ptr(q_start), _ptr(cos), _ptr(sin), code, cache_code, rope_code, tokens, seqs, hq, hkv, d, rot,
        rows, stride, pos_offset, ks[0], ks[1], vs[0], vs[1], q_strides[0], q_strides[1], *out_strides, pages, page_size,
        *cache_strides, width, table_stride)
    _launch(_nkb.lib().nkb_paged_append, packed, device)
    return q_out


def _attention(q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, out, prefix_pages, prefix_len):
    device = _on_device(q, k_cache, v_cache, page_table, kv_len, q_start, out, prefix_pages)
    code, shape, qs = _rows(q, "q", 3)
    tokens, hq, d = shape
    cache_code, (pages, page_size, hkv, dim), cache_strides = _caches(k_cache, v_cache)
    if cache_code != code:
        raise TypeError(f"q is {q.dtype}, the caches are {k_cache.dtype}")
    if dim != d or hkv == 0 or hq % hkv:
        _fail(f"q {tuple(shape)} does not go with caches of {hkv} heads of {dim}")
    seqs, width, table_stride = _batch(page_table, kv_len, q_start, tokens)
    out, out_strides = _like(q, code, shape, out, "out")
    sizes = (code, tokens, seqs, hq, hkv, d, qs[0], qs[1], *out_strides, pages, page_size, *cache_strides, width,
             table_stride, window, sinks, prefix_len)
    need = _workspace(q_start is not None, *sizes)
    room = q.new_empty(need, dtype=torch.uint8) if need else None
    _launch(_nkb.lib().nkb_paged_attention, _ATTENTION.pack(
        q.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(), kv_len.data_ptr(),
        _ptr(q_start), _ptr(prefix_pages), _ptr(room), *sizes, need, 1.0 / math.sqrt(d) if scale is None else scale), device)
    return out


def paged_attention(q, k_cache, v_cache, page_table, kv_len, q_start=None, window=0, sinks=0, scale=None, out=None):
    """Attention of the new tokens' ``q`` (tokens, q_heads, head_dim) over their
    sequences' cached keys up to their own position; with ``window`` > 0 only the last
    ``window`` of them (the token itself among them) and the first ``sinks``.  ``scale``
    defaults to 1 / sqrt(head_dim).  Returns ``out`` (tokens, q_heads, head_dim); a token
    that sees no key gives zeros."""
    return _attention(q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks, scale, out, None, 0)


def prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, kv_len, q_start=None, scale=None,
                     out=None):
    """Attention of a batch whose sequences all begin with the same ``prefix_len``
    tokens, held once in ``prefix_pages`` (int32 page ids) and read once for the batch;
    ``page_table`` and ``kv_len`` describe what each sequence has after the prefix."""
    if prefix_len < 0:
        _fail("prefix_len must not be negative")
    _int32(prefix_pages, "prefix_pages")
    if k_cache.dim() == 4 and prefix_len > prefix_pages.shape[0] * k_cache.shape[1]:
        _fail(f"prefix of {prefix_len} tokens needs more than {prefix_pages.shape[0]} pages of {k_cache.shape[1]}")
    return _attention(q, k_cache, v_cache, page_table, kv_len, q_start, 0, 0, scale, out, prefix_pages, prefix_len)


def sample_tokens(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
    """One token (int32) per row of ``logits`` (rows, vocab), drawn with the row's
    ``u`` (fp32, in [0, 1)).  ``temperature``, ``top_p``, ``min_p`` (fp32) and ``top_k``
    (int32) are one value per row, or None for 1, 1, 0 and 0 (off).  Filters apply in
    the order temperature, top-k, top-p, min-p; a temperature of 0 takes the largest
    logit.  A row without a finite logit or +inf gives -1."""
    device = _on_device(logits, u, temperature, top_k, top_p, min_p, out)
    code, (rows, vocab), strides = _rows(logits, "logits", 2)
    for t, name in ((u, "u"), (temperature, "temperature"), (top_p, "top_p"), (min_p, "min_p")):
        if t is not None and (t.dtype is not _FLOAT32 or t.dim() != 1 or t.numel() != rows or not t.is_contiguous()):
            _fail(f"{name}: expected a contiguous float32 tensor of shape ({rows},), got {t.dtype} {tuple(t.shape)}")
    if top_k is not None:
        _int32(top_k, "top_k", rows)
    if out is None:
        out = logits.new_empty(rows, dtype=_INT32)
    else:
        _int32(out, "out", rows)
    packed = _SAMPLE.pack(logits.data_ptr(), u.data_ptr(), _ptr(temperature), _ptr(top_k), _ptr(top_p), _ptr(min_p),
                          out.data_ptr(), code, rows, vocab, strides[0])
    _launch(_nkb.lib().nkb_sample_tokens, packed, device)
    return out

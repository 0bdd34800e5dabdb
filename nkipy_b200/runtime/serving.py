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
torch stream, so a call can be captured into a CUDA graph.  The calls have no
gradient: where autograd records, tensors that require one are refused, and
tensors that are written in place count as changed.  A kernel whose
bounded wait runs out ends without its results; ``check_device_error`` tells.
"""

import ctypes
import functools
import importlib.util
import os
import struct

from nkipy_b200.spike import _nkb, get_spike_singleton

# nkb_paged_append_args, nkb_paged_attention_args and nkb_sample_args as bytes (8-byte
# fields only), for callers of the C calls that have no compiler
_APPEND = struct.Struct("=11Q3q6q3q8q8q2q")
_ATTENTION = struct.Struct("=9Q6q4q8q2q4qd")
_SAMPLE = struct.Struct("=7Q4q")


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


@functools.lru_cache(maxsize=1)
def _calls():
    """The module that takes torch tensors (csrc/torch_serving.cpp)."""
    import torch

    from nkipy_b200.build import built_for

    _nkb.lib()
    path = os.path.join(os.path.dirname(_nkb.LIB_PATH), "nkb_torch.so")
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: run `python -m nkipy_b200.build`")
    spec = importlib.util.spec_from_file_location("nkb_torch", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    if module.built_for != built_for(torch.__version__, torch.version.git_version):
        raise ImportError(f"{path} was built for {module.built_for}: run `python -m nkipy_b200.build`")
    return module


def paged_append(k, v, k_cache, v_cache, page_table, kv_len, q_start=None, q=None, cos=None, sin=None, pos_offset=0,
                 q_out=None):
    """Store the new tokens' ``k`` and ``v`` (tokens, kv_heads, head_dim) in their
    sequences' pages, in place.  With ``cos`` / ``sin`` (positions, rot_dim / 2) the
    first rot_dim dimensions of ``k``, and of ``q`` (tokens, q_heads, head_dim) when
    given, are rotated (half split) by the token's position + ``pos_offset`` on the
    way, in fp32.  Returns the rotated queries (``q_out``; may be ``q`` itself), or
    None without ``q``.  A row whose page is not in the cache, or whose position is
    outside the table, is not stored."""
    return _calls().paged_append(get_spike_singleton().device, k, v, k_cache, v_cache, page_table, kv_len, q_start, q, cos, sin,
                                 pos_offset, q_out)


def paged_attention(q, k_cache, v_cache, page_table, kv_len, q_start=None, window=0, sinks=0, scale=None, out=None):
    """Attention of the new tokens' ``q`` (tokens, q_heads, head_dim) over their
    sequences' cached keys up to their own position; with ``window`` > 0 only the last
    ``window`` of them (the token itself among them) and the first ``sinks``.  ``scale``
    defaults to 1 / sqrt(head_dim).  Returns ``out`` (tokens, q_heads, head_dim); a token
    that sees no key gives zeros."""
    return _calls().attention(get_spike_singleton().device, q, k_cache, v_cache, page_table, kv_len, q_start, window, sinks,
                              scale, out, None, 0)


def prefix_attention(q, k_cache, v_cache, prefix_pages, prefix_len, page_table, kv_len, q_start=None, scale=None,
                     out=None):
    """Attention of a batch whose sequences all begin with the same ``prefix_len``
    tokens, held once in ``prefix_pages`` (int32 page ids) and read once for the batch;
    ``page_table`` and ``kv_len`` describe what each sequence has after the prefix."""
    return _calls().attention(get_spike_singleton().device, q, k_cache, v_cache, page_table, kv_len, q_start, 0, 0, scale, out,
                              prefix_pages, prefix_len)


def sample_tokens(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
    """One token (int32) per row of ``logits`` (rows, vocab), drawn with the row's
    ``u`` (fp32, in [0, 1)).  ``temperature``, ``top_p``, ``min_p`` (fp32) and ``top_k``
    (int32) are one value per row, or None for 1, 1, 0 and 0 (off).  Filters apply in
    the order temperature, top-k, top-p, min-p; a temperature of 0 takes the largest
    logit.  A row without a finite logit or +inf gives -1."""
    return _calls().sample_tokens(get_spike_singleton().device, logits, u, temperature, top_k, top_p, min_p, out)


def check_device_error():
    """Wait for the device, and raise ``NkbError`` if a kernel of this process has given up a
    bounded wait since the last check (its results are then invalid; the device stays usable).
    The calls above do not look by themselves, as that would synchronise: call this where the
    host waits anyway, once per step or per some steps."""
    import torch

    with torch.cuda.device(get_spike_singleton().device):
        torch.cuda.synchronize()
        flag = ctypes.c_int()
        _nkb.call("nkb_device_error", ctypes.byref(flag))
    if flag.value:
        raise _nkb.NkbError(7, "a kernel's bounded wait expired; results are invalid")

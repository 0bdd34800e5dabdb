"""Backward-compatible entry points (reference: ``core/tensor_apis.py``)."""

from nkipy_b200.core.ops import (
    constant,
    conv2d,
    conv3d,
    full,
    paged_append,
    paged_attention,
    prefix_attention,
    rms_norm,
    sample_tokens,
    softmax,
    topk,
    zeros,
)

__all__ = ["constant", "conv2d", "conv3d", "topk", "rms_norm", "softmax", "zeros", "full", "paged_append",
           "paged_attention", "prefix_attention", "sample_tokens"]

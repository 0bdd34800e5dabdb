"""Serving calls at the edges of what they take, as far as that goes without a GPU."""

import numpy as np
import pytest

from nkipy_b200.core import tensor_apis as T
from nkipy_b200.core.trace import NKIPyKernel
from nkipy_b200.spike import _nkb
from tests.test_serving_cpu import packed, step_inputs


@pytest.mark.parametrize("scale", [float("inf"), -float("inf"), float("nan")])
def test_scale_that_is_not_finite(scale):
    assert _nkb.lib().nkb_paged_attention(packed("attention", dtype=0, scale=scale), None) == 1
    assert "scale must be finite" in _nkb.lib().nkb_last_error().decode()
    args, _ = step_inputs()
    q, (kc, vc, table, lens) = np.zeros((3, 4, 64), args[5].dtype), args[5:9]
    with pytest.raises(ValueError, match="finite"):
        T.paged_attention(q, kc, vc, table, lens, scale=scale)
    with pytest.raises(ValueError, match="finite"):
        NKIPyKernel.trace(lambda q, kc, vc, t, n: T.paged_attention(q, kc, vc, t, n, scale=scale)).specialize(q, kc, vc, table, lens)


def test_append_of_no_tokens_with_queries():
    """An empty step: arrays without elements have no address."""
    none = dict(tokens=0, seqs=0, k=0, v=0, q=0, q_out=0, q_heads=4, q_token=256, q_head=64, q_out_token=256, q_out_head=64)
    lib = _nkb.lib()
    assert lib.nkb_paged_append(packed("append", **none), None) == 0
    assert lib.nkb_paged_append(packed("append", **none, cos=16, sin=16, rot_dim=64, rope_rows=4, rope_stride=32), None) == 0
    assert lib.nkb_paged_append(packed("append", **{**none, "q_heads": -1}), None) == 1
    assert lib.nkb_paged_append(packed("append", q_heads=4), None) == 1

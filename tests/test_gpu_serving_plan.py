"""The serving ops of a traced kernel body on the device, against the NumPy
direct call: a whole served step (RMSNorm, projections, append, attention,
sampling), single tokens and chunks, with a window and with a shared prefix."""

import numpy as np
import pytest

from nkipy_b200 import workloads as W
from nkipy_b200.core import tensor_apis as T
from tests.test_serving_cpu import BF16, step_inputs
from tests.utils import BF16_RTOL, assert_close, on_device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("news,lens", [(None, (1, 20, 64)), ((3, 1, 20), (30, 20, 64))])
@pytest.mark.parametrize("form", ["all", "window", "prefix"])
def test_step(news, lens, form):
    """Caches equal the direct call's to bf16 rounding; tokens are equal where both sides' logits
    leave no doubt, so the step is drawn from greedily."""
    args, kwargs = step_inputs(seed=3, news=news, lens=lens, prefix=37 if form == "prefix" else 0)
    if form == "window":
        kwargs.update(window=16, sinks=2)
    args = list(args)
    args[12] = np.zeros(3, np.float32)
    host = [a.copy() for a in args]
    want = W.paged_step_kernel(*host, **kwargs)
    got = on_device(W.paged_step_kernel, *args, **kwargs)
    for i in (5, 6):
        assert_close(args[i], host[i], BF16_RTOL)
        same = host[i] == args[i]
        assert same.mean() > 0.98  # rows that the step did not write are untouched
    assert got.shape == want.shape and got.dtype == np.int32
    assert (np.asarray(got) == want).mean() >= 2 / 3


def test_attention_and_sampling_alone():
    rng = np.random.default_rng(4)
    q = rng.standard_normal((5, 4, 64)).astype(np.float16)
    kc, vc = (rng.standard_normal((9, 2, 16, 64)).astype(np.float16) for _ in range(2))  # heads ahead of slots
    table, lens = rng.permutation(9)[:8].reshape(2, 4).astype(np.int32), np.array([40, 60], np.int32)
    start = np.array([0, 2, 5], np.int32)

    def body(q, kc, vc, table, lens, start):
        return T.paged_attention(q, kc.transpose(0, 2, 1, 3), vc.transpose(0, 2, 1, 3), table, lens, start, window=9, sinks=3)

    assert_close(on_device(body, q, kc, vc, table, lens, start), body(q, kc, vc, table, lens, start), 2.0**-9)
    x = rng.standard_normal((6, 700)).astype(np.float32)
    u = np.linspace(0.05, 0.95, 6).astype(np.float32)
    k, p = np.array([1, 2, 3, 50, 0, 9], np.int32), np.array([1, 0.5, 0.9, 0.9, 0.3, 1], np.float32)

    def draw(x, u, k, p):
        return T.sample_tokens(x, u, None, k, p)

    np.testing.assert_array_equal(on_device(draw, x, u, k, p), draw(x, u, k, p))


def test_appended_rows_are_read_by_the_attention_that_follows():
    """Append and attend in one body: the new rows are seen, and the caches come back mutated."""
    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((3, 2, 64)).astype(BF16) for _ in range(2))
    q = rng.standard_normal((3, 4, 64)).astype(BF16)
    kc, vc = (rng.standard_normal((8, 16, 2, 64)).astype(BF16) for _ in range(2))
    table, lens = np.array([[5, 1], [0, 7], [3, 2]], np.int32), np.array([1, 17, 32], np.int32)

    def body(k, v, q, kc, vc, table, lens):
        T.paged_append(k, v, kc, vc, table, lens)
        return T.paged_attention(q, kc, vc, table, lens)

    host = [kc.copy(), vc.copy()]
    want = body(k, v, q, *host, table, lens)
    got = on_device(body, k, v, q, kc, vc, table, lens)
    assert_close(got, want, BF16_RTOL)
    np.testing.assert_array_equal(kc.view(np.uint16), host[0].view(np.uint16))
    np.testing.assert_array_equal(vc.view(np.uint16), host[1].view(np.uint16))

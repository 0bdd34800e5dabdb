"""Serving calls at the edges of what they take: padding tokens and empty
sequences among others.  References, bounds and helpers are those of
``test_gpu_serving``; after each call the device error flag is read."""

import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from nkipy_b200 import runtime as nk  # noqa: E402
from nkipy_b200.spike import _nkb  # noqa: E402
from tests.test_serving_cpu import packed  # noqa: E402
from tests.test_gpu_serving import (BF16, F16, Paged, attention_reference, check_attention, f64, ints,  # noqa: E402
                                    randn, run_attention, seen_by)

pytestmark = pytest.mark.gpu


def no_device_error():
    torch.cuda.synchronize()
    flag = ctypes.c_int()
    _nkb.call("nkb_device_error", ctypes.byref(flag))
    assert flag.value == 0


# ---------------------------------------------------------------------------
# tokens without keys
# ---------------------------------------------------------------------------
def run_padded(seed, front, news, lens, behind, hq, hkv, d, page, dtype, prefix=0, scale=None):
    """``front`` and ``behind`` tokens belong to no sequence; a sequence's length may be less than
    its new tokens, whose first ones then lie before its first key."""
    rng = np.random.default_rng(seed)
    n_pages = -(-prefix // page)
    cache = Paged(rng, lens, hkv, d, page, dtype, extra=n_pages)
    pages, at_p = cache.free[:n_pages], np.arange(prefix)
    place = torch.tensor(pages[at_p // page], dtype=torch.long, device="cuda"), torch.tensor(at_p % page, device="cuda")
    for c in (cache.k, cache.v):
        if prefix:
            c[place] = randn(rng, (prefix, hkv, d), dtype)
    pk, pv = f64(cache.k[place]), f64(cache.v[place])
    T = front + sum(news) + behind
    q = randn(rng, (T, hq, d), dtype)
    want, mag, at = np.zeros((T, hq, d)), np.zeros((T, hq, d)), front
    for b, (n, length) in enumerate(zip(news, lens)):
        cache.write(rng, b, np.arange(length), dtype)
        rows = np.arange(length)
        k, v = (np.concatenate([x, cache.read(c, b, rows)]) for x, c in ((pk, cache.k), (pv, cache.v)))
        seen = np.concatenate([np.ones((n, prefix), bool), seen_by(np.arange(length - n, length), length, 0, 0)], 1)
        if n and seen.shape[1]:
            want[at : at + n], mag[at : at + n] = attention_reference(f64(q[at : at + n]), k, v, seen,
                                                                          1 / math.sqrt(d) if scale is None else scale, hkv)
        at += n
    start = ints((front + np.cumsum([0] + list(news))).tolist())
    args = (cache.device_table(), ints(lens))
    out = torch.full_like(q, 9.0)
    for _ in range(3):
        if prefix:
            got = nk.prefix_attention(q, cache.k, cache.v, ints(pages), prefix, *args, q_start=start, scale=scale,
                                      out=out.fill_(9.0))
        else:
            got = nk.paged_attention(q, cache.k, cache.v, *args, q_start=start, scale=scale, out=out.fill_(9.0))
        no_device_error()
        check_attention(got, want, mag, dtype)
        assert bool((got[:front] == 0).all()) and bool((got[at:] == 0).all())


EMPTY = [0, 0, 3, 0, 130, 0, 0, 17, 0, 0, 0, 0]
PADDED = [
    # front, news, lens, behind, hq, hkv, d, page, dtype
    (0, [448], [4448], 64, 32, 8, 128, 16, BF16),  # a real unit and then empty ones, cut into shares
    (64, [448], [4448], 0, 32, 8, 64, 16, F16),
    (0, [1] * 300, [0, 5] * 150, 0, 16, 8, 64, 16, BF16),  # every second sequence is empty
    (0, [40] * 12, EMPTY, 0, 32, 8, 128, 16, BF16),
    (33, [20, 1, 300] * 4, EMPTY, 500, 8, 8, 64, 32, F16),
    (0, [64] * 6, [0] * 6, 0, 32, 8, 128, 16, BF16),  # no key at all
    (0, [9] * 64, [3, 0] * 32, 0, 32, 8, 128, 16, BF16),
    (0, [64, 64, 64], [256, 0, 0], 1000, 8, 8, 128, 16, BF16),
    (5, [200], [12], 5, 16, 2, 64, 8, F16),  # most tokens lie before the first key
]


@pytest.mark.parametrize("case", range(len(PADDED)))
def test_padding(case):
    run_padded(700 + case, *PADDED[case])


@pytest.mark.parametrize("prefix", [20, 700])
@pytest.mark.parametrize("case", range(len(PADDED)))
def test_padding_after_a_prefix(case, prefix):
    run_padded(800 + case, *PADDED[case], prefix=prefix)


# ---------------------------------------------------------------------------
# the C call's workspace
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("offset", [0, 16])
@pytest.mark.parametrize("prefix, news, d", [(0, [200, 3], 128), (0, [200, 3], 64), (300, [30, 2], 64), (300, [1, 1], 128)])
def test_workspace_at_any_16_byte_boundary(offset, prefix, news, d):
    """Units cut into partials, with a workspace that starts at an odd multiple of 16 bytes: the torch call's
    outputs, and nothing written in front of it or behind it."""
    rng = np.random.default_rng(900)
    hq, hkv, page, lens, pages = 4, 2, 16, [3000, 40], -(-prefix // 16)
    cache = Paged(rng, lens, hkv, d, page, BF16, extra=pages, fill=0.0)
    for b, n in enumerate(lens):
        cache.write(rng, b, np.arange(n), BF16)
    q, table, kv_len, ids = randn(rng, (sum(news), hq, d), BF16), cache.device_table(), ints(lens), ints(cache.free[:pages])
    start = None if max(news) == 1 else ints(np.cumsum([0] + news).tolist())
    if prefix:
        want = nk.prefix_attention(q, cache.k, cache.v, ids, prefix, table, kv_len, q_start=start)
    else:
        want = nk.paged_attention(q, cache.k, cache.v, table, kv_len, q_start=start)
    out = torch.zeros_like(q)
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    values = dict(q=at(q), out=at(out), k_cache=at(cache.k), v_cache=at(cache.v), page_table=at(table), kv_len=at(kv_len),
                  q_start=at(start), prefix_pages=at(ids) if prefix else 0, tokens=sum(news), seqs=2, q_heads=hq, kv_heads=hkv,
                  head_dim=d, q_token=hq * d, q_head=d, out_token=hq * d, out_head=d, pages=cache.k.shape[0], page_size=page,
                  table_width=table.shape[1], table_stride=table.shape[1], prefix_len=prefix, scale=1 / math.sqrt(d))
    for c, x in (("k", cache.k), ("v", cache.v)):
        values.update({f"{c}_page": x.stride(0), f"{c}_slot": x.stride(1), f"{c}_cache_head": x.stride(2)})
    need = ctypes.c_size_t()
    _nkb.call("nkb_paged_attention_workspace", packed("attention", **values), ctypes.byref(need))
    room = torch.full((need.value + 512,), 77, dtype=torch.uint8, device="cuda")
    first = (-room.data_ptr()) % 256 + offset
    values.update(workspace=room.data_ptr() + first, workspace_bytes=need.value)
    _nkb.call("nkb_paged_attention", packed("attention", **values), torch.cuda.current_stream().cuda_stream)
    no_device_error()
    assert torch.equal(out, want)
    assert bool((room[:first] == 77).all()) and bool((room[first + need.value :] == 77).all())


# ---------------------------------------------------------------------------
# scale
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [0.0, -0.125, -1.0, 1e-42, 1e-60, 3.0])
@pytest.mark.parametrize("news, pasts, dtype, page", [([1, 1], [9, 300], BF16, 16), ([70, 200], [0, 90], BF16, 16),
                                                      ([70, 3], [5, 900], F16, 64), ([20, 1], [3, 70], BF16, 24)])
def test_scale_of_any_sign(scale, news, pasts, dtype, page):
    """Every form: uniform weights for 0 (and for what is as good as 0), the least product first for a negative one."""
    for q_start in [True] + [False] * (max(news) == 1):
        run_attention(1000, news, pasts, 0, 0, 4, 2, 64, page, dtype, scale=scale, q_start=q_start)
        run_attention(1001, news, pasts, 50, 3, 4, 2, 128, page, dtype, scale=scale, q_start=q_start)
    no_device_error()


@pytest.mark.parametrize("scale", [0.0, -0.25])
@pytest.mark.parametrize("news", [[1, 1], [30, 5]])
def test_scale_of_any_sign_after_a_prefix(scale, news):
    run_padded(1002, 0, news, [n + 40 for n in news], 0, 4, 2, 64, 16, BF16, prefix=300, scale=scale)


@pytest.mark.parametrize("scale", [float("inf"), float("nan")])
def test_scale_that_is_not_finite(scale):
    rng = np.random.default_rng(1003)
    cache = Paged(rng, [20], 2, 64, 16, BF16)
    with pytest.raises(RuntimeError, match="scale must be finite"):
        nk.paged_attention(randn(rng, (1, 4, 64), BF16), cache.k, cache.v, cache.device_table(), ints([20]), scale=scale)


# ---------------------------------------------------------------------------
# calls without tokens
# ---------------------------------------------------------------------------
def test_append_of_no_tokens_with_queries():
    cache = Paged(np.random.default_rng(1100), [20], 2, 64, 16, BF16, fill=3.0)
    none = lambda heads: torch.zeros((0, heads, 64), dtype=BF16, device="cuda")  # noqa: E731
    cos = torch.ones((30, 32), device="cuda")
    table, start = cache.device_table(), ints([0, 0])
    for rope in (dict(), dict(cos=cos, sin=cos)):
        got = nk.paged_append(none(2), none(2), cache.k, cache.v, table, ints([20]), q_start=start, q=none(4), **rope)
        assert got.shape == (0, 4, 64) and got.dtype == BF16
        got = nk.paged_append(none(2), none(2), cache.k, cache.v, table[:0], ints([]), q=none(4), **rope)
        assert got.shape == (0, 4, 64)
    assert bool((cache.k == 3).all())

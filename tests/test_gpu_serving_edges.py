"""Serving calls at the edges of what they take: padding tokens and empty
sequences among others.  References, bounds and helpers are those of
``test_gpu_serving``; after each call the device error flag is read."""

import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from nkipy_b200 import runtime as nk  # noqa: E402
from nkipy_b200 import workloads as W  # noqa: E402
from nkipy_b200.core import tensor_apis as T  # noqa: E402
from nkipy_b200.spike import _nkb  # noqa: E402
from tests.test_serving_cpu import packed, step_inputs  # noqa: E402
from tests.test_serving_edges_cpu import move_inputs, move_rows  # noqa: E402
from tests.test_gpu_serving import (BF16, F16, F32, Paged, attention_reference, check_attention, f64, ints,  # noqa: E402
                                    randn, run_attention, seen_by)
from tests.utils import on_device  # noqa: E402

pytestmark = pytest.mark.gpu


def no_device_error():
    nk.check_device_error()


def test_a_wait_that_runs_out_is_reported():
    """A counter that nothing advances, with a limit of 2 ms, on a stream of its own: one error, then none."""
    x, u = torch.zeros((2, 9), device="cuda"), torch.zeros(2, device="cuda")
    nk.sample_tokens(x, u)
    nk.check_device_error()
    counter, limit = torch.zeros(1, dtype=torch.int32, device="cuda"), ctypes.c_uint64()
    _nkb.call("nkb_get_wait_limit_us", ctypes.byref(limit))
    torch.cuda.synchronize()
    try:
        _nkb.call("nkb_set_wait_limit_us", 2000)
        _nkb.call("nkb_wait_probe", counter.data_ptr(), 1, torch.cuda.Stream().cuda_stream)
        with pytest.raises(_nkb.NkbError, match="bounded wait expired"):
            nk.check_device_error()
    finally:
        _nkb.call("nkb_set_wait_limit_us", limit.value)
    nk.check_device_error()
    assert nk.sample_tokens(x, u).tolist() == [0, 0]


# ---------------------------------------------------------------------------
# tokens without keys
# ---------------------------------------------------------------------------
def run_padded(seed, front, news, lens, behind, hq, hkv, d, page, dtype, prefix=0, scale=None, single=False):
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
    start = None if single else ints((front + np.cumsum([0] + list(news))).tolist())
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


@pytest.mark.parametrize("prefix", [700, 6000])
def test_single_tokens_after_a_prefix(prefix):
    """A short prefix shares the SMs with the sequences' own keys, a long one takes all."""
    run_padded(900, 0, [1] * 130, [0, 1, 70, 5, 300] * 26, 0, 64, 4, 64, 16, BF16, prefix=prefix, single=True)


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


def test_calls_without_tokens_at_any_strides():
    """An array without elements has no layout."""
    cache = Paged(np.random.default_rng(1101), [20], 2, 64, 16, BF16)
    table, start = cache.device_table(), ints([0, 0])
    for make in (lambda *s: torch.empty_strided(s, (0,) * len(s), dtype=BF16, device="cuda"),
                 lambda *s: torch.tensor(np.zeros(s)).to(BF16).cuda()):
        got = nk.paged_append(make(0, 2, 64), make(0, 2, 64), cache.k, cache.v, table, ints([20]), q_start=start, q=make(0, 4, 64))
        assert got.shape == (0, 4, 64)
        assert nk.paged_attention(make(0, 4, 64), cache.k, cache.v, table, ints([20]), q_start=start).shape == (0, 4, 64)
        none = torch.empty_strided((0, 3), (0, 0), dtype=torch.int32, device="cuda")
        assert nk.paged_attention(make(0, 4, 64), cache.k, cache.v, none, ints([])).shape == (0, 4, 64)
        assert nk.sample_tokens(make(0, 9), torch.zeros(0, device="cuda")).shape == (0,)


# ---------------------------------------------------------------------------
# NaN and infinities in what a token sees
# ---------------------------------------------------------------------------
INF, NAN = float("inf"), float("nan")
SEEN = [
    # news, pasts, hq, hkv, d, page, dtype, prefix
    ([1, 1, 1], [699, 2, 1299], 8, 2, 128, 16, BF16, 0),  # single tokens, cut
    ([1] * 200, [99] * 200, 16, 8, 64, 16, F16, 0),  # and some whole
    ([70, 3], [300, 900], 6, 2, 64, 32, F16, 0),  # tiles, cut
    ([130, 3], [300, 900], 8, 2, 128, 16, BF16, 0),
    ([3, 130], [900, 300], 8, 2, 128, 16, BF16, 0),
    ([7] * 40, range(140, 180), 16, 8, 128, 16, BF16, 0),  # tiles, whole
    ([31, 9], [2, 260], 4, 2, 20, 5, F32, 0),  # any layout
    ([1, 1], [2, 260], 4, 2, 64, 48, BF16, 0),
    ([1] * 3, [3, 0, 200], 8, 2, 128, 16, BF16, 700),  # a prefix
    ([5, 40], [3, 200], 8, 2, 64, 16, F16, 300),
    ([3], [20], 4, 2, 20, 5, F32, 40),
]


class Seen:
    """A call of one of the forms above: ``run`` repeats it with the present contents."""

    def __init__(self, case, seed):
        news, pasts, self.hq, self.hkv, d, page, dtype, prefix = SEEN[case]
        self.news, self.pasts, self.d, self.dtype, self.prefix = list(news), list(pasts), d, dtype, prefix
        self.rng = rng = np.random.default_rng(seed)
        self.lens = [a + b for a, b in zip(self.news, self.pasts)]
        pages = -(-prefix // page)
        self.cache = cache = Paged(rng, self.lens, self.hkv, d, page, dtype, extra=pages)
        for b, n in enumerate(self.lens):
            cache.write(rng, b, np.arange(n), dtype)
        at = np.arange(prefix)
        self.before = cache.free[:pages]
        self.where_before = (torch.tensor(self.before[at // page], dtype=torch.long, device="cuda"),
                             torch.tensor(at % page, device="cuda"))
        for c in (cache.k, cache.v):
            if prefix:
                c[self.where_before] = randn(rng, (prefix, self.hkv, d), dtype)
        self.first = np.cumsum([0] + self.news)
        self.q = randn(rng, (self.first[-1], self.hq, d), dtype)

    def run(self):
        start = None if max(self.news) == 1 else ints(self.first.tolist())
        args = (self.cache.device_table(), ints(self.lens))
        if self.prefix:
            out = nk.prefix_attention(self.q, self.cache.k, self.cache.v, ints(self.before), self.prefix, *args, q_start=start)
        else:
            out = nk.paged_attention(self.q, self.cache.k, self.cache.v, *args, q_start=start)
        no_device_error()
        return out

    def keys(self, b, j):
        """Where key j of sequence b lies, the shared ones first."""
        if j < self.prefix:
            return self.where_before[0][j], self.where_before[1][j]
        pages, slots = self.cache.where(b, [j - self.prefix])
        return pages[0], slots[0]


@pytest.mark.parametrize("case", range(len(SEEN)))
def test_a_query_that_is_nan(case):
    """Its row is NaN, whether its unit is cut or not, and no other changes."""
    x = Seen(case, 1200)
    plain = x.run()
    T = x.q.shape[0]
    for t, h in {(0, 0), (T - 1, x.hq - 1), (T // 2, x.hq // 2)}:
        kept = x.q[t, h].clone()
        x.q[t, h, 0] = NAN
        got = x.run()
        assert bool(got[t, h].isnan().all()), (t, h)
        got[t, h] = plain[t, h]
        assert torch.equal(got, plain)
        x.q[t, h] = kept


@pytest.mark.parametrize("case", range(len(SEEN)))
def test_a_key_that_is_nan_or_infinite(case):
    """Whatever its place in a block of keys: the rows that see it are NaN, the others as without it."""
    x = Seen(case, 1300)
    for value in (NAN, INF):
        x.q[..., 0] = x.q[..., 0].abs() + 0.5  # +inf in a key's first dimension is a score of +inf
        plain = x.run()
        b = len(x.news) - 1
        n = x.prefix + x.lens[b]
        rows = slice(int(x.first[b]), int(x.first[b + 1]))
        for j in sorted({*range(max(0, n // 3), n // 3 + 9), 0, n - 1}):
            at = x.keys(b, j)
            kept = x.cache.k[at].clone()
            x.cache.k[at[0], at[1], :, 0] = value
            got = x.run()
            x.cache.k[at] = kept
            sees = torch.zeros(len(plain), dtype=torch.bool, device="cuda")
            if j < x.prefix:
                sees[:] = True
            else:
                sees[rows] = torch.arange(x.pasts[b], x.lens[b], device="cuda") >= j - x.prefix
            assert bool(got[sees].isnan().all()), (j, value)
            assert torch.equal(got[~sees], plain[~sees])


@pytest.mark.parametrize("case", range(len(SEEN)))
def test_scores_of_minus_infinity(case):
    """A key with such a score has no weight; a row that has only such scores is zero."""
    x = Seen(case, 1400)
    x.q[..., 0] = -(x.q[..., 0].abs() + 0.5)
    b = len(x.news) - 1
    n = x.prefix + x.lens[b]
    gone = [j for j in range(0, n - x.news[b], 3)]
    for j in gone:
        at = x.keys(b, j)
        x.cache.k[at[0], at[1], :, 0] = INF
    got = x.run()
    rows = slice(int(x.first[b]), int(x.first[b + 1]))
    seen = seen_by(np.arange(x.prefix + x.pasts[b], n), n, 0, 0)
    seen[:, gone] = False
    at = [x.keys(b, j) for j in range(n)]
    pages, slots = (torch.stack([a[i] for a in at]) for i in (0, 1))
    k, v = f64(x.cache.k[pages, slots]), f64(x.cache.v[pages, slots])
    want, mag = attention_reference(f64(x.q[rows]), k, v, seen, 1 / math.sqrt(x.d), x.hkv)
    check_attention(got[rows], want, mag, x.dtype)
    for j in range(n):
        at = x.keys(b, j)
        x.cache.k[at[0], at[1], :, 0] = INF
    assert bool((x.run()[rows] == 0).all())


@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("dtype, d, page", [(BF16, 128, 16), (F16, 64, 16), (F32, 20, 5)])
def test_rows_that_see_nothing_beside_values_that_are_not_finite(dtype, d, page, value):
    rng = np.random.default_rng(1500)
    cache = Paged(rng, [12, 30], 2, d, page, dtype)
    for b, n in enumerate([12, 30]):
        cache.write(rng, b, np.arange(n), dtype)
    pages, slots = cache.where(0, [3])
    cache.v[pages[0], slots[0]] = value
    q = randn(rng, (60, 4, d), dtype)
    got = nk.paged_attention(q, cache.k, cache.v, cache.device_table(), ints([12, 30]), q_start=ints([0, 40, 50]))
    no_device_error()
    assert bool((got[:28] == 0).all()) and bool((got[50:] == 0).all())  # before the first key, and of no sequence
    assert not bool(got[31:40].isfinite().any()) and bool(got[40:50].isfinite().all())


# ---------------------------------------------------------------------------
# starts that go back
# ---------------------------------------------------------------------------
def test_starts_that_go_back_after_a_prefix():
    """More pairs than the list has room for: the tokens that are not listed are zeros, and nothing is read for them."""
    rng = np.random.default_rng(1600)
    T, d, page = 1000, 64, 16
    cache = Paged(rng, [0, T], 1, d, page, BF16, extra=2)
    cache.write(rng, 1, np.arange(T), BF16)
    for c in (cache.k, cache.v):
        c[torch.tensor(cache.free[:2], dtype=torch.long)] = randn(rng, (2, page, 1, d), BF16)
    q = randn(rng, (T, 32, d), BF16)
    got = nk.prefix_attention(q, cache.k, cache.v, ints(cache.free[:2]), 20, cache.device_table(), ints([0, T]),
                              q_start=ints([500, 0, T]))
    no_device_error()
    assert bool(got.isfinite().all()) and bool((got[600:] == 0).all())


# ---------------------------------------------------------------------------
# autograd
# ---------------------------------------------------------------------------
def test_gradients_are_refused_and_writes_are_seen():
    rng = np.random.default_rng(1700)
    cache = Paged(rng, [20], 2, 64, 16, BF16, fill=1.0)
    k, q, table, lens = randn(rng, (1, 2, 64), BF16), randn(rng, (1, 4, 64), BF16), cache.device_table(), ints([20])
    with pytest.raises(RuntimeError, match="q: requires a gradient"):
        nk.paged_attention(q.clone().requires_grad_(), cache.k, cache.v, table, lens)
    with torch.no_grad():
        nk.paged_attention(q.clone().requires_grad_(), cache.k, cache.v, table, lens)
    w = torch.ones((), dtype=BF16, device="cuda", requires_grad=True)
    loss = (w * cache.k).sum()  # keeps the cache for its backward pass
    versions = [cache.k._version, cache.v._version, q._version]
    nk.paged_append(k, k, cache.k, cache.v, table, lens, q=q, q_out=q)
    assert [cache.k._version, cache.v._version, q._version] == [x + 1 for x in versions]
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    out, tokens = torch.empty_like(q), torch.empty(1, dtype=torch.int32, device="cuda")
    nk.paged_attention(q, cache.k, cache.v, table, lens, out=out)
    nk.sample_tokens(torch.zeros((1, 9), device="cuda"), torch.zeros(1, device="cuda"), out=tokens)
    assert out._version == 1 and tokens._version == 1
    with torch.inference_mode():
        x = torch.empty_like(q)
        nk.paged_attention(q, cache.k, cache.v, table, lens, out=x)
    nk.paged_attention(q, cache.k, cache.v, table, lens, out=x)  # has no version to raise
    assert torch.equal(x, out)


# ---------------------------------------------------------------------------
# written tensors
# ---------------------------------------------------------------------------
def test_written_tensors_that_share_memory_are_refused():
    """Repeated elements and overlaps would be written by several blocks at once; nothing is launched."""
    zeros = lambda *s: torch.zeros(s, device="cuda", dtype=BF16)  # noqa: E731
    table, lens = torch.zeros((4, 1), dtype=torch.int32, device="cuda"), ints([1] * 4)
    qkv, both, room = zeros(4, 6, 8), zeros(3, 2, 16, 2, 8), zeros(9, 2, 8)
    q, k, v = qkv[:, :2], qkv[:, 2:4].contiguous(), qkv[:, 4:].contiguous()
    kc, vc = both[:, 0], both[:, 1]  # side by side
    append = lambda k, v, kc, vc, q, out: nk.paged_append(k, v, kc, vc, table, lens, q=q, q_out=out)  # noqa: E731
    attend = lambda q, kc, out: nk.paged_attention(q, kc, kc, table, lens, out=out)  # noqa: E731
    for call, what in (
        (lambda: append(k, v, kc[:1].expand(3, 16, 2, 8), vc, None, None), "k_cache: written"),
        (lambda: append(k, v, kc, vc[:, :1].expand(3, 16, 2, 8), None, None), "v_cache: written"),
        (lambda: append(k, v, both[0, :1], both[0, :1], None, None), "k_cache: .* v_cache"),
        (lambda: append(k, v, kc, vc, q, q[:1].expand(4, 2, 8)), "q_out: written"),
        (lambda: append(k, v, kc, vc, k, k), "q_out: .* shares memory with k"),
        (lambda: append(k, v, kc, vc, room[:4], room[1:5]), "q_out: .* part of its memory with q"),
        (lambda: append(room[:4], v, room[:4].view(1, 4, 2, 8), vc[:1, :4], None, None), "k_cache: .* k"),
        (lambda: attend(q, kc, q[:, :1].expand(4, 2, 8)), "out: written"),
        (lambda: attend(room[:4], kc, room[1:5]), "out: .* part of its memory with q"),
    ):
        with pytest.raises(ValueError, match=what):
            call()
    # what may share: an output that is its input, parts of one projection, keys and values of one allocation
    table.copy_(torch.tensor([[0], [1], [2], [-1]], dtype=torch.int32))
    append(qkv[:, 2:4], qkv[:, 4:], kc, vc, q, q)
    append(k, v, kc, vc, room[:4], room[4:8])
    attend(q, kc, q)
    attend(room[:4], kc, room[:4])
    no_device_error()


# ---------------------------------------------------------------------------
# the last positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("dtype, hq", [(BF16, 4), (F32, 2)])
def test_positions_up_to_the_limit(n, dtype, hq):
    """A page table of 2^31 - 256 positions, full: a window over the last ones, and the first tokens."""
    page, d, N = 8, 64, 2**31 - 256
    window, sinks, last = 60, 3, 20
    rng = np.random.default_rng(1800)
    table = torch.full((1, N // page), -1, dtype=torch.int32, device="cuda")
    order = rng.permutation(last + 1)
    table[0, 0], table[0, -last:] = int(order[0]), ints(order[1:])
    kc, vc = (randn(rng, (last + 1, page, 1, d), dtype) for _ in range(2))
    k, v, q = randn(rng, (n, 1, d), dtype), randn(rng, (n, 1, d), dtype), randn(rng, (n, hq, d), dtype)
    start = None if n == 1 else ints([0, n])
    nk.paged_append(k, v, kc, vc, table, ints([N]), q_start=start)
    rows = lambda c: np.concatenate([f64(c[order[0]])[:sinks], f64(c[order[1:]]).reshape(-1, 1, d)])  # noqa: E731
    assert np.array_equal(rows(kc)[-n:], f64(k)) and np.array_equal(rows(vc)[-n:], f64(v))
    at = np.concatenate([np.arange(sinks), N - last * page + np.arange(last * page)])
    pos = np.arange(N - n, N)[:, None]
    seen = (at <= pos) & ((at > pos - window) | (at < sinks))
    want, mag = attention_reference(f64(q), rows(kc), rows(vc), seen, 1 / math.sqrt(d), 1)
    got = nk.paged_attention(q, kc, vc, table, ints([N]), q_start=start, window=window, sinks=sinks)
    no_device_error()
    check_attention(got, want, mag, dtype)


# ---------------------------------------------------------------------------
# kernel bodies
# ---------------------------------------------------------------------------
def test_rows_that_move_inside_the_caches():
    args = move_inputs()
    host = [a.copy() for a in args]
    move_rows(*host)
    on_device(move_rows, *args)
    for got, want in zip(args[:2], host[:2]):
        np.testing.assert_array_equal(got.view(np.uint16), want.view(np.uint16))


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("vocab", [6, 5000, 500001])
def test_infinite_logits_at_any_temperature(vocab):
    """Only the infinite logits have a weight, as at any other temperature; in a cluster and in one long row."""
    x = torch.zeros((3, vocab), device="cuda")
    x[:, 1], x[:, 3], x[:, 4], x[:, 5] = INF, INF, -INF, NAN
    u, t = torch.tensor([0.2, 0.7, 0.7], device="cuda"), torch.tensor([1.0, 1e30, INF], device="cuda")
    for k, p, m in ((None, None, None), (ints([4] * 3), None, None), (None, torch.full((3,), 0.9, device="cuda"), None),
                    (None, None, torch.full((3,), 0.1, device="cuda")), (ints([1] * 3), None, None)):
        want = [1, 1, 1] if k is not None and int(k[0]) == 1 else [1, 3, 3]
        assert nk.sample_tokens(x, u, t, k, p, m).tolist() == want
    assert nk.sample_tokens(x, u, torch.zeros(3, device="cuda")).tolist() == [1, 1, 1]


def rows64(args, n_heads, n_kv_heads, q_start=None, last=None, prefix_pages=None, prefix_len=0, window=0, sinks=0, eps=1e-6):
    """Where ``workloads.paged_step_kernel`` writes, and the keys, values and queries in 64 bits, each with a bound: with
    u = 2^-8 for a value rounded to bf16, the normalised rows and the projection's result are rounded once each (2 u of
    the terms' magnitudes), rotated rows once more."""
    u = 2.0**-8
    x, norm, w = (np.asarray(a).astype(np.float64) for a in args[:3])
    table, kv_len, cos, sin = args[7], args[8], args[9].astype(np.float64), args[10].astype(np.float64)
    page, d = args[5].shape[1], args[5].shape[3]
    starts = np.arange(len(kv_len) + 1) if q_start is None else q_start
    h = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm
    split = lambda a: [p.reshape(len(x), -1, d) for p in np.split(a, [n_heads * d, (n_heads + n_kv_heads) * d], -1)]  # noqa: E731
    (q, k, v), (mq, mk, mv) = split(h @ w), split(abs(h) @ abs(w))
    pos = np.concatenate([np.arange(n - (e - s), n) for s, e, n in zip(starts, starts[1:], kv_len)])
    seq = np.repeat(np.arange(len(kv_len)), np.diff(starts))
    c, s = cos[pos + prefix_len][:, None], sin[pos + prefix_len][:, None]

    def turned(a, m):
        (lo, hi), (ml, mh) = np.split(a, 2, -1), np.split(m, 2, -1)
        return (np.concatenate([lo * c - hi * s, lo * s + hi * c], -1),
                3 * u * np.concatenate([ml * abs(c) + mh * abs(s), ml * abs(s) + mh * abs(c)], -1))

    return seq, pos, (table[seq, pos // page], pos % page), turned(k, mk), (v, 2 * u * mv), turned(q, mq)


def step_parts(x, norm_weight, qkv_weight, o_weight, head_weight, cache_k, cache_v, page_table, kv_len, cos, sin, u, temperature,
               top_k, top_p, min_p, q_start=None, last=None, prefix_pages=None, prefix_len=0, n_heads=4, n_kv_heads=2, window=0,
               sinks=0, eps=1e-6):
    """``workloads.paged_step_kernel`` with what lies between its calls: queries, attention, logits and tokens."""
    tokens, d = x.shape[0], cache_k.shape[3]
    h = W.qk_rmsnorm(x, norm_weight, eps)
    q, k, v = np.split((h @ qkv_weight).astype(x.dtype), [n_heads * d, (n_heads + n_kv_heads) * d], axis=-1)
    q, k, v = q.reshape(tokens, n_heads, d), k.reshape(tokens, n_kv_heads, d), v.reshape(tokens, n_kv_heads, d)
    q = T.paged_append(k, v, cache_k, cache_v, page_table, kv_len, q_start=q_start, q=q, cos=cos, sin=sin, pos_offset=prefix_len)
    if prefix_len:
        attn = T.prefix_attention(q, cache_k, cache_v, prefix_pages, prefix_len, page_table, kv_len, q_start=q_start)
    else:
        attn = T.paged_attention(q, cache_k, cache_v, page_table, kv_len, q_start=q_start, window=window, sinks=sinks)
    y = x + attn.reshape(tokens, n_heads * d) @ o_weight
    if last is not None:
        y = np.take(y, last, axis=0)
    logits = (y @ head_weight).astype(x.dtype)
    return q, attn, logits, T.sample_tokens(logits, u, temperature, top_k, top_p, min_p)


STEPS = [(None, (1, 20, 64)), ((3, 1, 20), (30, 20, 64)), ((64, 2, 9), (64, 40, 9))]


def step_case(form, news, lens, seed):
    args, kwargs = step_inputs(seed=seed, news=news, lens=lens, prefix=37 if form == "prefix" else 0)
    if form == "window":
        kwargs.update(window=16, sinks=2)
    args = list(args)
    args[12] = np.zeros(3, np.float32)  # greedy
    return args, kwargs


def check_written(args, old, where, keys, values):
    """Of the caches the new rows alone have changed, each within its bound."""
    for cache, before, (want, err) in zip(args[5:7], old, (keys, values)):
        assert np.all(abs(cache[where].astype(np.float64) - want) <= err)
        after = cache.copy()
        after[where] = before[where]
        np.testing.assert_array_equal(after.view(np.uint16), before.view(np.uint16))


@pytest.mark.parametrize("news, lens", STEPS)
@pytest.mark.parametrize("form", ["all", "window", "prefix"])
def test_rows_of_a_step(form, news, lens):
    args, kwargs = step_case(form, news, lens, 8)
    old = [args[i].copy() for i in (5, 6)]
    _, _, where, keys, values, _ = rows64(args, **kwargs)
    tokens = np.asarray(on_device(W.paged_step_kernel, *args, **kwargs))
    check_written(args, old, where, keys, values)
    assert tokens.shape == (3,) and tokens.min() >= 0 and tokens.max() < args[4].shape[1]


@pytest.mark.parametrize("news, lens", STEPS)
@pytest.mark.parametrize("form", ["all", "window", "prefix"])
def test_parts_of_a_step(form, news, lens):
    """Each call of a step against 64 bits, on what the calls before it gave; the tokens are the logits' largest."""
    args, kwargs = step_case(form, news, lens, 9)
    old = [args[i].copy() for i in (5, 6)]
    seq, pos, where, keys, values, (want, err) = rows64(args, **kwargs)
    q, attn, logits, tokens = (np.asarray(a) for a in on_device(step_parts, *args, **kwargs))
    check_written(args, old, where, keys, values)
    q, attn, logits = (a.astype(np.float64) for a in (q, attn, logits))
    assert np.all(abs(q - want) <= err)
    u, (kc, vc), table = 2.0**-8, (a.astype(np.float64) for a in args[5:7]), args[7]
    page, hkv, d = kc.shape[1:]
    before = np.arange(kwargs.get("prefix_len", 0))
    for t, (b, p) in enumerate(zip(seq, pos)):
        at = np.arange(p + 1)
        pages, slots = table[b, at // page], at % page
        seen = seen_by(np.array([p]), p + 1, kwargs.get("window", 0), kwargs.get("sinks", 0))
        if len(before):
            pages, slots = np.concatenate([kwargs["prefix_pages"][before // page], pages]), np.concatenate([before % page, slots])
            seen = np.concatenate([np.ones((1, len(before)), bool), seen], 1)
        want, mag = attention_reference(q[t : t + 1], kc[pages, slots], vc[pages, slots], seen, 1 / math.sqrt(d), hkv)
        assert np.all(abs(attn[t] - want[0]) <= u * (mag[0] + abs(want[0])) + 2.0**-16 * mag[0])
    x, wo, head = (np.asarray(args[i]).astype(np.float64) for i in (0, 3, 4))
    a = attn.reshape(len(x), -1)
    y, dy = x + a @ wo, 2 * u * (abs(x) + abs(a) @ abs(wo))  # the product and the sum, rounded once each
    if "last" in kwargs:
        y, dy = y[kwargs["last"]], dy[kwargs["last"]]
    assert np.all(abs(logits - y @ head) <= dy @ abs(head) + u * abs(y) @ abs(head))
    np.testing.assert_array_equal(tokens, logits.argmax(1))

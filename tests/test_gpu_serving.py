"""The paged serving operators against plain implementations in 64 bits.

Tolerances.  u is the rounding of the stored type (2^-8 bf16, 2^-11 fp16, 2^-24
fp32).  ``paged_append`` rotates in fp32 and rounds once: u |y| plus 2^-22 of
the terms' magnitudes.  Attention may round each probability and its result:
u (sum_j p_j |v_j| + |out|), plus 2^-16 of sum_j p_j |v_j| for the fp32 scores
and exponentials (scores of magnitude up to 2^5 with 2^-23 relative error, and
their sums).  Tokens are whole numbers: the weights are fp32 exponentials, so
a draw may fall to a neighbour only where the 64-bit running sum is within
2^-20 of u or of top_p."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from nkipy_b200 import runtime as nk  # noqa: E402

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def f64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def randn(rng, shape, dtype):
    return torch.tensor(rng.standard_normal(shape), dtype=torch.float64).to(dtype).cuda()


class Paged:
    """A cache whose pages are shuffled, its page table, and where each position's row lies.  ``fill``
    is what the pages hold where no sequence has written."""

    def __init__(self, rng, lens, hkv, d, page, dtype, layout="slots", fill=float("nan"), spare=2, width=None, extra=0):
        counts = [-(-n // page) for n in lens]
        total = sum(counts) + spare + extra
        order = rng.permutation(total)
        self.page, self.lens = page, lens
        self.width = max([1] + counts) if width is None else width
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at : at + n]
            at += n
        self.free = order[at:].astype(np.int32)
        shape = (total, page, hkv, d) if layout == "slots" else (total, hkv, page, d)
        view = (lambda t: t) if layout == "slots" else (lambda t: t.transpose(1, 2))
        self.k = view(torch.full(shape, fill, dtype=dtype, device="cuda"))
        self.v = view(torch.full(shape, fill, dtype=dtype, device="cuda"))
        if layout == "interleaved":  # keys and values of a page side by side
            both = torch.full((total, 2) + shape[1:], fill, dtype=dtype, device="cuda")
            self.k, self.v = view(both[:, 0]), view(both[:, 1])

    def where(self, b, positions):
        positions = np.asarray(positions)
        return torch.tensor(self.table[b, positions // self.page], dtype=torch.long, device="cuda"), torch.tensor(
            positions % self.page, device="cuda")

    def write(self, rng, b, positions, dtype):
        if len(positions) == 0:
            return
        pages, slots = self.where(b, positions)
        for c in (self.k, self.v):
            c[pages, slots] = randn(rng, (len(positions),) + tuple(c.shape[2:]), dtype)

    def read(self, cache, b, positions):
        pages, slots = self.where(b, positions)
        return f64(cache[pages, slots])

    def device_table(self):
        return ints(self.table)


def starts(news):
    return np.cumsum([0] + list(news)).tolist()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def append_reference(x, pos, cos, sin):
    """Rotated rows in 64 bits, and the magnitudes of their terms."""
    half = cos.shape[1]
    c, s = cos[np.clip(pos, 0, len(cos) - 1)][:, None], sin[np.clip(pos, 0, len(sin) - 1)][:, None]
    lo, hi, rest = x[..., :half], x[..., half : 2 * half], x[..., 2 * half :]
    y = np.concatenate([lo * c - hi * s, lo * s + hi * c, rest], -1)
    mag = np.concatenate([abs(lo * c) + abs(hi * s), abs(lo * s) + abs(hi * c), abs(rest)], -1)
    return y, mag


APPEND = [
    # news, pasts, hq, hkv, d, rot, page, dtype, cache dtype, layout
    ([1, 1, 1], [0, 15, 16], 8, 2, 128, 128, 16, BF16, BF16, "slots"),
    ([1], [4096], 32, 8, 128, 128, 16, F16, F16, "heads"),
    ([5, 0, 17, 1], [3, 9, 0, 100], 6, 2, 64, 32, 16, F16, F16, "slots"),
    ([7, 30], [31, 2], 4, 4, 96, 96, 32, BF16, BF16, "interleaved"),
    ([3, 2], [1, 1], 3, 1, 20, 10, 5, F32, F32, "slots"),  # odd page size, rows not a multiple of 16 bytes
    ([9], [11], 5, 5, 80, 0, 64, BF16, BF16, "heads"),  # no rotation
    ([4, 4], [100, 7], 2, 1, 128, 64, 8, F32, BF16, "slots"),  # the cache's type differs
    ([6], [0], 0, 3, 48, 48, 16, BF16, F32, "slots"),  # no queries
    ([260], [5], 3, 1, 72, 24, 128, F16, F16, "slots"),
]


@pytest.mark.parametrize("rope_dtype", [F32, BF16])
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(case, rope_dtype):
    news, pasts, hq, hkv, d, rot, page, dtype, cdtype, layout = APPEND[case]
    rng = np.random.default_rng(100 + case)
    lens = [a + b for a, b in zip(news, pasts)]
    cache = Paged(rng, lens, hkv, d, page, cdtype, layout, fill=3.0)
    T = sum(news)
    qkv = randn(rng, (T, hq + 2 * hkv, d), dtype)  # q, k and v side by side, as a projection leaves them
    q, k, v = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
    ang = rng.uniform(0, 6, (max(lens) + 3, rot // 2))
    cos, sin = (torch.tensor(f(ang)).to(rope_dtype).cuda() for f in (np.cos, np.sin))
    before = [c.clone() for c in (cache.k, cache.v)]
    got = nk.paged_append(k, v, cache.k, cache.v, cache.device_table(), ints(lens), q_start=ints(starts(news)),
                          q=q if hq else None, cos=cos if rot else None, sin=sin if rot else None)
    pos = np.concatenate([np.arange(p, p + n) for n, p in zip(news, pasts)]).astype(int)
    c64, s64 = f64(cos), f64(sin)
    if hq:
        want, mag = append_reference(f64(q), pos, c64, s64)
        assert np.all(abs(f64(got) - want) <= UNIT[dtype] * abs(want) + 2.0**-22 * mag + 1e-38 + 2.0**-25 * (dtype is F16))
    else:
        assert got is None
    want_k, mag = append_reference(f64(k), pos, c64, s64)
    at = 0
    for b, (n, p) in enumerate(zip(news, pasts)):
        if n == 0:
            continue
        pages, slots = cache.where(b, np.arange(p, p + n))
        gk, gv = f64(cache.k[pages, slots]), f64(cache.v[pages, slots])
        wk, m = want_k[at : at + n], mag[at : at + n]
        assert np.all(abs(gk - wk) <= UNIT[cdtype] * abs(wk) + 2.0**-22 * m + 2.0**-25 * (cdtype is F16))
        np.testing.assert_array_equal(gv, f64(v[at : at + n].to(cdtype)))
        for c, old in zip((cache.k, cache.v), before):  # nothing else was written
            c[pages, slots] = old[pages, slots]
        at += n
    for c, old in zip((cache.k, cache.v), before):
        assert torch.equal(c, old)


def test_append_single_tokens_without_q_start():
    rng = np.random.default_rng(1)
    lens = [1, 16, 17, 33]
    cache = Paged(rng, lens, 2, 64, 16, BF16)
    k, v = randn(rng, (4, 2, 64), BF16), randn(rng, (4, 2, 64), BF16)
    assert nk.paged_append(k, v, cache.k, cache.v, cache.device_table(), ints(lens)) is None
    for b, n in enumerate(lens):
        pages, slots = cache.where(b, [n - 1])
        assert torch.equal(cache.k[pages, slots][0], k[b]) and torch.equal(cache.v[pages, slots][0], v[b])


def test_append_drops_what_has_no_page():
    """Positions past the table, negative positions, page ids that the cache does not have, and
    tokens of no sequence: nothing is stored for them, and a token of no sequence has a zero query."""
    rng = np.random.default_rng(2)
    k, v = randn(rng, (9, 2, 64), F16), randn(rng, (9, 2, 64), F16)
    q = randn(rng, (9, 4, 64), F16)
    kc, vc = (torch.full((4, 16, 2, 64), 7.0, dtype=F16, device="cuda") for _ in range(2))
    table = ints([[0, -1], [1, 99], [2, 3]])
    # sequence 0: positions 15, 16 (page -1); 1: 31 (page 99) and 32 (past the table); 2: -1, 0
    cos = torch.ones((40, 32), device="cuda")
    sin = torch.zeros((40, 32), device="cuda")
    got = nk.paged_append(k, v, kc, vc, table, ints([17, 33, 1]), q_start=ints([0, 2, 4, 6]), q=q, cos=cos, sin=sin)
    want_k, want_v = (torch.full((4, 16, 2, 64), 7.0, dtype=F16, device="cuda") for _ in range(2))
    want_k[0, 15], want_v[0, 15], want_k[2, 0], want_v[2, 0] = k[0], v[0], k[5], v[5]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    assert torch.equal(got[:6], q[:6]) and bool((got[6:] == 0).all())


def test_append_in_place_queries_and_offset():
    """q_out may be q; pos_offset moves the rotation's position, not the slot."""
    rng = np.random.default_rng(3)
    cache = Paged(rng, [5], 1, 32, 16, F32)
    q, k, v = randn(rng, (2, 3, 32), F32), randn(rng, (2, 1, 32), F32), randn(rng, (2, 1, 32), F32)
    ang = rng.uniform(0, 6, (50, 16))
    cos, sin = torch.tensor(np.cos(ang)).float().cuda(), torch.tensor(np.sin(ang)).float().cuda()
    want, mag = append_reference(f64(q), np.array([33, 34]), f64(cos), f64(sin))
    out = nk.paged_append(k, v, cache.k, cache.v, cache.device_table(), ints([5]), q_start=ints([0, 2]), q=q, cos=cos,
                          sin=sin, pos_offset=30, q_out=q)
    assert out.data_ptr() == q.data_ptr()
    assert np.all(abs(f64(q) - want) <= 2.0**-22 * mag)
    pages, slots = cache.where(0, [3, 4])
    assert torch.equal(cache.v[pages, slots], v)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def attention_reference(q, k, v, seen, scale, hkv):
    """out and sum_j p_j |v_j| in 64 bits; q (n, hq, d), k and v (keys, hkv, d), seen (n, keys)."""
    n, hq, d = q.shape
    out, mag = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    g = hq // hkv
    v = np.where(seen.any(0)[:, None, None], v, 0.0)
    k = np.where(seen.any(0)[:, None, None], k, 0.0)
    for h in range(hq):
        s = np.where(seen, q[:, h] @ k[:, h // g].T * scale, -np.inf)
        top = s.max(1, initial=-np.inf, keepdims=True)
        e = np.where(seen, np.exp(s - np.where(top == -np.inf, 0, top)), 0.0)
        total = e.sum(1, keepdims=True)
        p = e / np.where(total > 0, total, 1)
        out[:, h], mag[:, h] = p @ v[:, h // g], p @ abs(v[:, h // g])
    return out, mag


def seen_by(pos, keys, window, sinks):
    i, j = pos[:, None], np.arange(keys)[None]
    seen = j <= i
    if window:
        seen = seen & ((j > i - window) | (j < sinks))
    return seen


def check_attention(got, want, mag, dtype):
    bound = UNIT[dtype] * (mag + abs(want)) + 2.0**-16 * mag + 2.0**-25 * (dtype is F16)
    err = abs(f64(got) - want)
    assert np.all(np.isfinite(f64(got)))
    assert np.all(err <= bound), (float(err.max()), float((err / bound).max()))


def run_attention(seed, news, pasts, window, sinks, hq, hkv, d, page, dtype, layout="slots", scale=None, q_start=True):
    """Every cached key that no query sees holds NaN."""
    rng = np.random.default_rng(seed)
    lens = [a + b for a, b in zip(news, pasts)]
    cache = Paged(rng, lens, hkv, d, page, dtype, layout)
    T = sum(news)
    q = randn(rng, (T, hq, d), dtype)
    want, mag, at = np.zeros((T, hq, d)), np.zeros((T, hq, d)), 0
    for b, (n, p) in enumerate(zip(news, pasts)):
        seen = seen_by(np.arange(p, p + n), p + n, window, sinks)
        if n == 0:
            continue
        cache.write(rng, b, np.flatnonzero(seen.any(0)), dtype)
        k, v = cache.read(cache.k, b, np.arange(p + n)), cache.read(cache.v, b, np.arange(p + n))
        want[at : at + n], mag[at : at + n] = attention_reference(f64(q[at : at + n]), k, v, seen,
                                                                  1 / math.sqrt(d) if scale is None else scale, hkv)
        at += n
    got = nk.paged_attention(q, cache.k, cache.v, cache.device_table(), ints(lens),
                             q_start=ints(starts(news)) if q_start else None, window=window, sinks=sinks, scale=scale)
    check_attention(got, want, mag, dtype)
    return got


DECODE = [
    # lengths, window, sinks, hq, hkv, d, page, dtype, layout
    ([1], 0, 0, 1, 1, 64, 16, BF16, "slots"),
    ([1, 2, 15, 16, 17, 33], 0, 0, 8, 2, 128, 16, BF16, "slots"),
    ([500], 0, 0, 32, 8, 128, 16, F16, "heads"),
    ([700, 3, 1300], 0, 0, 6, 2, 96, 64, BF16, "interleaved"),
    ([700, 3, 1300], 100, 4, 10, 2, 64, 32, F16, "slots"),
    ([257, 64, 63, 65], 64, 0, 7, 1, 128, 8, BF16, "slots"),
    ([200, 5], 1, 0, 4, 4, 64, 16, BF16, "slots"),  # a window of the token alone
    ([200, 5], 1, 19, 4, 4, 64, 16, BF16, "slots"),  # and first tokens, more than a page
    ([200, 40], 30, 500, 4, 2, 64, 16, F16, "heads"),  # more first tokens than there are
    ([90, 77], 0, 0, 40, 2, 64, 16, BF16, "slots"),  # 20 query heads per key head
    ([90, 77], 20, 3, 33, 1, 128, 16, F16, "slots"),
    ([130], 0, 0, 4, 2, 40, 16, BF16, "slots"),  # a head dimension under 64
    ([61, 9], 12, 2, 4, 2, 20, 5, F32, "slots"),  # no tensor-core form: type, page size, row size
    ([61, 9], 0, 0, 4, 2, 256, 16, BF16, "slots"),
    ([61, 9], 0, 0, 4, 2, 64, 48, F16, "slots"),
    ([5000, 1, 2500, 4097] * 5, 2048, 4, 8, 2, 128, 128, BF16, "slots"),
    ([20000], 0, 0, 8, 1, 64, 256, BF16, "slots"),
]


@pytest.mark.parametrize("case", range(len(DECODE)))
@pytest.mark.parametrize("q_start", [False, True])
def test_decode(case, q_start):
    lens, window, sinks, hq, hkv, d, page, dtype, layout = DECODE[case]
    run_attention(200 + case, [1] * len(lens), [n - 1 for n in lens], window, sinks, hq, hkv, d, page, dtype, layout,
                  q_start=q_start)


CHUNKS = [
    # news, pasts, window, sinks, hq, hkv, d, page, dtype, layout
    ([2], [0], 0, 0, 1, 1, 64, 16, BF16, "slots"),
    ([130], [0], 0, 0, 4, 2, 128, 16, BF16, "slots"),
    ([33, 0, 1, 127, 64], [0, 5, 300, 128, 1], 0, 0, 8, 2, 128, 16, F16, "heads"),
    ([300, 20], [100, 700], 50, 4, 6, 2, 64, 32, BF16, "slots"),
    ([300, 20], [100, 700], 50, 4, 6, 2, 64, 32, F16, "interleaved"),
    ([257], [0], 128, 0, 5, 1, 128, 8, BF16, "slots"),
    ([257], [1], 127, 200, 3, 3, 96, 64, BF16, "slots"),
    ([70, 3], [5, 2000], 0, 0, 40, 2, 64, 16, F16, "slots"),
    ([70, 3], [5, 900], 33, 1, 33, 1, 128, 128, BF16, "slots"),
    ([100], [28], 0, 0, 4, 2, 40, 16, BF16, "slots"),
    ([31, 9], [2, 60], 12, 2, 4, 2, 20, 5, F32, "slots"),
    ([31, 9], [2, 60], 0, 0, 4, 2, 256, 16, BF16, "slots"),
    ([31, 9], [2, 60], 7, 3, 4, 2, 64, 48, F16, "heads"),
    ([3], [9000], 0, 0, 8, 1, 128, 64, BF16, "slots"),  # few rows, many keys
    ([1000, 600], [0, 24], 256, 4, 8, 2, 128, 16, BF16, "slots"),
    ([1, 1, 90], [511, 0, 38], 0, 0, 128, 1, 64, 16, BF16, "slots"),  # 128 query heads per key head
]


@pytest.mark.parametrize("case", range(len(CHUNKS)))
def test_chunks(case):
    run_attention(300 + case, *CHUNKS[case])


def test_scale_and_large_scores():
    """Scores of some hundreds: the running maximum carries them."""
    run_attention(400, [1, 1], [99, 300], 0, 0, 8, 2, 64, 16, BF16, scale=8.0)
    run_attention(401, [60, 1], [99, 300], 0, 0, 8, 2, 64, 16, BF16, scale=8.0)


@pytest.mark.parametrize("news", [[1, 1, 1, 1], [3, 2, 4, 1]])
def test_rows_that_see_nothing(news):
    """Length 0, positions before the first key, and tokens of no sequence give zeros."""
    rng = np.random.default_rng(5)
    lens = [0, 40, 1, 0]
    cache = Paged(rng, lens, 2, 64, 16, BF16)
    cache.write(rng, 1, np.arange(40), BF16)
    cache.write(rng, 2, np.arange(1), BF16)
    T = sum(news) + (2 if news[0] > 1 else 0)
    q = randn(rng, (T, 4, 64), BF16)
    want, mag = np.zeros((T, 4, 64)), np.zeros((T, 4, 64))
    s = starts(news)
    for b in (1, 2):
        pos = np.arange(lens[b] - news[b], lens[b])
        k, v = cache.read(cache.k, b, np.arange(lens[b])), cache.read(cache.v, b, np.arange(lens[b]))
        want[s[b] : s[b + 1]], mag[s[b] : s[b + 1]] = attention_reference(
            f64(q[s[b] : s[b + 1]]), k, v, seen_by(pos, lens[b], 0, 0), 0.125, 2)
    got = nk.paged_attention(q, cache.k, cache.v, cache.device_table(), ints(lens),
                             q_start=ints(s) if news[0] > 1 else None, out=torch.full_like(q, 9.0))
    check_attention(got, want, mag, BF16)


@pytest.mark.parametrize("n", [1, 40])
def test_pages_the_cache_does_not_have_read_as_zeros(n):
    rng = np.random.default_rng(6)
    cache = Paged(rng, [100], 2, 64, 16, F16)
    cache.write(rng, 0, np.arange(100), F16)
    q = randn(rng, (n, 4, 64), F16)
    k, v = cache.read(cache.k, 0, np.arange(100)), cache.read(cache.v, 0, np.arange(100))
    for i, bad in ((1, -1), (4, 12345)):
        cache.table[0, i] = bad
        k[16 * i : 16 * i + 16], v[16 * i : 16 * i + 16] = 0, 0
    want, mag = attention_reference(f64(q), k, v, seen_by(np.arange(100 - n, 100), 100, 0, 0), 0.125, 2)
    got = nk.paged_attention(q, cache.k, cache.v, cache.device_table(), ints([100]), q_start=ints([0, n]))
    check_attention(got, want, mag, F16)


@pytest.mark.parametrize("n", [1, 50])
def test_length_past_the_table(n):
    """Keys past the page table do not exist; positions stay what kv_len says."""
    rng = np.random.default_rng(7)
    cache = Paged(rng, [64], 1, 64, 16, BF16)
    cache.write(rng, 0, np.arange(64), BF16)
    q = randn(rng, (n, 2, 64), BF16)
    k, v = cache.read(cache.k, 0, np.arange(64)), cache.read(cache.v, 0, np.arange(64))
    want, mag = attention_reference(f64(q), k, v, seen_by(np.arange(90 - n, 90), 64, 60, 3), 0.125, 1)
    got = nk.paged_attention(q, cache.k, cache.v, cache.device_table(), ints([90]), q_start=ints([0, n]), window=60, sinks=3)
    check_attention(got, want, mag, BF16)


def test_strided_queries_and_outputs():
    rng = np.random.default_rng(8)
    news, lens = [1, 70], [50, 90]
    cache = Paged(rng, lens, 2, 64, 16, BF16)
    for b in range(2):
        cache.write(rng, b, np.arange(lens[b]), BF16)
    wide = randn(rng, (71, 9, 72), BF16)
    q = wide[:, 1:5, :64]
    plain = nk.paged_attention(q.contiguous(), cache.k, cache.v, cache.device_table(), ints(lens), q_start=ints([0, 1, 71]))
    room = torch.full((71, 7, 80), 5.0, dtype=BF16, device="cuda")
    table = torch.full((2, 11), -7, dtype=torch.int32, device="cuda")
    table[:, : cache.width] = cache.device_table()
    got = nk.paged_attention(q, cache.k, cache.v, table[:, : cache.width], ints(lens), q_start=ints([0, 1, 71]),
                             out=room[:, 2:6, 8:72])
    assert got.data_ptr() == room[:, 2:6, 8:72].data_ptr() and torch.equal(got, plain)
    assert bool((room[:, :2] == 5).all()) and bool((room[:, 6:] == 5).all())
    assert bool((room[:, 2:6, :8] == 5).all()) and bool((room[:, 2:6, 72:] == 5).all())
    # rows that start at odd elements take another form of the kernel, with the same bounds
    odd = wide[:, 1:5, 3:67]
    a = nk.paged_attention(odd, cache.k, cache.v, cache.device_table(), ints(lens), q_start=ints([0, 1, 71]))
    b = nk.paged_attention(odd.contiguous(), cache.k, cache.v, cache.device_table(), ints(lens), q_start=ints([0, 1, 71]))
    assert float((a.float() - b.float()).abs().max()) <= 2.0**-6


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements whose last pages are read and written."""
    page, hkv, d = 128, 8, 128
    pages = 2**31 // (page * hkv * d) + 3
    kc, vc = (torch.zeros((pages, page, hkv, d), dtype=BF16, device="cuda") for _ in range(2))
    rng = np.random.default_rng(9)
    table = ints([[pages - 1, 0], [pages - 2, pages - 3]])
    k, v = randn(rng, (400, hkv, d), BF16), randn(rng, (400, hkv, d), BF16)
    news = [200, 200]
    nk.paged_append(k, v, kc, vc, table, ints(news), q_start=ints([0, 200, 400]))
    assert torch.equal(kc[pages - 1], k[:128]) and torch.equal(vc[pages - 3, :72], v[328:])
    for n in (1, 200):
        q = randn(rng, (2 * n, 16, d), BF16)
        got = nk.paged_attention(q, kc, vc, table, ints(news), q_start=ints([0, n, 2 * n]))
        for b in range(2):
            want, mag = attention_reference(f64(q[b * n : b * n + n]), f64(k[200 * b : 200 * b + 200]),
                                            f64(v[200 * b : 200 * b + 200]),
                                            seen_by(np.arange(200 - n, 200), 200, 0, 0), 1 / math.sqrt(d), hkv)
            check_attention(got[b * n : b * n + n], want, mag, BF16)


PREFIX = [
    # prefix, news, pasts, hq, hkv, d, page, dtype, layout
    (100, [1, 1, 1], [0, 20, 77], 8, 2, 128, 16, BF16, "slots"),
    (1, [1], [5], 4, 1, 64, 16, F16, "slots"),
    (1000, [1] * 9, [3, 0, 200, 16, 17, 64, 63, 1, 90], 10, 2, 64, 32, BF16, "heads"),
    (333, [2, 1, 5], [10, 0, 31], 6, 2, 96, 16, BF16, "slots"),
    (640, [150], [2], 4, 4, 128, 64, F16, "interleaved"),
    (37, [1, 3], [4, 5], 4, 2, 20, 5, F32, "slots"),
    (5000, [1] * 40, list(range(40)), 32, 2, 128, 128, BF16, "slots"),
    (700, [1, 1], [9, 3], 128, 1, 64, 16, BF16, "slots"),
    (0, [1, 1], [9, 3], 4, 2, 64, 16, BF16, "slots"),
]


@pytest.mark.parametrize("case", range(len(PREFIX)))
def test_prefix(case):
    prefix, news, pasts, hq, hkv, d, page, dtype, layout = PREFIX[case]
    rng = np.random.default_rng(500 + case)
    lens = [a + b for a, b in zip(news, pasts)]
    n_pages = -(-prefix // page)
    cache = Paged(rng, lens, hkv, d, page, dtype, layout, extra=n_pages)
    T = sum(news)
    q = randn(rng, (T, hq, d), dtype)
    pages = cache.free[:n_pages]
    where = np.arange(prefix)
    at_p = torch.tensor(pages[where // page], dtype=torch.long, device="cuda"), torch.tensor(where % page, device="cuda")
    for c in (cache.k, cache.v):
        if prefix:
            c[at_p] = randn(rng, (prefix, hkv, d), dtype)
    pk, pv = f64(cache.k[at_p]), f64(cache.v[at_p])
    want, mag, at = np.zeros((T, hq, d)), np.zeros((T, hq, d)), 0
    for b, (n, p) in enumerate(zip(news, pasts)):
        cache.write(rng, b, np.arange(p + n), dtype)
        k = np.concatenate([pk, cache.read(cache.k, b, np.arange(p + n))])
        v = np.concatenate([pv, cache.read(cache.v, b, np.arange(p + n))])
        seen = np.concatenate([np.ones((n, prefix), bool), seen_by(np.arange(p, p + n), p + n, 0, 0)], 1)
        want[at : at + n], mag[at : at + n] = attention_reference(f64(q[at : at + n]), k, v, seen, 1 / math.sqrt(d), hkv)
        at += n
    one = all(n == 1 for n in news)
    got = nk.prefix_attention(q, cache.k, cache.v, ints(pages), prefix, cache.device_table(), ints(lens),
                              q_start=None if one else ints(starts(news)))
    check_attention(got, want, mag, dtype)


SHARES = [
    # news, pasts, window, sinks, hq, hkv, d, page, dtype, layout
    ([5] * 12, range(40, 52), 0, 0, 4, 2, 64, 16, BF16, "slots"),  # fewer units than CTAs: one each
    ([200, 3], [3000, 0], 0, 0, 4, 2, 128, 32, F16, "slots"),  # few long ones: cut
    ([7] * 40, range(40), 0, 0, 16, 8, 64, 16, BF16, "slots"),  # some units per CTA
    ([70, 1] * 20, [30, 700] * 20, 60, 2, 32, 4, 128, 16, BF16, "slots"),
    ([7] * 20, [6000] + [10] * 19, 0, 0, 8, 8, 64, 128, BF16, "slots"),  # one much longer than a share: cut
    ([2] * 300, range(300), 0, 0, 2, 1, 64, 16, F16, "slots"),  # a long list
    ([3] * 120, range(120), 0, 0, 8, 8, 128, 16, BF16, "slots"),  # many units per CTA
]


@pytest.mark.parametrize("case", range(len(SHARES)))
def test_shares_of_work(case):
    news, pasts, *rest = SHARES[case]
    run_attention(400 + case, news, list(pasts), *rest)


@pytest.mark.parametrize("prefix, news, hq, hkv", [
    (40, [1] * 300, 64, 8),  # several rounds of whole units
    (40, [3] * 90, 8, 8),    # with units of the sequences' own
    (20, [1, 2], 4, 2),
    (3000, [2, 1, 1], 4, 2),
    (600, [1] * 130, 16, 1),
])
def test_prefix_shares_of_work(prefix, news, hq, hkv):
    d, page = 64, 16
    rng = np.random.default_rng(prefix + len(news))
    n_pages = -(-prefix // page)
    cache = Paged(rng, news, hkv, d, page, BF16, "slots", extra=n_pages)
    pages, where = cache.free[:n_pages], np.arange(prefix)
    at_p = torch.tensor(pages[where // page], dtype=torch.long, device="cuda"), torch.tensor(where % page, device="cuda")
    for c in (cache.k, cache.v):
        c[at_p] = randn(rng, (prefix, hkv, d), BF16)
    pk, pv, T = f64(cache.k[at_p]), f64(cache.v[at_p]), sum(news)
    q = randn(rng, (T, hq, d), BF16)
    want, mag, at = np.zeros((T, hq, d)), np.zeros((T, hq, d)), 0
    for b, n in enumerate(news):
        cache.write(rng, b, np.arange(n), BF16)
        k, v = (np.concatenate([p, cache.read(c, b, np.arange(n))]) for p, c in ((pk, cache.k), (pv, cache.v)))
        seen = np.concatenate([np.ones((n, prefix), bool), seen_by(np.arange(n), n, 0, 0)], 1)
        want[at : at + n], mag[at : at + n] = attention_reference(f64(q[at : at + n]), k, v, seen, 1 / math.sqrt(d), hkv)
        at += n
    one = all(n == 1 for n in news)
    got = nk.prefix_attention(q, cache.k, cache.v, ints(pages), prefix, cache.device_table(), ints(news),
                              q_start=None if one else ints(starts(news)))
    check_attention(got, want, mag, BF16)


def test_prefix_alone():
    """Sequences that have nothing of their own yet see the prefix."""
    rng = np.random.default_rng(10)
    cache = Paged(rng, [0, 0], 2, 64, 16, BF16, extra=3)
    q = randn(rng, (2, 4, 64), BF16)
    for c in (cache.k, cache.v):
        c[torch.tensor(cache.free[:3], dtype=torch.long)] = randn(rng, (3, 16, 2, 64), BF16)
    pk, pv = (f64(c[torch.tensor(cache.free[:3], dtype=torch.long)]).reshape(48, 2, 64)[:40] for c in (cache.k, cache.v))
    want, mag = attention_reference(f64(q), pk, pv, np.ones((2, 40), bool), 0.125, 2)
    got = nk.prefix_attention(q, cache.k, cache.v, ints(cache.free[:3]), 40, cache.device_table(), ints([0, 0]))
    check_attention(got, want, mag, BF16)


def test_attention_on_another_stream_and_in_a_graph():
    """A call issued on a side stream, and one captured and replayed with other lengths."""
    rng = np.random.default_rng(11)
    cache = Paged(rng, [300, 200], 2, 64, 16, BF16)
    for b, n in enumerate([300, 200]):
        cache.write(rng, b, np.arange(n), BF16)
    q, lens, table = randn(rng, (2, 8, 64), BF16), ints([300, 200]), cache.device_table()
    logits, u = randn(rng, (2, 5000), F32), torch.tensor([0.3, 0.9], device="cuda")

    def step():
        return nk.paged_attention(q, cache.k, cache.v, table, lens, window=100, sinks=4), nk.sample_tokens(logits, u)

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    lens.copy_(ints([17, 120]))
    u.copy_(torch.tensor([0.8, 0.1], device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in out]
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def draw64(x, u, temperature, top_k, top_p, min_p):
    """The definition in 64 bits, for one row."""
    x = np.where(np.isnan(x), -np.inf, x)
    if x.max() == -np.inf:
        return -1
    if temperature <= 0:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore"):
        e = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / temperature))
    e = np.where(x == -np.inf, 0.0, e)
    order = np.argsort(-x, kind="stable")
    k = len(x) if top_k <= 0 else min(top_k, len(x))
    s = np.where(np.arange(len(x)) < k, e[order], 0)
    if top_p < 1:
        before = np.cumsum(s) - s
        s = np.where((before < top_p * s.sum()) | (np.arange(len(x)) == 0), s, 0)
    w = np.zeros(len(x))
    w[order] = s
    w = np.where(e >= min(min_p, 1.0), w, 0)
    c = np.cumsum(w)
    at = min(max(u, 0.0) * c[-1], c[-1] * (1 - 1e-15))
    return int(np.argmax(c > at))


def check_sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    rows = logits.shape[0]
    dev = lambda v, t=torch.float32: None if v is None else torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    got = nk.sample_tokens(logits, dev(u), dev(temperature), dev(top_k, torch.int32), dev(top_p), dev(min_p)).cpu().numpy()
    x = f64(logits)
    eps = 2.0**-20
    for r in range(rows):
        f32 = lambda v, d: d if v is None else float(np.float32(v[r]))  # noqa: E731
        t, p, m, uu = f32(temperature, 1.0), f32(top_p, 1.0), f32(min_p, 0.0), f32(u, 0.0)
        k = 0 if top_k is None else top_k[r]
        near = {draw64(x[r], uu + du, t, k, p + dp if p < 1 else p, m * (1 + dm))
                for du in (0, -eps, eps) for dp in (0, -eps, eps) for dm in (0, -eps, eps)}
        assert int(got[r]) in near, (r, int(got[r]), near)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 50257])
@pytest.mark.parametrize("spread", [0.5, 3.0])
def test_sample(vocab, dtype, spread):
    rng = np.random.default_rng(600 + vocab)
    rows = 12
    logits = (randn(rng, (rows, vocab), F32) * spread).to(dtype)
    u = rng.uniform(size=rows).tolist()
    temperature = [1.0, 0.7, 1.5, 0.0, 1.0, 1.0, 0.3, 2.0, 1.0, 1.0, 5.0, 1e-3]
    top_k = [0, 1, 50, 5, 0, 1, 7, vocab, vocab + 5, 1000, 0, 3]
    top_p = [1.0, 0.9, 0.5, 0.9, 0.95, 1.0, 0.01, 0.8, 0.0, 0.99, 0.999, 0.5]
    min_p = [0.0, 0.0, 0.05, 0.1, 0.2, 1.0, 0.0, 0.01, 0.0, 2.0, 0.0, 0.0]
    check_sample(logits, u, temperature, top_k, top_p, min_p)
    check_sample(logits, u)
    check_sample(logits, u, top_k=top_k)
    check_sample(logits, u, top_p=top_p)
    check_sample(logits, u, min_p=min_p)
    check_sample(logits, u, temperature=temperature)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, vocab", [(40, 9001), (100, 5000), (300, 700), (320, 20001)])
def test_sample_many_rows(rows, vocab, dtype):
    """Weights are whole numbers: a row's token is the same however many rows go with it."""
    rng = np.random.default_rng(700 + vocab)
    logits = (randn(rng, (rows, vocab), F32) * 2).to(dtype)
    some = lambda values, t: torch.tensor([values[i] for i in rng.integers(len(values), size=rows)], dtype=t, device="cuda")  # noqa: E731
    given = [torch.tensor(rng.uniform(size=rows), dtype=torch.float32, device="cuda"), some([1.0, 0.3, 2.0, 0.0], torch.float32),
             some([0, 1, 20, 128, 300], torch.int32), some([1.0, 0.95, 0.5], torch.float32), some([0.0, 0.02], torch.float32)]
    got = nk.sample_tokens(logits, *given).tolist()
    assert got == [x for r in range(0, rows, 8) for x in nk.sample_tokens(logits[r:r + 8], *(g[r:r + 8] for g in given)).tolist()]
    host = [g[:8].tolist() for g in given]
    assert check_sample(logits[:8], *host).tolist() == got[:8]


def test_sample_ties():
    """Equal logits rank by index: whole rows of one value, and a threshold inside a run of equals."""
    x = torch.zeros((4, 5000), device="cuda")
    x[1, 2500:] = 1.0
    x[2, ::7] = 2.0
    x[3] = -5.0
    for u in (0.0, 0.25, 0.999):
        for k, p in ((0, 1.0), (10, 1.0), (0, 0.1), (600, 0.5), (3000, 0.9)):
            check_sample(x, [u] * 4, top_k=[k] * 4, top_p=[p] * 4)
    got = nk.sample_tokens(x, torch.full((4,), 0.9999, device="cuda"), top_k=ints([10] * 4))
    assert got.tolist() == [9, 2509, 63, 9]


def test_sample_infinities():
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(torch.float32).min
    x = torch.full((8, 300), -inf, device="cuda")
    x[1] = nan
    x[2, 17] = 0.0
    x[3, 5], x[3, 9], x[3, 250] = inf, inf, 3.0
    x[4] = low  # a mask of the type's lowest value, everywhere
    x[5] = low
    x[5, 200] = 1.0
    x[6, ::2], x[6, 1::2] = nan, 0.5
    x[7, 299] = -3.0e38
    got = check_sample(x, [0.6] * 8)
    assert got[0] == -1 and got[1] == -1 and got[2] == 17 and got[3] == 9 and got[5] == 200 and got[7] == 299
    check_sample(x, [0.6] * 8, top_k=[3] * 8, top_p=[0.7] * 8, min_p=[0.1] * 8)
    got = check_sample(x, [0.6] * 8, temperature=[0.0] * 8)
    assert got.tolist() == [-1, -1, 17, 5, 0, 200, 1, 299]
    check_sample(x, [0.0] * 8, temperature=[1e-30, 1e30, inf, 1.0, 2.0, 1e-40, 1e-40, 3.0])


def test_sample_random_numbers_at_the_ends():
    x = torch.zeros((5, 1000), device="cuda")
    u = torch.tensor([0.0, 1.0 - 2.0**-24, 1.0, -1.0, float("nan")], device="cuda")
    assert nk.sample_tokens(x, u).tolist() == [0, 999, 999, 0, 0]


def test_sample_strided_rows_and_large_vocabulary():
    rng = np.random.default_rng(12)
    wide = randn(rng, (3, 10000), BF16)
    check_sample(wide[:, 3:8004], [0.1, 0.5, 0.9], top_k=[40] * 3, top_p=[0.9] * 3)
    big = randn(rng, (2, 300001), F32) * 2
    check_sample(big, [0.3, 0.7], top_k=[0, 20000], top_p=[0.95, 0.99])


def test_sample_follows_the_distribution():
    """Draws over an even grid of u hit each token in proportion to its kept weight, exactly to the grid."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5, 3.0, -2.0]], device="cuda")
    n = 4096
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = nk.sample_tokens(x.expand(n, 7).contiguous(), u, top_k=ints([4] * n)).cpu().numpy()
    e = np.exp(f64(x)[0])
    e[[0, 3, 6]] = 0
    want = e / e.sum() * n
    assert np.all(abs(np.bincount(got, minlength=7) - want) <= 1)


# ---------------------------------------------------------------------------
# refusals (the Python layer; the C entries' are tested without a GPU)
# ---------------------------------------------------------------------------
def test_refusals():
    rng = np.random.default_rng(13)
    cache = Paged(rng, [20, 20], 2, 64, 16, BF16)
    q, table, lens = randn(rng, (2, 4, 64), BF16), cache.device_table(), ints([20, 20])
    k, v = randn(rng, (2, 2, 64), BF16), randn(rng, (2, 2, 64), BF16)
    ok = dict(q=q, k_cache=cache.k, v_cache=cache.v, page_table=table, kv_len=lens)
    for change, error in [
        (dict(q=q.half()), TypeError), (dict(q=q.double()), TypeError), (dict(q=q[0]), ValueError),
        (dict(q=q[:, :3]), ValueError), (dict(q=q.cpu()), ValueError), (dict(kv_len=lens.long()), TypeError),
        (dict(kv_len=lens[:1]), ValueError), (dict(page_table=table[0]), ValueError), (dict(q=q[..., ::2]), ValueError),
        (dict(v_cache=cache.v[:-1]), ValueError), (dict(q_start=ints([0, 2])), ValueError),
        (dict(q=q[:1]), ValueError), (dict(out=q.float()), ValueError), (dict(window=-1), RuntimeError),
        (dict(sinks=-1), RuntimeError),
    ]:
        with pytest.raises(error):
            nk.paged_attention(**{**ok, **change})
    with pytest.raises(ValueError):
        nk.prefix_attention(q, cache.k, cache.v, ints([0]), 17, table, lens)
    with pytest.raises(ValueError):
        nk.prefix_attention(q, cache.k, cache.v, ints([0]), -1, table, lens)
    cos = torch.ones((4, 33), device="cuda")
    with pytest.raises(ValueError):
        nk.paged_append(k, v, cache.k, cache.v, table, lens, cos=cos, sin=cos)  # rotates more than head_dim
    with pytest.raises(ValueError):
        nk.paged_append(k, v, cache.k, cache.v, table, lens, cos=cos[:, :8])
    with pytest.raises(ValueError):
        nk.paged_append(k, v[:1], cache.k, cache.v, table, lens)
    with pytest.raises(TypeError):
        nk.paged_append(k.double(), v.double(), cache.k, cache.v, table, lens)
    x, u = torch.zeros((2, 10), device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(ValueError):
        nk.sample_tokens(x, u[:1])
    with pytest.raises(ValueError):
        nk.sample_tokens(x, u, temperature=u.double())
    with pytest.raises(TypeError):
        nk.sample_tokens(x, u, top_k=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError):
        nk.sample_tokens(x.double(), u)


def test_empty_calls():
    cache = Paged(np.random.default_rng(14), [], 2, 64, 16, BF16)
    none = torch.zeros((0, 2, 64), dtype=BF16, device="cuda")
    table, lens = torch.zeros((0, 1), dtype=torch.int32, device="cuda"), ints([])
    nk.paged_append(none, none, cache.k, cache.v, table, lens)
    assert nk.paged_attention(none, cache.k, cache.v, table, lens).shape == (0, 2, 64)
    assert nk.sample_tokens(torch.zeros((0, 9), device="cuda"), torch.zeros(0, device="cuda")).shape == (0,)

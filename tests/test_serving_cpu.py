"""The paged serving ops without a GPU: the NumPy direct call against
independent 64-bit statements, the traced form and its plan, and what the C
entries and the ops refuse."""

import ctypes

import ml_dtypes
import numpy as np
import pytest

from nkipy_b200 import workloads as W
from nkipy_b200.core import tensor_apis as T
from nkipy_b200.core.trace import NKIPyKernel
from nkipy_b200.planner.lower import Lowering
from nkipy_b200.runtime import serving as S
from nkipy_b200.spike import _nkb

BF16 = np.dtype(ml_dtypes.bfloat16)


def step_inputs(seed=0, news=None, lens=(1, 20, 64), hq=4, hkv=2, d=64, hidden=64, vocab=500, page=16, prefix=0):
    rng = np.random.default_rng(seed)
    B = len(lens)
    n = sum(news) if news else B
    w = lambda *s: (rng.standard_normal(s, dtype=np.float32) * 0.1).astype(BF16)  # noqa: E731
    extra = -(-prefix // page)
    width = max(-(-x // page) for x in lens)
    pages = rng.permutation(B * width + extra).astype(np.int32)
    cos, sin = W.rope_tables(prefix + max(lens) + 1, d)
    args = (w(n, hidden), np.ones(hidden, BF16), w(hidden, (hq + 2 * hkv) * d), w(hq * d, hidden), w(hidden, vocab),
            w(len(pages), page, hkv, d), w(len(pages), page, hkv, d), pages[: B * width].reshape(B, width),
            np.array(lens, np.int32), cos, sin, rng.random(B, dtype=np.float32), np.array([1.0, 0.7, 0.0], np.float32)[:B],
            np.array([0, 5, 9], np.int32)[:B], np.array([0.9, 1.0, 0.5], np.float32)[:B],
            np.array([0.0, 0.05, 0.1], np.float32)[:B])
    kwargs = dict(n_heads=hq, n_kv_heads=hkv)
    if news:
        kwargs["q_start"] = np.cumsum([0] + list(news)).astype(np.int32)
        kwargs["last"] = (kwargs["q_start"][1:] - 1).astype(np.int32)
    if prefix:
        kwargs.update(prefix_pages=pages[B * width :], prefix_len=prefix)
    return args, kwargs


def test_direct_call_of_attention():
    """Window and first tokens, ragged chunks, a sequence without new tokens and one that sees nothing."""
    rng = np.random.default_rng(1)
    hq, hkv, d, page = 6, 2, 24, 5
    q = rng.standard_normal((9, hq, d)).astype(np.float32)
    kc, vc = (rng.standard_normal((12, page, hkv, d)).astype(np.float32) for _ in range(2))
    table = rng.permutation(12).reshape(3, 4).astype(np.int32)
    q_start, kv_len = np.array([0, 4, 4, 7], np.int32), np.array([17, 3, 1], np.int32)
    for window, sinks in ((0, 0), (5, 0), (3, 2)):
        got = T.paged_attention(q, kc, vc, table, kv_len, q_start, window=window, sinks=sinks)
        want = np.zeros_like(q, dtype=np.float64)
        for b in range(3):
            for i, t in enumerate(range(q_start[b], q_start[b + 1])):
                p = kv_len[b] - (q_start[b + 1] - q_start[b]) + i
                keys = [j for j in range(p + 1) if not window or j > p - window or j < sinks]
                if not keys:
                    continue
                rows = [(table[b, j // page], j % page) for j in keys]
                for h in range(hq):
                    k = np.array([kc[r][h // 3] for r in rows], np.float64)
                    v = np.array([vc[r][h // 3] for r in rows], np.float64)
                    e = np.exp(k @ q[t, h].astype(np.float64) / np.sqrt(d))
                    want[t, h] = e @ v / e.sum()
        np.testing.assert_allclose(got, want, rtol=0, atol=2e-6)
        assert not got[4:6].any() and not got[7:].any()  # positions -2 and -1, and tokens of no sequence


def test_direct_call_of_prefix_is_one_long_sequence():
    rng = np.random.default_rng(2)
    hq, hkv, d, page, P = 4, 2, 16, 8, 21
    q = rng.standard_normal((2, hq, d)).astype(np.float32)
    kc, vc = (rng.standard_normal((16, page, hkv, d)).astype(np.float32) for _ in range(2))
    prefix, table, kv_len = np.array([9, 3, 12], np.int32), np.array([[1, 2], [4, 5]], np.int32), np.array([1, 11], np.int32)
    got = T.prefix_attention(q, kc, vc, prefix, P, table, kv_len)
    for b in range(2):  # the same rows in one contiguous cache of page size 1
        flat = lambda c: np.concatenate([c[prefix].reshape(-1, hkv, d)[:P], c[table[b]].reshape(-1, hkv, d)])[:, None]  # noqa: E731
        n = P + kv_len[b]
        want = T.paged_attention(q[b : b + 1], flat(kc), flat(vc), np.arange(P + 16)[None], np.array([n]))
        np.testing.assert_allclose(got[b : b + 1], want, rtol=0, atol=1e-6)


def test_direct_call_of_sampling():
    x = np.log(np.array([[0.1, 0.4, 0.2, 0.3]] * 6, np.float32))
    one = np.ones(6, np.float32)
    u = np.array([0.05, 0.15, 0.55, 0.75, 0.0, 0.999], np.float32)
    assert T.sample_tokens(x, u).tolist() == [0, 1, 2, 3, 0, 3]
    assert T.sample_tokens(x, u, top_k=np.full(6, 2, np.int32)).tolist() == [1, 1, 1, 3, 1, 3]
    assert T.sample_tokens(x, u, top_p=one * 0.5).tolist() == [1, 1, 1, 3, 1, 3]
    assert T.sample_tokens(x, u, min_p=one * 0.6).tolist() == [1, 1, 1, 3, 1, 3]
    assert T.sample_tokens(x, u, temperature=one * 0).tolist() == [1] * 6
    assert T.sample_tokens(np.full((1, 4), -np.inf, np.float32), u[:1]).tolist() == [-1]


@pytest.mark.parametrize("news", [None, (3, 1, 20)])
@pytest.mark.parametrize("prefix", [0, 37])
def test_step_traces_to_one_launch_per_op(news, prefix):
    args, kwargs = step_inputs(news=news, prefix=prefix)
    kernel = NKIPyKernel.trace(W.paged_step_kernel)
    kernel.specialize(*args, **kwargs)
    plan = Lowering(kernel._code).run()
    counts = plan.kernel_counts()
    assert counts["paged_append"] == counts["paged_attention"] == counts["sample_tokens"] == 1
    assert {a.param_name for a in kernel._code.aliases} == {"cache_k", "cache_v"}
    # the caches are written in place: the only copies are the no-op ones of mutated parameters
    assert counts["copy_bytes"] == 2 and "ew" not in counts
    # the projection's q, k and v columns are read where they lie
    append = next(s for s in plan.steps if s.kernel == "paged_append")
    assert len({b for b, _ in append.bufs[:3]}) == 1


def test_direct_call_of_the_step_mutates_the_caches():
    args, kwargs = step_inputs()
    before = args[5].copy()
    tokens = W.paged_step_kernel(*args, **kwargs)
    assert tokens.shape == (3,) and tokens.dtype == np.int32 and (tokens >= 0).all()
    changed = np.argwhere((before != args[5]).any((2, 3)))
    want = {(args[7][b, (n - 1) // 16], (n - 1) % 16) for b, n in enumerate(args[8])}
    assert {tuple(c) for c in changed} == want


def test_ops_refuse():
    args, _ = step_inputs()
    kc, vc, table, lens = args[5:9]
    q = np.zeros((3, 4, 64), BF16)
    k = np.zeros((3, 2, 64), BF16)
    for bad in (dict(q=q.astype(np.float32)), dict(q=q[:, :3]), dict(q=q[:2]), dict(kv_len=lens[:2]), dict(window=-1),
                dict(page_table=table[0]), dict(v_cache=vc[:-1]), dict(q_start=np.zeros(3, np.int32))):
        with pytest.raises(ValueError):
            T.paged_attention(**{**dict(q=q, k_cache=kc, v_cache=vc, page_table=table, kv_len=lens), **bad})
    with pytest.raises(ValueError):
        T.prefix_attention(q, kc, vc, np.array([0], np.int32), 17, table, lens)
    for bad in (dict(v=k[:2]), dict(k=k[:, :1]), dict(cos=np.ones((4, 40), np.float32), sin=np.ones((4, 40), np.float32)),
                dict(cos=np.ones((4, 8), np.float32)), dict(q=q[:2])):
        with pytest.raises(ValueError):
            T.paged_append(**{**dict(k=k, v=k, k_cache=kc, v_cache=vc, page_table=table, kv_len=lens), **bad})
    x, u = np.zeros((2, 5), np.float32), np.zeros(2, np.float32)
    for bad in (dict(u=u[:1]), dict(temperature=np.ones(2, np.int32)), dict(top_k=u), dict(logits=x.astype(np.int32))):
        with pytest.raises(ValueError):
            T.sample_tokens(**{**dict(logits=x, u=u), **bad})


def test_traced_ops_refuse():
    args, _ = step_inputs()
    kc, vc, table, lens = args[5:9]
    q = np.zeros((3, 4, 64), BF16)
    k = np.zeros((3, 2, 64), BF16)
    with pytest.raises(TypeError, match="int32"):
        NKIPyKernel.trace(lambda q, kc, vc, t, n: T.paged_attention(q, kc, vc, t, n)).specialize(
            q, kc, vc, table.astype(np.int16), lens)
    with pytest.raises(TypeError, match="in place"):
        NKIPyKernel.trace(lambda k, t, n: T.paged_append(k, k, kc, vc, t, n)).specialize(k, table, lens)


# ---------------------------------------------------------------------------
# the C entries: every refusal is made before a launch
# ---------------------------------------------------------------------------
FIELDS = {
    "append": ("k v q q_out k_cache v_cache page_table kv_len q_start cos sin dtype cache_dtype rope_dtype tokens seqs q_heads "
               "kv_heads head_dim rot_dim rope_rows rope_stride pos_offset k_token k_head v_token v_head q_token q_head "
               "q_out_token q_out_head pages page_size k_page k_slot k_cache_head v_page v_slot v_cache_head table_width "
               "table_stride").split(),
    "attention": ("q out k_cache v_cache page_table kv_len q_start prefix_pages workspace dtype tokens seqs q_heads kv_heads "
                  "head_dim q_token q_head out_token out_head pages page_size k_page k_slot k_cache_head v_page v_slot "
                  "v_cache_head table_width table_stride window sinks prefix_len workspace_bytes scale").split(),
    "sample": "logits u temperature top_k top_p min_p tokens dtype rows vocab row_stride".split(),
}
GOOD = {
    "append": dict(k=16, v=16, k_cache=16, v_cache=16, page_table=16, kv_len=16, dtype=1, cache_dtype=1, tokens=2, seqs=2,
                   kv_heads=1, head_dim=64, k_token=64, k_head=64, v_token=64, v_head=64, pages=4, page_size=16, k_page=1024,
                   k_slot=64, k_cache_head=64, v_page=1024, v_slot=64, v_cache_head=64, table_width=2, table_stride=2),
    "attention": dict(q=16, out=16, k_cache=16, v_cache=16, page_table=16, kv_len=16, dtype=1, tokens=2, seqs=2, q_heads=2,
                      kv_heads=1, head_dim=64, q_token=128, q_head=64, out_token=128, out_head=64, pages=4, page_size=16,
                      k_page=1024, k_slot=64, k_cache_head=64, v_page=1024, v_slot=64, v_cache_head=64, table_width=2,
                      table_stride=2, scale=1.0),
    "sample": dict(logits=16, u=16, tokens=16, dtype=0, rows=1, vocab=10, row_stride=10),
}
STRUCTS = {"append": S._APPEND, "attention": S._ATTENTION, "sample": S._SAMPLE}
ENTRY = {"append": "nkb_paged_append", "attention": "nkb_paged_attention", "sample": "nkb_sample_tokens"}


def packed(kind, **change):
    values = {**dict.fromkeys(FIELDS[kind], 0), **GOOD[kind], **change}
    if kind == "attention":
        values["scale"] = float(values["scale"])
    return STRUCTS[kind].pack(*(values[f] for f in FIELDS[kind]))


@pytest.mark.parametrize("kind,change,status,text", [
    ("append", dict(tokens=-1), 1, "out of range"),
    ("append", dict(dtype=3), 4, "float32, bfloat16 or float16"),
    ("append", dict(cache_dtype=10), 4, "float32, bfloat16 or float16"),
    ("append", dict(rot_dim=7, cos=16, sin=16, rope_rows=4), 1, "rot_dim"),
    ("append", dict(rot_dim=66, cos=16, sin=16, rope_rows=4), 1, "rot_dim"),
    ("append", dict(rot_dim=64), 1, "cos and sin"),
    ("append", dict(q=16), 1, "go together"),
    ("append", dict(q=16, q_out=16), 1, "go together"),
    ("append", dict(k=0), 1, "NULL"),
    ("append", dict(tokens=3), 1, "one token per sequence"),
    ("append", dict(page_size=0), 1, "page_size"),
    ("append", dict(table_stride=1), 1, "overlap"),
    ("append", dict(table_width=1 << 30, table_stride=1 << 30), 1, "2^31"),
    ("attention", dict(q_heads=3, kv_heads=2), 1, "multiple"),
    ("attention", dict(dtype=5), 4, "float32, bfloat16 or float16"),
    ("attention", dict(head_dim=257), 4, "256"),
    ("attention", dict(window=-1), 1, "negative"),
    ("attention", dict(sinks=-1), 1, "negative"),
    ("attention", dict(prefix_len=5, prefix_pages=16, window=3), 4, "window over a shared prefix"),
    ("attention", dict(prefix_len=5, dtype=0), 1, "prefix needs its pages"),
    ("attention", dict(kv_len=0, dtype=0), 1, "NULL"),
    ("attention", dict(tokens=1), 1, "one token per sequence"),
    ("attention", dict(), 1, "workspace of 0 bytes"),
    ("attention", dict(workspace=24, workspace_bytes=1 << 40), 1, "unaligned workspace"),
    ("sample", dict(rows=-1), 1, "out of range"),
    ("sample", dict(vocab=0), 1, "out of range"),
    ("sample", dict(vocab=(1 << 21) + 1, row_stride=1 << 22), 4, "2^21"),
    ("sample", dict(dtype=3), 4, "float32, bfloat16 or float16"),
    ("sample", dict(u=0), 1, "NULL"),
    ("sample", dict(rows=2, row_stride=9), 1, "overlap"),
])
def test_c_entries_refuse(kind, change, status, text):
    lib = _nkb.lib()
    assert getattr(lib, ENTRY[kind])(packed(kind, **change), None) == status
    assert text in lib.nkb_last_error().decode()


def test_c_entries_without_arguments():
    lib = _nkb.lib()
    for entry in ENTRY.values():
        assert getattr(lib, entry)(None, None) == 1
    assert lib.nkb_paged_attention_workspace(None, None) == 1


def test_empty_c_calls_launch_nothing():
    lib = _nkb.lib()
    assert lib.nkb_paged_append(packed("append", tokens=0, seqs=0), None) == 0
    assert lib.nkb_paged_attention(packed("attention", tokens=0, seqs=0), None) == 0
    assert lib.nkb_sample_tokens(packed("sample", rows=0), None) == 0


def test_workspace_depends_on_the_sizes_alone():
    need = ctypes.c_size_t()
    lib = _nkb.lib()
    sizes = {}
    for name, change in (("bf16", {}), ("arrays", dict(q=17, k_cache=0)), ("f32", dict(dtype=0)), ("chunk", dict(q_start=16)),
                         ("prefix", dict(prefix_len=40)), ("empty", dict(tokens=0, seqs=0))):
        assert lib.nkb_paged_attention_workspace(packed("attention", **change), ctypes.byref(need)) == 0
        sizes[name] = need.value
    assert sizes["bf16"] == sizes["arrays"] > 0 and sizes["f32"] == sizes["empty"] == 0
    assert sizes["chunk"] > 0 and sizes["prefix"] > 0


@pytest.mark.parametrize("kernel,ints,floats", [
    ("paged_append", [1] + [0] * 29, []), ("paged_append", [1 << 11] + [0] * 30, []), ("paged_append", [3] + [0] * 30, []),
    ("paged_attention", [1] + [0] * 24, []), ("paged_attention", [-1] + [0] * 24, [1.0]),
    ("sample_tokens", [1] + [0] * 3, []),
])
def test_plan_steps_are_checked(kernel, ints, floats):
    """Malformed steps fail when a plan is loaded (with a GPU) or as an uninitialised runtime (without)."""
    text = "\n".join(["NKBPLAN 1", "name x", "inputs 1", "input 0 64", "outputs 0", "consts 0", "scratch 0", "buffers 1",
                      "buffer 0 in 0", "steps 1",
                      " ".join(["step", kernel, "1", "0", "0", str(len(ints))] + [str(i) for i in ints]
                               + [str(len(floats))] + [str(f) for f in floats]), "end"]) + "\n"
    plan = ctypes.c_void_p()
    status = _nkb.lib().nkb_plan_load(text.encode(), len(text), 0, ctypes.byref(plan))
    assert status in (1, 3, 4, 6)

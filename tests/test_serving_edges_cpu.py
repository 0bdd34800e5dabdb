"""Serving calls at the edges of what they take, as far as that goes without a GPU."""

import numpy as np
import pytest

from nkipy_b200.core import tensor_apis as T
from nkipy_b200.core.trace import NKIPyKernel
from nkipy_b200.planner.lower import Lowering
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


def test_tensors_that_require_a_gradient_are_refused():
    torch = pytest.importorskip("torch")
    from nkipy_b200.runtime import serving

    calls = serving._calls()
    x, u = torch.zeros(2, 3), torch.zeros(2)
    q, cache, table = torch.zeros(2, 2, 8), torch.zeros(1, 16, 2, 8), torch.zeros(2, 1, dtype=torch.int32)
    cos = torch.zeros(4, 4)
    sample = lambda *a: calls.sample_tokens(0, *a, None, None)  # noqa: E731
    attend = lambda q, k, v: calls.attention(0, q, k, v, table, table[:, 0], None, 0, 0, None, None, None, 0)  # noqa: E731
    append = lambda k, v, kc, q, cos: calls.paged_append(0, k, v, kc, kc, table, table[:, 0], None, q, cos, cos, 0, None)  # noqa: E731
    for call, args, names in ((sample, [x, u, u, None, u], ["logits", "u", "temperature", "", "top_p"]),
                              (attend, [q, cache, cache], ["q", "k_cache", "v_cache"]),
                              (append, [q, q, cache, q, cos], ["k", "v", "k_cache", "q", "cos"])):
        for i, name in enumerate(names):
            if not name:
                continue
            given = list(args)
            given[i] = given[i].clone().requires_grad_()
            with pytest.raises(RuntimeError, match=f"^{name}: requires a gradient"):
                call(*given)
            with torch.no_grad(), pytest.raises(ValueError, match="cuda:0"):  # then the device is looked at
                call(*given)


# ---------------------------------------------------------------------------
# the build of the module behind the torch calls
# ---------------------------------------------------------------------------
@pytest.fixture
def torch_build(tmp_path, monkeypatch):
    """The builder with a torch package and an output folder of its own; compiler commands are counted, not run."""
    from nkipy_b200 import build

    package, out = tmp_path / "torch", tmp_path / "_lib"
    (package / "lib").mkdir(parents=True)
    (out / "obj").mkdir(parents=True)
    (package / "lib" / "libc10_cuda.so").touch()
    (package / "version.py").write_text("__version__ = '2.0.0'\ngit_version = 'abc'\n")
    commands = []

    def run(cmd, **kwargs):
        commands.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return build.subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "OUT_DIR", str(out))
    monkeypatch.setattr(build, "OBJ_DIR", str(out / "obj"))
    monkeypatch.setattr(build, "TORCH_LIB", str(out / "nkb_torch.so"))
    monkeypatch.setattr(build.subprocess, "run", run)
    found = type("Spec", (), {"submodule_search_locations": [str(package)]})
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: found)
    return build, package, commands


def test_module_is_built_again_for_another_torch(torch_build):
    build, package, commands = torch_build
    for _ in range(2):
        build._build_torch(False)
    assert len(commands) == 1
    (package / "version.py").write_text("__version__ = '2.1.0'\ngit_version = 'abc'\n")
    for _ in range(2):
        build._build_torch(False)
    assert len(commands) == 2


def test_no_module_for_a_torch_without_cuda(torch_build, capsys):
    build, package, commands = torch_build
    (package / "lib" / "libc10_cuda.so").unlink()
    build._build_torch(False)  # builds nothing and raises nothing
    assert not commands and "no CUDA" in capsys.readouterr().err


def test_module_of_another_torch_is_not_used(monkeypatch):
    pytest.importorskip("torch")
    from nkipy_b200.runtime import serving

    serving._calls()
    serving._calls.cache_clear()
    monkeypatch.setattr("torch.version.git_version", "another")
    with pytest.raises(ImportError, match="was built for torch"):
        serving._calls()
    monkeypatch.undo()
    serving._calls()


# ---------------------------------------------------------------------------
# positions
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kind, change", [
    ("append", dict(page_size=1, table_width=2**31 - 1, table_stride=2**31 - 1)),
    ("attention", dict(page_size=1, table_width=2**31 - 1, table_stride=2**31 - 1)),
    ("attention", dict(page_size=2**31 - 255, table_width=1, table_stride=1)),
    ("append", dict(table_width=1 << 60, table_stride=1 << 60)),  # times the page size it is a multiple of 2^64
    ("attention", dict(prefix_len=2**31 - 255, prefix_pages=16)),
])
def test_positions_that_blocks_of_keys_could_not_count(kind, change):
    entry = {"append": "nkb_paged_append", "attention": "nkb_paged_attention"}[kind]
    assert getattr(_nkb.lib(), entry)(packed(kind, **change), None) == 1
    assert "2^31 - 256 positions" in _nkb.lib().nkb_last_error().decode()


# ---------------------------------------------------------------------------
# appends that read the caches
# ---------------------------------------------------------------------------
def move_rows(kc, vc, table, lens):
    """The first rows of the caches' page 6 become the new tokens' rows, twice (the second time of the changed caches)."""
    T.paged_append(kc[6, :3], vc[6, :3], kc, vc, table, lens)
    T.paged_append(kc[6, 3:6], vc[6, 3:6], kc, vc, table, lens - 1)


def move_inputs():
    rng = np.random.default_rng(6)
    kc, vc = (rng.standard_normal((8, 16, 2, 64)).astype(np.float16) for _ in range(2))
    # page 6 itself is written: a row that is read by the first append, and one that is read by the second
    return kc, vc, np.array([[6, 1], [6, 7], [3, 6]], np.int32), np.array([2, 5, 19], np.int32)


def test_rows_that_move_inside_the_caches():
    """The rows are those of before the append, although some of them are written by it."""
    kc, vc, table, lens = move_inputs()
    want = [c.copy() for c in (kc, vc)]
    for c in want:
        c[6, [1, 4, 2]] = c[6, :3].copy()
        c[6, [0, 3, 1]] = c[6, 3:6].copy()
    move_rows(kc, vc, table, lens)
    assert all((a == b).all() for a, b in zip((kc, vc), want))


def test_rows_that_move_inside_the_caches_are_copied_first():
    kernel = NKIPyKernel.trace(move_rows)
    kernel.specialize(*move_inputs())
    plan = Lowering(kernel._code).run()
    appends = [s for s in plan.steps if s.kernel == "paged_append"]
    assert len(appends) == 2
    same = {0, 1} | {b for s in appends for b, _ in s.bufs[2:4]}  # the caches' buffers, as inputs and as results
    for s in appends:
        assert not {b for b, _ in s.bufs[:2]} & same


def test_one_cache_for_keys_and_values_is_refused():
    kc, _, table, lens = move_inputs()
    k = np.zeros((3, 2, 64), np.float16)
    with pytest.raises(ValueError, match="one tensor"):
        T.paged_append(k, k, kc, kc, table, lens)
    with pytest.raises(ValueError, match="one tensor"):
        NKIPyKernel.trace(lambda k, kc, t, n: T.paged_append(k, k, kc, kc, t, n)).specialize(k, kc, table, lens)


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def test_infinite_logits_at_an_infinite_temperature():
    """Only the infinite logits have a weight, as at any other temperature."""
    x = np.array([[0.0, np.inf, 1.0, np.inf, -np.inf, np.nan]] * 2, np.float32)
    for t in (1.0, 1e30, np.inf):
        assert T.sample_tokens(x, np.array([0.2, 0.7], np.float32), np.full(2, t, np.float32)).tolist() == [1, 3]

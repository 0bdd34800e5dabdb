"""The compiled module behind the serving calls, as far as it goes without a GPU:
it is built with the library, and what is not a tensor of this process's device
is refused by name before anything is launched."""

import pytest

torch = pytest.importorskip("torch")

from nkipy_b200.runtime import serving  # noqa: E402


@pytest.fixture(scope="module")
def calls():
    return serving._calls()


def test_built_beside_the_library(calls):
    from nkipy_b200 import build

    assert calls.__file__ == build.TORCH_LIB


def test_tensors_of_another_device(calls):
    x, u = torch.zeros(2, 3), torch.zeros(2)
    with pytest.raises(ValueError, match="logits.*cuda:0.*cpu"):
        calls.sample_tokens(0, x, u, None, None, None, None, None)
    cache, table = torch.zeros(1, 16, 2, 8), torch.zeros(2, 1, dtype=torch.int32)
    q = torch.zeros(2, 2, 8)
    with pytest.raises(ValueError, match="q: .*cuda:0.*cpu"):
        calls.attention(0, q, cache, cache, table, table[:, 0], None, 0, 0, None, None, None, 0)
    with pytest.raises(ValueError, match="k: .*cuda:0.*cpu"):
        calls.paged_append(0, q, q, cache, cache, table, table[:, 0], None, None, None, None, 0, None)


@pytest.mark.parametrize("value", [3, "x", [1.0]])
def test_what_is_not_a_tensor(calls, value):
    with pytest.raises(TypeError, match="logits: expected a tensor"):
        calls.sample_tokens(0, value, torch.zeros(2), None, None, None, None, None)


def test_what_is_missing(calls):
    with pytest.raises(TypeError, match="logits: expected a tensor, got None"):
        calls.sample_tokens(0, None, None, None, None, None, None, None)
    with pytest.raises(TypeError, match="q: expected a tensor, got None"):
        calls.attention(0, *([None] * 12))
    with pytest.raises(TypeError, match="arguments"):
        calls.attention(0)
    with pytest.raises(TypeError):
        calls.sample_tokens("0", *([None] * 7))

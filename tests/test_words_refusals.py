"""Calls that the training step on words refuses, checked without a GPU: before anything is computed or changed; and what
`quantize_params` takes for a matrix."""
import pytest

pytest.importorskip("torch")

from clusternet_amd import maxout_step as ms  # noqa: E402


def _words():
    return ms.TokenInput.__new__(ms.TokenInput)  # never looked at


def test_step_refuses_words():
    """It would leave the table as it is."""
    with pytest.raises(TypeError, match="token_step"):
        ms.step(_words(), None, [None] * 6, 0.1)


@pytest.mark.parametrize("count", [0, 1, 3])
def test_token_step_refuses_other_than_two_momenta(count):
    """One would leave the second matrix as it is."""
    with pytest.raises(ValueError):
        ms.token_step(_words(), None, [None] * 6, [None] * count, 0.1, 0.1)


@pytest.mark.parametrize("shape", [(6,), (1, 6), (6, 1)])
def test_biases_are_not_quantised(monkeypatch, shape):
    """Biases may be rows or columns of one, as `forward` takes them."""
    import torch
    monkeypatch.setattr(ms.L, "quantize_4bit", lambda t, group, zero_points: ("4 bits", t))
    params = [torch.ones(6, 6), torch.ones(shape), torch.ones(3, 6), torch.ones(shape), torch.ones(3, 6), torch.ones(shape)]
    got = ms.quantize_params(params)
    for i, (g, t) in enumerate(zip(got, params)):
        assert g is t if i % 2 else g[0] == "4 bits" and g[1] is t

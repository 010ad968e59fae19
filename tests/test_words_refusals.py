"""Calls that the training step on words refuses, checked without a GPU: before anything is computed or changed."""
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

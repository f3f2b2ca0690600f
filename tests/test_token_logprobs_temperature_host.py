"""The temperatures that the log probabilities' entry points take (CPU: refused before a launch)."""

import pytest

from testt_amd import _ext

A = 4096       # an aligned address that is never read


@pytest.mark.parametrize("t", [0.0, -1.0, float("nan"), float("inf"), 9e-31, 1e-39, 1.1e30])
def test_temperature_out_of_range(t):
    """Below 1e-30 its reciprocal, or log2(e) times it, is no fp32 number any more: NaN for every row."""
    with pytest.raises(_ext.SoupkError, match="status 1:"):
        _ext.call("soupk_token_logprobs_fwd", A, 0, A, 4, 4, 0, 8, 8, t, 0, A, A, A, A, None, None, None, 0,
                  None)
    with pytest.raises(_ext.SoupkError, match="status 1:"):
        _ext.call("soupk_token_logprobs_bwd", A, 0, A, 4, 4, 0, 8, 8, t, 0, A, A, A, None, A, None, None,
                  A, None)


@pytest.mark.parametrize("t", [1e-30, 1.0, 1e30])
def test_the_ends_are_taken(t):
    _ext.call("soupk_token_logprobs_fwd", None, 0, None, 0, 1, 0, 8, 8, t, 2, *(None,) * 7, 0, None)

"""cached_importance says why there are no scores."""

import warnings

import pytest
import torch

from table_moe.utils import ModalityContext
from table_moe.utils.importance import cached_importance


class Cache:
    def __init__(self, result):
        self.result = result

    def importance(self, q, table, lengths, **kw):
        if isinstance(self.result, Exception):
            raise self.result
        return self.result


@pytest.mark.parametrize("error", [ValueError("q must be float16 or bfloat16"), RuntimeError("not on a device")])
def test_a_refusal_warns(error):
    with pytest.warns(RuntimeWarning, match=str(error)):
        assert cached_importance(Cache(error), None, None, None) is None
    assert ModalityContext.get_attn_weights() is None


def test_scores_do_not_warn():
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        y = cached_importance(Cache(torch.ones(2, 3)), None, None, None)
    assert y.shape == (2, 3) and torch.equal(ModalityContext.get_attn_weights(), torch.ones(6))
    ModalityContext.set_attn_weights(None)


def test_a_warning_that_is_an_error_leaves_no_scores():
    """Where warnings are raised, the scores of the call before are gone all the same."""
    cached_importance(Cache(torch.ones(2, 3)), None, None, None)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(RuntimeWarning):
            cached_importance(Cache(ValueError("no")), None, None, None)
    assert ModalityContext.get_attn_weights() is None

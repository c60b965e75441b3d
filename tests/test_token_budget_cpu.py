"""A budget of tokens: what is left out has a default, what is named is taken or refused."""

import pytest

from qwen3_runtime_b200 import TokenBudget


def test_first_tokens_that_are_named_are_not_lowered():
    """More first tokens than are kept: refused, four as well as three or five; left out they are four, or what there is."""
    for keep in (1, 2, 3):
        assert TokenBudget(keep).first == keep and TokenBudget(keep, first=None).first == keep
        for first in (4, 5):
            with pytest.raises(ValueError, match="cannot keep"):
                TokenBudget(keep, first=first)
    assert TokenBudget(4).first == TokenBudget(4, first=4).first == 4 and TokenBudget(100) == TokenBudget(100, first=4)

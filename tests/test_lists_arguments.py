"""Arguments of the softmax operators over lists that the binding refuses or converts, without a GPU."""

from __future__ import annotations

import pytest
import torch

from silvic_b200 import lists


def test_more_lists_than_a_call_takes_are_refused():
    """A count that its 32 bits would cut."""
    assert lists.lists_arg(torch.empty(2 ** 32 - 1, 0), None).num_lists == 2 ** 32 - 1
    for rows in (2 ** 32, 2 ** 32 + 3):
        with pytest.raises(ValueError, match="lists"):
            lists.lists_arg(torch.empty(rows, 0), None)
        with pytest.raises(ValueError, match="lists"):
            lists.lists_arg(torch.empty(4), torch.empty(rows + 1, dtype=torch.int32, device="meta"))

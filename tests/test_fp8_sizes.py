"""Sizes of the 8-bit float entries and of the balance loss that do not fit into 32 bits, without a GPU."""
import pytest
import torch

from metaltile_b200 import ops


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("call", [
    lambda: ops.moe_balance(torch.ones(0, 8), torch.empty(0, 2 ** 32 + 2, dtype=torch.int32)),               # would be two slots a row
    lambda: ops.moe_balance_grad(torch.ones(4, 8), _i(8), _i(1), 2 ** 32 + 2),
    lambda: ops.moe_balance_grad(torch.ones(4, 8), _i(8), _i(1), 2 - 2 ** 32),
    lambda: ops.moe_balance_grad(torch.ones(4, 8), _i(8), _i(1), -1),
])
def test_a_number_of_slots_that_32_bits_do_not_hold_is_refused(call):
    with pytest.raises(ValueError, match="k must be below"):
        call()

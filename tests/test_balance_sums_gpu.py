"""The sums over rows of moe_balance are 64-bit ones from the warps on."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e,warps", [(1024, 16), (1023, 16), (512, 16), (256, 32)])
def test_sums_over_many_warps_round_once(e, warps):
    """A row whose n experts have equal logits, the others minus infinity, has the probability 1/n rounded to f32 exactly; with one row for each warp of the grid nothing is
    added in 32 bits, so that a mean is the sum of these f32 numbers rounded once: the 64-bit sums err by 2^-53 a row, which turns a rounding in some 2^-17 of all cases."""
    from metaltile_b200 import ops
    rows = torch.cuda.get_device_properties(0).multi_processor_count * warps
    gen = torch.Generator(device="cuda").manual_seed(e)
    n = torch.randint(1, e + 1, (rows, 1), device="cuda", generator=gen)
    on = torch.rand(rows, e, device="cuda", generator=gen).argsort(dim=1) < n
    logits = torch.where(on, 0.0, -float("inf"))
    idx = torch.zeros(rows, 1, device="cuda", dtype=torch.int32)
    _, _, mean, counted = ops.moe_balance(logits, idx)
    p = torch.where(on, (1.0 / n.double()).float().double(), 0.0)
    want = (p.sum(dim=0) / rows).float()
    assert int(counted) == rows and torch.equal(mean, want), int((mean != want).sum())

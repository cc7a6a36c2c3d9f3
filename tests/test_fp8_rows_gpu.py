"""fp8_quantize on rows of every length that it takes."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pow2", [False, True])
def test_a_row_of_more_blocks_than_one_launch_takes(pow2):
    """65535 CTAs of 32 blocks side by side are a launch: here one block more than that, and a ragged one."""
    from metaltile_b200 import ops
    blocks = 65535 * 32
    gen = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(1, 128 * 4369, device="cuda", generator=gen).bfloat16()       # 65535 * 32 = 480 * 4369
    want, s = ref.quantize(base, 1, pow2)
    tail = base[:, 999:999 + 128 + 40]
    x = torch.cat([base.repeat(1, 480), tail], dim=1)
    assert ref.blocks(x.shape[1]) == blocks + 2
    codes, scales = ops.fp8_quantize(x, pow2=pow2)
    assert torch.equal(codes[:, :base.shape[1]].double(), want) and torch.equal(scales[:, :s.shape[1]].double(), s)
    body = codes[0, :128 * blocks].view(torch.uint8).reshape(480, -1)
    assert bool((body[1:] == body[:1]).all()) and bool((scales[0, :blocks].reshape(480, -1) == scales[0, :4369]).all())
    last, ls = ref.quantize(tail, 1, pow2)
    assert torch.equal(codes[:, 128 * blocks:].double(), last) and torch.equal(scales[:, blocks:].double(), ls)

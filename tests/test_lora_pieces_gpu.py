"""What the pieces that adapters' operands are cut into hold, where it is hardest to hold: ranks of very different size, values next to the borders of the pieces, infinities."""
import pytest
import torch

import lora_ref as ref
from test_lora_gpu import TYPES, Case, _close

pytestmark = pytest.mark.gpu

# Every kernel: warp-level with each block of ranks, in one block and several, tiles of 16 and 32 rows, values one by one on a side and on both; tiles of 128 rows back alone (1200 rows of
# 520 + 264) and both ways; CUDA cores
KERNELS = [(40, 256, 128, 8, 2), (64, 256, 136, 16, 2), (33, 512, 256, 32, 2), (60, 256, 264, 64, 1), (65, 256, 256, 72, 2), (1300, 264, 2056, 16, 2), (70, 1001, 515, 16, 2), (90, 2049, 415, 24, 4),
           (36, 691, 384, 64, 4), (40, 384, 691, 40, 2), (2400, 1032, 1040, 16, 2), (2400, 2048, 128, 32, 3), (1200, 520, 264, 64, 1), (20, 255, 127, 5, 2)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", KERNELS)
def test_ranks_of_different_size(size, dt):
    """a's ranks differ by up to 2^16 and b undoes it: the least of h count as much as the largest."""
    c = Case(*size, dt, seed=12)
    s = 2.0 ** torch.linspace(-8, 8, size[3], device="cuda").round()
    c.a, c.b = (c.a.float() / s[:, None]).to(TYPES[dt]), (c.b.float() * s).to(TYPES[dt])
    c.check()


@pytest.mark.parametrize("k,n", [(64, 264), (61, 131)])
def test_f16_gradients_of_values_below_a_step_of_eight_bits(k, n):
    """A row an adapter, so that db is one product: what eight bits leave of either factor is nearly a step, and so is the product of these rests."""
    rows, rank = 64, 16
    c = Case(rows, k, n, rank, rows, "f16", ids=list(range(rows)), seed=13, base=False)
    g = torch.Generator(device="cuda").manual_seed(14)
    h = 1 + 2.0 ** -7 - torch.rand(rows, rank, device="cuda", generator=g) * 2.0 ** -9
    c.dy = ((1 + 2.0 ** -7 - 2.0 ** -10) * 2.0 ** torch.randint(-3, 4, (rows, n), device="cuda", generator=g)).half()
    _, _, db = c.grad(h)
    want = c.scales.double()[:, None, None] * c.dy.double()[:, :, None] * h.double()[:, None, :]
    # rounded once; two pieces of h; the sums of the pieces' four products and the scale
    _close(db, want, (ref.STEP[torch.float16] + 2.0 ** -16 + 8 * ref.F32) * want)

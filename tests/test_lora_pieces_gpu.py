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

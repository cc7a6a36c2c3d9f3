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


# One step of 8 bits, with rests that are as large as they can be: what is left out of the products of their pieces is too.
BELOW = (1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -17, 1 + 3 * 2.0 ** -8 - 2.0 ** -17, 1 + 2.0 ** -8 - 2.0 ** -23)


@pytest.mark.parametrize("size", [s for s in KERNELS if s[0] < 100])
def test_f32_products_of_values_below_a_step_of_eight_bits(size):
    """One product a value of h: the pairs of small pieces that are left out are below 2^-24 of it, the rounding and what a tensor core cuts off of the small products 2^-24 together each."""
    rows, k, n, rank, adapters = size
    c = Case(*size, "f32", ids=[i % adapters for i in range(rows)], seed=15, base=False, scales=False)
    v = torch.tensor(BELOW, device="cuda", dtype=torch.float64)
    c.x.zero_()
    at = torch.arange(rows, device="cuda") * 7 % k
    c.x[torch.arange(rows, device="cuda"), at] = v[torch.arange(rows, device="cuda") % 4].float()
    c.a = v[(torch.arange(adapters * rank * k, device="cuda") // 3) % 4].float().view(adapters, rank, k)
    _, h = c.forward()
    want = ref.low(c.x, c.a, c.ids)
    _close(h, want, 1.5 * 2.0 ** -23 * want)


@pytest.mark.parametrize("size", [(300, 4096, 4096, 16, 2), (300, 4096, 4100, 64, 1), (300, 4095, 4100, 24, 1), (40, 4096, 4096, 8, 1), (200, 4096, 4096, 80, 1), (1300, 4096, 4096, 32, 2)])
def test_f32_sums_keep_what_three_pieces_hold(size):
    """Each value of a sum of thousands is a product of 24 bits.  Some fifty additions of partial sums stand behind a result, each off by a step of 2^-23 at most: 2^-20.2 of a result's root mean
    square, and once more where it goes through both products.  Two pieces in place of three would be 2^-17.8 (test_a_lost_piece_shows)."""
    c = Case(*size, "f32", seed=16, base=False)
    out, h = c.forward()
    got = (h, out, *c.grad(h))
    want_out, want_h = ref.lora(c.x, c.a, c.b, c.ids, c.scales, None)
    for one, want in zip(got, (want_h, want_out, *ref.lora_grad(c.dy, c.x, c.a, c.b, c.ids, c.scales, None))):
        assert (one.double() - want).square().mean().sqrt() <= 2.0 ** -19 * want.square().mean().sqrt()

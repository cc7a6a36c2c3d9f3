"""An infinity in x or dy: what it gives is what the formulas say, in every type and for every rank."""
import pytest
import torch

import lora_ref as ref
from test_lora_gpu import TYPES, Case
from test_lora_pieces_gpu import KERNELS

pytestmark = pytest.mark.gpu


def _same(got, want):
    """Infinities and NaN where the formula has them, and infinities of its sign."""
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)].double(), want[torch.isinf(want)])


# ranks that fill their block and ranks that do not (24 of 32, 4 and 6 of 8, 40 and 56 of 64)
RANKS = [(40, 256, 128, 4, 2), (40, 256, 128, 6, 2), (33, 512, 256, 24, 2), (60, 256, 264, 56, 1), (65, 256, 256, 200, 2), (90, 2049, 415, 40, 4), (40, 384, 691, 12, 2), (1200, 520, 264, 40, 1),
         (2400, 2048, 128, 24, 3), (2400, 1032, 1040, 8, 2)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", KERNELS + RANKS)
def test_infinities_of_a_row_are_those_of_the_formula(size, dt):
    rows, k, n, rank, adapters = size
    c = Case(*size, dt, ids=[i % (adapters + 1) for i in range(rows)], seed=17)
    inf = float("inf")
    # weights whose products are of one sign, so that sums of infinities stay infinities; a number of one bit among them, and of 24
    c.a, c.b = c.a.abs() + 2.0 ** -6, c.b.abs() + 2.0 ** -6
    c.a[:, :, 3], c.b[:, 2, :] = 1.0, 0.5
    c.a[:, ::2, 5], c.b[:, 4, ::3] = 0.0, 0.0                        # infinity times zero is no number
    row = torch.arange(0, rows, 3, device="cuda")
    at = torch.arange(len(row), device="cuda")
    c.x[row, at % 7], c.dy[row, at % 5] = inf, -inf
    c.x[row[1::4], (at % 7)[1::4]] = -inf
    c.dy[row[::5], (at % 5)[::5]] = inf
    out, h = c.forward()
    want, want_h = ref.lora(c.x, c.a, c.b, c.ids, c.scales, c.base)
    assert torch.isinf(want).any() and torch.isnan(want).any()
    _same(h, want_h)
    _same(out, want)
    dx, da, db = c.grad(h)
    want, want_a, want_b = ref.lora_grad(c.dy, c.x, c.a, c.b, c.ids, c.scales, c.dbase)
    assert torch.isinf(want).any() and torch.isnan(want).any()
    _same(dx, want)
    for got, one in ((da, want_a), (db, want_b)):                    # no infinity is lost, and none comes from rows of others
        assert torch.equal(torch.isfinite(got), torch.isfinite(one))


@pytest.mark.parametrize("size", KERNELS[:4] + [KERNELS[6]])
def test_f32_values_that_no_16_bit_number_reaches(size):
    """The largest of f32 lies half a step above the largest of bf16."""
    rows, k, n, rank, adapters = size
    c = Case(*size, "f32", ids=[i % adapters for i in range(rows)], seed=18, scales=False, base=False)
    c.x.zero_()
    c.x[torch.arange(rows), torch.arange(rows) % k] = torch.finfo(torch.float32).max
    c.a.fill_(0.5)
    out, h = c.forward()
    want = torch.finfo(torch.float32).max / 2
    assert torch.isfinite(h).all() and ((h.double() - want).abs() <= 1.5 * 2.0 ** -23 * want).all()
    assert torch.isfinite(out).any()

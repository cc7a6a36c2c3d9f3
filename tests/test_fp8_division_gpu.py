"""The quotients behind scales and codes of f32 rows, against divisions in 64 bits (which decide every f32 rounding here: two f32 numbers whose quotient is not on the border
between two f32 numbers, or two codes, are at least 2^-49 of it away)."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu
CHUNK = 1 << 20


@pytest.mark.parametrize("exponent", [0, -60, -82, 100])
def test_scales_of_every_mantissa(exponent):
    """-82: on both sides of the least scale, 2^-90, which 2^-81.2 has as a maximum."""
    from metaltile_b200 import ops
    for start in range(0, 1 << 23, CHUNK):
        bits = torch.arange(start, start + CHUNK, device="cuda", dtype=torch.int32) | ((127 + exponent) << 23)
        amax = bits.view(torch.float32)
        for sign in (1.0, -1.0):
            _, scales = ops.fp8_quantize((amax * sign)[:, None])
            want = (amax.double() / 448).float().clamp_min(2.0 ** -90)
            assert torch.equal(scales[:, 0], want), int((scales[:, 0] != want).sum())


def test_codes_next_to_every_kind_of_border_at_every_mantissa():
    """For each maximum seven values that are the border between two codes times the held scale, rounded to f32 or the next f32 on either side."""
    from metaltile_b200 import ops
    t = ref.table().to("cuda")
    borders = (t[1:] + t[:-1]) / 2
    borders = torch.cat([borders, borders[:-1].flip(0), t[100:126]])
    for i, start in enumerate(range(0, 1 << 23, CHUNK)):
        amax = (torch.arange(start, start + CHUNK, device="cuda", dtype=torch.int32) | (127 << 23)).view(torch.float32)
        scale = (amax.double() / 448).float()
        gen = torch.Generator(device="cuda").manual_seed(i)
        pick = torch.randint(0, borders.numel(), (CHUNK, 7), device="cuda", generator=gen)
        v = (scale.double()[:, None] * borders[pick]).float()
        v = (v.view(torch.int32) + torch.randint(-1, 2, v.shape, device="cuda", generator=gen, dtype=torch.int32)).view(torch.float32)
        x = torch.cat([amax[:, None], torch.minimum(v, amax[:, None])], dim=1)
        x[:, 1::2] *= -1
        codes, scales = ops.fp8_quantize(x)
        assert torch.equal(scales[:, 0], scale)
        want = ref.nearest(x.double() / scale.double()[:, None])
        bad = codes.double() != want
        assert not bad.any(), (int(bad.sum()), x[bad][:4], codes.double()[bad][:4], want[bad][:4])

"""The codes of add_rms_norm_fp8 against definitions that share no code with it: the quantizer's in 64 bits on its own f32 rows, and the whole formula in 64 bits."""
import pytest
import torch

import fp8_ref
import lora_ref as ref

pytestmark = pytest.mark.gpu
SIZES = [(1, 1), (3, 7), (5, 129), (130, 264), (333, 2880), (2, 4095), (600, 4096), (149, 8200), (3, 16392), (2, 40003)]


def _inputs(rows, k, dt):
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + k)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return (make(rows, k) * (1 + make(k).abs() ** 3)).to(dt), (1 + 0.3 * make(k)).to(dt)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("rows,k", SIZES)
def test_codes_of_f32_rows_are_those_of_the_definition(rows, k, pow2):
    from metaltile_b200 import ops
    x, w = _inputs(rows, k, torch.float32)
    y = torch.empty_like(x)                                          # f32: what the codes are made from
    codes, scales, _ = ops.add_rms_norm_fp8(x, w, 1e-5, pow2=pow2, out=y)
    want, want_scales = fp8_ref.quantize(y, pow2=pow2)
    assert torch.equal(scales.double(), want_scales) and torch.equal(codes.double(), want)


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k", SIZES)
def test_codes_of_the_whole_formula_but_next_to_a_border(rows, k, dt, pow2):
    from metaltile_b200 import ops
    x, w = _inputs(rows, k, dt)
    codes, scales, _ = ops.add_rms_norm_fp8(x, w, 1e-5, pow2=pow2)
    y = ref.norm(x, w, 1e-5)
    off = (ref.ROW / 2 + 6) * ref.F32                                # of y in f32, as norm_bound has it
    # the scale is that of y within `off`, held in f32 (a power of two: the next one of a value within it)
    least, most = fp8_ref.quantize((y * (1 - off)).double(), pow2=pow2)[1], fp8_ref.quantize((y * (1 + off)).double(), pow2=pow2)[1]
    s = scales.double()
    assert (s >= least * (1 - 2.0 ** -24)).all() and (s <= most * (1 + 2.0 ** -24)).all()
    q = y / fp8_ref.spread(s, rows, k, 1)
    lo, hi = fp8_ref.nearest(q * (1 - off)), fp8_ref.nearest(q * (1 + off))
    got = codes.double()
    assert (got >= torch.minimum(lo, hi)).all() and (got <= torch.maximum(lo, hi)).all()
    assert (lo != hi).double().mean() < 2e-3                         # and few lie so near to one

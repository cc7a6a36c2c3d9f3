"""The 8-bit float entries and the balance loss on tensors whose offsets pass 32 bits: a few rows over and over, whose results have to be those of the first time."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _repeats(t, rows):
    """Every `rows` rows hold the same."""
    v = t.reshape(-1, rows, t.shape[-1])
    return bool((v[1:] == v[:1]).all())


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize(block_rows):
    from metaltile_b200 import ops
    base = torch.randn(128, 60000, device="cuda", generator=_gen(1)).bfloat16()
    x = base.repeat(282, 1)
    assert x.numel() > 2 ** 31
    codes, scales = ops.fp8_quantize(x, block_rows=block_rows)
    want, s = ref.quantize(base, block_rows)
    assert torch.equal(codes[:128].double(), want) and _repeats(codes.view(torch.uint8), 128)
    assert torch.equal(scales[:s.shape[0]].double(), s) and _repeats(scales, s.shape[0])


@pytest.mark.parametrize("kernel", [2, 3])
def test_mm(kernel):
    from metaltile_b200 import ops
    k, n = 160, 56000
    base, bs = (torch.randn(250, k, device="cuda", generator=_gen(1)) * 100).clamp(-448, 448).to(F8), torch.rand(250, 2, device="cuda", generator=_gen(2)) + 0.5
    w, ws = (torch.randn(n, k, device="cuda", generator=_gen(3)) * 100).clamp(-448, 448).to(F8), torch.rand(ref.blocks(n), 2, device="cuda", generator=_gen(4)) + 0.5
    x, xs = base.view(torch.uint8).repeat(160, 1).view(F8), bs.repeat(160, 1)
    ops.context(0).set_option("fp8_kernel", kernel)
    try:
        out = ops.fp8_mm(x, w, ws, xs)
    finally:
        ops.context(0).set_option("fp8_kernel", 0)
    assert out.numel() > 2 ** 31 and _repeats(out, 250)
    ref.mm_close(out[:250], base, bs, w, ws)


@pytest.mark.parametrize("kernel", [2, 3])
def test_gather(kernel):
    from metaltile_b200 import ops
    e, n, k = 72, 8192, 4096
    base, bs = (torch.randn(8, n, k, device="cuda", generator=_gen(1)) * 100).clamp(-448, 448).to(F8), torch.rand(8, n // 128, k // 128, device="cuda", generator=_gen(2)) + 0.5
    w, ws = base.view(torch.uint8).repeat(9, 1, 1).view(F8), bs.repeat(9, 1, 1)
    assert w.numel() > 2 ** 31
    x = (torch.randn(24, k, device="cuda", generator=_gen(3)) * 100).clamp(-448, 448).to(F8)
    xs = torch.rand(24, k // 128, device="cuda", generator=_gen(4)) + 0.5
    off = torch.arange(0, 3 * e + 1, 3, device="cuda", dtype=torch.int32)
    ops.context(0).set_option("fp8_kernel", kernel)
    try:
        out = ops.fp8_gather_mm(x.view(torch.uint8).repeat(9, 1).view(F8), w, ws, off, xs.repeat(9, 1))
    finally:
        ops.context(0).set_option("fp8_kernel", 0)
    assert _repeats(out, 24)
    for i in (0, 7):
        ref.mm_close(out[3 * i:3 * i + 3], x[3 * i:3 * i + 3], xs[3 * i:3 * i + 3], base[i], bs[i])
    assert ops.context(0).status_word() == 0


def test_balance():
    from metaltile_b200 import ops
    e, k, rows, times = 1024, 2, 1000, 2200
    base = torch.randn(rows, e, device="cuda", generator=_gen(1)).bfloat16()
    idx = torch.topk(base.float(), k).indices.int()
    z = base.repeat(times, 1)
    assert z.numel() > 2 ** 31
    loss, counts, mean, n = ops.moe_balance(z, idx.repeat(times, 1))
    want_loss, want_counts, want_mean, _ = ref.balance(base, idx, 1.0, None)
    assert int(n) == rows * times and torch.equal(counts.long(), want_counts * times)
    each = (64 + 8 + e // 32 + 5) * 2.0 ** -24                        # of a probability, and 34 additions and roundings of a mean
    sums = each + 34 * 2.0 ** -24
    assert ((mean.double() - want_mean).abs() <= sums * want_mean).all() and abs(float(loss) - float(want_loss)) <= (sums + 2.0 ** -23) * float(want_loss)
    grad = ops.moe_balance_grad(z, counts, n, k)
    assert _repeats(grad, rows)
    want = ref.balance_grad(base, idx, 1.0, 1.0, None) / times
    p, f = ref.softmax(base), want_counts.double() / (rows * k)
    size = e / (rows * times) * p * (f + (p @ f)[:, None])
    assert ((grad[:rows].double() - want).abs() <= ref.STEP[torch.bfloat16] * want.abs() + 2 * each * size + ref.TINY[torch.bfloat16]).all()

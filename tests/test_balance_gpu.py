"""moe_balance and moe_balance_grad against their definitions in 64 bits."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(rows, e, k, dt, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(rows, e, device="cuda", generator=g) + spread * torch.randn(e, device="cuda", generator=g)
    return z.to(TYPES[dt]), torch.topk(z, k, dim=1).indices.to(torch.int32)


def _check(z, idx, coef, mask, grad_loss):
    from metaltile_b200 import ops
    rows, e = z.shape
    loss, counts, mean, n = ops.moe_balance(z, idx, coef=coef, mask=mask)
    grad = ops.moe_balance_grad(z, counts, n, idx.shape[1], grad_loss=grad_loss, coef=coef, mask=mask)
    want_loss, want_counts, want_mean, want_n = ref.balance(z, idx, coef, mask)
    assert int(n) == want_n and torch.equal(counts.long(), want_counts)
    # A probability: the difference to the largest logit (|z| <= 64 here) rounds by 2^-24 of itself, which exp turns into a relative error of 64 * 2^-24; exp and the quotient
    # err by 4 steps, the sum of the row by one for each expert of a lane and each of the five exchanges; all within `each` of the probability.
    # A mean adds up to 32 f32 additions in a warp, the rounding of a CTA's part and that of the result.
    each = (64 + 8 + e // 32 + 5) * 2.0 ** -24
    sums = each + (min(rows, 32) + 2) * 2.0 ** -24
    assert ((mean.double() - want_mean).abs() <= sums * want_mean).all()
    assert abs(float(loss) - float(want_loss)) <= (sums + 2.0 ** -23) * float(want_loss)
    g = float(grad_loss) if grad_loss is not None else 1.0
    want = ref.balance_grad(z, idx, coef, g, mask)
    # p (f - sum f p): the sum errs by `each` and an addition for each expert of a lane; both are multiplied by three more rounded factors
    keep = torch.ones(rows, dtype=torch.bool, device="cuda") if mask is None else mask.bool()
    p = torch.where(keep[:, None], ref.softmax(torch.where(keep[:, None], z, torch.zeros_like(z))), 0.0)
    f = want_counts.double() / max(want_n * idx.shape[1], 1)
    size = abs(g) * coef * e / max(want_n, 1) * p * (f + (p @ f)[:, None])
    tol = ref.STEP[z.dtype] * want.abs() + 2 * each * size + ref.TINY[z.dtype]
    assert grad.dtype == z.dtype and ((grad.double() - want).abs() <= tol).all(), float(((grad.double() - want).abs() / tol).max())
    assert torch.equal(grad[~keep], torch.zeros_like(grad[~keep]))
    again = ops.moe_balance(z, idx, coef=coef, mask=mask)
    assert torch.equal(again[0], loss) and torch.equal(again[2], mean)                # the same call, the same bits
    assert ops.context(0).status_word() == 0


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,e,k", [(1, 1, 1), (1, 8, 2), (3, 7, 7), (5, 32, 4), (64, 33, 8), (9, 60, 6), (130, 64, 8), (33, 65, 1), (77, 68, 4), (200, 100, 8), (257, 128, 8),
                                      (1, 128, 8), (31, 132, 3), (300, 160, 6), (41, 256, 8), (1000, 256, 8), (17, 257, 2), (19, 260, 32), (8, 1023, 32), (12, 1024, 32),
                                      (5000, 128, 8), (256, 64, 2), (257, 64, 2), (200000, 8, 2), (160001, 33, 1)])
def test_balance(rows, e, k, dt):
    _check(*_case(rows, e, k, dt, rows + e), 0.01, None, torch.tensor(1.7, device="cuda"))


@pytest.mark.parametrize("e", [8, 60, 128, 256])
@pytest.mark.parametrize("dt", TYPES)
def test_masked_rows_hold_anything(e, dt):
    z, idx = _case(700, e, 4, dt, e)
    at = torch.arange(700, device="cuda")
    mask = at % 100 < 37
    z[~mask] = float("nan")
    idx[~mask] = -1
    _check(z, idx, 1.0, mask, None)
    _check(z, idx, 1.0, mask.to(torch.uint8) * 255, torch.tensor([0.25], device="cuda"))


def test_no_rows_and_no_counted_rows_give_zeros():
    from metaltile_b200 import ops
    z, idx = _case(40, 16, 2, "bf16")
    for zz, ii, mask in ((z, idx, torch.zeros(40, dtype=torch.bool, device="cuda")), (z[:0], idx[:0], None)):
        loss, counts, mean, n = ops.moe_balance(zz, ii, mask=mask)
        assert float(loss) == 0 and int(n) == 0 and not counts.any() and not mean.any()
        grad = ops.moe_balance_grad(zz, counts, n, 2, mask=mask)
        assert grad.shape == zz.shape and not grad.any()


@pytest.mark.parametrize("dt", TYPES)
def test_experts_that_are_switched_off(dt):
    """Logits of minus infinity and of the type's lowest value, and rows that have nothing else."""
    low = torch.finfo(TYPES[dt]).min
    z, idx = _case(50, 64, 4, dt)
    z[:, 5:20] = -float("inf")
    z[::2, 20:30] = low
    z[7] = -float("inf")
    _check(z, idx, 0.5, None, None)
    z[9] = low                                       # equal lowest values are equal probabilities
    _check(z, idx, 0.5, None, None)


def test_uniform_routing_costs_coef_and_one_expert_costs_all():
    from metaltile_b200 import ops
    z, idx = torch.zeros(64, 8, device="cuda"), torch.arange(128, device="cuda", dtype=torch.int32).reshape(64, 2) % 8
    assert abs(float(ops.moe_balance(z, idx, coef=0.3)[0]) - 0.3) < 1e-7
    z[:, 3] = 50.0
    assert abs(float(ops.moe_balance(z, idx * 0 + 3, coef=0.3)[0]) - 0.3 * 8) < 1e-6


def test_the_same_expert_twice_counts_twice_and_one_outside_is_reported():
    from metaltile_b200 import ops
    ctx = ops.context(0)
    z, _ = _case(4, 8, 2, "f32")
    idx = torch.tensor([[1, 1], [1, 2], [7, 0], [3, 3]], device="cuda", dtype=torch.int32)
    assert ops.moe_balance(z, idx)[1].tolist() == [1, 3, 1, 2, 0, 0, 0, 1]
    idx[2, 1] = 8
    try:
        assert ops.moe_balance(z, idx)[1].tolist() == [0, 3, 1, 2, 0, 0, 0, 1] and ctx.status_word() == 0x907
    finally:
        ctx.status_clear()


@pytest.mark.parametrize("shift", [1, 2])
def test_logits_that_start_anywhere(shift):
    from metaltile_b200 import ops
    z, idx = _case(90, 128, 8, "bf16")
    held = torch.empty(z.numel() + 8, device="cuda", dtype=z.dtype)
    view = held[shift:shift + z.numel()].reshape(z.shape)
    view.copy_(z)
    _check(view, idx, 0.1, None, None)
    counts, n = ops.moe_balance(z, idx)[1::2]
    out = held[shift:shift + z.numel()].reshape(z.shape)
    assert ops.moe_balance_grad(z, counts, n, 8, out=out) is out


def test_a_captured_step_replays_with_new_inputs():
    from metaltile_b200 import ops
    cases = [_case(600, 128, 8, "bf16", i) for i in range(3)]
    want = []
    for z, idx in cases:
        loss, counts, mean, n = ops.moe_balance(z, idx)
        want.append((loss, counts, mean, ops.moe_balance_grad(z, counts, n, 8)))
    z, idx = (t.clone() for t in cases[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, counts, mean, n = ops.moe_balance(z, idx)
        grad = ops.moe_balance_grad(z, counts, n, 8)
    for (zz, ii), w in zip(cases, want):
        z.copy_(zz), idx.copy_(ii)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((loss, counts, mean, grad), w))


def test_refusals_of_sizes():
    from metaltile_b200 import MetalTileError, ops
    for e, k in ((1025, 8), (64, 33), (4, 5), (4, 0)):
        with pytest.raises(MetalTileError):
            ops.moe_balance(torch.zeros(3, e, device="cuda"), torch.zeros(3, k, device="cuda", dtype=torch.int32))
    with pytest.raises(MetalTileError, match="2\\^31"):               # counts are 32 bits
        ops.context(0).moe_balance(0, 0, None, 1.0, 0, 0, 0, 0, 2 ** 26, 64, 32, torch.float32)


def test_a_context_of_another_device_is_refused():
    from types import SimpleNamespace
    from metaltile_b200 import ops
    other = SimpleNamespace(device=1, _h=None)
    logits, idx = torch.zeros(3, 8, device="cuda"), torch.zeros(3, 2, device="cuda", dtype=torch.int32)
    _, counts, _, counted = ops.moe_balance(logits, idx)
    x = torch.zeros(4, 128, device="cuda")
    w, ws = ops.fp8_quantize(x, block_rows=128)
    xq, xs = ops.fp8_quantize(x)
    off = torch.tensor([0, 4], device="cuda", dtype=torch.int32)
    for call in (lambda: ops.moe_balance(logits, idx, ctx=other), lambda: ops.moe_balance_grad(logits, counts, counted, 2, ctx=other),
                 lambda: ops.fp8_quantize(x, ctx=other), lambda: ops.fp8_mm(x, w, ws, ctx=other), lambda: ops.fp8_gather_mm(xq, w[None], ws[None], off, xs, ctx=other)):
        with pytest.raises(ValueError, match="another device"):
            call()

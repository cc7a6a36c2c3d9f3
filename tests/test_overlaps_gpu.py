"""Results of norms and adapters over operands: whole and in place where the documentation has it, refused elsewhere, a shifted view of the same memory like the memory itself."""
import pytest
import torch

from test_lora_gpu import Case

pytestmark = pytest.mark.gpu


def _two(rows, width, dt, shift):
    """Two matrices in one piece of memory, the second `shift` values behind the first."""
    both = torch.randn(rows * width + shift, device="cuda").to(dt)
    return both, both[:rows * width].view(rows, width), both[shift:].view(rows, width)


@pytest.mark.parametrize("shift", [1, 8, 256, 9 * 256])
def test_adapters_refuse_results_that_lie_over_operands(shift):
    from metaltile_b200 import MetalTileError
    c = Case(10, 256, 256, 16, 2, "bf16")
    _, h = c.forward()
    for name in ("x", "base"):
        both, first, second = _two(10, 256, torch.bfloat16, shift)
        kept = both.clone()
        for one, out in ((first, second), (second, first)):
            held = getattr(c, name)
            setattr(c, name, one)
            with pytest.raises(MetalTileError, match="lie over"):
                c.forward(out=out)
            setattr(c, name, held)
        assert torch.equal(both, kept)
    for name in ("dy", "x", "dbase"):
        both, first, second = _two(10, 256, torch.bfloat16, shift)
        kept = both.clone()
        for one, out in ((first, second), (second, first)):
            held = getattr(c, name)
            setattr(c, name, one)
            with pytest.raises(MetalTileError, match="lie over"):
                c.grad(h, out=out)
            setattr(c, name, held)
        assert torch.equal(both, kept)
    weights = torch.randn(2 * 16 * 256 + 10 * 256, device="cuda").bfloat16()
    c.a = weights[:2 * 16 * 256].view(2, 16, 256)
    with pytest.raises(MetalTileError, match="lie over"):
        c.forward(out=weights[2 * 16 * 256 - shift:][:10 * 256].view(10, 256))
    want = c.forward()[0]
    assert torch.equal(c.forward(out=weights[2 * 16 * 256:].view(10, 256))[0], want)         # side by side


@pytest.mark.parametrize("shift", [1, 8, 256, 9 * 256])
def test_norms_refuse_results_that_lie_over_operands(shift):
    from metaltile_b200 import MetalTileError, ops
    w, other, free = torch.ones(256, device="cuda"), torch.randn(10, 256, device="cuda"), torch.empty(10, 256, device="cuda")
    both, first, second = _two(10, 256, torch.float32, shift)
    kept = both.clone()
    for one, out in ((first, second), (second, first)):
        for call in (lambda: ops.add_rms_norm(one, w, 1e-5, out=out), lambda: ops.add_rms_norm(one, w, 1e-5, residual=other, sum_out=out),
                     lambda: ops.add_rms_norm(other, w, 1e-5, residual=one, out=out), lambda: ops.add_rms_norm(other, w, 1e-5, residual=free, sum_out=one, out=out),
                     lambda: ops.add_rms_norm_fp8(one, w, 1e-5, out=out), lambda: ops.add_rms_norm_fp8(one, w, 1e-5, residual=other, sum_out=out),
                     lambda: ops.add_rms_norm_grad(one, other, w, 1e-5, out=out), lambda: ops.add_rms_norm_grad(other, one, w, 1e-5, out=out),
                     lambda: ops.add_rms_norm_grad(other, free, w, 1e-5, dsum=one, out=out)):
            with pytest.raises(MetalTileError, match="lie over"):
                call()
    assert torch.equal(both, kept)
    row = torch.randn(1, 256, device="cuda")
    with pytest.raises(MetalTileError, match="lie over"):
        ops.add_rms_norm(row, w, 1e-5, out=w.view(1, 256))


def test_operands_of_no_rows_lie_over_nothing():
    from metaltile_b200 import _lib, ops
    w, dw = torch.ones(256, device="cuda"), torch.empty(256, device="cuda")
    inside = w.data_ptr() + 64
    assert _lib.load().mtc_add_rms_norm_grad(ops.context(0)._handle, None, inside, inside, w.data_ptr(), 1e-5, None, inside, dw.data_ptr(), 0, 256, _lib.F32, None, 0) == 0
    assert not dw.any()

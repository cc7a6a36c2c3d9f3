"""The 8-bit float ops without a GPU: refusals, workspace sizes, and that the formulas the GPU tests compare with agree with differences."""
import pytest
import torch

import fp8_ref as ref
from metaltile_b200 import _lib, ops

F8 = torch.float8_e4m3fn


def _codes(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(F8)


def _f(*shape):
    return torch.ones(*shape)


MM = dict(x=_codes(3, 256), w=_codes(130, 256), w_scales=_f(2, 2), x_scales=_f(3, 2))
GATHER = dict(x=_codes(3, 256), w=_codes(4, 130, 256), w_scales=_f(4, 2, 2), expert_offsets=torch.zeros(5, dtype=torch.int32), x_scales=_f(3, 2))


@pytest.mark.parametrize("change,error,word", [
    (dict(x_scales=None), ValueError, "x_scales"), (dict(x=_f(3, 256)), ValueError, "x_scales"), (dict(x=_codes(3, 256).view(torch.uint8)), TypeError, "codes"),
    (dict(w=_codes(130, 255)), ValueError, r"\[N, K\]"), (dict(w=_f(130, 256)), TypeError, "float8"), (dict(w_scales=_f(1, 2)), ValueError, "w_scales"),
    (dict(w_scales=_f(2, 2).double()), TypeError, "float32"), (dict(x_scales=_f(3, 1)), ValueError, "x_scales"), (dict(x_scales=_f(2, 2)), ValueError, "x_scales"),
    (dict(w=_codes(256, 130).T), ValueError, "contiguous"), (dict(x=torch.zeros(3, 0, dtype=torch.uint8).view(F8)), ValueError, "at least one"),
    (dict(out_dtype=torch.float64), TypeError, "out_dtype"), (dict(), ValueError, "CUDA device"),
])
def test_mm_refuses(change, error, word):
    with pytest.raises(error, match=word):
        ops.fp8_mm(**{**MM, **change})


@pytest.mark.parametrize("change,error,word", [
    (dict(w=_codes(130, 256)), ValueError, r"\[E, n_out"), (dict(w_scales=_f(2, 2)), ValueError, "w_scales"), (dict(x_scales=_f(4, 2)), ValueError, "x_scales"),
    (dict(expert_offsets=torch.zeros(4, dtype=torch.int32)), ValueError, "E \\+ 1"), (dict(expert_offsets=torch.zeros(5, dtype=torch.int64)), TypeError, "int32"),
    (dict(x=_f(3, 256)), TypeError, "float8"), (dict(out_dtype=torch.int32), TypeError, "out_dtype"), (dict(), ValueError, "CUDA device"),
])
def test_gather_refuses(change, error, word):
    with pytest.raises(error, match=word):
        ops.fp8_gather_mm(**{**GATHER, **change})


@pytest.mark.parametrize("kw,error,word", [
    (dict(x=_f(4, 128), block_rows=64), ValueError, "block_rows"), (dict(x=_f(128), block_rows=128), ValueError, "at least one"),
    (dict(x=_f(4, 0)), ValueError, "at least one"), (dict(x=_f(4, 128).double()), KeyError, "dtype"), (dict(x=_f(128, 4).T), ValueError, "contiguous"),
    (dict(x=_f(4, 128), rows=torch.zeros(2, dtype=torch.int64)), TypeError, "int32"),
    (dict(x=_f(128, 128), rows=torch.zeros(2, dtype=torch.int32), block_rows=128), ValueError, "block_rows 1"), (dict(x=_f(4, 128)), ValueError, "CUDA device"),
])
def test_quantize_refuses(kw, error, word):
    with pytest.raises(error, match=word):
        ops.fp8_quantize(**kw)


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("call,error,word", [
    (lambda: ops.moe_balance(_f(4, 8), _i(3, 2)), ValueError, "topk_idx"), (lambda: ops.moe_balance(_f(4, 8), _i(4, 2).long()), TypeError, "int32"),
    (lambda: ops.moe_balance(_f(4, 8), _i(4, 2), mask=_f(4)), TypeError, "mask"), (lambda: ops.moe_balance(_f(4, 8), _i(4, 2), mask=_i(3).bool()), ValueError, "mask"),
    (lambda: ops.moe_balance(_f(4, 8).double(), _i(4, 2)), KeyError, "dtype"), (lambda: ops.moe_balance(_f(4, 8), _i(4, 2)), ValueError, "CUDA device"),
    (lambda: ops.moe_balance_grad(_f(4, 8), _i(7), _i(1), 2), ValueError, "counts"), (lambda: ops.moe_balance_grad(_f(4, 8), _i(8), _i(2), 2), ValueError, "n_counted"),
    (lambda: ops.moe_balance_grad(_f(4, 8), _i(8), _i(1), 2, grad_loss=_f(2)), TypeError, "grad_loss"),
    (lambda: ops.moe_balance_grad(_f(4, 8), _i(8), _i(1), 2, grad_loss=_f(1).half()), TypeError, "grad_loss"),
    (lambda: ops.moe_balance_grad(_f(4, 8), _i(8), _i(1), 2), ValueError, "CUDA device"),
])
def test_balance_refuses(call, error, word):
    with pytest.raises(error, match=word):
        call()


def test_entries_without_a_context_are_refused():
    lib = _lib.load()
    assert lib.mtc_fp8_quantize(None, None, None, None, None, None, 1, 1, 1, 128, 1, 0, 0) < 0
    assert lib.mtc_fp8_mm(None, None, None, None, None, None, None, 1, 1, 128, 3, 0, None, 0) < 0
    assert lib.mtc_fp8_gather_mm(None, None, None, None, None, None, None, None, 1, 1, 128, 1, 0, None, 0) < 0
    assert lib.mtc_moe_balance(None, None, None, None, None, 1.0, None, None, None, None, 1, 8, 2, 0, None, 0) < 0
    assert lib.mtc_moe_balance_grad(None, None, None, None, None, None, None, 1.0, None, 1, 8, 2, 0) < 0


def test_workspaces_cover_what_the_call_stages():
    lib = _lib.load()
    for m, k in ((1, 16), (3, 130), (2048, 4096), (70000, 40000)):
        assert lib.mtc_fp8_mm_workspace(None, m, 64, k, 2, 2) >= m * k + 4 * m * -(-k // 128)
    assert lib.mtc_moe_balance_workspace(None, 0, 8) == 0 and lib.mtc_moe_balance_workspace(None, 65536, 1024) > 65536 * 8


@pytest.mark.parametrize("args,want", [
    ((1, 4096, 4096, 0), "tile"), ((64, 14336, 4096, 0), "tile"), ((65, 4096, 4096, 0), "tile"), ((65, 4097, 4096, 0), "pair"), ((256, 2048, 4096, 0), "tile"),
    ((257, 2048, 4096, 0), "pair"), ((2048, 28672, 4096, 0), "pair"), ((1, 64, 130, 0), "cuda_core"), ((2048, 4096, 4088, 0), "cuda_core"),
    ((32, 768, 2048, 128), "tile"), ((7167, 768, 2048, 128), "tile"), ((7168, 768, 2048, 128), "pair"), ((60000, 768, 2048, 1025), "tile"), ((64, 64, 100, 8), "cuda_core"),
    ((8, 2 ** 20, 16, 2 ** 12), "cuda_core"), ((0, 64, 64, 0), None), ((2 ** 31 - 1, 64, 64, 0), None), ((1, 64, 2 ** 31 - 8, 0), None),
])
def test_kernels_on_both_sides_of_the_rules(args, want):
    name = _lib.load().mtc_fp8_kernel(None, *args).decode()
    assert name == ("" if want is None else ("fp8_gather_mm_" if args[3] else "fp8_mm_") + want)


def test_the_table_of_codes_is_the_types():
    values = torch.arange(127, dtype=torch.uint8).view(F8).double()
    assert torch.equal(values, ref.table())
    x = torch.randn(4096, dtype=torch.float32, generator=torch.Generator().manual_seed(1)) * 100
    assert torch.equal(ref.nearest(x.double()), x.to(F8).double())


@pytest.mark.parametrize("masked", [False, True])
def test_balance_gradient_agrees_with_differences(masked):
    gen = torch.Generator().manual_seed(2)
    z = torch.randn(6, 5, dtype=torch.float64, generator=gen)
    idx = torch.topk(z, 2, dim=1).indices
    mask = torch.tensor([1, 0, 1, 1, 0, 1]).bool() if masked else None
    g, h = ref.balance_grad(z, idx, 0.7, 1.3, mask), 1e-6
    for t in range(6):
        for e in range(5):
            d = torch.zeros_like(z)
            d[t, e] = h
            slope = 1.3 * (ref.balance(z + d, idx, 0.7, mask)[0] - ref.balance(z - d, idx, 0.7, mask)[0]) / (2 * h)
            assert abs(slope - g[t, e]) < 1e-9

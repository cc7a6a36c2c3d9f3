"""The norm with the residual's addition and low-rank adapters without a GPU: refusals, workspaces, and that the formulas the GPU tests compare with agree with
differences and with automatic ones."""
import pytest
import torch

import lora_ref as ref
from metaltile_b200 import _lib, ops


def _f(*shape):
    return torch.ones(*shape)


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


X, W = _f(3, 64), _f(64)


@pytest.mark.parametrize("call,error,word", [
    (lambda: ops.add_rms_norm(_f(3, 0), _f(0), 1e-5), ValueError, "at least one"), (lambda: ops.add_rms_norm(X, _f(63), 1e-5), ValueError, r"\[K\]"),
    (lambda: ops.add_rms_norm(X, W.half(), 1e-5), TypeError, "share one dtype"), (lambda: ops.add_rms_norm(X.double(), W.double(), 1e-5), KeyError, "dtype"),
    (lambda: ops.add_rms_norm(X, W, 1e-5, residual=_f(2, 64)), ValueError, "shape of x"), (lambda: ops.add_rms_norm(X, W, 1e-5, residual=X.half()), TypeError, "share"),
    (lambda: ops.add_rms_norm(_f(64, 3).T, W, 1e-5), ValueError, "contiguous"), (lambda: ops.add_rms_norm(X, W, "a"), TypeError, "real number"),
    (lambda: ops.add_rms_norm(X, W, 1e-5), ValueError, "CUDA device"), (lambda: ops.add_rms_norm(None, W, 1e-5), TypeError, "Tensor"),
    (lambda: ops.add_rms_norm_fp8(X, _f(63), 1e-5), ValueError, r"\[K\]"), (lambda: ops.add_rms_norm_fp8(X, W, 1e-5), ValueError, "CUDA device"),
    (lambda: ops.add_rms_norm_grad(_f(2, 64), X, W, 1e-5), ValueError, "shape of sum"), (lambda: ops.add_rms_norm_grad(X, X, W.half(), 1e-5), TypeError, "share"),
    (lambda: ops.add_rms_norm_grad(X, X, W, 1e-5, dsum=_f(3, 63)), ValueError, "shape of sum"), (lambda: ops.add_rms_norm_grad(X, X, W, 1e-5), ValueError, "CUDA device"),
])
def test_norms_refuse(call, error, word):
    with pytest.raises(error, match=word):
        call()


LORA = dict(x=_f(5, 64), a=_f(2, 8, 64), b=_f(2, 32, 8), rows=_i(5), offsets=_i(3))


@pytest.mark.parametrize("change,error,word", [
    (dict(x=_f(5, 0)), ValueError, "at least one"), (dict(x=_f(5, 64).double()), KeyError, "dtype"), (dict(a=_f(2, 8, 63)), ValueError, r"\[adapters, rank, K\]"),
    (dict(a=_f(8, 64)), ValueError, r"\[adapters, rank, K\]"), (dict(a=_f(0, 8, 64), b=_f(0, 32, 8)), ValueError, r"\[adapters, rank, K\]"),
    (dict(b=_f(2, 32, 7)), ValueError, r"\[adapters, N, rank\]"), (dict(b=_f(3, 32, 8)), ValueError, r"\[adapters, N, rank\]"), (dict(a=_f(2, 8, 64).half()), TypeError, "share"),
    (dict(rows=_i(4)), ValueError, "rows must"), (dict(rows=_i(5).long()), TypeError, "int32"), (dict(offsets=_i(2)), ValueError, "offsets must"),
    (dict(offsets=_i(3).long()), TypeError, "int32"), (dict(scales=_f(3)), ValueError, "scales must"), (dict(scales=_f(2).half()), TypeError, "scales must"),
    (dict(base=_f(5, 31)), ValueError, "base must"), (dict(base=_f(5, 32).half()), TypeError, "base must"), (dict(a=_f(2, 64, 8).transpose(1, 2)), ValueError, "contiguous"),
    (dict(), ValueError, "CUDA device"),
])
def test_adapters_refuse(change, error, word):
    with pytest.raises(error, match=word):
        ops.lora_mm(**{**LORA, **change})


@pytest.mark.parametrize("change,error,word", [
    (dict(dy=_f(5, 31)), ValueError, "dy must"), (dict(dy=_f(4, 32)), ValueError, "dy must"), (dict(dy=_f(5, 32).half()), TypeError, "dy must"),
    (dict(hidden=_f(5, 7)), ValueError, "hidden must"), (dict(hidden=_f(5, 8).half()), TypeError, "hidden must"), (dict(base=_f(5, 32)), ValueError, "base must"),
    (dict(), ValueError, "CUDA device"),
])
def test_adapters_gradients_refuse(change, error, word):
    with pytest.raises(error, match=word):
        ops.lora_grad(**{**LORA, "dy": _f(5, 32), "hidden": _f(5, 8), **change})


def test_entries_without_a_context_are_refused():
    lib, null = _lib.load(), None
    assert lib.mtc_add_rms_norm(null, null, null, null, null, 0.0, null, null, 1, 8, 0) < 0
    assert lib.mtc_add_rms_norm_fp8(null, null, null, null, null, 0.0, null, null, null, null, 1, 8, 0, 0) < 0
    assert lib.mtc_add_rms_norm_grad(null, null, null, null, null, 0.0, null, null, null, 1, 8, 0, null, 0) < 0
    assert lib.mtc_lora_mm(*[null] * 11, 1, 8, 8, 8, 1, 0) < 0
    assert lib.mtc_lora_grad(*[null] * 14, 1, 8, 8, 8, 1, 0, null, 0) < 0


def test_workspaces_cover_what_the_calls_keep():
    lib = _lib.load()
    assert lib.mtc_add_rms_norm_grad_workspace(None, 0, 64, 2) == 0 and lib.mtc_add_rms_norm_grad_workspace(None, 1, 64, 2) >= 264
    assert lib.mtc_add_rms_norm_grad_workspace(None, 9, 0, 2) == lib.mtc_add_rms_norm_grad_workspace(None, 9, 64, 7) == 0
    for rows, rank in ((1, 1), (70000, 64), (1 << 30, 1024)):
        assert lib.mtc_lora_grad_workspace(None, rows, 64, 64, rank, 3, 2) >= 4 * rows * rank
    assert lib.mtc_lora_grad_workspace(None, 1, 64, 64, 0, 3, 2) == 0 and lib.mtc_lora_grad_workspace(None, -1, 64, 64, 1, 3, 2) == 0


def _slope(f, v, at, h=1e-6):
    d = torch.zeros_like(v)
    d.view(-1)[at] = h
    return (f(v + d) - f(v - d)) / (2 * h)


@pytest.mark.parametrize("stream", [False, True])
def test_norm_gradients_agree_with_differences(stream):
    gen = torch.Generator().manual_seed(1)
    s, dy, w = torch.randn(3, 7, dtype=torch.float64, generator=gen), torch.randn(3, 7, dtype=torch.float64, generator=gen), torch.randn(7, dtype=torch.float64, generator=gen)
    dsum = torch.randn(3, 7, dtype=torch.float64, generator=gen) if stream else None
    dx, dw = ref.norm_grad(dy, s, w, 1e-5, dsum)
    loss = lambda v, u: (ref.norm(v, u, 1e-5) * dy).sum() + (0 if dsum is None else (v * dsum).sum())  # noqa: E731
    for i in range(s.numel()):
        assert abs(_slope(lambda v: loss(v, w), s, i) - dx.view(-1)[i]) < 1e-8
    for i in range(7):
        assert abs(_slope(lambda u: loss(s, u), w, i) - dw[i]) < 1e-8


@pytest.mark.parametrize("scaled", [False, True])
def test_adapter_gradients_agree_with_differences(scaled):
    gen = torch.Generator().manual_seed(2)
    r = lambda *shape: torch.randn(*shape, dtype=torch.float64, generator=gen)  # noqa: E731
    x, a, b, base, dy, dbase = r(6, 5), r(3, 2, 5), r(3, 4, 2), r(6, 4), r(6, 4), r(6, 5)
    ids, scales = torch.tensor([2, 0, 3, 2, 0, 2]), r(3) if scaled else None
    dx, da, db = ref.lora_grad(dy, x, a, b, ids, scales, dbase)
    loss = lambda x, a, b: (ref.lora(x, a, b, ids, scales, base)[0] * dy).sum() + (x * dbase).sum()  # noqa: E731
    for grad, v, f in ((dx, x, lambda v: loss(v, a, b)), (da, a, lambda v: loss(x, v, b)), (db, b, lambda v: loss(x, a, v))):
        for i in range(v.numel()):
            assert abs(_slope(f, v, i) - grad.reshape(-1)[i]) < 1e-8
    assert not da[1].any() and not db[1].any()                       # nobody has it


def test_groups_are_those_of_the_rows():
    rows, offsets = ref.group(torch.tensor([1, 3, 0, 1, 3, 1]), 3)
    assert rows.tolist() == [2, 0, 3, 5, 1, 4] and offsets.tolist() == [0, 1, 4, 4, 6]

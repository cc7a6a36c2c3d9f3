"""add_rms_norm, add_rms_norm_fp8 and add_rms_norm_grad against their definitions in 64 bits."""
import pytest
import torch

import lora_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# one value to rows that no thread keeps in registers, whole eights or not; a warp a row up to 512 values, one turn and two
SIZES = [(1, 1), (3, 7), (1, 8), (5, 64), (9, 120), (2, 129), (7, 256), (130, 264), (33, 512), (4, 520), (3, 1000), (1, 2880), (333, 2880), (2, 4095), (1, 4096), (150, 4096),
         (16, 8192), (149, 8200), (1, 14336), (5, 16384), (3, 16392), (2, 40000), (2, 40003), (1500, 96), (700, 1032)]


def _inputs(rows, k, dt, seed=0, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 7 + k)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    t = TYPES[dt]
    return (make(rows, k) * (1 + make(k).abs() ** 3)).to(t), (make(rows, k) * 2).to(t) if residual else None, (1 + 0.3 * make(k)).to(t), make(rows, k).to(t)


def _close(got, want, tol):
    off = (got.double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k", SIZES)
def test_norm(rows, k, dt):
    from metaltile_b200 import ops
    for residual in (True, False):
        x, r, w, _ = _inputs(rows, k, dt, 1, residual)
        y, s = ops.add_rms_norm(x, w, 1e-5, residual=r)
        if residual:
            assert s.dtype == x.dtype and torch.equal(s, (x.float() + r.float()).to(x.dtype))
        else:
            assert s is x
        assert y.dtype == x.dtype and y.shape == x.shape
        _close(y, ref.norm(s, w, 1e-5), ref.norm_bound(s, w, 1e-5))
    assert ops.context(0).status_word() == 0


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k", SIZES)
def test_codes_are_those_of_the_f32_results(rows, k, dt, pow2):
    from metaltile_b200 import ops
    x, r, w, _ = _inputs(rows, k, dt, 2, rows % 2 == 1)
    out = torch.empty_like(x)
    codes, scales, s = ops.add_rms_norm_fp8(x, w, 1e-5, residual=r, pow2=pow2, out=out)
    y, s2 = ops.add_rms_norm(x, w, 1e-5, residual=r)
    assert torch.equal(out, y) and torch.equal(s, s2)
    y32, _ = ops.add_rms_norm(s.float(), w.float(), 1e-5)
    want, want_scales = ops.fp8_quantize(y32, pow2=pow2)
    assert torch.equal(scales, want_scales) and torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
    again = ops.add_rms_norm_fp8(x, w, 1e-5, residual=r, pow2=pow2)
    assert torch.equal(again[0].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(again[1], scales)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k", SIZES + [(2000, 512), (3000, 4096)])
def test_gradients(rows, k, dt):
    from metaltile_b200 import ops
    for stream in (True, False):
        s, d, w, dy = _inputs(rows, k, dt, 3, stream)
        dx, dw = ops.add_rms_norm_grad(dy, s, w, 1e-5, dsum=d)
        want, want_w = ref.norm_grad(dy, s, w, 1e-5, d)
        tol, tol_w = ref.norm_grad_bounds(dy, s, w, 1e-5, d, -(-rows // 148) + 2)            # at least 148 shares, where there are as many rows
        assert dx.dtype == dw.dtype == s.dtype and dw.shape == (k,)
        _close(dx, want, tol)
        _close(dw, want_w, tol_w)
        again = ops.add_rms_norm_grad(dy, s, w, 1e-5, dsum=d)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("k", [1000, 4096, 4099])
def test_in_place_and_unaligned(k, dt):
    from metaltile_b200 import ops
    x, r, w, dy = _inputs(40, k, dt, 4)
    y, s = ops.add_rms_norm(x, w, 1e-6, residual=r)
    dx, dw = ops.add_rms_norm_grad(dy, s, w, 1e-6, dsum=r)
    stream, hidden = r.clone(), x.clone()
    got = ops.add_rms_norm(hidden, w, 1e-6, residual=stream, sum_out=stream, out=hidden)
    assert got[0] is hidden and got[1] is stream and torch.equal(hidden, y) and torch.equal(stream, s)
    for place in ("dy", "dsum"):
        g, d = dy.clone(), r.clone()
        got = ops.add_rms_norm_grad(g, s, w, 1e-6, dsum=d, out=g if place == "dy" else d)
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
    off = lambda v: torch.cat([v.new_zeros(1), v.reshape(-1)])[1:].view(v.shape)  # noqa: E731
    sums, bound = ref.norm(s, w, 1e-6), ref.norm_bound(s, w, 1e-6)
    _close(ops.add_rms_norm(off(x), off(w), 1e-6, residual=off(r))[0], sums, bound)
    codes, scales, _ = ops.add_rms_norm_fp8(off(x), w, 1e-6, residual=r)
    y32, _ = ops.add_rms_norm(off(s.float()), w.float(), 1e-6)
    want, want_scales = ops.fp8_quantize(y32)
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, want_scales)
    tol, tol_w = ref.norm_grad_bounds(dy, s, w, 1e-6, r, 40)
    got = ops.add_rms_norm_grad(off(dy), off(s), w, 1e-6, dsum=r)
    want = ref.norm_grad(dy, s, w, 1e-6, r)
    _close(got[0], want[0], tol)
    _close(got[1], want[1], tol_w)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("k", [256, 4096, 4099])
def test_special_values_stay_in_their_row(k, dt):
    from metaltile_b200 import ops
    x, r, w, _ = _inputs(8, k, dt, 5)
    clean = ops.add_rms_norm(x, w, 1e-5, residual=r)[0]
    clean_codes, clean_scales, _ = ops.add_rms_norm_fp8(x, w, 1e-5, residual=r)
    x[1, 3], x[2, k // 2], x[4], r[4], x[6, 0] = float("nan"), float("inf"), 0.0, 0.0, float("-inf")
    r[6, 0] = float("inf")                                           # their sum is a NaN
    y, _ = ops.add_rms_norm(x, w, 1e-5, residual=r)
    assert torch.isnan(y[1]).all() and torch.isnan(y[6]).all() and not y[4].any()
    assert torch.isnan(y[2, k // 2]) and not y[2, :k // 2].any()     # inf / inf, and the others over inf
    codes, scales, _ = ops.add_rms_norm_fp8(x, w, 1e-5, residual=r)
    values = codes.float()
    assert torch.isnan(values[1]).all() and torch.isnan(values[6]).all() and not values[4].any() and (scales[[1, 4, 6]] == 2.0 ** -90).all()
    for i in (0, 3, 5, 7):
        assert torch.equal(y[i], clean[i]) and torch.equal(values[i], clean_codes[i].float()) and torch.equal(scales[i], clean_scales[i])
    zero, _ = ops.add_rms_norm(torch.zeros_like(x), w, 0.0)
    assert torch.isnan(zero).all()                                   # 0 / 0, as the formula has it


def test_no_rows():
    from metaltile_b200 import ops
    x, w = torch.empty(0, 64, device="cuda"), torch.ones(64, device="cuda")
    y, s = ops.add_rms_norm(x, w, 1e-5, residual=x)
    codes, scales, _ = ops.add_rms_norm_fp8(x, w, 1e-5)
    dx, dw = ops.add_rms_norm_grad(x, x, w, 1e-5)
    assert y.shape == s.shape == codes.shape == dx.shape == (0, 64) and scales.shape == (0, 1) and dw.shape == (64,) and not dw.any()


def test_shapes_of_more_dimensions_and_refusals():
    from metaltile_b200 import MetalTileError, _lib, ops
    x, _, w, _ = _inputs(6, 300, "bf16", 6)
    y, _ = ops.add_rms_norm(x, w, 1e-5)
    codes, scales, _ = ops.add_rms_norm_fp8(x.view(2, 3, 300), w, 1e-5)
    assert torch.equal(ops.add_rms_norm(x.view(2, 3, 300), w, 1e-5)[0].view(6, 300), y) and codes.shape == (2, 3, 300) and scales.shape == (2, 3, 3)
    for call in (lambda: ops.add_rms_norm(x, w, 1e-5, sum_out=torch.empty_like(x)), lambda: ops.add_rms_norm(x, w, 1e-5, out=torch.empty(5, 300, device="cuda", dtype=x.dtype))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        ops.add_rms_norm(x, w, 1e-5, out=torch.empty_like(x, dtype=torch.float32))
    t = torch.empty_like(x)
    with pytest.raises(MetalTileError):
        ops.add_rms_norm(x, w, 1e-5, residual=x, sum_out=t, out=t)
    ctx = ops.context(0)
    lib, p = _lib.load(), x.data_ptr()
    assert lib.mtc_add_rms_norm_grad(ctx._handle, None, p, p, p, 1e-5, None, p, p, 6, 300, _lib.BF16, None, 0) == -3
    assert lib.mtc_add_rms_norm(ctx._handle, None, p, None, p, 1e-5, None, None, 6, 300, _lib.BF16) == -8
    assert lib.mtc_add_rms_norm(ctx._handle, None, p, None, p, 1e-5, None, p, 6, (1 << 30) + 1, _lib.BF16) == -8
    assert lib.mtc_add_rms_norm(ctx._handle, None, p, None, p, 1e-5, None, p, 6, 300, 7) == -6


def test_another_stream_and_a_graph():
    from metaltile_b200 import ops
    x, r, w, dy = _inputs(70, 4096, "bf16", 7)
    want = (*ops.add_rms_norm(x, w, 1e-5, residual=r), *ops.add_rms_norm_fp8(x, w, 1e-5, residual=r)[:2], *ops.add_rms_norm_grad(dy, x, w, 1e-5, dsum=r))
    run = lambda: (*ops.add_rms_norm(x, w, 1e-5, residual=r), *ops.add_rms_norm_fp8(x, w, 1e-5, residual=r)[:2], *ops.add_rms_norm_grad(dy, x, w, 1e-5, dsum=r))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for t in held:
        t.view(torch.uint8).zero_()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, got, held):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(a.view(torch.uint8), c.view(torch.uint8))


@pytest.mark.parametrize("dt,k", [("bf16", 16392), ("f16", 16391)])
def test_rows_whose_offsets_pass_32_bits(dt, k):
    from metaltile_b200 import ops
    rows, t = 132000, TYPES[dt]
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(rows, k, device="cuda", dtype=t).normal_(generator=g)
    r = torch.empty(rows, k, device="cuda", dtype=t).normal_(generator=g)
    w = (1 + 0.2 * torch.randn(k, device="cuda", generator=g)).to(t)
    at = torch.cat([torch.arange(3, device="cuda"), torch.arange(rows - 20, rows, device="cuda")])
    y, s = ops.add_rms_norm(x, w, 1e-5, residual=r)
    assert torch.equal(s[at], (x[at].float() + r[at].float()).to(t))
    _close(y[at], ref.norm(s[at], w, 1e-5), ref.norm_bound(s[at], w, 1e-5))
    del y
    codes, scales, _ = ops.add_rms_norm_fp8(s, w, 1e-5)
    want, want_scales = ops.fp8_quantize(ops.add_rms_norm(s[at].float(), w.float(), 1e-5)[0])
    assert torch.equal(codes[at].view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales[at], want_scales)
    del codes
    dx, _ = ops.add_rms_norm_grad(x, s, w, 1e-5, out=r)
    _close(dx[at], ref.norm_grad(x[at], s[at], w, 1e-5)[0], ref.norm_grad_bounds(x[at], s[at], w, 1e-5, None, 1)[0])

"""fp8_quantize, fp8_mm and fp8_gather_mm against their definitions in 64 bits."""
import threading

import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _x(rows, k, dt, seed=0):
    g = _gen(seed)
    return (torch.randn(rows, k, device="cuda", generator=g) * (1 + torch.randn(k, device="cuda", generator=g).abs() ** 3)).to(TYPES[dt])


def _codes(*shape, seed=0):
    return (torch.randn(*shape, device="cuda", generator=_gen(seed)) * 120).clamp(-448, 448).to(F8)


def _scales(*shape, seed=0):
    return (torch.rand(*shape, device="cuda", generator=_gen(seed)) + 0.5) * 2.0 ** -9


def _operands(m, n, k, seed=0, experts=None):
    lead = () if experts is None else (experts,)
    return (_codes(m, k, seed=seed), _scales(m, ref.blocks(k), seed=seed + 1), _codes(*lead, n, k, seed=seed + 2),
            _scales(*lead, ref.blocks(n), ref.blocks(k), seed=seed + 3))


def _same_codes(codes, want):
    got = codes.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    bad = (got != want) & ~torch.isnan(want)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


@pytest.fixture(params=[0, 2, 3], ids=["by shape", "tiles", "pairs"])
def kernel(request):
    """The products by each of their kernels, wherever it takes the shape."""
    from metaltile_b200 import ops
    ops.context(0).set_option("fp8_kernel", request.param)
    yield request.param
    ops.context(0).set_option("fp8_kernel", 0)


# ---- the quantizer ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 128), (3, 7), (5, 127), (2, 129), (17, 200), (33, 2880), (1, 4096), (257, 1024)])
def test_quantize_rows(rows, k, dt, pow2):
    from metaltile_b200 import ops
    x = _x(rows, k, dt, rows + k)
    codes, scales = ops.fp8_quantize(x, pow2=pow2)
    want, s = ref.quantize(x, 1, pow2)
    assert codes.dtype == F8 and codes.shape == x.shape and torch.equal(scales.double(), s)
    _same_codes(codes, want)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 130), (300, 272), (2, 130, 136), (3, 1, 64), (2, 2, 127, 129)])
def test_quantize_blocks(shape, dt):
    from metaltile_b200 import ops
    x = _x(torch.Size(shape[:-1]).numel(), shape[-1], dt, sum(shape)).reshape(shape)
    codes, scales = ops.fp8_quantize(x, block_rows=128, pow2=shape[-1] % 2 == 0)
    flat, c, s = x.reshape(-1, *shape[-2:]), codes.reshape(-1, *shape[-2:]), scales.reshape(-1, *scales.shape[-2:])
    assert scales.shape == (*shape[:-2], ref.blocks(shape[-2]), ref.blocks(shape[-1]))
    for i in range(flat.shape[0]):                                   # a block never reaches into the next matrix
        want, ws = ref.quantize(flat[i], 128, shape[-1] % 2 == 0)
        assert torch.equal(s[i].double(), ws)
        _same_codes(c[i], want)


@pytest.mark.parametrize("dt", TYPES)
def test_quotients_on_a_border_between_codes(dt):
    """x = amax * (2 i + 1) / 2^j: with a scale rounded to f32 the quotient is next to a border, or on one."""
    from metaltile_b200 import ops
    amax = (1 + torch.arange(128, device="cuda") / 128.0)[:, None]
    t = torch.cat([torch.arange(1, 64, 2, device="cuda") / 64.0, torch.arange(17, 32, 2, device="cuda") * 0.875 / 28, torch.arange(1, 33, device="cuda") / 448.0])
    x = torch.cat([amax, amax * t, -amax * t], dim=1)
    x = torch.nn.functional.pad(x, (0, 128 - x.shape[1] % 128))
    x = x.to(TYPES[dt]).reshape(-1, 128)
    for pow2 in (False, True):
        codes, scales = ops.fp8_quantize(x, pow2=pow2)
        want, s = ref.quantize(x, 1, pow2)
        assert torch.equal(scales.double(), s)
        _same_codes(codes, want)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dt,bits", [("bf16", 8), ("f16", 11)])
def test_every_mantissa_in_a_block_of_every_maximum(dt, bits, block_rows):
    """16-bit types decide codes by a factor that depends on which side of amax / 448 its scale is rounded to: every pair of mantissas, over as many binary
    orders as a code has, and subnormal ones."""
    from metaltile_b200 import ops
    half = 1 << (bits - 1)
    top = torch.arange(half, 2 * half, device="cuda", dtype=torch.float64)
    x = top[None, :, None] * torch.exp2(-torch.arange(16384 // half, device="cuda", dtype=torch.float64) % 17)         # [1, mantissa, order]
    x = torch.where(x > top[:, None, None], x / 2, x).reshape(half, -1, 128)
    x[:, :, 0] = top[:, None]
    for scale in (2.0 ** -5, 2.0 ** -20 if dt == "f16" else 2.0 ** -130):
        v = (x * scale).to(TYPES[dt]).reshape(-1, 128)
        codes, scales = ops.fp8_quantize(v, block_rows=block_rows)
        want, s = ref.quantize(v, block_rows)
        assert torch.equal(scales.double(), s)
        _same_codes(codes, want)


@pytest.mark.parametrize("dt", TYPES)
def test_quantize_special_values(dt):
    from metaltile_b200 import ops
    inf, nan = float("inf"), float("nan")
    fi = torch.finfo(TYPES[dt])
    x = torch.zeros(9, 256, device="cuda", dtype=torch.float64)
    x[1, 5] = inf
    x[2, 7], x[2, 8] = -inf, 3.0
    x[3, 200], x[3, 201] = nan, -2.5
    x[4] = nan
    x[5, 0], x[5, 1] = fi.max, fi.min
    x[6, 0], x[6, 1] = fi.smallest_normal, -fi.smallest_normal / 2
    x[7, :] = fi.tiny
    x[8, 3] = -0.0
    x = x.to(TYPES[dt])
    for pow2 in (False, True):
        codes, scales = ops.fp8_quantize(x, pow2=pow2)
        want, s = ref.quantize(x, 1, pow2)
        assert torch.equal(scales.double(), s)
        _same_codes(codes, want)


@pytest.mark.parametrize("dt", TYPES)
def test_quantize_in_another_order_and_unaligned(dt):
    from metaltile_b200 import ops
    x = _x(37, 264, dt)
    order = torch.randint(0, 37, (91,), device="cuda", generator=_gen(4)).to(torch.int32)
    codes, scales = ops.fp8_quantize(x, rows=order)
    plain, ps = ops.fp8_quantize(x)
    assert torch.equal(codes.view(torch.uint8), plain.view(torch.uint8)[order.long()]) and torch.equal(scales, ps[order.long()])
    held = torch.empty(x.numel() + 1, device="cuda", dtype=x.dtype)                 # rows that start off a 16-byte boundary
    held[1:] = x.reshape(-1)
    codes, scales = ops.fp8_quantize(held[1:].reshape(x.shape))
    assert torch.equal(codes.view(torch.uint8), plain.view(torch.uint8)) and torch.equal(scales, ps)
    assert ops.fp8_quantize(x[:0])[0].shape == (0, 264) and ops.fp8_quantize(x, rows=order[:0])[1].shape == (0, 3)
    assert ops.fp8_quantize(x[:0], block_rows=128)[1].shape == (0, 3)
    assert ops.context(0).status_word() == 0


def test_an_index_outside_reads_row_0_and_is_reported():
    from metaltile_b200 import ops
    ctx = ops.context(0)
    x = _x(4, 128, "bf16")
    try:
        codes, _ = ops.fp8_quantize(x, rows=torch.tensor([3, 4, -1], device="cuda", dtype=torch.int32))
        plain = ops.fp8_quantize(x)[0]
        assert torch.equal(codes.view(torch.uint8), plain.view(torch.uint8)[[3, 0, 0]]) and ctx.status_word() == 0x906
    finally:
        ctx.status_clear()


# ---- the dense product ---------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 5, 16), (2, 128, 128), (3, 129, 130), (1, 300, 4096), (5, 64, 272), (16, 257, 1024), (17, 130, 144), (33, 640, 2880), (64, 256, 512),
          (100, 1000, 128), (129, 385, 400), (300, 520, 1040), (257, 256, 2048), (1, 4100, 96), (8, 129, 16384), (520, 128, 16), (256, 512, 7)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_mm(m, n, k, dt, kernel):
    from metaltile_b200 import ops
    x, xs, w, ws = _operands(m, n, k, m + n + k)
    out = ops.fp8_mm(x, w, ws, x_scales=xs, out_dtype=TYPES[dt])
    ref.mm_close(out, x, xs, w, ws)
    assert torch.equal(out, ops.fp8_mm(x, w, ws, x_scales=xs, out_dtype=TYPES[dt]))          # the same call, the same bits
    assert ops.context(0).status_word() == 0


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 4096, 1024), (1, 130, 2880), (3, 500, 200), (16, 129, 4096), (40, 256, 256), (200, 300, 136), (1, 7, 5)])
def test_mm_of_float_activations_is_that_of_their_codes(m, n, k, dt):
    from metaltile_b200 import ops
    x = _x(m, k, dt, m)
    _, _, w, ws = _operands(1, n, k, n)
    codes, scales = ops.fp8_quantize(x)
    out = ops.fp8_mm(x, w, ws)
    assert out.dtype == x.dtype and torch.equal(out, ops.fp8_mm(codes, w, ws, x_scales=scales, out_dtype=x.dtype))
    ref.mm_close(out, codes, scales, w, ws)


def test_mm_out_batches_defaults_and_nothing():
    from metaltile_b200 import ops
    x, xs, w, ws = _operands(6, 200, 256)
    out = torch.full((6, 200), 7.0, device="cuda", dtype=torch.float16)
    assert ops.fp8_mm(x, w, ws, x_scales=xs, out=out) is out
    ref.mm_close(out, x, xs, w, ws)
    batched = ops.fp8_mm(x.reshape(2, 3, 256), w, ws, x_scales=xs.reshape(2, 3, 2))
    assert batched.dtype == torch.bfloat16 and batched.shape == (6, 200)
    assert ops.fp8_mm(x[:0], w, ws, x_scales=xs[:0]).shape == (0, 200) and ops.fp8_mm(x, w[:0], ws[:0], x_scales=xs).shape == (6, 0)
    with pytest.raises(ValueError):
        ops.fp8_mm(x, w, ws, x_scales=xs, out=out[:5])
    with pytest.raises(TypeError):
        ops.fp8_mm(x, w, ws, x_scales=xs, out=out, out_dtype=torch.float32)
    with pytest.raises(ValueError):
        ops.fp8_mm(x, w.cpu(), ws, x_scales=xs)


def _shifted(t, by):
    """The same values `by` bytes behind a 256-byte boundary."""
    raw = t.contiguous().view(torch.uint8).reshape(-1)
    held = torch.empty(raw.numel() + 256, device="cuda", dtype=torch.uint8)
    view = held[by:by + raw.numel()]
    view.copy_(raw)
    return view.view(t.dtype).reshape(t.shape)


@pytest.mark.parametrize("m", [1, 16, 200])
@pytest.mark.parametrize("by", [1, 4, 16])
def test_mm_operands_that_start_anywhere(m, by):
    from metaltile_b200 import ops
    x, xs, w, ws = _operands(m, 260, 512)
    want = ops.fp8_mm(x, w, ws, x_scales=xs, out_dtype=torch.float32)
    for args in ((_shifted(x, by), w), (x, _shifted(w, by))):
        out = torch.empty(m * 260 + 4, device="cuda")[1:1 + m * 260].reshape(m, 260)
        ops.fp8_mm(args[0], args[1], ws, x_scales=xs, out=out)
        ref.mm_close(out, x, xs, w, ws)
    assert torch.allclose(out, want, rtol=1e-3, atol=1e-3)


@pytest.mark.parametrize("m", [1, 9, 40, 300])
def test_mm_special_values(m, kernel):
    """NaN codes and scales reach their rows and columns and no others; zeros and scales far apart are as the definition has them."""
    from metaltile_b200 import ops
    x, xs, w, ws = _operands(m, 300, 400, 11)
    x, w = x.clone(), w.clone()
    row, col = m // 2, 137
    x.view(torch.uint8)[row, 333] = 0x7F
    w.view(torch.uint8)[col, 5] = 0xFF
    xs[0, 1], ws[2, 3] = 0.0, 2.0 ** 60
    out = ops.fp8_mm(x, w, ws, x_scales=xs, out_dtype=torch.float32)
    nan = torch.zeros(m, 300, dtype=torch.bool, device="cuda")
    nan[row], nan[:, col] = True, True
    assert torch.equal(torch.isnan(out), nan)
    x.view(torch.uint8)[row, 333], w.view(torch.uint8)[col, 5] = 0, 0
    keep = ~nan
    want, size = ref.mm(x, xs, w, ws)
    assert ((out.double() - want).abs() <= 200 * 2.0 ** -23 * size + 2.0 ** -24 * want.abs())[keep].all()
    assert torch.isinf(ops.fp8_mm(x, w, ws * 2.0 ** 60, x_scales=xs, out_dtype=torch.float16)[:, 256:]).any()        # past the type: infinities


# ---- the grouped product ------------------------------------------------------------------------------------------
def _check_groups(out, x, xs, w, ws, off, untouched):
    owned = torch.zeros(x.shape[0], dtype=torch.bool, device="cuda")
    for e in range(w.shape[0]):
        r = slice(off[e], off[e + 1])
        owned[r] = True
        if off[e + 1] > off[e]:
            ref.mm_close(out[r], x[r], xs[r], w[e], ws[e])
    assert torch.equal(out[~owned], untouched[~owned])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("counts,n,k,lead,tail", [
    ([1], 130, 256, 0, 0), ([0, 0, 5], 129, 144, 0, 0), ([3, 0, 1, 0, 0, 7], 256, 400, 2, 3), ([1] * 32, 96, 128, 0, 0), ([130, 0, 257, 64], 200, 272, 0, 5),
    ([16, 17, 15, 1, 33], 384, 1024, 1, 0), ([0, 0, 0], 64, 64, 0, 4), ([300, 20], 1000, 130, 0, 0), ([64, 65, 63, 128, 129, 127, 32, 31, 33], 257, 512, 0, 1),
    ([1000, 1, 0, 600], 512, 640, 3, 2), ([1, 0, 2] * 70, 130, 160, 1, 1), ([2] * 1030, 64, 128, 0, 0),
])
def test_gather(counts, n, k, lead, tail, dt, kernel):
    from metaltile_b200 import ops
    m = sum(counts) + lead + tail
    x, xs, w, ws = _operands(m, n, k, m + n, experts=len(counts))
    off = [lead]
    for c in counts:
        off.append(off[-1] + c)
    out = torch.full((m, n), -3.0, device="cuda", dtype=TYPES[dt])
    before = out.clone()
    ops.fp8_gather_mm(x, w, ws, torch.tensor(off, device="cuda", dtype=torch.int32), xs, out=out)
    _check_groups(out, x, xs, w, ws, off, before)
    assert ops.context(0).status_word() == 0


def test_gather_nothing_and_defaults():
    from metaltile_b200 import ops
    x, xs, w, ws = _operands(4, 64, 128, experts=3)
    off = torch.tensor([0, 1, 1, 4], device="cuda", dtype=torch.int32)
    assert ops.fp8_gather_mm(x, w, ws, off, xs).dtype == torch.bfloat16
    assert ops.fp8_gather_mm(x[:0], w, ws, off * 0, xs[:0]).shape == (0, 64)
    assert ops.fp8_gather_mm(x, w[:, :0].contiguous(), ws[:, :0].contiguous(), off, xs).shape == (4, 0)


@pytest.mark.parametrize("off", [[0, 3, 2, 6], [0, 2, 4, 9], [0, -1, 3, 6]])
def test_gather_offsets_that_make_no_sense_are_reported(off, kernel):
    """Nothing outside the rows is read or written; the rows of ranges that hold are right."""
    from metaltile_b200 import ops
    ctx = ops.context(0)
    x, xs, w, ws = _operands(6, 130, 256, experts=3)
    held = torch.full((10, 130), 5.0, device="cuda")
    try:
        ops.fp8_gather_mm(x, w, ws, torch.tensor(off, device="cuda", dtype=torch.int32), xs, out=held[:6])
        torch.cuda.synchronize()
        assert ctx.status_word() == 0x901 and torch.equal(held[6:], torch.full((4, 130), 5.0, device="cuda"))
    finally:
        ctx.status_clear()


@pytest.mark.parametrize("m,e", [(64, 9), (700, 33), (1500, 200)])
def test_gather_offsets_that_hold_the_rows_many_times_over(m, e, kernel):
    """Ranges that overlap make more chunks than the launch was sized for: they end, are reported, and write no row of another tensor."""
    from metaltile_b200 import ops
    ctx = ops.context(0)
    x, xs, w, ws = _operands(m, 160, 256, experts=e)
    off = torch.tensor([m * (i % 2) for i in range(e + 1)], device="cuda", dtype=torch.int32)
    held = torch.full((m + 8, 160), 5.0, device="cuda")
    try:
        ops.fp8_gather_mm(x, w, ws, off, xs, out=held[4:-4])
        torch.cuda.synchronize()
        assert ctx.status_word() == 0x901
        assert (held[:4] == 5).all() and (held[-4:] == 5).all() and held.isfinite().all()
    finally:
        ctx.status_clear()


# ---- streams, graphs, threads --------------------------------------------------------------------------------------
@pytest.mark.parametrize("m,n,k", [(1, 2048, 2048), (40, 512, 2880), (300, 384, 1024)])
def test_mm_on_another_stream_and_in_graphs(m, n, k, kernel):
    """Two captured graphs replay in turn and at once with new inputs, each with its own workspace."""
    from metaltile_b200 import ops
    x = [_x(m, k, "bf16", i) for i in range(4)]
    _, _, w, ws = _operands(1, n, k)
    want = [ops.fp8_mm(v, w, ws) for v in x]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(ops.fp8_mm(x[0], w, ws), want[0])
    side.synchronize()
    inputs, outs, graphs = [torch.empty_like(x[0]) for _ in range(2)], [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        inputs[i].copy_(x[i])
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs.append(ops.fp8_mm(inputs[i], w, ws))
        graphs.append(g)
    for a, b in ((0, 1), (2, 3), (3, 0)):
        inputs[0].copy_(x[a]), inputs[1].copy_(x[b])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[a]) and torch.equal(outs[1], want[b])


def test_a_captured_layer_replays_with_other_routing(kernel):
    """Offsets are read on the device: the same graph serves other rows, other experts, and none."""
    from metaltile_b200 import ops
    e, k = 6, 2
    _, _, w, ws = _operands(1, 256, 384, 4, experts=e)
    cases = []
    for i in range(3):
        x = _x(150, 384, "bf16", i)
        logits = torch.randn(150, e, device="cuda", generator=_gen(i)) + torch.tensor([0.0, 9.0, 0.0, -9.0, 0.0, 3.0], device="cuda") * i
        idx, _ = ops.moe_router_topk(logits, k)
        cases.append((x, idx))

    def layer(x, idx):
        order, _, off, _ = ops.moe_sort(idx, e)
        codes, scales = ops.fp8_quantize(x, rows=order)
        return codes, scales, off, ops.fp8_gather_mm(codes, w, ws, off, scales)

    x, idx = (t.clone() for t in cases[0])
    layer(x, idx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        codes, scales, off, out = layer(x, idx)
    for xx, ii in cases:
        x.copy_(xx), idx.copy_(ii)
        graph.replay()
        torch.cuda.synchronize()
        _check_groups(out, codes, scales, w, ws, off.tolist(), out)


def test_a_product_right_behind_the_quantizer_of_its_weights():
    """The context keeps a product from requesting weights that are still being written."""
    from metaltile_b200 import ops
    mats = [(torch.randn(1024, 2048, device="cuda", generator=_gen(i)) * 0.02).bfloat16() for i in range(4)]
    x = _x(3, 2048, "bf16")
    want = []
    for m in mats:
        w, ws = ops.fp8_quantize(m, block_rows=128)
        torch.cuda.synchronize()
        want.append(ops.fp8_mm(x, w, ws))
        torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for m in mats:
            w, ws = ops.fp8_quantize(m, block_rows=128)
            got.append(ops.fp8_mm(x, w, ws))
            got.append(ops.fp8_mm(x, w, ws))
        assert all(torch.equal(g, want[i // 2]) for i, g in enumerate(got))


def test_a_product_captured_behind_a_quantizer_leaves_the_next_one_waiting():
    """The captured product does not run: the first that does is the one to wait for the weights."""
    from metaltile_b200 import ops
    m = (torch.randn(2048, 2048, device="cuda", generator=_gen(9)) * 0.02).bfloat16()
    xq, xs = ops.fp8_quantize(_x(2, 2048, "bf16"))
    w, ws = ops.fp8_quantize(m, block_rows=128)
    torch.cuda.synchronize()
    want = ops.fp8_mm(xq, w, ws, xs)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(3):
            torch.cuda._sleep(20_000_000)                            # the quantizer is still to come when the products are launched
            w, ws = ops.fp8_quantize(m, block_rows=128)
            graph = torch.cuda.CUDAGraph()
            graph.capture_begin()
            captured = ops.fp8_mm(xq, w, ws, xs)
            graph.capture_end()
            got = ops.fp8_mm(xq, w, ws, xs)
            graph.replay()
            stream.synchronize()
            assert torch.equal(got, want) and torch.equal(captured, want)


def test_calls_of_two_threads_at_once():
    from metaltile_b200 import ops
    jobs = []
    for i, (m, n, k) in enumerate(((4, 1024, 2048), (130, 512, 1040))):
        x, (_, _, w, ws) = _x(m, k, "bf16", i), _operands(1, n, k, i)
        jobs.append((x, w, ws, ops.fp8_mm(x, w, ws)))
    torch.cuda.synchronize()
    wrong = []

    def work(x, w, ws, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = ops.fp8_mm(x, w, ws)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want):
                    wrong.append(x.shape)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_gradient_of_x_is_the_product_with_the_matrix_the_other_way_round():
    from metaltile_b200 import ops
    _, _, w, ws = _operands(1, 384, 640, 5)
    dy = _x(50, 384, "bf16", 3)
    dyq, dys = ops.fp8_quantize(dy)
    wt, wst = w.T.contiguous(), ws.T.contiguous()
    torch.cuda.synchronize()                                         # weights are there before a product that may request them early
    dx = ops.fp8_mm(dy, wt, wst, out_dtype=torch.float32)
    want = (dyq.double() * ref.spread(dys, 50, 384, 1)) @ (w.double() * ref.spread(ws, 384, 640, 128))
    size = (dyq.double() * ref.spread(dys, 50, 384, 1)).abs() @ (w.double() * ref.spread(ws, 384, 640, 128)).abs()
    assert ((dx.double() - want).abs() <= 140 * 2.0 ** -23 * size).all()


def test_a_whole_layer_of_experts():
    """router -> balance -> sort -> codes in expert order -> gate, up -> SwiGLU -> codes -> down -> unpermute: every stage from what the one before gave."""
    from metaltile_b200 import ops
    tokens, hidden, inter, e, k = 70, 256, 384, 8, 2
    x = _x(tokens, hidden, "bf16", 1)
    logits = torch.randn(tokens, e, device="cuda", generator=_gen(2)).bfloat16()
    stacks = [ops.fp8_quantize((torch.randn(e, n, c, device="cuda", generator=_gen(5 + i)) * 0.05).bfloat16(), block_rows=128)
              for i, (n, c) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    idx, wts = ops.moe_router_topk(logits, k)
    loss, counts, _, n = ops.moe_balance(logits, idx)
    order, inv, off, _ = ops.moe_sort(idx, e)
    assert torch.equal(off[1:] - off[:-1], counts) and int(n) == tokens and float(loss) > 0.99
    codes, scales = ops.fp8_quantize(x, rows=order)
    gate, up = (ops.fp8_gather_mm(codes, *s, off, scales) for s in stacks[:2])
    act = ops.swiglu(gate, up)
    ac, asc = ops.fp8_quantize(act)
    down = ops.fp8_gather_mm(ac, *stacks[2], off, asc)
    out = ops.moe_unpermute(down, inv, wts)
    at = off.tolist()
    for got, (c, s), (w, ws) in ((gate, (codes, scales), stacks[0]), (up, (codes, scales), stacks[1]), (down, (ac, asc), stacks[2])):
        for i in range(e):
            r = slice(at[i], at[i + 1])
            if at[i + 1] > at[i]:
                ref.mm_close(got[r], c[r], s[r], w[i], ws[i])
    want = (down.double()[inv.long()] * wts.double()[:, :, None]).sum(dim=1)
    size = (down.double()[inv.long()] * wts.double()[:, :, None]).abs().sum(dim=1)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * 2.0 ** -24 * size).all()

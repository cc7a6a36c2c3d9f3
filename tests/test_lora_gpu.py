"""lora_mm and lora_grad against their definitions in 64 bits."""
import pytest
import torch

import lora_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Case:
    def __init__(self, rows, k, n, rank, adapters, dt, ids=None, seed=0, scales=True, base=True):
        g = torch.Generator(device="cuda").manual_seed(seed + rows + 3 * k + 5 * n + 7 * rank)
        make, t = lambda *s: torch.randn(*s, device="cuda", generator=g), TYPES[dt]  # noqa: E731
        self.x, self.dy = make(rows, k).to(t), make(rows, n).to(t)
        self.a, self.b = (make(adapters, rank, k) / k ** 0.5).to(t), (make(adapters, n, rank) / rank ** 0.5).to(t)
        self.base, self.dbase = (make(rows, n).to(t), make(rows, k).to(t)) if base else (None, None)
        self.scales = torch.rand(adapters, device="cuda", generator=g) + 0.5 if scales else None
        self.ids = torch.randint(0, adapters + 1, (rows,), device="cuda", generator=g) if ids is None else torch.as_tensor(ids, device="cuda")
        self.rows, self.offsets = ref.group(self.ids, adapters)
        self.adapters = adapters

    def forward(self, **kw):
        from metaltile_b200 import ops
        return ops.lora_mm(self.x, self.a, self.b, self.rows, self.offsets, scales=self.scales, **{"base": self.base, "hidden": True, **kw})

    def grad(self, hidden, **kw):
        from metaltile_b200 import ops
        return ops.lora_grad(self.dy, self.x, self.a, self.b, self.rows, self.offsets, hidden, scales=self.scales, **{"base": self.dbase, **kw})

    def check(self):
        from metaltile_b200 import ops
        dt, ids = self.x.dtype, self.ids
        out, h = self.forward()
        want, want_h = ref.lora(self.x, self.a, self.b, ids, self.scales, self.base)
        dh = ref.low_bound(self.x, self.a, ids)
        assert out.dtype == dt and out.shape == want.shape and h.dtype == torch.float32
        _close(h, want_h, dh)
        _close(out, want, ref.high_bound(want, want_h, dh, self.b.transpose(1, 2), ids, self.scales, self.base, dt))
        got = self.grad(h)
        w = ref.lora_grad(self.dy, self.x, self.a, self.b, ids, self.scales, self.dbase)
        u, bt = ref.low(self.dy, self.b.transpose(1, 2), ids), self.b.transpose(1, 2)
        du = ref.low_bound(self.dy, bt, ids)
        _close(got[0], w[0], ref.high_bound(w[0], u, du, self.a, ids, self.scales, self.dbase, dt))
        _close(got[1], w[1], ref.outer_bound(w[1], u, du, self.x, ids, self.scales, self.adapters, dt))
        _close(got[2], w[2], ref.outer_bound(w[2].transpose(1, 2), want_h, dh, self.dy, ids, self.scales, self.adapters, dt).transpose(1, 2))
        again, h2 = self.forward()
        assert torch.equal(again, out) and torch.equal(h2, h)                    # the same call, the same bits
        for a, b in zip(self.grad(h), got):
            assert torch.equal(a, b)
        assert torch.equal(self.forward(hidden=False), out)
        assert ops.context(0).status_word() == 0


def _close(got, want, tol):
    """A result that rounds beyond the largest value of its type is an infinity there (round to nearest: from half a step, max * eps / 4, above it on); nearer
    to that border than `tol` it may be either."""
    most = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    got = got.double()
    over, may = want.abs() - tol > most, want.abs() + tol >= most
    assert (got == torch.copysign(torch.full_like(want, float("inf")), want))[over].all()
    off = torch.where(may & torch.isinf(got) & (got.sign() == want.sign()), 0.0, (got - want).abs())
    assert (off <= tol).all(), float((off / tol).max())


# one row to hundreds; whole eights, odd sizes; ranks on both sides of what tensor cores take at once; one adapter to more than there are rows
SIZES = [(1, 8, 8, 8, 1), (1, 4096, 4096, 16, 4), (2, 64, 96, 16, 1), (3, 7, 5, 3, 2), (5, 256, 264, 8, 3), (7, 130, 131, 1, 2), (16, 512, 256, 32, 2), (17, 1024, 512, 64, 1),
         (33, 2880, 760, 24, 3), (40, 328, 1000, 40, 5), (64, 4096, 1024, 16, 32), (65, 256, 256, 72, 2), (100, 264, 520, 128, 3), (128, 1032, 2056, 16, 7), (200, 512, 768, 8, 1),
         (30, 96, 72, 200, 2), (333, 720, 1904, 24, 3), (500, 1024, 1024, 64, 4), (9, 4100, 4100, 16, 2), (20, 4096, 33, 4, 2), (61, 24, 16, 12, 9),
         # rows that are no whole 16-byte pieces; hundreds of rows, which other kernels take
         (70, 1001, 515, 16, 2), (700, 257, 263, 32, 3), (50, 131, 1030, 64, 2), (33, 77, 99, 8, 2), (90, 2049, 4095, 24, 4), (40, 333, 250, 4, 2), (30, 101, 55, 72, 2),
         (1100, 512, 264, 64, 1), (2100, 264, 520, 16, 2), (2100, 128, 72, 32, 3), (1500, 1032, 328, 48, 1), (1030, 96, 160, 80, 2), (1500, 72, 64, 8, 2), (700, 264, 136, 2, 2),
         # whole pieces on one side alone
         (36, 691, 384, 64, 4), (40, 384, 691, 64, 2), (210, 264, 331, 24, 3), (210, 331, 264, 40, 3), (700, 130, 264, 16, 2), (700, 264, 130, 128, 1), (24, 77, 512, 200, 2), (900, 512, 36, 8, 2),
         # clusters of 4 and 2 CTAs, and the most rows of 8
         (1300, 264, 2056, 16, 2), (2500, 96, 72, 40, 3), (240, 1536, 1032, 64, 1), (600, 264, 2048, 32, 2), (2600, 2048, 264, 8, 1), (1250, 130, 77, 16, 4),
         (2400, 1032, 1040, 16, 2), (2400, 2048, 72, 32, 3), (2350, 520, 1600, 24, 1), (1200, 512, 264, 64, 1), (2310, 40, 2056, 32, 1)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_adapters(size, dt):
    Case(*size, dt).check()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("adapters", [1, 31, 32, 33, 100, 1000])
def test_more_adapters_than_rows_and_adapters_without_any(adapters, dt):
    Case(24, 256, 128, 8, adapters, dt).check()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("ids", [[2] * 50, [0] * 50, [3] * 50, [0] * 16 + [3] * 34, [1] * 33 + [0] * 17, [0, 1, 2, 3] * 12 + [2, 0], [3] * 49 + [1]])
def test_rows_of_one_adapter_of_none_and_mixed(ids, dt):
    Case(50, 264, 136, 16, 3, dt, ids=ids).check()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", [(20, 256, 128, 16, 2), (20, 255, 127, 3, 2)])
def test_without_scales_and_base(size, dt):
    Case(*size, dt, scales=False, base=False).check()


@pytest.mark.parametrize("dt", TYPES)
def test_in_place_leaves_rows_without_an_adapter_alone(dt):
    for n in (128, 127):
        c = Case(40, 256, n, 16, 3, dt, seed=3)
        out, h = c.forward()
        base, dbase = c.base.clone(), c.dbase.clone()
        none = c.ids == 3
        base[none], dbase[none] = float("nan"), float("nan")         # nobody looks at them
        got, _ = c.forward(base=base, out=base)
        assert got is base and torch.equal(base[~none], out[~none]) and torch.isnan(base[none]).all()
        dx, _, _ = c.grad(h)
        got, _, _ = c.grad(h, base=dbase, out=dbase)
        assert torch.equal(dbase[~none], dx[~none]) and torch.isnan(dbase[none]).all()


# (the second size reaches tiles of 128 rows back, the fourth both ways; the third has rows that are no whole pieces)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", [(60, 256, 128, 16, 3), (2100, 256, 128, 32, 3), (60, 255, 127, 16, 3), (2400, 2048, 128, 32, 3)])
def test_rows_without_an_adapter_hold_anything(size, dt):
    c = Case(*size, dt, seed=4)
    want, h = c.forward()
    grads = c.grad(h)
    none = c.ids == 3
    c.x[none], c.dy[none] = float("nan"), float("inf")
    got, h2 = c.forward()
    assert torch.equal(got, want) and torch.equal(h2, h) and not h[none].any()
    h2[none] = float("nan")
    for a, b in zip(c.grad(h2), grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,n", [(48, 128), (2100, 128), (48, 127), (2400, 2048)])
def test_special_values_stay_in_their_row(rows, n, dt):
    c = Case(rows, 256, n, 16, 2, dt, seed=5)
    want, _ = c.forward()
    c.x[5, 7], c.x[20, 100] = float("nan"), float("inf")
    c.ids[5], c.ids[20] = 0, 1
    c.rows, c.offsets = ref.group(c.ids, 2)
    got, h = c.forward()
    assert torch.isnan(got[5]).all() and not torch.isfinite(got[20]).any()
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[5] = rest[20] = False
    clean = ref.lora(c.x[rest], c.a, c.b, c.ids[rest], c.scales, c.base[rest])[0]
    assert torch.isfinite(got[rest]).all() and (got[rest].double() - clean).abs().max() < 0.05


@pytest.mark.parametrize("rows,n", [(40, 256), (2100, 256), (40, 255), (2400, 2048)])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_large_and_small_values(dt, rows, n):
    """What a row goes through may be far outside of 16-bit floats."""
    c = Case(rows, 512, n, 16, 2, dt, seed=6)
    up = 2.0 ** torch.randint(-10, 9, (rows, 1), device="cuda").float()
    c.x = (c.x.float() * up * 16).to(TYPES[dt])
    c.dy = (c.dy.float() * up * 16).to(TYPES[dt])
    c.a, c.b = (c.a.float() * 512).to(TYPES[dt]), (c.b.float() / 64).to(TYPES[dt])
    c.scales = c.scales / 512
    c.check()


def test_no_rows():
    c = Case(0, 64, 32, 8, 3, "bf16")
    out, h = c.forward()
    dx, da, db = c.grad(h)
    assert out.shape == (0, 32) and h.shape == (0, 8) and dx.shape == (0, 64) and not da.any() and not db.any()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("size", [(40, 256, 128, 16, 3), (40, 255, 127, 5, 3)])
def test_bad_offsets_and_rows_are_reported(size, dt):
    from metaltile_b200 import ops
    ctx = ops.context(0)
    c = Case(*size, dt, ids=[0] * 10 + [1] * 10 + [2] * 20)
    good, h = c.forward()
    grads = c.grad(h)
    try:
        for offsets in ([0, 30, 10, 40], [0, 10, 20, 2000], [0, 10, -5, 40], [35, 20, 10, 0]):
            ctx.status_clear()
            c.offsets = torch.tensor(offsets, dtype=torch.int32, device="cuda")
            c.forward()
            assert ctx.status_word() == 0x901
            c.grad(h)
        ctx.status_clear()
        c.offsets = torch.tensor([0, 10, 20, 40], dtype=torch.int32, device="cuda")
        c.rows = c.rows.clone()
        c.rows[3], c.rows[25] = 40, -1
        out, _ = c.forward()
        assert ctx.status_word() == 0x908
        keep = [i for i in range(40) if i not in (3, 25)]
        assert torch.equal(out[keep], good[keep])
        c.grad(h)
    finally:
        ctx.status_clear()
    c.rows, c.offsets = ref.group(c.ids, 3)
    assert torch.equal(c.forward()[0], good)
    for a, b in zip(c.grad(h), grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("size", [(90, 256, 128, 16, 3), (90, 255, 127, 16, 3), (90, 255, 127, 5, 3), (2100, 128, 64, 32, 1), (2400, 2048, 64, 32, 1), (1300, 128, 64, 64, 1)])
def test_places_before_the_first_adapter_have_none(size, dt):
    """Any places outside of the ranges belong to no adapter, those in front as well."""
    rows, k, n, rank, adapters = size
    c = Case(*size, dt, seed=7)
    want, h = c.forward()
    dx, da, db = c.grad(h)
    none = int((c.ids == adapters).sum())
    c.rows = torch.cat([c.rows[rows - none // 2:], c.rows[:rows - none // 2]]).contiguous()          # half of them in front
    c.offsets = c.offsets + none // 2
    got, h2 = c.forward()
    assert torch.equal(got, want) and torch.equal(h2, h)
    for a, b in zip(c.grad(h), (dx, da, db)):
        assert torch.equal(a, b)
    base = c.base.clone()
    base[c.ids == adapters] = float("nan")
    got, _ = c.forward(base=base, out=base)
    assert torch.isnan(got[c.ids == adapters]).all() and torch.equal(got[c.ids != adapters], want[c.ids != adapters])


@pytest.mark.parametrize("dt,rows", [("bf16", 66000), ("f32", 33000)])
def test_rows_whose_offsets_pass_32_bits(dt, rows):
    from metaltile_b200 import ops
    k, n, rank, t = 33008, 64, 8, TYPES[dt]
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(rows, k, device="cuda", dtype=t).normal_(generator=g)
    dy = torch.randn(rows, n, device="cuda", generator=g).to(t)
    a, b = (torch.randn(3, rank, k, device="cuda", generator=g) / 180).to(t), torch.randn(3, n, rank, device="cuda", generator=g).to(t)
    ids = torch.randint(0, 4, (rows,), device="cuda", generator=g)
    order, offsets = ref.group(ids, 3)
    out, h = ops.lora_mm(x, a, b, order, offsets, hidden=True)
    dx, da, db = ops.lora_grad(dy, x, a, b, order, offsets, h)
    at = torch.cat([torch.arange(40, device="cuda"), torch.arange(rows - 200, rows, device="cuda")])
    want, want_h = ref.lora(x[at], a, b, ids[at], None, None)
    dh = ref.low_bound(x[at], a, ids[at])
    _close(out[at], want, ref.high_bound(want, want_h, dh, b.transpose(1, 2), ids[at], None, None, t))
    u, du = ref.low(dy[at], b.transpose(1, 2), ids[at]), ref.low_bound(dy[at], b.transpose(1, 2), ids[at])
    want = ref.high(u, a, ids[at], None, None, k)
    _close(dx[at], want, ref.high_bound(want, u, du, a, ids[at], None, None, t))
    # a column of the weights' gradient over all rows
    u = ref.low(dy, b.transpose(1, 2), ids)
    cols = torch.tensor([0, 77, k - 1], device="cuda")
    want = ref.outer(u, x[:, cols], ids, None, 3)
    tol = ref.outer_bound(want, u, ref.low_bound(dy, b.transpose(1, 2), ids), x[:, cols], ids, None, 3, t)
    _close(da[:, :, cols], want, tol)
    assert ops.context(0).status_word() == 0


@pytest.mark.parametrize("rows", [2200, 2500])
def test_beside_other_tensor_memory_kernels_on_another_stream(rows):
    from metaltile_b200 import ops
    c = Case(rows, 1024, 2048, 16, 2, "bf16", seed=11)
    want, h = c.forward()
    grads = c.grad(h)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2048, 1024, device="cuda", generator=g).to(torch.bfloat16)
    w, s = ops.fp8_quantize((torch.randn(2048, 1024, device="cuda", generator=g) * 0.02).to(torch.bfloat16), block_rows=128)
    y = ops.fp8_mm(x, w, s)
    y16 = ops.fp8_mm(x[:16].contiguous(), w, s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[0]):
            outs.append((c.forward()[0], want))
            outs.append((c.grad(h)[0], grads[0]))
        with torch.cuda.stream(streams[1]):
            outs.append((ops.fp8_mm(x, w, s), y))
            outs.append((ops.fp8_mm(x[:16].contiguous(), w, s), y16))
    torch.cuda.synchronize()
    for got, one in outs:
        assert torch.equal(got, one)


def test_groups_of_moe_sort():
    from metaltile_b200 import ops
    c = Case(100, 256, 128, 16, 5, "bf16")
    want, h = c.forward()
    c.rows, _, c.offsets, _ = ops.moe_sort(c.ids.to(torch.int32)[:, None].contiguous(), 6)
    assert torch.equal(c.forward()[0], want)


def test_unaligned_operands():
    c = Case(20, 256, 128, 16, 2, "bf16")
    off = lambda v: torch.cat([v.new_zeros(1), v.reshape(-1)])[1:].view(v.shape)  # noqa: E731
    for name in ("x", "a", "b", "base", "dy", "dbase"):
        d = Case(20, 256, 128, 16, 2, "bf16")
        setattr(d, name, off(getattr(c, name)))
        d.check()


def test_refusals():
    from metaltile_b200 import MetalTileError, ops
    c = Case(20, 64, 64, 8, 2, "bf16")
    out, h = c.forward()
    for bad in (c.x, out.new_zeros(0)[:0]):
        with pytest.raises((MetalTileError, ValueError)):                        # its rows are read by other tiles; not the result's shape
            c.forward(out=bad)
    for bad in (c.x, c.dy):
        with pytest.raises(MetalTileError):                                      # read again for the weights
            c.grad(h, out=bad)
    with pytest.raises(MetalTileError):                                          # a rank of more than 1024
        ops.lora_mm(c.x, c.x.new_zeros(2, 1025, 64), c.x.new_zeros(2, 64, 1025), c.rows, c.offsets)
    c.check()                                                                    # nothing was written or left behind


def test_another_stream_and_graphs_that_run_at_once():
    c, d = Case(300, 1024, 768, 16, 3, "bf16", seed=1), Case(300, 1024, 768, 16, 3, "bf16", seed=2)

    def step(v):
        out, h = v.forward()
        return (out, h, *v.grad(h))

    wants = [step(c), step(d)]
    streams, graphs, held = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for v, g in zip((c, d), graphs):
        with torch.cuda.graph(g):
            held.append(step(v))
    torch.cuda.synchronize()
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for want, got in zip(wants, held):
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_a_layer_with_norm_eight_bit_product_and_adapters():
    """The operators as a layer uses them, forward and back, against the same in 64 bits from what is held between them."""
    from metaltile_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(9)
    make, t = lambda *s: torch.randn(*s, device="cuda", generator=g), torch.bfloat16  # noqa: E731
    c = Case(70, 512, 384, 16, 3, "bf16", seed=8)
    x, stream, w = make(70, 512).to(t), make(70, 512).to(t), (1 + 0.1 * make(512)).to(t)
    codes, w_scales = ops.fp8_quantize((make(384, 512) * 0.05).to(t), block_rows=128)
    y = torch.empty_like(x)
    q, q_scales, s = ops.add_rms_norm_fp8(x, w, 1e-5, residual=stream, sum_out=stream, out=y)
    base = ops.fp8_mm(q, codes, w_scales, x_scales=q_scales, out_dtype=t)
    shared = base.clone()
    c.x, c.base = y, base
    out, h = c.forward(out=base)
    want, want_h = ref.lora(y, c.a, c.b, c.ids, c.scales, shared)
    _close(out, want, ref.high_bound(want, want_h, ref.low_bound(y, c.a, c.ids), c.b.transpose(1, 2), c.ids, c.scales, shared, t))
    _close(y, ref.norm(s, w, 1e-5), ref.norm_bound(s, w, 1e-5))
    wt, wt_scales = codes.view(torch.uint8).T.contiguous().view(torch.float8_e4m3fn), w_scales.T.contiguous()
    c.dbase = ops.fp8_mm(c.dy, wt, wt_scales)
    dy_norm, da, db = c.grad(h)
    dx, dw = ops.add_rms_norm_grad(dy_norm, s, w, 1e-5, dsum=stream)
    want, want_w = ref.norm_grad(dy_norm, s, w, 1e-5, stream)
    tol, tol_w = ref.norm_grad_bounds(dy_norm, s, w, 1e-5, stream, 70)
    _close(dx, want, tol)
    _close(dw, want_w, tol_w)
    assert ops.context(0).status_word() == 0

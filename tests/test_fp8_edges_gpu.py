"""Bad offsets and special values by every kernel of the 8-bit float products, the CUDA-core one among them: what is in order has to be right, and nothing else touched."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(*shape, seed=0):
    return (torch.randn(*shape, device="cuda", generator=_gen(seed)) * 120).clamp(-448, 448).to(F8)


def _scales(*shape, seed=0):
    return (torch.rand(*shape, device="cuda", generator=_gen(seed)) + 0.5) * 2.0 ** -9


def _operands(m, n, k, seed=0, experts=None):
    lead = () if experts is None else (experts,)
    return (_codes(m, k, seed=seed), _scales(m, ref.blocks(k), seed=seed + 1), _codes(*lead, n, k, seed=seed + 2),
            _scales(*lead, ref.blocks(n), ref.blocks(k), seed=seed + 3))


@pytest.fixture(params=[0, 1, 2, 3], ids=["by shape", "CUDA cores", "tiles", "pairs"])
def kernel(request):
    from metaltile_b200 import ops
    ops.context(0).set_option("fp8_kernel", request.param)
    yield request.param
    ops.context(0).set_option("fp8_kernel", 0)


def _owners(off, m):
    """The experts that a row belongs to once offsets are unsigned and clamped to the rows."""
    at = [min(o % 2 ** 32, m) for o in off]
    return [[e for e in range(len(off) - 1) if at[e] <= r < at[e + 1]] for r in range(m)]


@pytest.mark.parametrize("m,off", [(6, [0, 3, 2, 6]), (6, [0, 2, 4, 9]), (6, [0, -1, 3, 6]), (6, [1, 4, 4, 2, 5]), (90, [70, 80, 10, 60, 500]), (700, [0, 300, -5, 650, 640, 690]),
                                   (40, [41, 50, 60])])
@pytest.mark.parametrize("k", [256, 200])
def test_offsets_that_make_no_sense(m, off, k, kernel):
    """Rows of one range are its product, rows of none stay what they were, rows of several hold the product of one of them or parts of both; the rows in front of `out` and
    behind it belong to somebody else."""
    from metaltile_b200 import ops
    ctx, n = ops.context(0), 130
    x, xs, w, ws = _operands(m, n, k, m + k, experts=len(off) - 1)
    held = torch.full((m + 16, n), -7.0, device="cuda")
    out = held[8:-8]
    try:
        ops.fp8_gather_mm(x, w, ws, torch.tensor(off, device="cuda", dtype=torch.int32), xs, out=out)
        torch.cuda.synchronize()
        assert ctx.status_word() == 0x901
    finally:
        ctx.status_clear()
    assert (held[:8] == -7).all() and (held[-8:] == -7).all()
    owners = _owners(off, m)
    for e in range(len(off) - 1):
        rows = [r for r in range(m) if owners[r] == [e]]
        if rows:
            ref.mm_close(out[rows], x[rows], xs[rows], w[e], ws[e])
    nobody = [r for r in range(m) if not owners[r]]
    assert (out[nobody] == -7).all()
    for r in (r for r in range(m) if len(owners[r]) > 1):
        ok = torch.zeros(n, dtype=torch.bool, device="cuda")
        for e in owners[r]:
            want, size = ref.mm(x[r:r + 1], xs[r:r + 1], w[e], ws[e])
            ok |= ((out[r].double() - want[0]).abs() <= ref.STEP[torch.float32] * want[0].abs() + (128 + ref.blocks(k) + 4) * 2.0 ** -23 * size[0])
        assert ok.all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("counts,n,k", [([3, 0, 1, 0, 0, 7], 130, 400), ([1] * 9, 64, 130), ([70, 0, 33], 129, 256)])
def test_groups(counts, n, k, dt, kernel):
    from metaltile_b200 import ops
    m = sum(counts) + 5
    x, xs, w, ws = _operands(m, n, k, m + n, experts=len(counts))
    off = [2]
    for c in counts:
        off.append(off[-1] + c)
    out = torch.full((m, n), -3.0, device="cuda", dtype=TYPES[dt])
    ops.fp8_gather_mm(x, w, ws, torch.tensor(off, device="cuda", dtype=torch.int32), xs, out=out)
    for e in range(len(counts)):
        if counts[e]:
            r = slice(off[e], off[e + 1])
            ref.mm_close(out[r], x[r], xs[r], w[e], ws[e])
    assert (out[:2] == -3).all() and (out[off[-1]:] == -3).all() and ops.context(0).status_word() == 0


@pytest.mark.parametrize("m,n,k", [(1, 5, 16), (3, 129, 130), (5, 64, 272), (17, 130, 144), (70, 300, 400)])
def test_products(m, n, k, kernel):
    from metaltile_b200 import ops
    x, xs, w, ws = _operands(m, n, k, m + n + k)
    for dt in TYPES.values():
        ref.mm_close(ops.fp8_mm(x, w, ws, x_scales=xs, out_dtype=dt), x, xs, w, ws)


@pytest.mark.parametrize("k", [400, 393])
@pytest.mark.parametrize("m", [1, 9, 40])
def test_special_values(m, k, kernel):
    """NaN codes and NaN scales reach their rows and columns and no others; scales of zero take their block out; infinite results are infinite."""
    from metaltile_b200 import ops
    x, xs, w, ws = _operands(m, 300, k, 11)
    row, col = m // 2, 137
    x.view(torch.uint8)[row, 333] = 0x7F
    w.view(torch.uint8)[col, 5] = 0xFF
    xs[0, 1], ws[2, 3], ws[0, 2] = 0.0, 2.0 ** 60, float("nan")
    out = ops.fp8_mm(x, w, ws, x_scales=xs, out_dtype=torch.float32)
    nan = torch.zeros(m, 300, dtype=torch.bool, device="cuda")
    nan[row], nan[:, col], nan[:, :128] = True, True, True
    assert torch.equal(torch.isnan(out), nan)
    x.view(torch.uint8)[row, 333], w.view(torch.uint8)[col, 5], ws[0, 2] = 0, 0, 1.0
    want, size = ref.mm(x, xs, w, ws)
    tol = ref.STEP[torch.float32] * want.abs() + (128 + ref.blocks(k) + 4) * 2.0 ** -23 * size
    assert ((out.double() - want).abs() <= tol)[~nan].all()
    big = ops.fp8_mm(x, w, ws * 2.0 ** 40, x_scales=xs, out_dtype=torch.float16)[:, 256:]
    over = want[:, 256:] * 2.0 ** 40
    assert torch.equal(torch.isinf(big), over.abs() >= 65520.0) and torch.equal(torch.sign(big.double())[torch.isinf(big)], torch.sign(over)[torch.isinf(big)])

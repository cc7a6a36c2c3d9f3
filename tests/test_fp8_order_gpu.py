"""The 8-bit float products between other work: launches right behind each other, chunks that a launch was sized for and that do not come, long predecessors."""
import pytest
import torch

import fp8_ref as ref

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


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


def test_kernels_that_follow_each_other_on_the_same_SMs():
    """A CTA leaves only when the tensor core's last arrivals at its barriers have come: short ends (few columns) and other kernels in the same shared memory right behind them."""
    from metaltile_b200 import ops
    ctx = ops.context(0)
    cases = [(3, 300, 8, 640), (3, 257, 264, 128), (2, 20, 8, 512), (3, 40, 130, 4096), (2, 200, 64, 128), (3, 1000, 16, 384)]
    args = [_operands(m, n, k, 10 * i) for i, (_, m, n, k) in enumerate(cases)]
    e = 5
    x, xs, w, ws = _operands(300, 24, 256, 99, experts=e)
    off = torch.tensor([0, 130, 130, 131, 290, 300], device="cuda", dtype=torch.int32)

    def one(i):
        ctx.set_option("fp8_kernel", cases[i][0])
        return ops.fp8_mm(args[i][0], args[i][2], args[i][3], x_scales=args[i][1])

    def grouped(kernel):
        ctx.set_option("fp8_kernel", kernel)
        return ops.fp8_gather_mm(x, w, ws, off, xs)

    try:
        torch.cuda.synchronize()
        want, groups = [one(i) for i in range(len(cases))], [grouped(2), grouped(3)]
        for (_, m, n, k), a, o in zip(cases, args, want):
            ref.mm_close(o, *a)
        got = [[one(i) for i in range(len(cases))] + [grouped(2), grouped(3)] for _ in range(60)]
        assert all(torch.equal(g, v) for row in got for g, v in zip(row, want + groups))
        assert ctx.status_word() == 0
    finally:
        ctx.set_option("fp8_kernel", 0)


@pytest.mark.parametrize("kernel", [2, 3])
def test_far_fewer_chunks_than_a_launch_is_sized_for(kernel):
    """The number of chunks is counted on the device; where rows belong to nobody it is far below what the host reckons with."""
    from metaltile_b200 import ops
    ctx = ops.context(0)
    x, xs, w, ws = _operands(4000, 200, 384, 7, experts=64)
    offs = [torch.full((65,), 17, dtype=torch.int32), torch.tensor([5] * 30 + [9] * 35, dtype=torch.int32), torch.tensor([0] * 64 + [3], dtype=torch.int32)]
    ctx.set_option("fp8_kernel", kernel)
    try:
        for off in offs:
            on_device = off.cuda()
            out = torch.full((4000, 200), -3.0, device="cuda", dtype=torch.bfloat16)
            for _ in range(50):
                ops.fp8_gather_mm(x, w, ws, on_device, xs, out=out)
            at = off.tolist()
            for e in range(64):
                r = slice(at[e], at[e + 1])
                if at[e + 1] > at[e]:
                    ref.mm_close(out[r], x[r], xs[r], w[e], ws[e])
            assert (out[:at[0]] == -3).all() and (out[at[-1]:] == -3).all()
        assert ctx.status_word() == 0
    finally:
        ctx.set_option("fp8_kernel", 0)


@pytest.mark.parametrize("m,n,k", [(1, 2048, 2048), (40, 512, 2880), (64, 14336, 512), (300, 384, 1024)])
def test_a_product_behind_a_kernel_that_lets_it_start_long_before_its_end(m, n, k):
    """A barrier of peers one of which does not come (its limit of polls ends it after some hundredths of a second) lets the next kernels of the stream start at once: no role of
    theirs may count that time against the limit of its own waits."""
    from metaltile_b200 import ops
    ctx = ops.context(0)
    _, _, w, ws = _operands(1, n, k)
    x = torch.randn(m, k, device="cuda", generator=_gen(5)).bfloat16()
    codes, scales = ops.fp8_quantize(x)
    want = ops.fp8_mm(x, w, ws)
    mine, absent = (torch.zeros(64, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream().cuda_stream
    ctx.set_option("peer_poll_limit", 300000)
    try:
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        ctx.peer_barrier([mine.data_ptr(), absent.data_ptr()], 0, mine.data_ptr(), mine.data_ptr() + 128, stream=stream)
        got = [ops.fp8_mm(codes, w, ws, x_scales=scales, out_dtype=x.dtype), ops.fp8_mm(x, w, ws)]
        end.record()
        torch.cuda.synchronize()
        assert start.elapsed_time(end) > 30 and ctx.status_word() == 0x602             # the barrier's report, and none of the products'
        assert all(torch.equal(g, want) for g in got)
    finally:
        ctx.set_option("peer_poll_limit", 1 << 22)
        ctx.status_clear()

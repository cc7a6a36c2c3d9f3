"""The products in 8-bit floating point and the router's balance loss, as cases that can be timed and compared.

Every case is one call, or the calls of one step, of ``metaltile_b200.ops``.  Kinds:

``quantize``  float rows or a float weight matrix -> e4m3 codes with an f32 scale for each block of 128 (``ops.fp8_quantize``)
``mm``        activations times a weight matrix in that format (``ops.fp8_mm``), from codes or from float activations
``gather``    the same product of rows sorted by expert with stacked expert matrices (``ops.fp8_gather_mm``)
``balance``   the balance loss of a router with its per-expert counts, and the gradient of the logits (``ops.moe_balance``,
              ``ops.moe_balance_grad``): one training step of the router

The plain forms are elementary torch operations in 32 bits; the quotient that a code is rounded from, which may lie next to a border
between two codes, and the sums over all rows of a batch are in 64.
"""
import math

import torch

own = False                                     # True: the package's operators, False: their plain forms

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_B = 128                                        # values that share a scale
_LEAST = 2.0 ** -90                             # the least scale


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # The activations of one token before a projection: the smallest call there is, launch and host time count.
        dict(name="quantize_m1", kind="quantize", rows=1, k=4096, block_rows=1, pow2=False, top_k=0, dtype="bf16"),
        # A prompt's tokens put into expert order and quantized at once, in front of the experts' products (scales powers of two).
        dict(name="quantize_sorted", kind="quantize", rows=512, k=2048, block_rows=1, pow2=True, top_k=8, dtype="bf16"),
        # A feed-forward matrix quantized while a model is loaded: blocks of 128 x 128.
        dict(name="quantize_weight", kind="quantize", rows=14336, k=4096, block_rows=128, pow2=False, top_k=0, dtype="bf16"),
        # One attention projection for one token, from its float activations: single-user generation.
        dict(name="mm_m1", kind="mm", m=1, n=4096, k=4096, codes=False, dtype="bf16"),
        # The gate or up projection for sixteen users that decode together.
        dict(name="mm_m16", kind="mm", m=16, n=14336, k=4096, codes=True, dtype="bf16"),
        # A short prompt of no round length on a model whose rows end inside a block (2880 = 22.5 blocks).
        dict(name="mm_ragged", kind="mm", m=333, n=7616, k=2880, codes=True, dtype="f16"),
        # A long prompt through the fused gate and up matrices.
        dict(name="mm_2048", kind="mm", m=2048, n=28672, k=4096, codes=True, dtype="bf16"),
        # A layer of many small experts while four users decode: few experts are hit, each by a row or two.
        dict(name="gather_4", kind="gather", tokens=4, top_k=8, experts=128, n=768, k=2048, dtype="bf16"),
        # The same layer with a prompt of 512 tokens: a few dozen rows an expert.
        dict(name="gather_512", kind="gather", tokens=512, top_k=8, experts=128, n=768, k=2048, dtype="bf16"),
        # The down product of a layer of few experts over a long prompt: hundreds of rows an expert, ragged, f32 sums kept.
        dict(name="gather_4096", kind="gather", tokens=4096, top_k=2, experts=8, n=4096, k=1536, dtype="f32"),
        # The router of that layer of many experts in a training step of 4096 tokens.
        dict(name="balance_4096", kind="balance", rows=4096, experts=128, top_k=8, masked=False, dtype="bf16"),
        # A large batch of padded sequences with f32 logits.
        dict(name="balance_65536", kind="balance", rows=65536, experts=256, top_k=8, masked=True, dtype="f32"),
    ]


_MOST_OPS = 2048 * 28672 * 4096                 # of the largest listed product
_MOST_VALUES = 14336 * 4096                     # of the largest listed matrix


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _length(rng, lo, hi):
    """A row length: whole blocks half of the time, else any multiple of 16."""
    step = _B if rng.random() < 0.5 else 16
    return max(step, _log(rng, lo, hi) // step * step)


def draw(rng):
    kind = rng.choice(("quantize", "mm", "mm", "mm", "gather", "gather", "balance"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "quantize":
        block_rows = rng.choice((1, 1, _B))
        top_k = rng.choice((0, 2, 8)) if block_rows == 1 else 0
        k = _length(rng, 256, 14336)
        most = max(1, min(14336, _MOST_VALUES // k) // max(1, top_k))
        return dict(kind=kind, rows=_log(rng, 1, most), k=k, block_rows=block_rows, pow2=rng.random() < 0.5, top_k=top_k, dtype=dtype)
    if kind == "mm":
        n, k = _log(rng, 256, 28672), _length(rng, 256, 14336)
        m = _log(rng, 1, min(2048, _MOST_OPS // (n * k)))
        return dict(kind=kind, m=m, n=n, k=k, codes=rng.random() < 0.6, dtype=dtype)
    if kind == "gather":
        experts, top_k = rng.choice((8, 16, 32, 64, 128)), rng.choice((1, 2, 4, 8))
        n, k = _log(rng, 256, 4096), _length(rng, 256, 2048)
        while experts * n * k > 128 * 768 * 2048:
            n = max(128, n // 2)
        return dict(kind=kind, tokens=_log(rng, 1, 8192 // top_k), top_k=top_k, experts=experts, n=n, k=k, dtype=dtype)
    return dict(kind=kind, rows=_log(rng, 1, 65536), experts=rng.choice((8, 16, 60, 64, 128, 160, 256)), top_k=rng.choice((1, 2, 6, 8)),
                masked=rng.random() < 0.5, dtype=dtype)


# ---- inputs ------------------------------------------------------------------------------------------------------
class _Maker:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(shape, device="cuda", generator=self.gen)

    def activations(self, rows, k, dtype):
        """Normal, with channels that are louder than the others, as activations have them."""
        return (self.normal(rows, k) * (1 + 2 * self.normal(k).abs() ** 3)).to(_DT[dtype])

    def weights(self, *shape):
        """Codes and scales of normal weights: the values matter little here, so the codes are drawn as rounded normals."""
        codes = (self.normal(*shape) * 120).clamp(-448, 448).to(torch.float8_e4m3fn)
        scales = (0.5 + torch.rand(*shape[:-2], -(-shape[-2] // _B), -(-shape[-1] // _B), device="cuda", generator=self.gen)) * 2e-4
        return codes, scales

    def routed(self, tokens, experts, top_k, spread=1.0):
        """The top_k experts of each token of a router that favours some."""
        logits = self.normal(tokens, experts) + spread * self.normal(experts)
        return logits, torch.topk(logits, top_k, dim=1).indices.to(torch.int32)


def prepare(case, seed):
    make, kind = _Maker(seed), case["kind"]
    state = dict(case)
    if kind == "quantize":
        state["x"] = make.activations(case["rows"], case["k"], case["dtype"])
        if case["block_rows"] != 1:
            state["x"] = (make.normal(case["rows"], case["k"]) * 0.02).to(_DT[case["dtype"]])
        state["order"] = None
        if case["top_k"]:
            state["order"] = torch.randperm(case["rows"] * case["top_k"], device="cuda", generator=make.gen).div(case["top_k"], rounding_mode="floor").to(torch.int32)
    elif kind == "mm":
        x = make.activations(case["m"], case["k"], case["dtype"])
        state["x"], state["x_scales"] = _quantize(x, 1, False, None) if case["codes"] else (x, None)
        state["w"], state["w_scales"] = make.weights(case["n"], case["k"])
    elif kind == "gather":
        _, idx = make.routed(case["tokens"], case["experts"], case["top_k"])
        owner, order = torch.sort(idx.reshape(-1).long(), stable=True)
        state["owner"] = owner
        counts = torch.zeros(case["experts"], dtype=torch.int64, device="cuda").index_add_(0, owner, torch.ones_like(owner))
        state["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        x = make.activations(case["tokens"], case["k"], "bf16")[order // case["top_k"]]
        state["x"], state["x_scales"] = _quantize(x, 1, False, None)
        state["w"], state["w_scales"] = make.weights(case["experts"], case["n"], case["k"])
    else:
        logits, idx = make.routed(case["rows"], case["experts"], case["top_k"])
        state["logits"], state["idx"] = logits.to(_DT[case["dtype"]]), idx
        state["coef"] = 0.01
        state["grad_loss"] = make.normal(1).abs()[0] + 0.5          # the scale that a loss gets on its way back
        state["mask"] = None
        if case["masked"]:                                          # sequences of 512 rows whose ends are padding
            length = torch.randint(1, 513, (-(-case["rows"] // 512),), device="cuda", generator=make.gen)
            at = torch.arange(case["rows"], device="cuda")
            state["mask"] = at % 512 < length[at // 512]
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _blocks(x, block_rows):
    """x [R, K] with zeros behind its ends as [R / block_rows, block_rows, K / 128, 128]."""
    r, k = x.shape
    x = torch.nn.functional.pad(x, (0, -k % _B, 0, -r % block_rows))
    return x.reshape(x.shape[0] // block_rows, block_rows, x.shape[1] // _B, _B)


def _quantize(x, block_rows, pow2, order):
    if order is not None:
        x = x[order.long()]
    r, k = x.shape
    v = _blocks(x.float(), block_rows)
    scale = (v.abs().amax(dim=(1, 3)).double() / 448).float().clamp_min(_LEAST)      # rounded once: torch divides by a number in two steps
    if pow2:
        mantissa, exponent = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), exponent - (mantissa == 0.5).int())
    q = (v.double() / scale.double()[:, None, :, None]).clamp(-448.0, 448.0)
    # to the nearest of e4m3's values, ties to the even one: steps of 2^(e-3) from 2^e on, of 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    q = torch.round(q / step) * step
    return q.float().to(torch.float8_e4m3fn).reshape(-1, v.shape[2] * _B)[:r, :k].contiguous(), scale


def _values(codes, scales, block_rows):
    """What codes [R, K] stand for, in the type of the scales."""
    r, k = codes.shape
    s = scales.repeat_interleave(block_rows, dim=0)[:r] if block_rows != 1 else scales
    return codes.to(scales.dtype) * s.repeat_interleave(_B, dim=1)[:, :k]


def _balance(s):
    z, idx, mask, e = s["logits"].float(), s["idx"].long(), s["mask"], s["experts"]
    rows = z.shape[0]
    valid = torch.ones(rows, dtype=torch.bool, device=z.device) if mask is None else mask
    top = z.amax(dim=1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(dim=1, keepdim=True)
    p = torch.where(valid[:, None] & (total > 0), p / total, torch.zeros_like(p))
    n = valid.sum()
    each = valid[:, None].expand(-1, idx.shape[1]).reshape(-1).to(torch.int32)
    counts = torch.zeros(e, dtype=torch.int32, device=z.device).index_add_(0, idx.reshape(-1), each)
    safe = n.clamp_min(1).double()
    mean = p.double().sum(dim=0) / safe
    share = counts.double() / (safe * idx.shape[1])
    loss = s["coef"] * e * (share * mean).sum()
    share = share.float()
    grad = (s["grad_loss"].double() * s["coef"] * e / safe).float() * p * (share - (p * share).sum(dim=1, keepdim=True))
    return loss.float(), counts, mean.float(), n.to(torch.int32), grad.to(s["logits"].dtype)


def _plain(s):
    kind = s["kind"]
    if kind == "quantize":
        return _quantize(s["x"], s["block_rows"], s["pow2"], s["order"])
    if kind == "balance":
        return _balance(s)
    if kind == "mm":
        codes, scales = (s["x"], s["x_scales"]) if s["x_scales"] is not None else _quantize(s["x"], 1, False, None)
        return (_values(codes, scales, 1) @ _values(s["w"], s["w_scales"], _B).T).to(_DT[s["dtype"]])
    x = _values(s["x"], s["x_scales"], 1)
    out = torch.zeros(x.shape[0], s["n"], device="cuda")
    for e in range(s["experts"]):               # no host copy of the offsets: every expert meets all rows, the others' as zeros
        out += (x * (s["owner"] == e)[:, None]) @ _values(s["w"][e], s["w_scales"][e], _B).T
    return out.to(_DT[s["dtype"]])


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    if not own:
        return _plain(s)
    from metaltile_b200 import ops

    kind = s["kind"]
    if kind == "quantize":
        return ops.fp8_quantize(s["x"], block_rows=s["block_rows"], pow2=s["pow2"], rows=s["order"])
    if kind == "mm":
        return ops.fp8_mm(s["x"], s["w"], s["w_scales"], x_scales=s["x_scales"], out_dtype=_DT[s["dtype"]])
    if kind == "gather":
        return ops.fp8_gather_mm(s["x"], s["w"], s["w_scales"], s["offsets"], x_scales=s["x_scales"], out_dtype=_DT[s["dtype"]])
    loss, counts, mean, n = ops.moe_balance(s["logits"], s["idx"], coef=s["coef"], mask=s["mask"])
    grad = ops.moe_balance_grad(s["logits"], counts, n, s["top_k"], grad_loss=s["grad_loss"], coef=s["coef"], mask=s["mask"])
    return loss, counts, mean, n, grad


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def _scales(rows, k, block_rows=1):
    return 4 * -(-rows // block_rows) * -(-k // _B)


def work(case):
    c, size = case, _SIZE[case["dtype"]]
    if c["kind"] == "quantize":
        rows = c["rows"] * max(1, c["top_k"])
        return {"bytes": c["rows"] * c["k"] * size + rows * c["k"] + _scales(rows, c["k"], c["block_rows"]) + (4 * rows if c["top_k"] else 0), "flops": 3 * rows * c["k"]}
    if c["kind"] == "mm":
        x = c["m"] * c["k"] + _scales(c["m"], c["k"]) if c["codes"] else c["m"] * c["k"] * size
        return {"bytes": x + c["n"] * c["k"] + _scales(c["n"], c["k"], _B) + c["m"] * c["n"] * size, "flops": 2 * c["m"] * c["n"] * c["k"]}
    if c["kind"] == "gather":
        rows = c["tokens"] * c["top_k"]
        hit = c["experts"] * (1 - (1 - c["top_k"] / c["experts"]) ** c["tokens"])       # experts that a uniform router reaches
        return {"bytes": int(hit * (c["n"] * c["k"] + _scales(c["n"], c["k"], _B))) + rows * c["k"] + _scales(rows, c["k"]) + rows * c["n"] * size,
                "flops": 2 * rows * c["n"] * c["k"]}
    cells = c["rows"] * c["experts"]
    return {"bytes": 2 * cells * size + 4 * c["rows"] * c["top_k"] + (c["rows"] if c["masked"] else 0) + 8 * c["experts"], "flops": 14 * cells}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------
def _e4m3(v):
    """The finite values of e4m3 from the bits: sign, four bits of exponent (bias 7), three of mantissa."""
    codes = torch.arange(127, dtype=torch.float64, device=v.device)
    exponent, mantissa = torch.div(codes, 8, rounding_mode="floor"), codes % 8
    table = torch.where(exponent == 0, mantissa * 2.0 ** -9, (8 + mantissa) * torch.exp2(exponent - 10))
    a = v.abs().contiguous()
    up = torch.searchsorted(table, a).clamp(max=126)
    down = (up - 1).clamp(min=0)
    low, high = table[down], table[up]
    take_up = (a - low > high - a) | ((a - low == high - a) & (up % 2 == 0))
    return torch.where(take_up, high, low) * torch.sign(v)


def _exact_quantize(x, block_rows, pow2, order):
    x = x if order is None else x[order.long()]
    r, k = x.shape
    scales = torch.empty(-(-r // block_rows), -(-k // _B), dtype=torch.float64, device=x.device)
    codes = torch.empty(r, k, dtype=torch.float64, device=x.device)
    for b in range(scales.shape[1]):
        v = x[:, b * _B:(b + 1) * _B].double()
        most = v.abs().amax(dim=1)
        if block_rows != 1:
            most = torch.nn.functional.pad(most, (0, -r % block_rows)).reshape(-1, block_rows).amax(dim=1)
        s = torch.clamp((most / 448).float().double(), min=_LEAST)          # a scale is held in 32 bits: codes are relative to what is held
        if pow2:
            s = ((s.view(torch.int64) + (2 ** 52 - 1)) >> 52 << 52).view(torch.float64)       # the next power of two: no mantissa
        scales[:, b] = s
        codes[:, b * _B:(b + 1) * _B] = _e4m3(v / s.repeat_interleave(block_rows)[:r, None])
    return codes, scales


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "quantize":
        return _exact_quantize(s["x"], s["block_rows"], s["pow2"], s["order"])
    if kind == "mm":
        if s["x_scales"] is None:
            codes, scales = _exact_quantize(s["x"], 1, False, None)
        else:
            codes, scales = s["x"].double(), s["x_scales"].double()
        out = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        row_block = torch.arange(case["n"], device="cuda") // _B
        for b in range(scales.shape[1]):
            cut = slice(b * _B, (b + 1) * _B)
            out += codes[:, cut] @ s["w"][:, cut].double().T * scales[:, b:b + 1] * s["w_scales"].double()[row_block, b]
        return out
    if kind == "gather":
        out = torch.zeros(s["x"].shape[0], case["n"], dtype=torch.float64, device="cuda")
        at = s["offsets"].tolist()
        row_block = torch.arange(case["n"], device="cuda") // _B
        for e in range(case["experts"]):
            rows = slice(at[e], at[e + 1])
            for b in range(s["x_scales"].shape[1]):
                cut = slice(b * _B, (b + 1) * _B)
                out[rows] += (s["x"][rows, cut].double() @ s["w"][e][:, cut].double().T * s["x_scales"][rows, b:b + 1].double()
                              * s["w_scales"][e].double()[row_block, b])
        return out
    rows = slice(None) if s["mask"] is None else torch.nonzero(s["mask"]).reshape(-1)
    z, idx, e = s["logits"].double()[rows], s["idx"][rows].long(), case["experts"]
    n, k = idx.shape
    p = torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True))
    counts = torch.bincount(idx.reshape(-1), minlength=e)
    f, mean = counts.double() / (n * k), p.mean(dim=0)
    g = torch.zeros(case["rows"], e, dtype=torch.float64, device="cuda")
    g[rows] = s["grad_loss"].double() * s["coef"] * e / n * p * (f - (p @ f)[:, None])
    return s["coef"] * e * (f @ mean), None, mean, None, g

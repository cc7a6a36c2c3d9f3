"""What stands in front of a projection and beside it, as cases that can be timed and compared: the norm with the residual's addition and low-rank adapters.

Every case is one call, or the calls of one step, of ``metaltile_b200.ops``.  Kinds:

``norm``       residual stream + root-mean-square norm, results in the type of the activations (``ops.add_rms_norm``)
``norm_fp8``   the same with the normalised rows as e4m3 codes with an f32 scale for each block of 128 (``ops.add_rms_norm_fp8``)
``norm_grad``  its gradients (``ops.add_rms_norm_grad``)
``lora``       low-rank adapters of many requests added to the result of a shared projection (``ops.lora_mm``)
``train``      one training step of such adapters: the same with what the gradients need kept, and the gradients (``ops.lora_grad``)

The plain forms are elementary torch operations in 32 bits; what an e4m3 code is rounded from, which may lie next to a border between two
codes, and the sums over all rows of a batch are in 64.
"""
import math

import torch

own = False                                     # True: the package's operators, False: their plain forms

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_B = 128                                        # values that share a scale
_LEAST = 2.0 ** -90                             # the least scale
_EPS = 1e-5


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # The norm in front of a layer's projections for one token: the smallest call there is, launch and host time count.
        dict(name="norm_m1", kind="norm", rows=1, k=4096, residual=True, dtype="bf16"),
        # The same for a long prompt.
        dict(name="norm_2048", kind="norm", rows=2048, k=4096, residual=True, dtype="bf16"),
        # A short prompt of no round length whose rows end inside a block of the codes (2880 = 22.5 blocks), scales powers of two.
        dict(name="fp8_ragged", kind="norm_fp8", rows=333, k=2880, residual=True, pow2=True, dtype="f16"),
        # A batch of long prompts in front of 8-bit products.
        dict(name="fp8_8192", kind="norm_fp8", rows=8192, k=4096, residual=True, pow2=False, dtype="bf16"),
        # Fine-tuning in full precision on one short sequence.
        dict(name="grad_ragged", kind="norm_grad", rows=333, k=2880, residual=False, dtype="f32"),
        # A training batch, with the gradient that comes down the residual stream.
        dict(name="grad_8192", kind="norm_grad", rows=8192, k=4096, residual=True, dtype="bf16"),
        # One token of one user beside an attention projection.
        dict(name="lora_m1", kind="lora", rows=1, k=4096, n=4096, rank=16, adapters=4, run=1, none=0.0, dtype="bf16"),
        # Sixty-four users that decode together, each with one of 32 adapters, beside a gate or up projection.
        dict(name="lora_m64", kind="lora", rows=64, k=4096, n=14336, rank=16, adapters=32, run=1, none=0.1, dtype="bf16"),
        # A few prompts of no round length, some of them without an adapter, and a rank that is no power of two.
        dict(name="lora_ragged", kind="lora", rows=333, k=2880, n=7616, rank=24, adapters=3, run=47, none=0.2, dtype="f16"),
        # Prompts of eight users with adapters of a high rank.
        dict(name="lora_2048", kind="lora", rows=2048, k=4096, n=4096, rank=64, adapters=8, run=256, none=0.0, dtype="bf16"),
        # Fine-tuning in full precision, a small model and a low rank.
        dict(name="train_512", kind="train", rows=512, k=2048, n=768, rank=8, adapters=1, run=512, none=0.0, dtype="f32"),
        # Four fine-tuning jobs that share a batch.
        dict(name="train_4096", kind="train", rows=4096, k=4096, n=4096, rank=16, adapters=4, run=512, none=0.0, dtype="bf16"),
    ]


_MOST_BYTES = 8192 * 4096 * 2                   # of the largest listed activations


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _length(rng, lo, hi):
    """A row length: whole blocks half of the time, else any multiple of 8, and sometimes any number."""
    v, step = _log(rng, lo, hi), rng.choice((_B, _B, _B, 8, 8, 1))
    return max(step, v // step * step)


def draw(rng):
    kind = rng.choice(("norm", "norm_fp8", "norm_grad", "lora", "lora", "lora", "train", "train"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    size = _SIZE[dtype]
    if kind in ("norm", "norm_fp8", "norm_grad"):
        k = _length(rng, 64, 14336)
        case = dict(kind=kind, rows=_log(rng, 1, max(1, min(16384, _MOST_BYTES // (k * size)))), k=k, residual=rng.random() < 0.7, dtype=dtype)
        return dict(case, pow2=rng.random() < 0.5) if kind == "norm_fp8" else case
    rank, k, n = rng.choice((4, 8, 8, 16, 16, 16, 24, 32, 64)), _length(rng, 256, 14336), _length(rng, 256, 14336)
    most = max(1, min(4096, _MOST_BYTES // 2 // (max(k, n) * size), 2048 * 8192 * 64 // ((k + n) * rank)))
    if kind == "train":
        rows, adapters = _log(rng, min(32, most), most), rng.choice((1, 1, 2, 4, 8))
        return dict(kind=kind, rows=rows, k=k, n=n, rank=rank, adapters=adapters, run=rng.choice((32, 100, 512)), none=rng.choice((0.0, 0.2)), dtype=dtype)
    rows = _log(rng, 1, most)
    adapters = rng.choice((1, 2, 4, 8, 16, 32, 64))
    while adapters * rank * (k + n) > 64 * 16 * 18432:
        adapters = max(1, adapters // 2)
    return dict(kind=kind, rows=rows, k=k, n=n, rank=rank, adapters=adapters, run=1 if rows <= 128 else rng.choice((16, 100, 256)), none=rng.choice((0.0, 0.1, 0.3)),
                dtype=dtype)


# ---- inputs ------------------------------------------------------------------------------------------------------
class _Maker:
    """Seeded inputs on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(int(seed))

    def normal(self, *shape):
        return torch.randn(shape, device="cuda", generator=self.gen)

    def uniform(self, *shape):
        return torch.rand(shape, device="cuda", generator=self.gen)

    def activations(self, rows, k, dtype):
        """Normal, with channels that are louder than the others, as activations have them."""
        return (self.normal(rows, k) * (1 + self.normal(k).abs() ** 3)).to(_DT[dtype])

    def owners(self, case):
        """The adapter of every row, `adapters` for those that have none: runs of rows are a request."""
        requests = -(-case["rows"] // case["run"])
        ids = torch.randint(0, case["adapters"], (requests,), device="cuda", generator=self.gen)
        ids = torch.where(self.uniform(requests) < case["none"], torch.full_like(ids, case["adapters"]), ids)
        return ids.repeat_interleave(case["run"])[:case["rows"]]


def prepare(case, seed):
    make, kind = _Maker(seed), case["kind"]
    state, dt = dict(case), _DT[case["dtype"]]
    rows, k = case["rows"], case["k"]
    if kind in ("norm", "norm_fp8", "norm_grad"):
        state["x"] = make.activations(rows, k, case["dtype"])
        state["weight"] = (1 + 0.2 * make.normal(k)).to(dt)
        state["other"] = make.activations(rows, k, case["dtype"]) if case["residual"] else None      # the residual stream, or the gradient that comes down it
        state["dy"] = make.normal(rows, k).to(dt) if kind == "norm_grad" else None
        return state
    n, rank, adapters = case["n"], case["rank"], case["adapters"]
    state["x"] = make.normal(rows, k).to(dt)
    state["base"] = make.normal(rows, n).to(dt)                     # what the shared projection gave
    state["a"] = (make.normal(adapters, rank, k) / math.sqrt(k)).to(dt)
    state["b"] = (make.normal(adapters, n, rank) * (0.5 / math.sqrt(rank))).to(dt)
    state["scales"] = 0.5 + make.uniform(adapters)
    # A step sorts its rows once for all projections of all layers (``ops.moe_sort``); rows without an adapter come last.
    state["ids"] = make.owners(case)
    state["order"] = torch.sort(state["ids"], stable=True).indices.to(torch.int32)
    counts = (state["ids"][:, None] == torch.arange(adapters + 1, device="cuda")).sum(dim=0)
    state["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    if kind == "train":
        state["dy"] = make.normal(rows, n).to(dt)
        state["dx"] = make.normal(rows, k).to(dt)                   # the gradient that the shared projection gave
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _sum(s):
    return s["x"] if s["other"] is None else (s["x"].float() + s["other"].float()).to(s["x"].dtype)


def _norm(s):
    total = _sum(s)
    v = total.float()
    y = v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + _EPS) * s["weight"].float()
    return y.to(total.dtype), total


def _norm_fp8(s):
    total = _sum(s)
    r, k = total.shape
    v = total.double()
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + _EPS) * s["weight"].double()
    y = torch.nn.functional.pad(y, (0, -k % _B)).reshape(r, -1, _B)
    scale = (y.abs().amax(dim=2) / 448).float().clamp_min(_LEAST)
    if s["pow2"]:
        mantissa, exponent = torch.frexp(scale)
        scale = torch.ldexp(torch.ones_like(scale), exponent - (mantissa == 0.5).int())
    q = (y / scale.double()[:, :, None]).clamp(-448.0, 448.0)
    # to the nearest of e4m3's values, ties to the even one: steps of 2^(e-3) from 2^e on, of 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    q = torch.round(q / step) * step
    return q.float().to(torch.float8_e4m3fn).reshape(r, -1)[:, :k].contiguous(), scale, total


def _norm_grad(s):
    v, dy, w = s["x"].float(), s["dy"].float(), s["weight"].float()
    inv = torch.rsqrt((v * v).mean(dim=1, keepdim=True) + _EPS)
    n = v * inv
    g = dy * w
    dx = inv * (g - n * (g * n).mean(dim=1, keepdim=True))
    if s["other"] is not None:
        dx = dx + s["other"].float()
    return dx.to(s["x"].dtype), (dy * n).sum(dim=0, dtype=torch.float64).to(s["x"].dtype)


def _owned(s):
    """[rows, adapters], one where the row has the adapter."""
    return (s["ids"][:, None] == torch.arange(s["adapters"], device="cuda")).float()


def _low(v, w, owned):
    """v [rows, c] through every adapter's w [adapters, r, c], zeros where the row has another: [rows, adapters, r]."""
    return (v @ w.reshape(-1, w.shape[2]).T).reshape(v.shape[0], w.shape[0], w.shape[1]) * owned[:, :, None]


def _lora(s):
    x, a, b, owned = s["x"].float(), s["a"].float(), s["b"].float(), _owned(s)
    h = _low(x, a, owned)
    out = s["base"].float() + (h * s["scales"][:, None]).flatten(1) @ b.transpose(1, 2).reshape(-1, s["n"])
    return out.to(s["x"].dtype), h


def _train(s):
    out, h = _lora(s)
    x, dy, a, b = s["x"].float(), s["dy"].float(), s["a"].float(), s["b"].float()
    u = _low(dy, b.transpose(1, 2).contiguous(), _owned(s)) * s["scales"][:, None]
    dx = s["dx"].float() + u.flatten(1) @ a.reshape(-1, s["k"])
    da = (u.flatten(1).T @ x).reshape(a.shape)
    db = ((h * s["scales"][:, None]).flatten(1).T @ dy).reshape(s["adapters"], s["rank"], s["n"]).transpose(1, 2).contiguous()
    t = s["x"].dtype
    return out, h.sum(dim=1), dx.to(t), da.to(t), db.to(t)


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    kind = s["kind"]
    if not own:
        return _lora(s)[0] if kind == "lora" else {"norm": _norm, "norm_fp8": _norm_fp8, "norm_grad": _norm_grad, "train": _train}[kind](s)
    from metaltile_b200 import ops

    if kind == "norm":
        return ops.add_rms_norm(s["x"], s["weight"], _EPS, residual=s["other"])
    if kind == "norm_fp8":
        return ops.add_rms_norm_fp8(s["x"], s["weight"], _EPS, residual=s["other"], pow2=s["pow2"])
    if kind == "norm_grad":
        return ops.add_rms_norm_grad(s["dy"], s["x"], s["weight"], _EPS, dsum=s["other"])
    if kind == "lora":
        return ops.lora_mm(s["x"], s["a"], s["b"], s["order"], s["offsets"], scales=s["scales"], base=s["base"])
    out, hidden = ops.lora_mm(s["x"], s["a"], s["b"], s["order"], s["offsets"], scales=s["scales"], base=s["base"], hidden=True)
    dx, da, db = ops.lora_grad(s["dy"], s["x"], s["a"], s["b"], s["order"], s["offsets"], hidden, scales=s["scales"], base=s["dx"])
    return out, hidden, dx, da, db


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    c, size = case, _SIZE[case["dtype"]]
    cells = c["rows"] * c["k"]
    if c["kind"] in ("norm", "norm_fp8"):
        moved = cells * size * (3 if c["residual"] else 1)          # read x (and the stream), write the stream
        return {"bytes": moved + c["k"] * size + (cells * size if c["kind"] == "norm" else cells + 4 * c["rows"] * -(-c["k"] // _B)), "flops": 5 * cells}
    if c["kind"] == "norm_grad":
        return {"bytes": cells * size * (4 if c["residual"] else 3) + 2 * c["k"] * size, "flops": 11 * cells}
    r, k, n, rank = c["rows"], c["k"], c["n"], c["rank"]
    requests, having = -(-r // c["run"]), 1 - c["none"]
    hit = c["adapters"] * (1 - (1 - having / c["adapters"]) ** requests)        # adapters that a uniform draw reaches
    forward = r * size * (having * k + 2 * n) + hit * rank * (k + n) * size
    if c["kind"] == "lora":
        return {"bytes": int(forward), "flops": int(2 * having * r * rank * (k + n))}
    # x, a and b are there once for both directions; h goes out and the gradients read what is left of dy and the shared gradient
    back = r * size * (2 * k + having * n) + 4 * r * rank + c["adapters"] * rank * (k + n) * size
    return {"bytes": int(forward + back), "flops": int(6 * having * r * rank * (k + n))}


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


def _root_mean_square(x, weight):
    return weight * x / (torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + _EPS) ** 0.5


def _exact_norm(s):
    total = s["x"].double() if s["other"] is None else s["x"].double() + s["other"].double()
    held = total.to(s["x"].dtype).double()                          # the stream is held in the type of the activations, and the norm is of what is held
    return _root_mean_square(held, s["weight"].double()), total


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "norm":
        return _exact_norm(s)
    if kind == "norm_fp8":
        y, total = _exact_norm(s)
        codes = torch.empty_like(y)
        scales = torch.empty(y.shape[0], -(-y.shape[1] // _B), dtype=torch.float64, device="cuda")
        for b in range(scales.shape[1]):
            v = y[:, b * _B:(b + 1) * _B]
            scale = torch.clamp((v.abs().amax(dim=1) / 448).float().double(), min=_LEAST)        # a scale is held in 32 bits: codes are relative to what is held
            if case["pow2"]:
                scale = ((scale.view(torch.int64) + (2 ** 52 - 1)) >> 52 << 52).view(torch.float64)       # the next power of two: no mantissa
            scales[:, b] = scale
            codes[:, b * _B:(b + 1) * _B] = _e4m3(v / scale[:, None])
        return codes, scales, total
    if kind == "norm_grad":
        x, w = s["x"].double().requires_grad_(), s["weight"].double().requires_grad_()
        dx, dw = torch.autograd.grad(_root_mean_square(x, w), (x, w), s["dy"].double())
        return (dx if s["other"] is None else dx + s["other"].double()), dw
    train = kind == "train"
    x, a, b = (s[name].double().requires_grad_(train) for name in ("x", "a", "b"))
    out = s["base"].double()
    hidden = torch.zeros(case["rows"], case["rank"], dtype=torch.float64, device="cuda")
    for e in range(case["adapters"]):
        mine = torch.nonzero(s["ids"] == e).reshape(-1)
        h = x[mine] @ a[e].T
        hidden[mine] = h.detach()
        out = out.index_add(0, mine, s["scales"][e].double() * (h @ b[e].T))
    if not train:
        return out
    dx, da, db = torch.autograd.grad(out, (x, a, b), s["dy"].double())
    return out.detach(), hidden, dx + s["dx"].double(), da, db

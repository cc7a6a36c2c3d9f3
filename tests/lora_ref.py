"""The norm with the residual's addition and low-rank adapters in 64 bits, and how far a kernel may be from them."""
import torch

STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}           # half a step, relative to the value
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}        # half a step of subnormals (f32: one)
F32 = 2.0 ** -24
# f32 sums of a row: a thread adds up at most 64 values in turn here, five exchanges in a warp and five over the warps
ROW = 64 + 10


# ---- norms -------------------------------------------------------------------------------------------------------------
def norm(s, w, eps):
    s, w = s.double(), w.double()
    return s / torch.sqrt((s * s).mean(dim=-1, keepdim=True) + eps) * w


def norm_bound(s, w, eps):
    """y: the sum of squares errs by ROW roundings, its root by half of that; the division by K, the sum with eps, the root, the reciprocal and two products by one each."""
    y = norm(s, w, eps).abs()
    return (STEP[s.dtype] + (ROW / 2 + 6) * F32) * y + TINY[s.dtype]


def norm_grad(dy, s, w, eps, dsum=None):
    dy, s, w = dy.double(), s.double(), w.double()
    inv = 1 / torch.sqrt((s * s).mean(dim=-1, keepdim=True) + eps)
    n, g = s * inv, dy * w
    dx = inv * (g - n * (g * n).mean(dim=-1, keepdim=True))
    return dx if dsum is None else dx + dsum.double(), (dy * n).reshape(-1, s.shape[-1]).sum(dim=0)


def norm_grad_bounds(dy, s, w, eps, dsum, rows_a_worker):
    dx, dw = norm_grad(dy, s, w, eps, dsum)
    t = s.dtype
    dy, s, w = dy.double().abs(), s.double().abs(), w.double().abs()
    inv = 1 / torch.sqrt((s * s).mean(dim=-1, keepdim=True) + eps)
    n, g = s * inv, dy * w
    # n errs by ROW / 2 + 5 of its own size, the mean of g n by that and ROW of the sum of magnitudes, and everything is rounded four more times
    size = inv * (g + n * (g * n).mean(dim=-1, keepdim=True))
    if dsum is not None:
        size = size + dsum.double().abs()
    cells = (dy * n).reshape(-1, s.shape[-1]).sum(dim=0)
    return (STEP[t] * dx.abs() + 2 * (ROW + 10) * F32 * size + TINY[t], STEP[t] * dw.abs() + (ROW / 2 + 6 + rows_a_worker) * F32 * cells + TINY[t])


# ---- adapters ----------------------------------------------------------------------------------------------------------
# What a row goes through is held in two pieces of 8 bits and more where weights are 16-bit, in three where they are f32: 16 and 24 bits.
PIECES = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -16, torch.bfloat16: 2.0 ** -16}


def group(ids, adapters):
    """(rows, offsets) as moe_sort makes them."""
    order = torch.sort(ids, stable=True).indices.to(torch.int32)
    counts = torch.stack([(ids == e).sum() for e in range(adapters + 1)])
    return order, torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)


def low(v, w, ids):
    """v [rows, c] through the w [adapters, rank, c] of each row's adapter, zeros for none."""
    h = torch.zeros(v.shape[0], w.shape[1], dtype=torch.float64, device=v.device)
    for e in range(w.shape[0]):
        mine = torch.nonzero(ids == e).reshape(-1)
        h[mine] = v[mine].double() @ w[e].double().T
    return h


def high(h, w, ids, scales, base, width):
    out = torch.zeros(h.shape[0], width, dtype=torch.float64, device=h.device) if base is None else base.double().clone()
    for e in range(w.shape[0]):
        mine = torch.nonzero(ids == e).reshape(-1)
        out[mine] += (1.0 if scales is None else scales[e].double()) * (h[mine] @ w[e].double())
    return out


def outer(h, v, ids, scales, adapters):
    """sum over the rows of an adapter of h[t] (x) v[t], [adapters, rank, c]"""
    g = torch.zeros(adapters, h.shape[1], v.shape[1], dtype=torch.float64, device=h.device)
    for e in range(adapters):
        mine = torch.nonzero(ids == e).reshape(-1)
        g[e] = (1.0 if scales is None else scales[e].double()) * (h[mine].T @ v[mine].double())
    return g


def lora(x, a, b, ids, scales, base):
    h = low(x, a, ids)
    return high(h, b.transpose(1, 2), ids, scales, base, b.shape[1]), h


def lora_grad(dy, x, a, b, ids, scales, base):
    u, h = low(dy, b.transpose(1, 2), ids), low(x, a, ids)
    n = a.shape[0]
    return (high(u, a, ids, scales, base, a.shape[2]), outer(u, x, ids, scales, n), outer(h, dy, ids, scales, n).transpose(1, 2))


def low_bound(v, w, ids):
    """At most c / 16 + 32 additions of products or of partial sums stand behind a value, and a tensor core may cut off what a rounding would round: two steps each."""
    c = v.shape[1]
    return 2 * (c / 16 + 32) * F32 * low(v.abs(), w.abs(), ids)


def high_bound(want, h, dh, w, ids, scales, base, dt):
    size = high(h.abs(), w.abs(), ids, scales.abs() if scales is not None else None, None, w.shape[2])
    err = high(dh + PIECES[dt] * h.abs(), w.abs(), ids, scales.abs() if scales is not None else None, None, w.shape[2])
    total = size if base is None else size + base.double().abs()
    return STEP[dt] * want.abs() + err + 2 * (h.shape[1] + 8) * F32 * total + TINY[dt]


def outer_bound(want, h, dh, v, ids, scales, adapters, dt):
    s = scales.abs() if scales is not None else None
    rows = v.shape[0]
    err = outer(dh + PIECES[dt] * h.abs(), v.abs(), ids, s, adapters)
    return STEP[dt] * want.abs() + err + 2 * (rows / 16 + 80) * F32 * outer(h.abs(), v.abs(), ids, s, adapters) + TINY[dt]

"""The 8-bit float format, its products and the balance loss in 64 bits, from their definitions (tests only)."""
import torch

B = 128
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # half a step, relative to the value
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}    # ... and near zero


def blocks(n):
    return -(-n // B)


def table():
    """The finite values of the codes 0 .. 126."""
    c = torch.arange(127, dtype=torch.float64)
    e, m = torch.div(c, 8, rounding_mode="floor"), c % 8
    return torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))


def nearest(v):
    """v (float64) to the nearest value of e4m3, ties to the even code; NaN and infinities stay NaN."""
    t = table().to(v.device)
    a = v.abs().clamp(max=448.0).nan_to_num(0.0).contiguous()
    up = torch.searchsorted(t, a).clamp(max=126)
    down = (up - 1).clamp(min=0)
    lo, hi = t[down], t[up]
    r = torch.where((a - lo > hi - a) | ((a - lo == hi - a) & (up % 2 == 0)), hi, lo) * torch.sign(v)
    return torch.where(torch.isfinite(v), r, torch.full_like(r, float("nan")))


def quantize(x, block_rows=1, pow2=False):
    """x [R, K] -> (values of the codes float64 [R, K], scales float64)."""
    r, k = x.shape
    v = x.double()
    finite = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v))
    p = torch.nn.functional.pad(finite, (0, -k % B, 0, -r % block_rows))
    amax = p.reshape(p.shape[0] // block_rows, block_rows, p.shape[1] // B, B).amax(dim=(1, 3))
    s = (amax / 448).float().double().clamp(min=2.0 ** -90)      # held in f32 (a quotient in 64 bits rounds to 32 as the true one does)
    if pow2:
        s = ((s.view(torch.int64) + (2 ** 52 - 1)) >> 52 << 52).view(torch.float64)
    full = spread(s, r, k, block_rows)
    q = torch.where(torch.isfinite(v), v / full, torch.full_like(v, float("nan")))
    return nearest(q), s


def spread(s, r, k, block_rows):
    return s.double().repeat_interleave(block_rows, 0)[:r].repeat_interleave(B, 1)[:, :k]


def mm(x, xs, w, ws):
    """(out, sum of magnitudes), both float64 [M, N]."""
    a, b = x.double() * spread(xs, *x.shape, 1), w.double() * spread(ws, *w.shape, B)
    return a @ b.T, a.abs() @ b.abs().T


def mm_close(got, x, xs, w, ws):
    """Within what f32 sums and one rounding of the result allow.  A product of codes is exact; each of the (at most 128) additions inside a block, each of those
    over blocks and the product of the two scales err by at most a step (2^-23: additions may truncate) of the sum of magnitudes."""
    ref, size = mm(x, xs, w, ws)
    tol = STEP[got.dtype] * ref.abs() + (min(B, x.shape[1]) + blocks(x.shape[1]) + 4) * 2.0 ** -23 * size + TINY[got.dtype]
    bad = (got.double() - ref).abs() > tol
    assert got.shape == ref.shape and not bad.any(), (int(bad.sum()), float(((got.double() - ref).abs() / tol).max()))


def softmax(logits):
    z = logits.double()
    top = z.amax(dim=1, keepdim=True)
    p = torch.exp(z - torch.where(top == -float("inf"), torch.zeros_like(top), top))
    total = p.sum(dim=1, keepdim=True)
    return torch.where(total > 0, p / total, torch.zeros_like(p))


def balance(logits, idx, coef, mask=None):
    """(loss, counts, mean probabilities, rows) in 64 bits."""
    e = logits.shape[1]
    keep = torch.ones(logits.shape[0], dtype=torch.bool, device=logits.device) if mask is None else mask.bool()
    p, ids = softmax(logits[keep]), idx[keep].long().reshape(-1)
    n, k = int(keep.sum()), idx.shape[1]
    counts = torch.bincount(ids[(ids >= 0) & (ids < e)], minlength=e)
    mean = p.sum(dim=0) / max(n, 1)
    f = counts.double() / max(n * k, 1)
    return coef * e * (f * mean).sum(), counts, mean, n


def balance_grad(logits, idx, coef, grad_loss=1.0, mask=None):
    keep = torch.ones(logits.shape[0], dtype=torch.bool, device=logits.device) if mask is None else mask.bool()
    _, counts, _, n = balance(logits, idx, coef, mask)
    f, p = counts.double() / max(n * idx.shape[1], 1), softmax(logits)
    g = grad_loss * coef * logits.shape[1] / max(n, 1) * p * (f - (p @ f)[:, None])
    return torch.where(keep[:, None], g, torch.zeros_like(g))

"""How many bits the pieces of a f32 value hold that a sum of their products has, without a GPU."""
import pytest
import torch


def _pieces(v, n):
    out = []
    for _ in range(n):
        out.append(v.to(torch.bfloat16).double())
        v = (v - out[-1]).float()
    return out


@pytest.mark.parametrize("n", [2, 3])
def test_a_lost_piece_shows(n):
    """What the GPU tests' border of 2^-19 of a result's root mean square lies between: three pieces of a value are all of it, two are not."""
    g = torch.Generator().manual_seed(1)
    x, a = torch.randn(64, 4096, generator=g), torch.randn(32, 4096, generator=g) / 64
    p, q = _pieces(x, n), _pieces(a, n)
    got = sum(p[i] @ q[j].T for i in range(n) for j in range(n) if i + j < n)
    want = x.double() @ a.double().T
    off = (got - want).square().mean().sqrt() / want.square().mean().sqrt()
    assert off < 2.0 ** -25 if n == 3 else off > 2.0 ** -18.5
    assert (sum(_pieces(x, 3)) == x.double()).all()

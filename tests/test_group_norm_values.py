"""torch.ops.mineral.group_norm_act where a small error shows: groups whose values are all alike, saturated activations, and offsets
beyond 32 bits.

A group of equal values has no spread: its normalised values are zero, and an error of one spacing in its mean would be divided by
sqrt(eps).  u = 2^-24: a sum is at most 64 roundings deep here, so a mean is off by 64 u of it before its residual is taken off, and by
64 u of that afterwards: the normalised value is off by (64 u)^2 |x| / sqrt(eps)."""

import pytest
import torch

import test_group_norm_act as gn

DEV = 'cuda:0'
DT = gn.DT
U = gn.U
EPS = 1e-5


def ops():
    import mineral_amd.ops  # noqa: F401
    return torch.ops.mineral


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape,groups', [((5, 3), 1), ((5, 49), 1), ((40, 98), 2), ((9, 11), 1), ((7, 1000), 1), ((3, 5000), 2), ((64, 512), 8), ((3, 49, 12), 4), ((2, 676, 184), 8),
                                          ((2, 677, 184), 8), ((2, 37, 63), 7), ((1, 31, 33, 64), 32), ((2, 5, 2100), 1), ((1, 40, 2144), 32)])
@pytest.mark.parametrize('value', [1.0, 1000.0, -37.7, 0.1])
def test_groups_of_equal_values(dtype, shape, groups, value):
    dt = DT[dtype]
    x, w, b, dy = gn.make(shape, dt, 31)
    x = torch.full(shape, value).to(dt)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = ops().group_norm_act(leaves[0], groups, leaves[1], leaves[2], EPS, None)
    xhat = (64 * U) ** 2 * abs(value) / EPS ** 0.5
    half = torch.finfo(dt).eps / 2
    err = (y.detach().double().cpu() - b.double()).abs()
    assert bool((err <= half * b.double().abs() + (1 + half) * xhat * w.double().abs()).all()), float(err.max())
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(DEV))
    # the normalised values are zero: dx = (w dy - mean(w dy)) / sqrt(eps), d_weight = 0
    rows = tuple(range(x.dim() - 1))
    mag = (dy.double().abs()).sum(rows)
    assert bool((dw.double().cpu().abs() <= (1 + half) * 2 * xhat * mag).all())
    h = gn.parts_of(w.double() * dy.double(), groups)
    want = ((h - h.mean(dim=(1, 3), keepdim=True)) / EPS ** 0.5).reshape(shape)
    lim = (gn.D * U + 4 * xhat * xhat) * ((h.abs() + h.abs().mean(dim=(1, 3), keepdim=True)) / EPS ** 0.5).reshape(shape)
    gn.close(dx, want, lim, 'dx')


@pytest.mark.gpu
@pytest.mark.parametrize('shape,groups', [((4, 64), 2), ((3, 50, 24), 4)])
def test_slopes_in_the_tails_of_tanh(shape, groups):
    """fp32 gradients of units at |z| around 6 to 10, relative to themselves: with weights of zero, z is the bias, and d_bias the
    sum of dy times one slope.  The slope is off by (4|z| + 16) u of itself, a sum over at most 2^8 rows by 2^8 u."""
    x, _, _, dy = gn.make(shape, torch.float32, 32)
    C = shape[-1]
    b = torch.linspace(-10, 10, C)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, torch.zeros(C), b)]
    _, _, db = torch.autograd.grad(ops().group_norm_act(leaves[0], groups, leaves[1], leaves[2], EPS, 'Tanh'), leaves, dy.abs().to(DEV))
    want = dy.double().abs().sum(tuple(range(x.dim() - 1))) / torch.cosh(b.double()) ** 2
    err = (db.double().cpu() - want).abs() / want
    assert bool((err <= (4 * b.double().abs() + 16 + 256) * U).all()), err


@pytest.mark.gpu
def test_more_than_2_to_the_31_values_in_tokens():
    """Rows without a gradient between a few that have one: the same bits as those rows by themselves, up to the parameters' sums."""
    n, C, G, dt = 2 ** 21 + 3, 1024, 8, torch.bfloat16
    x, w, b, dy = gn.make((8, C), dt, 33)
    rows = torch.tensor([0, 1, 2, 3, n - 4, n - 3, n - 2, n - 1], device=DEV)
    xs, gs = torch.zeros(n, C, dtype=dt, device=DEV), torch.zeros(n, C, dtype=dt, device=DEV)
    xs[rows], gs[rows] = x.to(DEV), dy.to(DEV)

    def both(x, dy):
        leaves = [t.requires_grad_(True) for t in (x, w.to(DEV), b.to(DEV))]
        y = ops().group_norm_act(leaves[0], G, leaves[1], leaves[2], EPS, 'SiLU')
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    y, dx, dw, db = both(xs, gs)
    y8, dx8, dw8, db8 = both(x.to(DEV), dy.to(DEV))
    assert torch.equal(y[rows], y8) and torch.equal(dx[rows], dx8)
    by = gn.bounds(x.double(), G, w.double(), b.double(), dy.double(), EPS)
    gn.close(dw, dw8.double().cpu(), by[2] + torch.finfo(dt).eps / 2 * dw8.double().cpu().abs(), 'd_weight')
    gn.close(db, db8.double().cpu(), by[3] + torch.finfo(dt).eps / 2 * db8.double().cpu().abs(), 'd_bias')


@pytest.mark.gpu
def test_more_than_2_to_the_31_values_in_pixels():
    """Three equal samples, the last beyond 2^31: equal results."""
    L, C, dt = 2 ** 20 + 3, 1024, torch.bfloat16
    g = torch.Generator(device=DEV).manual_seed(34)
    one, dy = (torch.randn(1, L, C, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    w, b = (torch.randn(C, generator=g, device=DEV, dtype=dt) for _ in range(2))
    x = one.expand(3, L, C).contiguous().requires_grad_(True)
    y = ops().group_norm_act(x, 16, w, b, EPS, 'SiLU')
    (dx,) = torch.autograd.grad(y, x, dy.expand(3, L, C))
    for t in (y.detach(), dx):
        assert torch.equal(t[2], t[0]) and torch.equal(t[1], t[0])
    h = one[0, :, :64].double()
    z = (h - h.mean()) / (((h - h.mean()) ** 2).mean() + EPS).sqrt() * w[:64].double() + b[:64].double()
    err = (y.detach()[2, :, :64].double() - torch.nn.functional.silu(z)).abs()
    assert bool((err <= 2.0 ** -8 * z.abs() + 2.0 ** -12).all())

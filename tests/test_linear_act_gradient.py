"""What the gradient of torch.ops.mineral.linear_act has to survive: units in the tails of their activation, values that are not
finite, fp16 gradients near the type's largest value, and offsets beyond 32 bits.

Tolerances.  u = 2^-24.  A slope is evaluated in fp32, off by (4|z| + 16) u of itself (tanh, exponential: the rounded argument of an
exponential of up to 2|z|, and a dozen operations), for SiLU and GELU of the magnitudes of their two terms (GELU's arguments are
squared: 4 z^2).  Beside 16-bit types it is kept as its fourth root in steps of 1/30720, off by half a step, after two square roots of an
ulp each (2^-20 of the slope together, with the decoding).  dz is rounded to the type before the two products, eps/2 (and half a
spacing of its subnormals); d_bias sums it unrounded.  Results are rounded once more."""

import pytest
import torch

import test_linear_act as la

DEV = 'cuda:0'
DT = la.DT
U = la.U
STEP = 1 / 30720


def ops():
    import mineral_amd.ops  # noqa: F401
    return torch.ops.mineral


def slope64(z, act):
    z = z.clone().requires_grad_(True)
    (s,) = torch.autograd.grad(la.act64(z, act).sum(), z)
    return s.detach()


def slope_error(z, act, dt):
    """How far a slope at z may be off."""
    s, a = slope64(z, act), z.abs()
    if act == 'SiLU':
        g = torch.sigmoid(z)
        e = (4 * a + 16) * U * (g + a * g * (1 - g))
    elif act == 'GELU':
        e = (4 * a * a + 16) * U * (0.5 * torch.erfc(-z / 2 ** 0.5) + a * 0.4 * torch.exp(-z * z / 2))
    else:
        e = (4 * a + 16) * U * s
    if dt != torch.float32:
        q = (s.abs() + e) ** 0.25
        e = e + (q + STEP / 2) ** 4 - q ** 4 + 2.0 ** -20 * s.abs()
    return s, e


def half_spacing(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


TAILS = {'Tanh': (-12.0, 12.0), 'ELU': (-24.0, 1.0), 'SiLU': (-24.0, 24.0), 'GELU': (-6.0, 6.0)}


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('act', TAILS)
def test_tails_of_the_slopes(dtype, act):
    """One row and one input of one: z is the weight, and each unit's d_bias is its slope times dy."""
    dt = DT[dtype]
    z = torch.linspace(*TAILS[act], 4001).to(dt).unique()
    N, big = z.numel(), 2.0 ** 14
    x, w, b = torch.ones(1, 1, dtype=dt), z[:, None].clone(), torch.zeros(N, dtype=dt)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = ops().linear_act(*leaves, None, act)
    _, dw, db = torch.autograd.grad(y, leaves, torch.full((1, N), big, dtype=dt, device=DEV))
    s, e = slope_error(z.double(), act, dt)
    tiny = half_spacing(dt)
    half = la.half_of(dt) * (1 + 2.0 ** -10)
    err, lim = (db.double().cpu() - big * s).abs(), big * e + half * (big * (s.abs() + e)) + tiny
    assert bool((err <= lim).all()), f'd_bias: worst {float((err / lim).max()):.2f} of the bound at z = {float(z[(err / lim).argmax()]):.3f}'
    err, lim = (dw[:, 0].double().cpu() - big * s).abs(), lim + half * (big * (s.abs() + e)) + 2 * tiny
    assert bool((err <= lim).all()), f'd_weight: worst {float((err / lim).max()):.2f} of the bound at z = {float(z[(err / lim).argmax()]):.3f}'


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
def test_slopes_of_zero_and_one_are_exact(dtype):
    dt = DT[dtype]
    z = torch.tensor([-3.0, -0.5, 0.0, 0.5, 3.0]).to(dt)
    for act, want in (('ReLU', (z > 0).to(dt)), ('ELU', torch.where(z > 0, torch.ones_like(z), torch.zeros_like(z)))):
        leaves = [t.to(DEV).requires_grad_(True) for t in (torch.ones(1, 1, dtype=dt), z[:, None].clone(), torch.zeros(5, dtype=dt))]
        dy = torch.tensor([[1.0, -2.0, 3.0, 1.25, 1.75]], dtype=dt)
        _, dw, db = torch.autograd.grad(ops().linear_act(*leaves, None, act), leaves, dy.to(DEV))
        at = torch.ones_like(z, dtype=torch.bool) if act == 'ReLU' else z > 0
        assert torch.equal(db.cpu()[at], (want * dy[0])[at]) and torch.equal(dw[:, 0].cpu()[at], (want * dy[0])[at])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('act,z', [('SiLU', -300.0), ('ELU', -300.0), ('Tanh', 60.0), ('GELU', -40.0), ('SiLU', 1.0), ('ReLU', 2.0)])
def test_a_gradient_that_is_not_finite_stays_so(dtype, bad, act, z):
    """Also where the unit is saturated: zero times NaN or infinity is no number, as in torch."""
    dt = DT[dtype]
    dy = torch.ones(3, 2, dtype=dt)
    dy[1, 1] = bad
    x, w, b = torch.ones(3, 1, dtype=dt), torch.tensor([[1.0], [z]], dtype=dt), torch.zeros(2, dtype=dt)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops().linear_act(*leaves, None, act), leaves, dy.to(DEV))
    assert torch.isfinite(dx).cpu().flatten().tolist() == [True, False, True]
    assert torch.isfinite(dw).cpu().flatten().tolist() == [True, False] and torch.isfinite(db).cpu().tolist() == [True, False]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_the_rectifier_drops_what_it_cut(dtype, bad):
    """As in torch: no gradient passes a rectifier below zero, whatever it is."""
    dt = DT[dtype]
    dy = torch.ones(3, 2, dtype=dt)
    dy[1, 1] = bad
    x, w, b = torch.ones(3, 1, dtype=dt), torch.tensor([[1.0], [-2.0]], dtype=dt), torch.zeros(2, dtype=dt)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(ops().linear_act(*leaves, None, 'ReLU'), leaves, dy.to(DEV))
    assert torch.equal(dx.cpu(), torch.ones(3, 1, dtype=dt))
    assert dw.cpu().flatten().tolist() == [3.0, 0.0] and db.cpu().tolist() == [3.0, 0.0]


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['SiLU', 'GELU'])
@pytest.mark.parametrize('shape', [(1, 1, 1), (5, 40, 33), (70, 96, 128), (2100, 72, 264), (5000, 130, 520), (9000, 264, 1000), (1100, 1048, 1032), (16400, 200, 1024)])
def test_fp16_gradients_near_the_largest_value(act, shape):
    """Slopes of SiLU and GELU reach 1.13: dy slope passes 65504 where dy does not, while its products with small weights and inputs are
    ordinary numbers."""
    M, K, N = shape
    dt = torch.float16
    g = torch.Generator().manual_seed(21)
    sign = lambda *s: torch.randint(0, 2, s, generator=g).double() * 2 - 1  # noqa: E731
    # powers of two, so that z = 1.5 + x w is nearly 1.5 (slope over 1.04) and the results stay below 65504
    x = (2.0 ** -11 * (1 + torch.rand(M, K, generator=g).double()) * sign(M, K)).to(dt)
    w = (2.0 ** -11 * (1 + torch.rand(N, K, generator=g).double()) * sign(N, K)).to(dt)
    b, dy = torch.full((N,), 1.5).to(dt), (sign(M, N) * 65504).to(dt)
    print(f'large fp16 gradients {shape} {act}', flush=True)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    dx, dw, _ = torch.autograd.grad(ops().linear_act(*leaves, None, act), leaves, dy.to(DEV))
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    z = x @ w.t() + b
    s, e = slope_error(z, act, dt)
    e = e + 1.13 * (K + 16) * U * (x.abs() @ w.abs().t() + b)
    dz = dy * s
    assert float(dz.abs().max()) > 65504 * 1.03
    dze = dy.abs() * e + la.half_of(dt) * (dy.abs() * (s.abs() + e))
    for n, a, ref, lim in (('dx', dx, dz @ w, dze @ w.abs() + (N + 16) * U * ((dz.abs() + dze) @ w.abs())),
                           ('d_weight', dw, dz.t() @ x, dze.t() @ x.abs() + (M + 16) * U * ((dz.abs() + dze).t() @ x.abs()))):
        assert float(ref.abs().max()) < 65504
        err = (a.double().cpu() - ref).abs()
        lim = lim + la.half_of(dt) * (ref.abs() + lim) + half_spacing(dt)
        assert bool((err <= lim).all()), f'{n}: worst {float((err / lim).max()):.2f} of the bound'


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
def test_more_than_2_to_the_31_outputs(dtype):
    """All but the first and the last rows have no gradient; those are held to the definition."""
    dt, (M, K, N) = DT[dtype], (2 ** 21 + 5, 16, 1024)
    x, w, b, r, dy = la.make(8, K, N, dt, 22)
    rows = torch.tensor([0, 1, 2, 3, M - 4, M - 3, M - 2, M - 1], device=DEV)
    big = torch.zeros(M, K, dtype=dt, device=DEV)
    big[rows] = x.to(DEV)
    leaves = [big.requires_grad_(True), w.to(DEV).requires_grad_(True), b.to(DEV).requires_grad_(True)]
    y = ops().linear_act(*leaves, None, 'SiLU')
    g = torch.zeros(M, N, dtype=dt, device=DEV)
    g[rows] = dy.to(DEV)
    dx, dw, db = torch.autograd.grad(y, leaves, g)
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    z = x @ w.t() + b
    ze = (K + 16) * U * (x.abs() @ w.abs().t() + b.abs())
    la.close(y.detach()[rows], la.act64(z, 'SiLU'), 1.13 * ze + 16 * U * (z.abs() + 1), 'y')
    s, e = slope_error(z, 'SiLU', dt)
    dz, dze = dy * s, dy.abs() * (e + 1.13 * ze)
    dzr = dze + la.half_of(dt) * (dz.abs() + dze)
    la.close(dx[rows], dz @ w, dzr @ w.abs() + (N + 16) * U * (dz.abs() @ w.abs()), 'dx')
    assert not dx[4:M - 4].any()
    la.close(dw, dz.t() @ x, dzr.t() @ x.abs() + 32 * U * (dz.abs().t() @ x.abs()), 'd_weight')
    la.close(db, dz.sum(0), dze.sum(0) + 32 * U * dz.abs().sum(0), 'd_bias')

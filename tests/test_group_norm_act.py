"""torch.ops.mineral.group_norm_act against its definition in 64 bits, with torch's automatic gradient of that.

Tolerances.  u = 2^-24.  A sum in the kernels is at most D = 200 roundings deep at the sizes below (a thread's run, its lanes, its
parts), so the mean is off by D u mean|x| and the normalised value by D u (|xhat| + A) with A = rstd mean|x|.  The activations
and their slopes have slopes of at most 1.13 and are themselves within 16 u of |z| + 1.  Every gradient is a sum of products of such
factors; with X = |xhat| + A + 1 and W = |w| + |b| + 1 each of its terms is off by at most D u times the same expression over
absolute values, where |dz| <= 2 |dy| X W.  A result of a 16-bit type is off by eps/2 of itself more."""

import pytest
import torch

DEV = 'cuda:0'
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
ACTS = [None, 'SiLU', 'ELU', 'ReLU', 'Tanh', 'GELU']
D, U = 200, 2.0 ** -24


def ops():
    import mineral_amd.ops  # noqa: F401
    return torch.ops.mineral


def act64(z, name):
    F = torch.nn.functional
    return {None: lambda t: t, 'SiLU': F.silu, 'ELU': F.elu, 'ReLU': F.relu, 'Tanh': torch.tanh, 'GELU': F.gelu}[name](z)


def parts_of(x, G):
    n, C = x.shape[0], x.shape[-1]
    return x.reshape(n, -1, G, C // G)


def reference(x, G, w, b, eps, act):
    xg = parts_of(x, G)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    rstd = ((xg - mean) ** 2).mean(dim=(1, 3), keepdim=True).add(eps).rsqrt()
    xhat = ((xg - mean) * rstd).reshape(x.shape)
    z = xhat if w is None else xhat * w
    z = z if b is None else z + b
    return act64(z, act), xhat, rstd


def close(got, ref, bound, what):
    half = torch.finfo(got.dtype).eps / 2 * (1 + 2.0 ** -8) if got.dtype != torch.float32 else 0.0
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps if got.dtype != torch.float32 else 1e-37
    err = (got.double().cpu() - ref).abs()
    lim = half * ref.abs() + bound + tiny
    assert bool((err <= lim).all()), f'{what}: worst {float((err / lim).max()):.2f} of the bound'


def make(shape, dt, seed, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(*shape, generator=g) * 1.5 + shift).to(dt)
    return x, (torch.randn(C, generator=g) * 0.3 + 1).to(dt), (torch.randn(C, generator=g) * 0.3).to(dt), torch.randn(*shape, generator=g).to(dt)


def bounds(x, G, w, b, dy, eps):
    """The magnitudes of the header, as tensors in 64 bits."""
    _, xhat, rstd = reference(x, G, None, None, eps, None)
    xg = parts_of(x, G)
    spread = lambda t: t.expand(xg.shape).reshape(x.shape)  # noqa: E731
    A = spread(rstd * xg.abs().mean(dim=(1, 3), keepdim=True))
    X, W = xhat.abs() + A + 1, w.abs() + b.abs() + 1
    mean = lambda t: spread(parts_of(t, G).mean(dim=(1, 3), keepdim=True))  # noqa: E731
    y = D * U * 1.13 * X * W + 16 * U * (X * W + 1)
    dz = 2 * dy.abs() * X * W
    rows = tuple(range(x.dim() - 1))
    dx = D * U * 2 * spread(rstd) * (w.abs() * dz + mean(w.abs() * dz) + X * mean(w.abs() * dz * X))
    return y, dx, D * U * 2 * (dz * X).sum(rows), D * U * 2 * dz.sum(rows)


SHAPES = [((5, 24), 4), ((64, 512), 8), ((3, 7), 7), ((2, 9), 3), ((9, 1), 1), ((33, 130), 2), ((4, 640), 1), ((3, 5000), 2), ((1000, 96), 6), ((70, 48), 48),
          ((2, 3, 3, 32), 8), ((3, 49, 12), 4), ((2, 100, 70), 10), ((1, 31, 33, 64), 32), ((2, 5, 2100), 1), ((1, 3, 2100), 2), ((2, 500, 6), 2), ((4, 2, 30), 3), ((2, 676, 184), 8), ((1, 40, 2144), 32),
          ((70, 63), 1), ((40, 196), 2), ((9, 11), 1)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape,groups', SHAPES)
@pytest.mark.parametrize('shift', [0.0, 30.0])
def test_matches_the_definition(dtype, shape, groups, shift):
    x, w, b, dy = make(shape, DT[dtype], 1, shift)
    print(f'group_norm_act {dtype} {shape} {groups}', flush=True)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = ops().group_norm_act(leaves[0], groups, leaves[1], leaves[2], 1e-5, 'SiLU')
    got = torch.autograd.grad(y, leaves, dy.to(DEV))
    ref = [t.double().requires_grad_(True) for t in (x, w, b)]
    yr = reference(ref[0], groups, ref[1], ref[2], 1e-5, 'SiLU')[0]
    want = torch.autograd.grad(yr, ref, dy.double())
    by = bounds(x.double(), groups, w.double(), b.double(), dy.double(), 1e-5)
    close(y, yr.detach(), by[0], 'y')
    for n, a, r, lim in zip(('dx', 'd_weight', 'd_bias'), got, want, by[1:]):
        assert a.dtype == DT[dtype]
        close(a, r, lim, n)
    assert torch.equal(y, ops().group_norm_act(x.to(DEV), groups, w.to(DEV), b.to(DEV), 1e-5, 'SiLU'))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('shape,groups', [((37, 64), 4), ((3, 30, 24), 6)])
def test_activations_and_parameters(dtype, act, shape, groups):
    x, w, b, dy = make(shape, DT[dtype], 2)
    if act == 'ReLU':                       # its slope jumps at zero: keep every value away from it
        z = reference(x.double(), groups, w.double(), b.double(), 1e-5, None)[0]
        dy = torch.where(z.abs() > 1e-3, dy, torch.zeros((), dtype=dy.dtype))
    y64, dx64, dw64, db64 = bounds(x.double(), groups, w.double(), b.double(), dy.double(), 1e-5)
    for pw, pb in ((w, b), (w.float(), b.float()), (w, None), (None, b), (None, None)):
        params = [t for t in (pw, pb) if t is not None]
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, *params)]
        it = iter(leaves[1:])
        y = ops().group_norm_act(leaves[0], groups, None if pw is None else next(it), None if pb is None else next(it), 1e-5, act)
        got = torch.autograd.grad(y, leaves, dy.to(DEV))
        ref = [t.double().requires_grad_(True) for t in (x, *params)]
        it = iter(ref[1:])
        yr = reference(ref[0], groups, None if pw is None else next(it), None if pb is None else next(it), 1e-5, act)[0]
        want = torch.autograd.grad(yr, ref, dy.double())
        one, zero = torch.ones_like(w).double(), torch.zeros_like(b).double()
        by = bounds(x.double(), groups, one if pw is None else w.double(), zero if pb is None else b.double(), dy.double(), 1e-5)
        close(y, yr.detach(), by[0], f'y {act}')
        lims = [by[1]] + [l for l, t in zip(by[2:], (pw, pb)) if t is not None]
        for a, r, lim, leaf in zip(got, want, lims, leaves):
            assert a.dtype == leaf.dtype
            close(a, r, lim, f'gradient {act}')
    (gx,) = torch.autograd.grad(ops().group_norm_act(leaves[0], groups, w.to(DEV), b.to(DEV), 1e-5, act), leaves[0], dy.to(DEV))     # x alone
    assert gx.shape == x.shape


@pytest.mark.gpu
def test_gradient_matches_differences():
    x, w, b, dy = (t.to(DEV) for t in make((6, 20, 32), torch.float32, 3))
    g = torch.Generator(device=DEV).manual_seed(4)

    def loss(x, w, b):
        return (ops().group_norm_act(x, 4, w, b, 1e-5, 'Tanh').double() * dy).sum()

    xs = [x, w, b]
    leaves = [t.clone().requires_grad_(True) for t in xs]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i in range(3):
        d = torch.randn(xs[i].shape, device=DEV, generator=g)
        h = 2.0 ** -7
        up, down = list(xs), list(xs)
        up[i], down[i] = xs[i] + h * d, xs[i] - h * d
        diff = float(loss(*up) - loss(*down)) / (2 * h)
        want = float((grads[i].double() * d).sum())
        # truncation: the same difference of the 64-bit definition at the same points, minus its derivative, is part of the bound
        r = [t.double().cpu() for t in xs]
        rd = d.double().cpu()

        def ref(k):
            q = list(r)
            q[i] = (xs[i] + k * h * d).double().cpu()
            return float((reference(q[0], 4, q[1], q[2], 1e-5, 'Tanh')[0] * dy.double().cpu()).sum())
        by = bounds(r[0], 4, r[1], r[2], dy.double().cpu(), 1e-5)
        rounding = 2 * float((by[0] * dy.double().cpu().abs()).sum()) / (2 * h) + float((by[1 + i] * rd.abs()).sum())
        rl = [t.clone().requires_grad_(True) for t in r]
        exact = float((torch.autograd.grad((reference(rl[0], 4, rl[1], rl[2], 1e-5, 'Tanh')[0] * dy.double().cpu()).sum(), rl[i])[0] * rd).sum())
        truncation = abs((ref(1) - ref(-1)) / (2 * h) - exact)
        assert abs(diff - want) <= rounding + truncation, i


@pytest.mark.gpu
def test_one_bad_sample_stays_alone():
    x, w, b, dy = (t.to(DEV) for t in make((6, 40, 32), torch.float32, 5))
    for bad in (float('nan'), float('inf')):
        for shape in ((6, 40, 32), (240, 32)):
            clean = x.reshape(shape)
            broken = clean.clone()
            broken.view(-1)[0] = bad
            a, c = (t.clone().requires_grad_(True) for t in (broken, clean))
            ya, yc = ops().group_norm_act(a, 4, w, b, 1e-5, 'SiLU'), ops().group_norm_act(c, 4, w, b, 1e-5, 'SiLU')
            (ga,), (gc,) = (torch.autograd.grad(y, t, torch.ones_like(y)) for y, t in ((ya, a), (yc, c)))
            assert torch.equal(ya[1:], yc[1:]) and torch.equal(ga[1:], gc[1:])
            assert torch.equal(ya[0, ..., 8:], yc[0, ..., 8:]) and not torch.isfinite(ya[0, ..., :8]).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
def test_layouts_streams_and_graphs(dtype):
    for shape, groups in (((200, 96), 6), ((3, 300, 40), 5)):
        x, w, b, dy = (t.to(DEV) for t in make(shape, DT[dtype], 6))

        def both(x, dy):
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
            y = ops().group_norm_act(leaves[0], groups, leaves[1], leaves[2], 1e-5, 'ELU')
            return (y, *torch.autograd.grad(y, leaves, dy))

        want = [t.clone() for t in both(x, dy)]
        odd = torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)
        odd[1:] = x.reshape(-1)
        wide = torch.cat([x, x], -1)
        for xx in (odd[1:].view(shape), wide[..., :shape[-1]]):
            assert all(torch.equal(p, q) for p, q in zip(both(xx, dy), want))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = both(x, dy)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = both(x, dy)
        for _ in range(3):
            for t in held:
                t.detach().zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(held, want))
            assert all(torch.equal(p, q) for p, q in zip(both(x, dy), want))


@pytest.mark.gpu
def test_nothing_to_do_and_refusals_on_the_device():
    M = ops()
    w = torch.ones(8, device=DEV, requires_grad=True)
    for shape in ((0, 8), (3, 0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        y = M.group_norm_act(x, 2, w, None, 1e-5, 'SiLU')
        gx, gw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == shape and gx.shape == shape and torch.equal(gw, torch.zeros_like(w))
    x = torch.zeros(2, 8, device=DEV)
    with pytest.raises(NotImplementedError, match='act_type'):
        M.group_norm_act(x, 2, None, None, 1e-5, 'Mish')
    with pytest.raises(ValueError, match='tensors on'):
        M.group_norm_act(x, 2, torch.ones(8), None, 1e-5, None)


def test_refusals():
    """Argument checks, on CPU tensors: they come before the refusal of the CPU itself."""
    from mineral_amd import _hip
    x, w, b, _ = make((4, 8), torch.float32, 7)
    ok = dict(x=x, num_groups=2, weight=w, bias=b, eps=1e-5, act_type=None)
    with pytest.raises(NotImplementedError, match='CPU'):
        ops().group_norm_act(**ok)
    with pytest.raises(NotImplementedError, match='act_type'):
        ops().group_norm_act(**{**ok, 'act_type': 'Mish'})
    for change, text in ((dict(x=x.double()), 'dtype'), (dict(x=x[0]), 'channels'), (dict(num_groups=3), 'groups'), (dict(num_groups=0), 'groups'), (dict(eps=-1.0), 'eps'),
                         (dict(eps=float('nan')), 'eps'), (dict(weight=w[:4]), 'weight'), (dict(bias=b.half()), 'bias'), (dict(x=x.half(), weight=w.half()), 'one type')):
        with pytest.raises(ValueError, match=text):
            ops().group_norm_act(**{**ok, **change})
    a = _hip.GroupNorm(4, 1, 8, 2, 0, 0, 0, 1e-5)
    L = _hip.lib()
    assert L.mrl_group_norm_act_workspace_bytes(a, 0) == 0 and L.mrl_group_norm_act_workspace_bytes(a, 1) > 0
    assert L.mrl_group_norm_act(a, None, None, None, None, None, None, None, 0, None) == -1 and b'null' in L.mrl_last_error()
    assert L.mrl_group_norm_act(None, None, None, None, None, None, None, None, 0, None) == -1
    assert L.mrl_group_norm_act(a, 4, None, None, 16, None, None, None, 0, None) == -1 and b'aligned' in L.mrl_last_error()
    assert L.mrl_group_norm_act(a, 16, None, None, 16, 16, None, None, 0, None) == -1 and b'together' in L.mrl_last_error()
    assert L.mrl_group_norm_act_backward(a, 16, 16, None, None, 16, 16, 16, 16, 16, None, 0, None) == -2
    assert L.mrl_group_norm_act_backward(a, 16, 16, None, None, 16, 16, 16, 16, None, None, 0, None) == -1
    for bad in (_hip.GroupNorm(4, 1, 8, 3, 0, 0, 0, 1e-5), _hip.GroupNorm(4, 1, 8, 2, 3, 0, 0, 1e-5), _hip.GroupNorm(4, 1, 8, 2, 1, 2, 0, 1e-5),
                _hip.GroupNorm(4, 1, 8, 2, 0, 0, 9, 1e-5), _hip.GroupNorm(-1, 1, 8, 2, 0, 0, 0, 1e-5)):
        assert L.mrl_group_norm_act_workspace_bytes(bad, 0) == -1
    many = _hip.GroupNorm(1 << 24, 2, 8, 2, 0, 0, 0, 1e-5)
    assert L.mrl_group_norm_act(many, 16, None, None, 16, None, None, 16, 1 << 40, None) == -1 and b'2^24' in L.mrl_last_error()

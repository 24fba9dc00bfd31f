"""torch.ops.mineral.linear_act against its definition in 64 bits, with torch's automatic gradient of that.

Tolerances.  u = 2^-24.  A product of r terms is off by (r + 16) u of the sum of its terms' magnitudes, fp32 operands by 4 u more
(their six bf16 products drop 2^-23 of each).  Activations and their slopes have slopes of at most 1.13 and are themselves within
16 u of |z| + 1; beside bf16 the backward pass reads the slope off by 2^-12 of itself (at least 2^-26), beside fp16 by
2^-13 (at least 2^-20), and rounds dz.  A result is rounded once: eps/2."""

import pytest
import torch

DEV = 'cuda:0'
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
U = 2.0 ** -24


def ops():
    import mineral_amd.ops  # noqa: F401
    return torch.ops.mineral


def act64(z, name):
    F = torch.nn.functional
    return {None: lambda t: t, 'SiLU': F.silu, 'ELU': F.elu, 'ReLU': F.relu, 'Tanh': torch.tanh, 'GELU': F.gelu}[name](z)


def half_of(dt):
    return torch.finfo(dt).eps / 2


def make(M, K, N, dt, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return r(M, K).to(dt), (r(N, K) / max(K, 1) ** 0.5).to(dt), (r(N) * 0.3).to(dt), r(M, N).to(dt), r(M, N).to(dt)


def close(got, ref, bound, what):
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps if got.dtype != torch.float32 else 1e-37
    err = (got.double().cpu() - ref).abs()
    lim = half_of(got.dtype) * (1 + 2.0 ** -7) * ref.abs() + bound + tiny
    assert bool((err <= lim).all()), f'{what}: worst {float((err / lim).max()):.2f} of the bound'


def check(M, K, N, dt, act, seed, bias=True, residual=True, inputs=None):
    x, w, b, r, dy = inputs if inputs is not None else make(M, K, N, dt, seed)
    print(f'linear_act {dt} {M}x{K}x{N} {act}', flush=True)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b, r)]
    y = ops().linear_act(leaves[0], leaves[1], leaves[2] if bias else None, leaves[3] if residual else None, act)
    used = [t for t, k in zip(leaves, (True, True, bias, residual)) if k]
    got = torch.autograd.grad(y, used, dy.to(DEV))
    x, w, b, r, dy = (t.double() for t in (x, w, b, r, dy))
    ref = [t.requires_grad_(True) for t in (x, w, b, r)]
    z = ref[0] @ ref[1].t() + (ref[2] if bias else 0)
    yr = act64(z, act) + (ref[3] if residual else 0)
    want = torch.autograd.grad(yr, [t for t, k in zip(ref, (True, True, bias, residual)) if k], dy, retain_graph=True)
    (slope,) = torch.autograd.grad(act64(z, act), z, torch.ones_like(z))
    x, w, b, r, z, slope = (t.detach() for t in (x, w, b, r, z, slope))
    extra, h = (4 * U if dt == torch.float32 else 0.0), half_of(dt)
    ze = ((K + 16) * U + extra) * (x.abs() @ w.abs().t() + b.abs())
    close(y, yr.detach(), 1.13 * ze + 16 * U * (z.abs() + 1) + 4 * U * (z.abs() + r.abs()), 'y')
    se = 0 if act is None else 1.13 * ze + 16 * U * (z.abs() + 1) + {torch.float32: 0, torch.bfloat16: 2.0 ** -12 * slope.abs() + 2.0 ** -26, torch.float16: 2.0 ** -13 * slope.abs() + 2.0 ** -20}[dt]     # of the slope
    dz, dze = (dy * slope).abs(), dy.abs() * se
    dzr = dze + (0 if act is None else h * (dz + dze))                                   # and of the rounded dz
    lims = [dzr @ w.abs() + ((N + 16) * U + extra) * ((dz + dzr) @ w.abs()), dzr.t() @ x.abs() + ((M + 16) * U + extra) * ((dz + dzr).t() @ x.abs()),
            dze.sum(0) if act is not None else torch.zeros(N, dtype=torch.float64), torch.zeros(M, N, dtype=torch.float64)]
    lims[2] = lims[2] + (M + 16) * U * dz.sum(0)
    lims = [l for l, k in zip(lims, (True, True, bias, residual)) if k]
    for n, a, q, lim in zip(('dx', 'd_weight', 'd_bias', 'd_residual') if bias else ('dx', 'd_weight', 'd_residual'), got, want, lims):
        close(a, q, lim, n)
    return y


SHAPES = [(1, 1, 1), (1, 16, 8), (3, 5, 7), (33, 40, 31), (64, 512, 96), (130, 64, 130), (200, 333, 77), (65, 129, 257), (1000, 24, 16), (2, 1000, 3), (257, 96, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape', SHAPES)
def test_matches_the_definition(dtype, shape):
    check(*shape, DT[dtype], 'SiLU', 1)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape', [(2100, 72, 2040), (4200, 200, 1030), (8200, 130, 520)])
def test_large_tiles(dtype, shape):
    """Enough tiles for each tile size, ragged at both edges, and rows split over blocks in the weight's gradient."""
    check(*shape, DT[dtype], 'Tanh', 2)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape', [(13000, 264, 1000), (1100, 1048, 1032), (900, 1047, 1031), (700, 2056, 4104)])
def test_large_tiles_without_a_residual(dtype, shape):
    """The largest tiles forward, and those of 128 and 256 in the weight's gradient."""
    check(*shape, DT[dtype], 'SiLU', 4, residual=False)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('act', [None, 'SiLU', 'ELU', 'Tanh', 'GELU'])
@pytest.mark.parametrize('bias,residual', [(True, True), (True, False), (False, True), (False, False)])
def test_epilogues(dtype, act, bias, residual):
    x, w, b, r, dy = make(70, 48, 50, DT[dtype], 3)
    check(70, 48, 50, DT[dtype], act, 3, bias, residual, (x, w, b if bias else torch.zeros_like(b), r if residual else torch.zeros_like(r), dy))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
def test_rectifier_on_whole_numbers(dtype):
    """Small whole numbers and a bias of one half: every sum is exact and none is zero, so the slope has no doubt."""
    g = torch.Generator().manual_seed(4)
    i = lambda *s: torch.randint(-3, 4, s, generator=g).to(DT[dtype])  # noqa: E731
    x, w, dy = i(70, 20), i(50, 20), i(70, 50)
    b, r = torch.full((50,), 0.5).to(DT[dtype]), torch.zeros(70, 50).to(DT[dtype])
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = ops().linear_act(*leaves, r.to(DEV), 'ReLU')
    got = torch.autograd.grad(y, leaves, dy.to(DEV))
    z = x.double() @ w.double().t() + 0.5
    dz = dy.double() * (z > 0)
    for a, q in zip((y, *got), (z.clamp(min=0), dz @ w.double(), dz.t() @ x.double(), dz.sum(0))):
        assert torch.equal(a.cpu(), q.to(DT[dtype]))


@pytest.mark.gpu
def test_gradient_matches_differences():
    """Without an activation the layer is linear in each operand: a symmetric difference is the derivative up to rounding."""
    x, w, b, r, dy = (t.to(DEV) for t in make(90, 70, 60, torch.float32, 5))
    g = torch.Generator(device=DEV).manual_seed(6)
    xs = [x, w, b, r]
    loss = lambda *a: (ops().linear_act(*a, None).double() * dy).sum()  # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in xs]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i in range(4):
        d = torch.randn(xs[i].shape, device=DEV, generator=g)
        up, down = list(xs), list(xs)
        up[i], down[i] = xs[i] + d, xs[i] - d
        mag = [t.double().abs() for t in xs]
        mag[i] = mag[i] + d.double().abs()
        lim = 4 * (70 + 90 + 20) * U * float(((mag[0] @ mag[1].t() + mag[2] + mag[3]) * dy.double().abs()).sum())
        assert abs(float(loss(*up) - loss(*down)) / 2 - float((grads[i].double() * d).sum())) <= lim, i


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
def test_layouts_streams_and_graphs(dtype):
    x, w, b, r, dy = (t.to(DEV) for t in make(600, 64, 72, DT[dtype], 7))
    M = ops()
    want = M.linear_act(x, w, b, r, 'GELU')
    wide = torch.cat([x, x], 1)
    odd = torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)
    odd[1:] = x.reshape(-1)
    for xx in (wide[:, :64], wide[:, 64:], odd[1:].view(x.shape), x.t().contiguous().t()):
        assert torch.equal(M.linear_act(xx, w, b, r, 'GELU'), want)
    assert torch.equal(M.linear_act(x, w.t().contiguous().t(), b, r.t().contiguous().t(), 'GELU'), want)
    deep = M.linear_act(x.view(2, 3, 100, 64), w, b, r.view(2, 3, 100, 72), 'GELU')
    assert deep.shape == (2, 3, 100, 72) and torch.equal(deep.view(600, 72), want)
    assert torch.equal(M.linear_act(x[:1].expand(5, 64), w, b, None, None), M.linear_act(x[:1].repeat(5, 1), w, b, None, None))
    one = M.linear_act(x[0], w, b, None, 'SiLU')
    assert one.shape == (72,) and torch.equal(one, M.linear_act(x[:1], w, b, None, 'SiLU')[0])

    def both():
        leaves = [t.detach().requires_grad_(True) for t in (wide[:, :64], w, b, r)]
        y = M.linear_act(*leaves, 'SiLU')
        return (y, *torch.autograd.grad(y, leaves, dy))

    eager = [t.clone() for t in both()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for _ in range(3):
        for t in held[:4]:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager))
        assert all(torch.equal(p, q) for p, q in zip(both(), eager))
    # a gradient that arrives broadcast, and a broadcast residual
    leaf = x.clone().requires_grad_(True)
    y = M.linear_act(leaf, w, b, r[:1].expand(600, 72), 'SiLU')
    (g1,) = torch.autograd.grad(y.sum(), leaf, retain_graph=True)
    (g2,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.equal(g1, g2)


@pytest.mark.gpu
def test_only_what_is_asked_for():
    x, w, b, r, dy = (t.to(DEV) for t in make(300, 40, 50, torch.bfloat16, 8))
    M = ops()
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    full = torch.autograd.grad(M.linear_act(*leaves, 'SiLU'), leaves, dy)
    for i in range(4):
        args = [t if k == i else t.detach() for k, t in enumerate(leaves)]
        (g,) = torch.autograd.grad(M.linear_act(*args, 'SiLU'), args[i], dy)
        assert torch.equal(g, full[i])


@pytest.mark.gpu
def test_nothing_to_do_and_refusals_on_the_device():
    M = ops()
    for shape in ((0, 8, 4), (3, 0, 4), (3, 8, 0)):
        m, k, n = shape
        x, w, b = torch.ones(m, k, device=DEV, requires_grad=True), torch.ones(n, k, device=DEV, requires_grad=True), torch.ones(n, device=DEV, requires_grad=True)
        y = M.linear_act(x, w, b, None, 'SiLU')
        gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
        assert y.shape == (m, n) and gx.shape == x.shape and gw.shape == w.shape
        if m == 0:
            assert torch.equal(gw, torch.zeros_like(gw)) and torch.equal(gb, torch.zeros_like(gb))
        if k == 0:
            assert torch.equal(y, torch.nn.functional.silu(torch.ones(m, n, device=DEV)))
    x, w = torch.zeros(2, 8, device=DEV), torch.zeros(4, 8, device=DEV)
    with pytest.raises(NotImplementedError, match='act_type'):
        M.linear_act(x, w, None, None, 'Mish')
    with pytest.raises(ValueError, match='tensors on'):
        M.linear_act(x, w.cpu(), None, None, None)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows 2^30 elements apart."""
    x, w, b, r, _ = (t.to(DEV) for t in make(4, 32, 40, torch.bfloat16, 9))
    far = 2 ** 30
    big = torch.empty(3 * far + 32, dtype=torch.bfloat16, device=DEV)
    xx = big.as_strided((4, 32), (far, 1))
    xx.copy_(x)
    assert torch.equal(ops().linear_act(xx, w, b, r, 'SiLU'), ops().linear_act(x, w, b, r, 'SiLU'))


def test_refusals():
    """Argument checks, on CPU tensors: they come before the refusal of the CPU itself."""
    from mineral_amd import _hip
    x, w, b, r, _ = make(4, 8, 6, torch.float32, 10)
    ok = dict(x=x, weight=w, bias=b, residual=r, act_type=None)
    with pytest.raises(NotImplementedError, match='CPU'):
        ops().linear_act(**ok)
    with pytest.raises(NotImplementedError, match='act_type'):
        ops().linear_act(**{**ok, 'act_type': 'Mish'})
    for change, text in ((dict(x=x.double()), 'dtype'), (dict(weight=w[:, :4]), 'weight'), (dict(weight=w[0]), 'weight'), (dict(weight=w.half()), 'weight'),
                         (dict(bias=b[:3]), 'bias'), (dict(bias=b.half()), 'bias'), (dict(residual=r[:1]), 'residual'), (dict(residual=r.half()), 'residual')):
        with pytest.raises(ValueError, match=text):
            ops().linear_act(**{**ok, **change})
    L = _hip.lib()
    a = _hip.Linear(4, 8, 8, 6, 0, 0)
    assert L.mrl_linear_act(a, None, None, None, None, None, None, None) == -1 and b'null' in L.mrl_last_error()
    assert L.mrl_linear_act(None, None, None, None, None, None, None, None) == -1
    assert L.mrl_linear_act_backward_workspace_bytes(a) > 0
    assert L.mrl_linear_act_backward(a, 16, 16, None, 16, 16, 16, 16, None, 0, None) == -2
    a.act = 1
    assert L.mrl_linear_act_backward(a, 16, 16, None, 16, 16, 16, 16, 16, 1 << 30, None) == -1
    a.x_stride = 3
    assert L.mrl_linear_act(a, 16, 16, None, None, 16, None, None) == -1 and b'x_stride' in L.mrl_last_error()
    for bad in (_hip.Linear(4, 8, 8, 6, 3, 0), _hip.Linear(4, 8, 8, 6, 0, 6), _hip.Linear(-1, 8, 8, 6, 0, 0), _hip.Linear(4, 1 << 25, 1 << 25, 6, 0, 0), _hip.Linear(1 << 30, 8, 8, 256, 0, 0)):
        assert L.mrl_linear_act_backward_workspace_bytes(bad) == -1

"""The memory operators under what torch puts between a program and a kernel: dispatch modes, tracers, lazily negated tensors.
Each has to see one operator, not the allocations inside it, and to get the operator's own result."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

DEV = 'cuda:0'


def ops():
    import mineral_amd.ops  # noqa: F401
    return torch.ops.mineral


def inputs(device=DEV, dtype=torch.float32):
    """Name -> (call, differentiable inputs by position, all inputs)."""
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)  # noqa: E731
    M = ops()
    decay = (-torch.rand(3, generator=g)).to(device)
    state = torch.randn(2, 3, 8, 12, generator=g).to(device)
    resets = torch.zeros(2, 5, dtype=torch.bool, device=device)
    return {
        'linear_attention': (lambda q, k, v, l, s: M.linear_attention(q, k, v, l, resets, s, 0.5), (0, 1, 2, 4), [r(2, 5, 3, 8), r(2, 5, 3, 8), r(2, 5, 3, 12), decay, state]),
        'linear_attention_step': (lambda q, k, v, l, s: M.linear_attention_step(q, k, v, l, s, None, 0.5), (), [r(2, 3, 8), r(2, 3, 8), r(2, 3, 12), decay, state.clone()]),
        'group_norm_act': (lambda x, w, b: M.group_norm_act(x, 4, w, b, 1e-5, 'SiLU'), (0, 1, 2), [r(6, 32), r(32), r(32)]),
        'linear_act': (lambda x, w, b, y: M.linear_act(x, w, b, y, 'Tanh'), (0, 1, 2, 3), [r(6, 16), r(24, 16), r(24), r(6, 24)]),
    }


NAMES = ('linear_attention', 'linear_attention_step', 'group_norm_act', 'linear_act')
# what a differentiable call is made of
HALVES = {'linear_attention': ('linear_attention', '_linear_attention_backward'), 'group_norm_act': ('_group_norm_act_stats', '_group_norm_act_backward'),
          'linear_act': ('_linear_act_slope', '_linear_act_backward')}


def flat(out):
    return [out] if isinstance(out, torch.Tensor) else list(out)


def with_gradient(name, device=DEV, dtype=torch.float32):
    call, where, args = inputs(device, dtype)[name]

    def run(*args):
        args = [t.detach().requires_grad_(True) if i in where else t for i, t in enumerate(args)]
        out = flat(call(*args))
        return out + list(torch.autograd.grad(out, [args[i] for i in where], [torch.full_like(t, 0.5) for t in out]))
    return run, args


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.gpu
@pytest.mark.parametrize('name', NAMES)
def test_a_dispatch_mode_sees_the_operator(name):
    call, _, args = inputs()[name]
    want = flat(call(*[t.clone() for t in args]))
    with Seen() as seen:
        got = flat(call(*args))
    assert seen.names == [f'mineral.{name}.default']
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize('name', HALVES)
def test_a_dispatch_mode_sees_both_halves(name):
    run, args = with_gradient(name)
    want = run(*args)
    with Seen() as seen:
        got = run(*args)
    assert [n for n in seen.names if n.startswith('mineral.')] == [f'mineral.{h}.default' for h in HALVES[name]]
    assert not [n for n in seen.names if n.startswith('aten.empty.')]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize('name', NAMES)
def test_a_traced_call_runs_the_operator(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    call, _, args = inputs()[name]
    graph = make_fx(lambda *a: tuple(2 * t for t in flat(call(*a))))(*[t.clone() for t in args])
    assert f'mineral.{name}' in graph.code
    others = [t.clone() if i == 3 and 'attention' in name else t * 0.5 for i, t in enumerate(args)]      # other values than the traced ones
    want = [2 * t for t in flat(call(*[t.clone() for t in others]))]
    assert all(torch.equal(a, b) for a, b in zip(graph(*[t.clone() for t in others]), want))


@pytest.mark.gpu
@pytest.mark.parametrize('name', HALVES)
def test_a_traced_gradient_runs_the_operators(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    run, args = with_gradient(name)
    graph = make_fx(run)(*args)
    assert all(f'mineral.{h}.' in graph.code for h in HALVES[name])
    others = [t.clone() if i == 3 and 'attention' in name else t * 0.5 for i, t in enumerate(args)]
    assert all(torch.equal(a, b) for a, b in zip(graph(*others), run(*others)))


def negated(t):
    """The same values, held with the opposite sign and a note to negate them."""
    n = torch._neg_view(-t)
    assert n.is_neg() and torch.equal(n, t)
    return n


@pytest.mark.gpu
@pytest.mark.parametrize('name', NAMES)
def test_a_lazily_negated_tensor_is_read_with_its_sign(name):
    call, where, args = inputs()[name]
    for i, t in enumerate(args):
        plain, lazy = [a.clone() for a in args], [a.clone() for a in args]
        lazy[i] = negated(t)
        assert all(torch.equal(a, b) for a, b in zip(flat(call(*lazy)), flat(call(*plain)))), i
        assert all(torch.equal(a, b) for a, b in zip(lazy, plain)), i          # a state too
    if where:
        run, args = with_gradient(name)
        want = run(*args)
        got = run(*[negated(t) if i in where else t for i, t in enumerate(args)])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize('name', HALVES)
def test_a_gradient_that_arrives_lazily_negated(name):
    call, where, args = inputs()[name]
    args = [t.clone().requires_grad_(True) if i in where else t for i, t in enumerate(args)]
    leaves = [args[i] for i in where]
    out = flat(call(*args))
    g = [torch.linspace(-1, 1, t.numel(), device=DEV).view(t.shape) for t in out]
    want = torch.autograd.grad(out, leaves, g, retain_graph=True)
    got = torch.autograd.grad(out, leaves, [negated(t) for t in g])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def dual(name, device, i):
    """The call with a tangent on input i, inside a dual level."""
    import torch.autograd.forward_ad as fwd
    call, _, args = inputs(device)[name]
    with fwd.dual_level():
        return call(*[fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)])


@pytest.mark.parametrize('name', NAMES)
def test_a_forward_mode_derivative_is_refused(name):
    """Before anything else is asked, the device among it."""
    for i in range(len(inputs('cpu')[name][2])):
        with pytest.raises(NotImplementedError, match='forward-mode'):
            dual(name, 'cpu', i)
        with pytest.raises(NotImplementedError, match='forward-mode'), torch.no_grad():
            dual(name, 'cpu', i)


@pytest.mark.gpu
@pytest.mark.parametrize('name', NAMES)
def test_a_forward_mode_derivative_is_refused_on_the_device(name):
    import torch.autograd.forward_ad as fwd
    call, where, args = inputs()[name]
    for i in range(len(args)):
        with pytest.raises(NotImplementedError, match='forward-mode'):
            dual(name, DEV, i)
    # a tangent that arrives with the gradient
    if where:
        leaves = [t.clone().requires_grad_(True) if i in where else t for i, t in enumerate(args)]
        out = flat(call(*leaves))
        with fwd.dual_level():
            g = [fwd.make_dual(torch.ones_like(t), torch.ones_like(t)) for t in out]
            with pytest.raises(NotImplementedError, match='forward-mode'):
                torch.autograd.grad(out, [leaves[i] for i in where], g)
    # a dual level without tangents, and tangents that are switched off, change nothing
    want = flat(call(*[t.clone() for t in args]))
    with fwd.dual_level():
        assert all(torch.equal(a, b) for a, b in zip(flat(call(*[t.clone() for t in args])), want))
        with fwd._set_fwd_grad_enabled(False):
            assert all(torch.equal(a, b) for a, b in zip(flat(call(*[t.clone() for t in args])), want))


@pytest.mark.parametrize('name', HALVES)
def test_a_functional_jvp_is_refused(name):
    call, where, args = inputs('cpu')[name]
    with pytest.raises(NotImplementedError, match='forward-mode'):
        torch.func.jvp(lambda t: call(t, *args[1:]), (args[0],), (torch.ones_like(args[0]),))

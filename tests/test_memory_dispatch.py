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


def shapes(outs):
    return [(tuple(t.shape), t.dtype, t.is_contiguous()) for t in outs]


EXPECTED = {'linear_attention': [(2, 5, 3, 12), (2, 3, 8, 12)], 'linear_attention_step': [(2, 3, 12)], 'group_norm_act': [(6, 32)], 'linear_act': [(6, 24)]}


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('name', NAMES)
def test_shapes_of_tensors_without_data(name, dtype):
    call, where, args = inputs('meta', dtype)[name]
    out = flat(call(*args))
    assert [tuple(t.shape) for t in out] == EXPECTED[name] and all(t.is_meta and t.is_contiguous() for t in out)
    assert out[0].dtype == dtype and (len(out) == 1 or out[1].dtype == torch.float32)
    if where:
        run, args = with_gradient(name, 'meta', dtype)
        got = run(*args)
        assert shapes(got[len(out):]) == [(tuple(args[i].shape), args[i].dtype, True) for i in where]


@pytest.mark.parametrize('name', NAMES)
def test_a_trace_without_data_records_the_operator(name):
    """Tensors of a device that need not be there, and, with the gradient, of none."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    call, where, args = inputs('meta')[name]
    if name != 'linear_attention':          # whose resets are a constant of the call
        with FakeTensorMode():
            on_device = [torch.empty(t.shape, dtype=t.dtype, device=DEV) for t in args]
            assert f'torch.ops.mineral.{name}' in make_fx(lambda *a: tuple(2 * t for t in flat(call(*a))))(*on_device).code
    if where:
        run, args = with_gradient(name, 'meta')
        code = make_fx(run)(*args).code
        assert all(f'torch.ops.mineral.{h}.' in code for h in HALVES[name]) and 'aten.empty.' not in code


def test_symbolic_sizes():
    from torch.fx.experimental.proxy_tensor import make_fx
    M = ops()
    for name, fn, args in (('linear_act', lambda x, w: M.linear_act(x, w, None, None, 'SiLU'), [torch.empty(6, 16, device='meta'), torch.empty(24, 16, device='meta')]),
                           ('group_norm_act', lambda x: M.group_norm_act(x, 4, None, None, 1e-5, None), [torch.empty(6, 9, 32, device='meta')]),
                           ('linear_attention', lambda q, k, v, l: M.linear_attention(q, k, v, l)[1], [torch.empty(2, 5, 3, 8, device='meta')] * 2 + [torch.empty(2, 5, 3, 12, device='meta'), torch.empty(3, device='meta')])):
        graph = make_fx(fn, tracing_mode='symbolic')(*args)
        assert f'torch.ops.mineral.{name}' in graph.code
        more = [t.new_empty((7, *t.shape[1:])) if t.dim() > 2 or name == 'linear_act' and i == 0 else t for i, t in enumerate(args)]
        assert graph(*more).shape == fn(*more).shape and graph(*more).shape[0] == 7


def test_shapes_that_do_not_fit_are_refused_without_data():
    M = ops()
    e = lambda *s, **k: torch.empty(*s, device='meta', **k)  # noqa: E731
    for bad in (lambda: M.linear_act(e(4, 8), e(6, 7)), lambda: M.linear_act(e(4, 8), e(6, 8), e(5)), lambda: M.linear_act(e(4, 8), e(6, 8), None, e(1, 6)),
                lambda: M.linear_act(e(4, 8), e(6, 8, dtype=torch.half)), lambda: M.group_norm_act(e(4, 9), 2), lambda: M.group_norm_act(e(4, 8), 2, e(4)),
                lambda: M.linear_attention(e(2, 4, 2, 8), e(2, 4, 2, 8), e(2, 3, 2, 8), e(2)), lambda: M.linear_attention(e(2, 4, 2, 8), e(2, 4, 2, 8), e(2, 4, 2, 8), e(3)),
                lambda: M.linear_attention_step(e(2, 2, 8), e(2, 2, 8), e(2, 2, 8), e(2), e(2, 2, 8, 4)), lambda: M.linear_act(e(4, 8, dtype=torch.double), e(6, 8, dtype=torch.double))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize('name', NAMES)
def test_shape_functions_agree_with_the_kernels(name):
    call, where, args = inputs()[name]
    assert shapes(flat(call(*[t.clone() for t in args]))) == shapes(flat(inputs('meta')[name][0](*[t.to('meta') for t in args])))
    if where:
        run, args = with_gradient(name)
        meta, margs = with_gradient(name, 'meta')
        assert shapes(run(*args)) == shapes(meta(*margs))


@pytest.mark.gpu
@pytest.mark.parametrize('name', NAMES)
def test_torchs_own_checks_of_an_operator(name):
    _, where, args = inputs()[name]
    M = ops()
    full = {'linear_attention': lambda: (*args[:4], None, args[4], 0.5), 'linear_attention_step': lambda: (*args[:4], args[4], None, 0.5),
            'group_norm_act': lambda: (args[0], 4, *args[1:], 1e-5, 'SiLU'), 'linear_act': lambda: (*args, 'Tanh')}[name]()
    full = tuple(t.clone().requires_grad_(True) if any(t is args[i] for i in where) else t for t in full)
    torch.library.opcheck(getattr(M, name).default, full, test_utils=('test_schema', 'test_autograd_registration', 'test_faketensor'))


@pytest.mark.gpu
@pytest.mark.parametrize('name', HALVES)
def test_a_compiled_call_gives_the_same(name):
    """Ahead-of-time traced, forward and backward, and run as the trace stands."""
    call, where, args = inputs()[name]
    compiled = torch.compile(lambda *a: flat(call(*a)), backend='aot_eager', fullgraph=True)

    def run(fn):
        leaves = [t.clone().requires_grad_(True) if i in where else t for i, t in enumerate(args)]
        out = flat(fn(*leaves))
        return [t.detach() for t in out] + list(torch.autograd.grad(out, [leaves[i] for i in where], [torch.ones_like(t) for t in out]))
    assert all(torch.equal(a, b) for a, b in zip(run(compiled), run(call)))


@pytest.mark.gpu
def test_a_compiled_step_updates_its_state():
    call, _, args = inputs()['linear_attention_step']
    compiled = torch.compile(lambda *a: call(*a), backend='aot_eager', fullgraph=True)
    mine, theirs = args[4].clone(), args[4].clone()
    with torch.no_grad():
        for _ in range(3):
            assert torch.equal(compiled(*args[:4], mine), call(*args[:4], theirs)) and torch.equal(mine, theirs)


@pytest.mark.gpu
def test_states_of_inference_mode():
    """Updated there, and outside refused before anything is written."""
    call, _, args = inputs()['linear_attention_step']
    want = args[4].clone()
    out = call(*args[:4], want)
    with torch.inference_mode():
        state = args[4].clone()
        assert torch.equal(call(*args[:4], state), out) and torch.equal(state, want)
        held = state.clone()
    with pytest.raises(RuntimeError, match='inference'):
        call(*args[:4], state)
    assert torch.equal(state, held)
    q, k, v, l = (t.clone() for t in args[:4])
    with torch.inference_mode():
        others = [t.clone() for t in (q, k, v, l)]
    with pytest.raises(RuntimeError, match='inference'):
        call(*others, state)
    assert torch.equal(state, held)


@pytest.mark.gpu
@pytest.mark.parametrize('name', HALVES)
def test_a_call_mapped_over_a_batch(name):
    """torch.vmap has no rule for the operators and calls them one by one."""
    call, where, args = inputs()[name]
    x = torch.stack([args[0], args[0] * 0.5, -args[0]])
    got = flat(torch.vmap(lambda t: call(t, *args[1:]))(x))
    want = [torch.stack(ts) for ts in zip(*(flat(call(t, *args[1:])) for t in x))]
    assert all(torch.equal(a, b) for a, b in zip(got, want))

"""The memory operators as a policy uses them together: a block in front of the towers projects observations to queries, keys and
values, attends over the rollout, normalises each head, projects back with a residual and adds a feed-forward part; acting, the
same block runs one step at a time.  Every stage is held to its own definition on what the stage before it gave (the bounds are
those of the single operators' tests), and the block's gradients to the chain of the stages' gradients, bit for bit."""

import pytest
import torch

import test_group_norm_act as gn
import test_linear_act as la
import test_linear_attention as at

DEV = 'cuda:0'
B, T, H, K, V, C, F = 6, 40, 4, 16, 24, 64, 128
SCALE = 0.25


def ops():
    import mineral_amd.ops  # noqa: F401
    return torch.ops.mineral


def params(dt, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    p = dict(w_qkv=r(H * (2 * K + V), C) / C ** 0.5, b_qkv=r(H * (2 * K + V)) * 0.1, gamma=1 + 0.1 * r(H * V), beta=0.1 * r(H * V), w_o=r(C, H * V) / (H * V) ** 0.5, b_o=r(C) * 0.1,
             w_1=r(F, C) / C ** 0.5, b_1=r(F) * 0.1, w_2=r(C, F) / F ** 0.5, b_2=r(C) * 0.1)
    p = {k: v.to(dt).to(DEV) for k, v in p.items()}
    log_decay = torch.log1p(-torch.exp2(-torch.linspace(1, 6, H))).to(DEV)
    return p, log_decay, r(B, T, C).to(dt).to(DEV), (torch.rand(B, T, generator=g) < 0.1).to(DEV), r(B, H, K, V).to(DEV), r(B, T, C).to(dt).to(DEV), r(B, H, K, V).to(DEV)


def block(p, l, x, resets, state, step=False, keep=None):
    """x [B,T,C] (or [B,C] acting) -> y like x, final state (acting: `state` is updated)."""
    M = ops()
    keep = {} if keep is None else keep
    rows = x.shape[:-1]
    qkv = keep['qkv'] = M.linear_act(x, p['w_qkv'], p['b_qkv'], None, None)
    q, k, v = keep['cut'] = [t.unflatten(-1, (H, -1)) for t in qkv.split([H * K, H * K, H * V], -1)]
    if step:
        o, final = M.linear_attention_step(q, k, v, l, state, resets, SCALE), state
    else:
        o, final = M.linear_attention(q, k, v, l, resets, state, SCALE)
    keep['o'], keep['final'] = o, final
    n = keep['n'] = M.group_norm_act(o.reshape(-1, H * V), H, p['gamma'], p['beta'], 1e-5, 'SiLU').view(*rows, H * V)
    h = keep['h'] = M.linear_act(n, p['w_o'], p['b_o'], x, None)
    f = keep['f'] = M.linear_act(h, p['w_1'], p['b_1'], None, 'SiLU')
    y = keep['y'] = M.linear_act(f, p['w_2'], p['b_2'], h, None)
    return y, final


def check_linear(y, x, w, b, r, act):
    x, w, b = (t.detach().double().cpu() for t in (x.reshape(-1, x.shape[-1]), w, b))
    z = x @ w.t() + b
    ref = la.act64(z, act)
    mag = x.abs() @ w.abs().t() + b.abs()
    k = x.shape[-1]
    ze = ((k + 16) * la.U + 4 * la.U) * mag
    bound = 1.13 * ze + 16 * la.U * (z.abs() + 1) + 4 * la.U * z.abs()
    if r is not None:
        r = r.detach().double().cpu().reshape(ref.shape)
        ref, bound = ref + r, bound + 4 * la.U * r.abs()
    la.close(y.detach().reshape(ref.shape), ref, bound, 'linear_act')


def check_stages(p, l, x, resets, state0, keep, dt):
    check_linear(keep['qkv'], x, p['w_qkv'], p['b_qkv'], None, None)
    q, k, v = (t.detach().double().cpu() for t in keep['cut'])
    if x.dim() == 2:
        q, k, v = q[:, None], k[:, None], v[:, None]
    r = resets.cpu() if x.dim() == 3 else resets.cpu()[:, None]
    s, lc = state0.double().cpu(), l.cpu()
    o, S = at.recurrence(q, k, v, lc, r, s, SCALE)
    mo, mS = at.recurrence(q.abs(), k.abs(), v.abs(), lc, r, s.abs(), SCALE)
    at.check(keep['o'].detach().reshape(o.shape), o, mo, dt, o.shape[1], K, 'o')
    at.check(keep['final'].detach(), S, mS, dt, o.shape[1], K, 'state')
    flat = keep['o'].detach().reshape(-1, H * V).double().cpu()
    w, b = p['gamma'].detach().double().cpu(), p['beta'].detach().double().cpu()
    ref = gn.reference(flat, H, w, b, 1e-5, 'SiLU')[0]
    gn.close(keep['n'].detach().reshape(ref.shape), ref, gn.bounds(flat, H, w, b, torch.zeros_like(flat), 1e-5)[0], 'n')
    check_linear(keep['h'], keep['n'], p['w_o'], p['b_o'], x, None)
    check_linear(keep['f'], keep['h'], p['w_1'], p['b_1'], None, 'SiLU')
    check_linear(keep['y'], keep['f'], p['w_2'], p['b_2'], keep['h'], None)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', at.DT)
def test_a_rollout_and_its_gradient(dtype):
    dt = at.DT[dtype]
    p, l, x, resets, state, dy, df = params(dt, 1)
    p = {k: v.requires_grad_(True) for k, v in p.items()}
    x, state = x.requires_grad_(True), state.requires_grad_(True)
    keep = {}
    y, final = block(p, l, x, resets, state, keep=keep)
    check_stages(p, l, x, resets, state.detach(), keep, dt)
    leaves = [x, state, *p.values()]
    got = dict(zip(('x', 'state', *p), torch.autograd.grad((y, final), leaves, (dy, df))))
    # the chain by hand, each stage differentiated by itself from detached inputs
    M, want = ops(), {}

    def stage(fn, inputs, g):
        ins = [t.detach().requires_grad_(True) for t in inputs]
        out = fn(*ins)
        return torch.autograd.grad(out, ins, g)
    k = {n: ([t.detach() for t in v] if n == 'cut' else v.detach()) for n, v in keep.items()}
    d = {n: v.detach() for n, v in p.items()}
    df_, want['w_2'], want['b_2'], dh = stage(lambda f, w, b, r: M.linear_act(f, w, b, r, None), (k['f'], d['w_2'], d['b_2'], k['h']), dy)
    dh2, want['w_1'], want['b_1'] = stage(lambda h, w, b: M.linear_act(h, w, b, None, 'SiLU'), (k['h'], d['w_1'], d['b_1']), df_)
    dn, want['w_o'], want['b_o'], dx = stage(lambda n, w, b, r: M.linear_act(n, w, b, r, None), (k['n'], d['w_o'], d['b_o'], x), dh + dh2)
    do, want['gamma'], want['beta'] = stage(lambda o, w, b: M.group_norm_act(o, H, w, b, 1e-5, 'SiLU'), (k['o'].reshape(-1, H * V), d['gamma'], d['beta']), dn.reshape(-1, H * V))
    dq, dk, dv, want['state'] = stage(lambda q, kk, v, s: M.linear_attention(q, kk, v, l, resets, s, SCALE), (*k['cut'], state), (do.view(B, T, H, V), df))
    dqkv = torch.cat([t.reshape(B, T, -1) for t in (dq, dk, dv)], -1)
    dx2, want['w_qkv'], want['b_qkv'] = stage(lambda a, w, b: M.linear_act(a, w, b, None, None), (x, d['w_qkv'], d['b_qkv']), dqkv)
    want['x'] = dx + dx2
    for n, g in want.items():
        assert torch.isfinite(g).all() and float(g.abs().max()) > 0, n
        assert torch.equal(got[n], g), n


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', at.DT)
def test_acting_step_by_step(dtype):
    dt = at.DT[dtype]
    p, l, x, resets, state, _, _ = params(dt, 2)
    with torch.no_grad():
        for t in range(8):
            before, keep = state.clone(), {}
            block(p, l, x[:, t], resets[:, t], state, step=True, keep=keep)
            check_stages(p, l, x[:, t], resets[:, t], before, keep, dt)


@pytest.mark.gpu
def test_acting_from_a_captured_graph():
    p, l, x, resets, state, _, _ = params(torch.bfloat16, 3)
    with torch.no_grad():
        xs, rs, live, eager = x[:, 0].clone(), resets[:, 0].clone(), state.clone(), state.clone()
        block(p, l, xs, rs, state.clone(), step=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, _ = block(p, l, xs, rs, live, step=True)
        live.copy_(state)
        for t in range(6):
            xs.copy_(x[:, t])
            rs.copy_(resets[:, t])
            graph.replay()
            torch.cuda.synchronize()
            want, _ = block(p, l, x[:, t], resets[:, t], eager, step=True)
            assert torch.equal(y, want) and torch.equal(live, eager), t

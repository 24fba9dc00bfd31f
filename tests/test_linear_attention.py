"""torch.ops.mineral.linear_attention / linear_attention_step against the recurrence in 64 bits.

Tolerances.  With A the same recurrence over absolute values (the sum of the magnitudes of all terms of an output), an output
is off by at most eps/2 of itself (its one rounding to its type, plus half a spacing of the subnormals) plus u A:
  * fp32 accumulation: a term passes through at most T + K + C sums and 8 weights of one rounding each: (T + K + 80) 2^-24;
  * 16-bit inputs: P and S enter an output's product as two bf16 terms, off by 2^-17 (a term meets one of them), and the product
    drops at most 2^-16 (both low terms, fp16): 2^-15 covers both.
The state is fp32 and is bounded by u A alone, where 16-bit inputs lose nothing beyond fp32's own rounding either (three terms,
2^-24, counted among the 80)."""

import ctypes as C

import pytest
import torch

DEV = 'cuda:0'
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def ops():
    import mineral_amd.ops  # noqa: F401
    return torch.ops.mineral


def recurrence(q, k, v, log_decay, resets, state, scale):
    """The definition, in float64, differentiable."""
    B, T, H, K = q.shape
    S = torch.zeros(B, H, K, v.shape[-1], dtype=torch.float64) if state is None else state
    lam = torch.exp(log_decay.double()).view(1, H, 1, 1)
    out = []
    for t in range(T):
        S = S * lam
        if resets is not None:
            S = torch.where(resets[:, t].bool().view(B, 1, 1, 1), torch.zeros((), dtype=torch.float64), S)
        S = S + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append((S * q[:, t, :, :, None]).sum(2) * scale)
    return (torch.stack(out, 1) if out else v.new_zeros(v.shape)), S


def unit(dtype, T, K):
    return (T + K + 80) * 2.0 ** -24 + (2.0 ** -15 if dtype != torch.float32 else 0.0)    # dtype: the output's


def check(got, ref, mag, dtype, T, K, what):
    """|got - ref| <= rounding of the output + u * magnitude, elementwise."""
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps if got.dtype != torch.float32 else 1e-37
    err = (got.double().cpu() - ref).abs()
    lim = half * ref.abs() * (1 + 2.0 ** -8) + unit(got.dtype, T, K) * mag + tiny
    bad = err > lim
    assert not bool(bad.any()), f'{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / lim).max()):.2f} of the bound'


def make(B, T, H, K, V, dt, seed, p_reset=0.1, initial=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = r(B, T, H, K).to(dt), r(B, T, H, K).to(dt), r(B, T, H, V).to(dt)
    log_decay = -torch.exp(torch.empty(H).uniform_(-6, 1, generator=g))
    resets = torch.rand(B, T, generator=g) < p_reset if p_reset > 0 else None
    state = r(B, H, K, V) if initial else None
    return q, k, v, log_decay, resets, state


def dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def doubles(*ts):
    return [None if t is None else (t if t.dtype in (torch.bool, torch.uint8) else t.double()) for t in ts]


SHAPES = [(1, 1, 1, 1, 1), (2, 2, 3, 5, 7), (3, 31, 2, 32, 32), (2, 33, 1, 16, 32), (2, 63, 2, 64, 64), (1, 64, 3, 64, 64), (2, 65, 2, 40, 72), (1, 130, 2, 128, 128),
          (2, 97, 1, 127, 3), (1, 700, 2, 64, 64), (1, 1025, 3, 24, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('resets,initial', [(0.0, False), (0.1, True)])
def test_forward_matches_the_recurrence(dtype, shape, resets, initial):
    B, T, H, K, V = shape
    x = make(*shape, DT[dtype], 1, resets, initial)
    print(f'forward {dtype} {shape} {resets}', flush=True)
    got, final = ops().linear_attention(*dev(*x), 0.3)
    assert got.dtype == DT[dtype] and final.dtype == torch.float32 and got.shape == (B, T, H, V)
    ref, S = recurrence(*doubles(*x), 0.3)
    q, k, v, l, r, s = doubles(*x)
    mag, Smag = recurrence(q.abs(), k.abs(), v.abs(), l, r, None if s is None else s.abs(), 0.3)
    check(got, ref, mag, DT[dtype], T, K, 'out')
    check(final, S, Smag, DT[dtype], T, K, 'final state')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape', [(1, 1, 1, 1, 1), (2, 5, 3, 8, 12), (2, 32, 2, 64, 64), (1, 65, 2, 40, 72), (2, 130, 2, 128, 64), (1, 600, 2, 32, 32), (1, 700, 1, 17, 65)])
@pytest.mark.parametrize('resets,initial', [(0.0, False), (0.1, True)])
def test_gradients_match_the_recurrence(dtype, shape, resets, initial):
    B, T, H, K, V = shape
    q, k, v, l, r, s = make(*shape, DT[dtype], 2, resets, initial)
    g = torch.Generator().manual_seed(3)
    do, df = torch.randn(B, T, H, V, generator=g).to(DT[dtype]), torch.randn(B, H, K, V, generator=g)

    def grads(q, k, v, s, do, df):
        leaves = [t.double().requires_grad_(True) for t in (q, k, v)] + ([] if s is None else [s.double().requires_grad_(True)])
        o, f = recurrence(*leaves[:3], l.double(), r, None if s is None else leaves[3], 0.3)
        return torch.autograd.grad((o, f), leaves, (do.double(), df.double()))

    ref = grads(q, k, v, s, do, df)
    mag = grads(q.abs(), k.abs(), v.abs(), None if s is None else s.abs(), do.abs(), df.abs())
    print(f'gradients {dtype} {shape} {resets}', flush=True)
    leaves = [t.to(DEV).requires_grad_(True) for t in ((q, k, v) if s is None else (q, k, v, s))]
    o, f = ops().linear_attention(*leaves[:3], *dev(l, r), None if s is None else leaves[3], 0.3)
    got = torch.autograd.grad((o, f), leaves, (do.to(DEV), df.to(DEV)))
    for n, a, b, m in zip(('dq', 'dk', 'dv', 'd_initial'), got, ref, mag):
        assert a.shape == b.shape
        check(a, b, m, DT[dtype], T, max(K, V), n)
    # only the state, or only one input, asks for its gradient
    o, f = ops().linear_attention(leaves[0].detach(), leaves[1], leaves[2].detach(), *dev(l, r, s), 0.3)
    (dk,) = torch.autograd.grad(f, leaves[1], df.to(DEV))
    zero = torch.zeros_like(do)
    check(dk, grads(q, k, v, s, zero, df)[1], grads(q.abs(), k.abs(), v.abs(), None if s is None else s.abs(), zero, df.abs())[1], DT[dtype], T, max(K, V), 'dk alone')


@pytest.mark.gpu
def test_gradients_match_differences():
    """The operator is linear in each of q, k, v and the state, so a symmetric difference is the directional derivative up to rounding."""
    q, k, v, l, r, s = dev(*make(2, 70, 2, 48, 56, torch.float32, 5))
    g = torch.Generator(device=DEV).manual_seed(6)
    do, df = torch.randn(v.shape, device=DEV, generator=g), torch.randn(s.shape, device=DEV, generator=g)

    def loss(q, k, v, s):
        o, f = ops().linear_attention(q, k, v, l, r, s, 0.3)
        return (o.double() * do).sum() + (f.double() * df).sum()

    xs = [q, k, v, s]
    leaves = [x.clone().requires_grad_(True) for x in xs]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i, n in enumerate('qkvs'):
        d = torch.randn(xs[i].shape, device=DEV, generator=g)
        up, down = list(xs), list(xs)
        up[i], down[i] = xs[i] + d, xs[i] - d
        diff = (loss(*up) - loss(*down)) / 2
        want = (grads[i].double() * d).sum()
        # both are sums of the same terms; magnitude: sum of |terms| of the loss at |x| + |d|, each off by (T + K + 80) 2^-24 twice
        mag = [x.abs().cpu().double() for x in xs]
        mag[i] = mag[i] + d.abs().cpu().double()
        om, fm = recurrence(*mag[:3], l.cpu().double(), r.cpu(), mag[3], 0.3)
        lim = 4 * unit(torch.float32, 70, 56) * float((om * do.abs().cpu()).sum() + (fm * df.abs().cpu()).sum())
        assert abs(float(diff - want)) <= lim, n


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
def test_steps_equal_the_sequence(dtype):
    B, T, H, K, V = 5, 12, 3, 40, 20
    x = make(B, T, H, K, V, DT[dtype], 7, 0.2, True)
    q, k, v, l, r, s = dev(*x)
    ref, S = recurrence(*doubles(*x), 0.5)
    d = doubles(*x)
    mag, Smag = recurrence(d[0].abs(), d[1].abs(), d[2].abs(), d[3], d[4], d[5].abs(), 0.5)
    state, outs = s.clone(), []
    for t in range(T):
        outs.append(ops().linear_attention_step(q[:, t], k[:, t], v[:, t], l, state, r[:, t], 0.5))
    check(torch.stack(outs, 1), ref, mag, DT[dtype], T, K, 'out')
    check(state, S, Smag, DT[dtype], T, K, 'state')
    # no resets given, a byte mask, and rows that a second call continues
    one = ops().linear_attention_step(q[:, 0], k[:, 0], v[:, 0], l, s.clone(), r[:, 0].to(torch.uint8), 0.5)
    assert torch.equal(one, outs[0])
    half = s.clone()
    ops().linear_attention_step(q[:, 0], k[:, 0], v[:, 0], l, half, None, 0.5)
    _, S1 = recurrence(d[0][:, :1], d[1][:, :1], d[2][:, :1], d[3], None, d[5], 0.5)
    _, M1 = recurrence(d[0][:, :1].abs(), d[1][:, :1].abs(), d[2][:, :1].abs(), d[3], None, d[5].abs(), 0.5)
    check(half, S1, M1, DT[dtype], 1, K, 'state without resets')


@pytest.mark.gpu
@pytest.mark.parametrize('K,V', [(1, 1), (3, 5), (32, 32), (64, 64), (128, 128), (100, 36), (7, 128), (128, 2), (33, 65)])
@pytest.mark.parametrize('dtype', DT)
def test_step_widths(dtype, K, V):
    x = make(7, 1, 2, K, V, DT[dtype], 8, 0.3, True)
    q, k, v, l, r, s = dev(*x)
    d = doubles(*x)
    ref, S = recurrence(*d, 0.7)
    mag, Smag = recurrence(d[0].abs(), d[1].abs(), d[2].abs(), d[3], d[4], d[5].abs(), 0.7)
    out = ops().linear_attention_step(q[:, 0], k[:, 0], v[:, 0], l, s, r[:, 0], 0.7)
    check(out, ref[:, 0], mag[:, 0], DT[dtype], 1, K, 'out')
    check(s, S, Smag, DT[dtype], 1, K, 'state')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T,at,end', [(50, 10, 20), (60, 0, 20), (200, 70, 70), (200, 64, 127), (900, 300, 640)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_what_a_reset_drops_leaks_nowhere(dtype, T, at, end, bad):
    """Token `at` and the state on entry hold `bad`; a new episode begins at `end + 1`.  Tokens before `at` (after the first reset)
    and after `end` are those of the clean inputs, bit for bit where the chunks are walked alike and to the bound otherwise."""
    B, H, K, V = 2, 2, 32, 48
    x = make(B, T, H, K, V, DT[dtype], 9, 0.0, True)
    q, k, v, l, _, s = x
    resets = torch.zeros(B, T, dtype=torch.bool)
    resets[:, 0] = True
    resets[:, end + 1] = True
    d = doubles(q, k, v, l)
    ref, S = recurrence(*d, resets, None, 1.0)
    mag, Smag = recurrence(d[0].abs(), d[1].abs(), d[2].abs(), d[3], resets, None, 1.0)
    for which in 'qkvs':
        xs = dict(q=q.clone(), k=k.clone(), v=v.clone(), s=s.clone())
        if which == 's':
            xs['s'][:, :, 0] = bad
        else:
            xs[which][:, at, :, 0] = bad
        print(f'masked {dtype} T={T} {which}={bad}', flush=True)
        leaves = [t.to(DEV).requires_grad_(True) for t in (xs['q'], xs['k'], xs['v'], xs['s'])]
        o, f = ops().linear_attention(*leaves[:3], *dev(l, resets), leaves[3], 1.0)
        clean = torch.ones(T, dtype=torch.bool)
        if which != 's':
            clean[at:end + 1] = False
        check(o[:, clean.to(DEV)], ref[:, clean], mag[:, clean], DT[dtype], T, K, f'out beside a bad {which}')
        check(f, S, Smag, DT[dtype], T, K, f'state after a bad {which}')
        if which != 's':
            assert not torch.isfinite(o[:, at]).all()
        # backwards: the other episodes' gradients are finite, and nothing reaches the state that the first token drops
        grads = torch.autograd.grad((o, f), leaves, (torch.ones_like(o), torch.ones_like(f)))
        later = torch.arange(T, device=DEV) > end
        for a in grads[:3]:
            assert torch.isfinite(a[:, later]).all()
        assert torch.equal(grads[3], torch.zeros_like(grads[3]))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
def test_layouts_and_strides(dtype):
    """Slices of a fused projection, head-major tensors, rows on odd addresses, a broadcast key: the same bits as contiguous ones."""
    B, T, H, K, V = 2, 75, 3, 16, 24
    q, k, v, l, r, s = dev(*make(B, T, H, K, V, DT[dtype], 11))
    want = ops().linear_attention(q, k, v, l, r, s, 0.25)
    fused = torch.cat([t.reshape(B, T, -1) for t in (q, k, v)], -1)
    fq, fk, fv = (t.unflatten(-1, (H, -1)) for t in fused.split([H * K, H * K, H * V], -1))
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    odd = []
    for t in (q, k, v):
        buf = torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)
        buf[1:] = t.reshape(-1)
        odd.append(buf[1:].view(t.shape))
    last = [torch.stack([t, t], -1)[..., 0] for t in (q, k, v)]      # the last dimension is not contiguous
    for xs in ((fq, fk, fv), heads_first, odd, last):
        got = ops().linear_attention(*xs, l, r, s, 0.25)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    k1 = k[:, :, :1].contiguous()
    got = ops().linear_attention(q, k1.expand(B, T, H, K), v, l, r.to(torch.uint8), s, 0.25)
    ref = ops().linear_attention(q, k1.expand(B, T, H, K).contiguous(), v, l, r, s, 0.25)
    assert torch.equal(got[0], ref[0])
    # a broadcast key's gradient is the sum over its heads
    a, b = k1.clone().requires_grad_(True), k1.expand(B, T, H, K).contiguous().requires_grad_(True)
    go = torch.randn_like(v)
    (ga,) = torch.autograd.grad(ops().linear_attention(q, a.expand(B, T, H, K), v, l, r, s, 0.25)[0], a, go)
    (gb,) = torch.autograd.grad(ops().linear_attention(q, b, v, l, r, s, 0.25)[0], b, go)
    assert torch.equal(ga, gb.sum(2, keepdim=True))
    # a gradient that arrives broadcast
    o, _ = ops().linear_attention(q, b, v, l, r, s, 0.25)
    (g1,) = torch.autograd.grad(o.sum(), b, retain_graph=True)
    (g2,) = torch.autograd.grad(o, b, torch.ones_like(o))
    assert torch.equal(g1, g2)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Two batch rows 2^31 + 64 elements apart in one allocation."""
    B, T, H, K, V = 2, 40, 1, 32, 32
    q, k, v, l, r, s = dev(*make(B, T, H, K, V, torch.bfloat16, 12))
    want = ops().linear_attention(q, k, v, l, r, s, 1.0)
    far = 2 ** 31 + 64
    big = torch.empty(far + T * H * K, dtype=torch.bfloat16, device=DEV)
    qq = big.as_strided((B, T, H, K), (far, H * K, K, 1))
    qq.copy_(q)
    got = ops().linear_attention(qq, k, v, l, r, s, 1.0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_extreme_decays():
    B, T, H, K, V = 1, 150, 4, 16, 16
    q, k, v, _, r, s = make(B, T, H, K, V, torch.float32, 13)
    l = torch.tensor([0.0, -1e-6, -30.0, -float('inf')])
    d = doubles(q, k, v, l, r, s)
    ref, S = recurrence(*d, 1.0)
    mag, Smag = recurrence(d[0].abs(), d[1].abs(), d[2].abs(), d[3], d[4], d[5].abs(), 1.0)
    got, final = ops().linear_attention(*dev(q, k, v, l, r, s), 1.0)
    check(got, ref, mag, torch.float32, T, K, 'out')
    check(final, S, Smag, torch.float32, T, K, 'state')


@pytest.mark.gpu
def test_nothing_to_do():
    q, k, v, l, r, s = dev(*make(2, 0, 3, 8, 8, torch.bfloat16, 14))
    o, f = ops().linear_attention(q, k, v, l, r, s, 1.0)
    assert o.shape == (2, 0, 3, 8) and torch.equal(f, s)
    o, f = ops().linear_attention(q, k, v, l, None, None, 1.0)
    assert torch.equal(f, torch.zeros_like(s))
    s2 = s.clone().requires_grad_(True)
    o, f = ops().linear_attention(q, k, v, l, r, s2, 1.0)
    (ds,) = torch.autograd.grad(f, s2, s)
    assert torch.equal(ds, s)
    e = dev(*make(0, 5, 3, 8, 8, torch.float32, 15))
    o, f = ops().linear_attention(*e, 1.0)
    assert o.shape == (0, 5, 3, 8) and f.shape == (0, 3, 8, 8)
    assert ops().linear_attention_step(e[0][:, 0], e[1][:, 0], e[2][:, 0], e[3], e[5], None, 1.0).shape == (0, 3, 8)


@pytest.mark.gpu
def test_streams_and_graphs():
    """On another stream, and captured: every replay, with eager work between, gives the eager bits."""
    q, k, v, l, r, s = dev(*make(1, 700, 2, 64, 64, torch.bfloat16, 16))
    do, df = torch.randn_like(v), torch.randn_like(s)

    def both(q, k, v, s):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, s)]
        o, f = ops().linear_attention(*leaves[:3], l, r, leaves[3], 0.2)
        return (o, f, *torch.autograd.grad((o, f), leaves, (do, df)))

    want = [t.clone() for t in both(q, k, v, s)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(q, k, v, s)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    state = s.clone()
    with torch.cuda.graph(graph):
        held = both(q, k, v, s)
        stepped = ops().linear_attention_step(q[:, 0], k[:, 0], v[:, 0], l, state, None, 0.2)
    eager = s.clone()
    for _ in range(3):
        for t in held:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        o = ops().linear_attention_step(q[:, 0], k[:, 0], v[:, 0], l, eager, None, 0.2)
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert torch.equal(stepped, o) and torch.equal(state, eager)
        assert all(torch.equal(a, b) for a, b in zip(both(q, k, v, s), want))


@pytest.mark.gpu
def test_refusals_on_the_device():
    q, k, v, l, r, s = dev(*make(2, 4, 2, 8, 8, torch.float32, 17))
    M = ops()
    with pytest.raises(NotImplementedError, match='log_decay'):
        M.linear_attention(q.requires_grad_(True), k, v, l.clone().requires_grad_(True), r, s, 1.0)
    with pytest.raises(NotImplementedError, match='no gradient'):
        M.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], l, s, None, 1.0)
    # what a step overwrites is not what an earlier call's gradient reads
    for mode in (torch.no_grad, torch.inference_mode):
        out, _ = M.linear_attention(q, k, v, l, r, s, 1.0)
        with mode():
            M.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], l, s, None, 1.0)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            out.sum().backward()
    q = q.detach()
    with pytest.raises(ValueError, match='in place'):
        M.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], l, s.transpose(2, 3), None, 1.0)
    with pytest.raises(ValueError, match='tensors on'):
        M.linear_attention(q, k, v, l, r.cpu(), s, 1.0)


def test_refusals():
    """Argument checks, on CPU tensors: they come before the refusal of the CPU itself."""
    from mineral_amd import _hip
    M = ops()
    q, k, v, l, r, s = make(2, 4, 2, 8, 12, torch.float32, 18)
    ok = dict(q=q, k=k, v=v, log_decay=l, resets=r, initial_state=s, scale=1.0)
    with pytest.raises(NotImplementedError, match='CPU'):
        M.linear_attention(**ok)
    wide = torch.zeros(2, 4, 2, 129)
    for change, text in ((dict(q=q.double()), 'dtype'), (dict(k=k.half()), 'one type'), (dict(k=k[:, :3]), 'dim_k'), (dict(v=v[:1]), 'dim_v'),
                         (dict(log_decay=l[:1]), 'log_decay'), (dict(log_decay=l.double()), 'log_decay'), (dict(resets=r.float()), 'resets'),
                         (dict(resets=r[:, :2]), 'resets'), (dict(initial_state=s.half()), 'state'), (dict(initial_state=s[:, :1]), 'state'), (dict(q=q[0]), 'dim_k'),
                         (dict(q=wide, k=wide), '128'), (dict(v=v[..., :0]), 'dim_v'), (dict(q=q[:, :, :0], k=k[:, :, :0], v=v[:, :, :0]), 'heads')):
        with pytest.raises(ValueError, match=text):
            M.linear_attention(**{**ok, **change})
    step = dict(q=q[:, 0], k=k[:, 0], v=v[:, 0], log_decay=l, state=s, resets=r[:, 0], scale=1.0)
    with pytest.raises(NotImplementedError, match='CPU'):
        M.linear_attention_step(**step)
    for change, text in ((dict(state=s.transpose(2, 3).contiguous().transpose(2, 3)), 'in place'), (dict(state=s[:1]), 'state'), (dict(resets=r), 'resets'), (dict(q=q), 'dim_k')):
        with pytest.raises(ValueError, match=text):
            M.linear_attention_step(**{**step, **change})
    # the C ABI
    L = _hip.lib()
    i3 = C.c_int64 * 3

    def desc(B=2, T=4, H=2, K=8, V=12, dtype=0):
        return _hip.Attention(B, T, H, K, V, dtype, 16, 16, 16, i3(T * H * K, H * K, K), i3(T * H * K, H * K, K), i3(T * H * V, H * V, V), 16, None, None, 1.0)
    a = desc()
    assert L.mrl_linear_attention_workspace_bytes(a, 0) == 0
    for bad in (desc(K=129), desc(V=0), desc(H=0), desc(T=-1), desc(T=1 << 30), desc(B=1 << 30), desc(B=1 << 22), desc(dtype=7)):
        assert L.mrl_linear_attention_workspace_bytes(bad, 0) == -1
    assert L.mrl_linear_attention(a, None, None, None, 0, None) == -1 and b'null output' in L.mrl_last_error()
    assert L.mrl_linear_attention(None, None, None, None, 0, None) == -1
    assert L.mrl_linear_attention_step(a, None, None, None) == -1 and b'steps' in L.mrl_last_error()
    assert L.mrl_linear_attention_backward(a, None, None, None, None, None, None, None, None, 0, None) == -1
    assert L.mrl_linear_attention_backward(a, 16, i3(0, 0, 0), None, 16, 16, None, 16, None, 0, None) == -1 and b'd_initial_state' in L.mrl_last_error()
    assert L.mrl_linear_attention(a, 8, 16, None, 0, None) == -1 and b'aligned' in L.mrl_last_error()
    assert L.mrl_linear_attention_backward(a, 16, i3(0, 0, 0), None, 16, 8, 16, None, None, 0, None) == -1 and b'aligned' in L.mrl_last_error()
    long = desc(T=4096)
    assert L.mrl_linear_attention_workspace_bytes(long, 0) > 0
    assert L.mrl_linear_attention(long, 16, 16, None, 0, None) == -2 and b'workspace' in L.mrl_last_error()


def test_header_and_binding_list_the_same_entry_points():
    import os
    import re
    from mineral_amd import _hip
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r'/\*.*?\*/', '', open(os.path.join(root, 'include', 'mineral_memory.h')).read(), flags=re.S)
    names = sorted(set(re.findall(r'\b(mrl_[a-z0-9_]+)\s*\(', text)))
    assert sorted(_hip.MEMORY_EXPORTS) == names
    assert all(hasattr(_hip.lib(), n) for n in names)

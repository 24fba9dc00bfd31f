"""The operators of a sequence memory in front of the policy towers, as they are measured: linear attention with a decay for
each head (over whole rollouts and prompts, with its gradient, and one step at a time), group norm with an activation on
channels-last data, and a linear layer with bias, activation and residual in its epilogue.

`listed()` and `draw()` give the cases, `prepare()` the inputs of one, `run()` one pass through the operator: in its plain form
(elementary torch operations in 32 bits, rounded once at the end) or, where `own` is set, through `torch.ops.mineral.*`.
`exact()` computes the same outputs in 64 bits from the operators' definitions, `work()` what a pass cannot do without.
"""

import math

import torch

own = False

DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
EPS = 1e-5


# ---- the cases ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a handful of environments acting through a narrow memory: nothing but latency
        dict(name='act 64 envs', op='attention', mode='step', dtype='bfloat16', batch=64, steps=1, heads=4, dim_k=32, dim_v=32, resets=0.05, initial=True),
        # the acting step of a large vectorised environment: the state of every environment is read and written once
        dict(name='act 8192 envs', op='attention', mode='step', dtype='float32', batch=8192, steps=1, heads=4, dim_k=64, dim_v=64, resets=0.02, initial=True),
        # one minibatch of a recurrent update: 2048 environments x 32 steps with episode ends inside, state carried in and out
        dict(name='rollout train', op='attention', mode='train', dtype='float32', batch=2048, steps=32, heads=4, dim_k=64, dim_v=64, resets=0.02, initial=True),
        # one long demonstration or prompt: few rows, a long axis
        dict(name='long prompt', op='attention', mode='forward', dtype='bfloat16', batch=1, steps=16384, heads=8, dim_k=128, dim_v=128, resets=0.0, initial=False),
        # whole episodes of odd length packed into a few rows, keys narrower than values, an odd number of heads
        dict(name='episodes train', op='attention', mode='train', dtype='float16', batch=3, steps=1021, heads=5, dim_k=40, dim_v=72, resets=0.003, initial=False),
        # the norm over each head's output for a handful of rows: nothing but latency
        dict(name='head norm 64 rows', op='norm', mode='forward', dtype='bfloat16', batch=64, pixels=1, channels=512, groups=8, act='SiLU'),
        # the norm over each head's output for a minibatch of tokens, both directions
        dict(name='head norm train', op='norm', mode='train', dtype='bfloat16', batch=65536, pixels=1, channels=512, groups=8, act='SiLU'),
        # frames of an encoder: 84 x 84 pixels, 32 channels in 8 groups, both directions
        dict(name='frames train', op='norm', mode='train', dtype='float32', batch=64, pixels=7056, channels=32, groups=8, act='SiLU'),
        # the layer of a policy acting for 64 environments: the weights are what is read
        dict(name='linear 64 rows', op='linear', mode='forward', dtype='bfloat16', batch=64, inputs=512, outputs=2048, act='SiLU', residual=False),
        # the wide layer of a feed-forward block on one minibatch, both directions
        dict(name='linear train', op='linear', mode='train', dtype='bfloat16', batch=32768, inputs=512, outputs=2048, act='SiLU', residual=True),
        # the second tower layer of the shipped configuration on one minibatch
        dict(name='tower layer', op='linear', mode='forward', dtype='float32', batch=32768, inputs=512, outputs=256, act='ELU', residual=False),
        # sizes that fit no tile, both directions
        dict(name='linear odd train', op='linear', mode='train', dtype='float16', batch=4099, inputs=333, outputs=777, act='Tanh', residual=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w['bytes'], w['flops'] / 50.0)


def draw(rng):
    most = {}
    for c in listed():
        key = (c['op'], c['mode'])
        most[key] = max(most.get(key, 0.0), _cost(c))
    op, mode = rng.choice([('attention', 'step'), ('attention', 'train'), ('attention', 'forward'), ('norm', 'train'), ('norm', 'forward'), ('linear', 'train'),
                           ('linear', 'forward')])
    top = max(v for k, v in most.items() if k[0] == op)
    while True:
        dtype = rng.choice(list(DTYPES))
        if op == 'attention':
            head = rng.choice([32, 64, 64, 128])
            odd = rng.random() < 0.4
            dim_k = rng.randrange(8, 129) if odd else head
            dim_v = rng.randrange(8, 129) if odd else head
            case = dict(op=op, mode=mode, dtype=dtype, batch=1, steps=1, heads=rng.randrange(1, 13), dim_k=dim_k, dim_v=dim_v,
                        resets=rng.choice([0.0, 0.003, 0.02, 0.1]), initial=mode == 'step' or rng.random() < 0.5)
            if mode == 'step':
                case['batch'] = _log_int(rng, 1, 8192)
            else:
                case['steps'] = _log_int(rng, 1, 16384)
                case['batch'] = _log_int(rng, 1, max(1, 65536 // case['steps']))
        elif op == 'norm':
            groups = rng.choice([1, 2, 4, 8, 16, 32])
            case = dict(op=op, mode=mode, dtype=dtype, batch=1, pixels=1, channels=groups, groups=groups, act=rng.choice(['SiLU', 'ELU', 'Tanh', 'none']))
            if rng.random() < 0.5:                 # tokens: a group is a head's width (a norm over two or three values has no gradient to speak of)
                case['channels'] *= _log_int(rng, 16, 128)
                case['batch'] = _log_int(rng, 1, 65536)
            else:
                case['channels'] *= _log_int(rng, 2, 128)
                case['pixels'] = rng.randrange(3, 85) ** 2
                case['batch'] = _log_int(rng, 1, 512)
        else:
            # the rectifier's gradient jumps at zero: it is measured forwards only
            act = rng.choice(['SiLU', 'ELU', 'Tanh', 'none'] + (['ReLU'] if mode == 'forward' else []))
            case = dict(op=op, mode=mode, dtype=dtype, batch=_log_int(rng, 1, 32768), inputs=_log_int(rng, 16, 2048), outputs=_log_int(rng, 16, 2048), act=act,
                        residual=rng.random() < 0.5)
        if _cost(case) <= top:
            return case


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def _normal(gen, shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device='cuda', dtype=torch.float32) * std + mean


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(int(seed))
    dt = DTYPES[case['dtype']]
    train = case['mode'] == 'train'
    s = dict(case=dict(case))
    if case['op'] == 'attention':
        B, T, H, K, V = (case[k] for k in ('batch', 'steps', 'heads', 'dim_k', 'dim_v'))
        # q, k and v as a fused projection leaves them: three slices of one tensor
        qkv = _normal(gen, (B, T, H * (2 * K + V))).to(dt)
        q, k, v = qkv.split([H * K, H * K, H * V], dim=-1)
        s['q'], s['k'], s['v'] = q.view(B, T, H, K), k.view(B, T, H, K), v.view(B, T, H, V)
        # a spread of memories over the heads, from about 16 steps to about 2000
        span = torch.linspace(4.0, 11.0, H, device='cuda', dtype=torch.float64)
        s['log_decay'] = torch.log1p(-torch.exp2(-span)).to(torch.float32)
        s['scale'] = 1.0 / math.sqrt(K)
        s['resets'] = torch.rand((B, T), generator=gen, device='cuda') < case['resets'] if case['resets'] > 0 else None
        s['initial'] = _normal(gen, (B, H, K, V)) if case['initial'] else None
        if case['mode'] == 'step':
            for n in ('q', 'k', 'v'):
                s[n] = s[n][:, 0]
            if s['resets'] is not None:
                s['resets'] = s['resets'][:, 0].contiguous()
        if train:
            s['d_out'] = _normal(gen, (B, T, H, V)).to(dt)
            s['d_final'] = _normal(gen, (B, H, K, V))
            for n in ('q', 'k', 'v', 'initial'):
                if s[n] is not None:
                    s[n] = s[n].detach().requires_grad_(True)
    elif case['op'] == 'norm':
        C = case['channels']
        shape = (case['batch'], C) if case['pixels'] == 1 else (case['batch'], case['pixels'], C)
        s['x'] = _normal(gen, shape, 1.5, 0.3).to(dt)
        s['weight'], s['bias'] = _normal(gen, (C,), 0.2, 1.0).to(dt), _normal(gen, (C,), 0.2).to(dt)
        if train:
            s['d_out'] = _normal(gen, shape).to(dt)
            for n in ('x', 'weight', 'bias'):
                s[n] = s[n].requires_grad_(True)
    else:
        M, K, N = case['batch'], case['inputs'], case['outputs']
        s['x'] = _normal(gen, (M, K)).to(dt)
        s['weight'], s['bias'] = _normal(gen, (N, K), 1.0 / math.sqrt(K)).to(dt), _normal(gen, (N,), 0.1).to(dt)
        s['residual'] = _normal(gen, (M, N)).to(dt) if case['residual'] else None
        if train:
            s['d_out'] = _normal(gen, (M, N)).to(dt)
            for n in ('x', 'weight', 'bias'):
                s[n] = s[n].requires_grad_(True)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------------
def run(state):
    form = _own if own else _plain
    return form[state['case']['op'], state['case']['mode'] == 'train', state['case']['mode'] == 'step'](state)


def _ops():
    import mineral_amd.ops  # noqa: F401  (registers the operators)
    return torch.ops.mineral


def _act_name(s):
    a = s['case']['act']
    return None if a == 'none' else a


def _own_attention(s):
    o, final = _ops().linear_attention(s['q'], s['k'], s['v'], s['log_decay'], s['resets'], s['initial'], s['scale'])
    return {'out': o, 'final': final}


def _own_attention_train(s):
    o, final = _ops().linear_attention(s['q'], s['k'], s['v'], s['log_decay'], s['resets'], s['initial'], s['scale'])
    leaves = [s[n] for n in ('q', 'k', 'v', 'initial') if s[n] is not None]
    grads = torch.autograd.grad((o, final), leaves, (s['d_out'], s['d_final']))
    return {'out': o, 'final': final, 'grads': list(grads)}


def _own_attention_step(s):
    o = _ops().linear_attention_step(s['q'], s['k'], s['v'], s['log_decay'], s['initial'], s['resets'], s['scale'])
    return {'out': o, 'state': s['initial']}


def _own_norm(s):
    return {'out': _ops().group_norm_act(s['x'], s['case']['groups'], s['weight'], s['bias'], EPS, _act_name(s))}


def _own_norm_train(s):
    y = _ops().group_norm_act(s['x'], s['case']['groups'], s['weight'], s['bias'], EPS, _act_name(s))
    return {'out': y, 'grads': list(torch.autograd.grad(y, (s['x'], s['weight'], s['bias']), s['d_out']))}


def _own_linear(s):
    return {'out': _ops().linear_act(s['x'], s['weight'], s['bias'], s['residual'], _act_name(s))}


def _own_linear_train(s):
    y = _ops().linear_act(s['x'], s['weight'], s['bias'], s['residual'], _act_name(s))
    return {'out': y, 'grads': list(torch.autograd.grad(y, (s['x'], s['weight'], s['bias']), s['d_out']))}


# ---- the plain form: elementary operations in 32 bits, rounded once at the end ---------------------------------------------------
def _act32(z, name):
    if name == 'SiLU':
        return z * torch.sigmoid(z)
    if name == 'ELU':
        return torch.where(z > 0, z, torch.expm1(z))
    if name == 'Tanh':
        return torch.tanh(z)
    if name == 'ReLU':
        return torch.clamp(z, min=0)
    return z


def _act32_slope(z, name):
    if name == 'SiLU':
        g = torch.sigmoid(z)
        return g * (1 + z * (1 - g))
    if name == 'ELU':
        return torch.where(z > 0, torch.ones_like(z), torch.exp(z))
    if name == 'Tanh':
        t = torch.tanh(z)
        return 1 - t * t
    if name == 'ReLU':
        return (z > 0).to(z.dtype)
    return torch.ones_like(z)


def _scan32(q, k, v, log_decay, clears, state, off):
    """Linear attention in chunks.  q, k [B,H,T,K], v [B,H,T,V], all fp32; clears [B,T] whole numbers: how often the state was
    cleared before token i reads it, and the same after the last token [B]; off: how many decays lie between the state on entry
    and the first token's reading (1 forwards, 0 backwards in time, where the decay follows the write).  Exponents in 64 bits."""
    seg, total = clears
    B, H, T, K = q.shape
    V = v.shape[-1]
    C = min(64, T)
    N = -(-T // C)
    pad = N * C - T
    l = log_decay.double()
    dev = q.device

    def power(n):                                  # decay ** n for each head, n a table of whole numbers
        return torch.exp(l.view(H, *([1] * n.dim())) * n.double()).float()

    far = T - off - torch.arange(T, device=dev)    # decays between token j's write and the end
    w = power(far) * (seg == total[:, None])[:, None]                              # [B,H,T]
    final = torch.matmul(k.transpose(2, 3).contiguous(), v * w[..., None])
    if state is not None:
        final = final + state * (power(torch.full((1,), T, device=dev)).view(1, H, 1, 1) * (total == 0).view(B, 1, 1, 1))

    def cut(x):
        return torch.nn.functional.pad(x, (0, 0, 0, pad)).view(B, H, N, C, x.shape[-1])
    qc, kc, vc = cut(q), cut(k), cut(v)
    # the padding continues the last token's segment
    sc = torch.cat([seg, total[:, None].expand(B, pad)], dim=1).view(B, N, C)
    # how often the state has been cleared when chunk c ends: what the next chunk's entry has seen
    ends = sc[:, :, -1] if off else torch.cat([sc[:, 1:, 0], total[:, None]], dim=1)
    i = torch.arange(C, device=dev)
    gap = (i[:, None] - i[None, :]).clamp(min=0)
    keep = (i[:, None] >= i[None, :]) & (sc[..., :, None] == sc[..., None, :])     # [B,N,C,C]
    p = torch.matmul(qc, kc.transpose(3, 4).contiguous()) * power(gap).view(1, H, 1, C, C) * keep[:, None]
    out = torch.matmul(p, vc)
    if N > 1 or state is not None:
        wl = power(C - off - i).view(1, H, 1, C) * (sc == ends[..., None])[:, None]
        local = torch.matmul(kc.transpose(3, 4).contiguous(), vc * wl[..., None])  # [B,H,N,K,V]
        first = torch.zeros(B, H, 1, K, V, device=dev) if state is None else state[:, :, None]
        parts = torch.cat([first, local[:, :, :-1]], dim=2).reshape(B, H, N, K * V)
        c = torch.arange(N, device=dev)
        seen = torch.cat([torch.zeros_like(ends[:, :1]), ends[:, :-1]], dim=1)      # at the entry of chunk c
        mix = power((C * (c[:, None] - c[None, :])).clamp(min=0)) * ((c[:, None] >= c[None, :]) & (seen[:, :, None] == seen[:, None, :]))[:, None]
        entry = torch.matmul(mix, parts).view(B, H, N, K, V)
        read = power(i + off).view(1, H, 1, C) * (sc == seen[..., None])[:, None]
        out = out + torch.matmul(qc, entry) * read[..., None]
    return out.reshape(B, H, N * C, V)[:, :, :T], final


def _heads_first(x):
    return x.detach().float().transpose(1, 2).contiguous()


def _clears32(resets, B, T, backwards):
    if resets is None:
        seg = torch.zeros(B, T, dtype=torch.int64, device='cuda')
        return seg, seg[:, 0]
    if not backwards:
        seg = torch.cumsum(resets.long(), dim=1)
        return seg, seg[:, -1]
    r = torch.flip(resets.long(), [1])
    seg = torch.cumsum(r, dim=1)
    return seg - r, seg[:, -1]


def _plain_attention_of(s):
    q, k, v = (_heads_first(s[n]) for n in ('q', 'k', 'v'))
    B, _, T, _ = q.shape
    state = None if s['initial'] is None else s['initial'].detach()
    o, final = _scan32(q * s['scale'], k, v, s['log_decay'], _clears32(s['resets'], B, T, False), state, 1)
    return q, k, v, state, {'out': o.transpose(1, 2).contiguous().to(s['q'].dtype), 'final': final}


def _plain_attention(s):
    with torch.no_grad():
        return _plain_attention_of(s)[4]


def _plain_attention_train(s):
    """The gradients are the same scan with the operands in other places: dq reads (d_out, v) against k forwards in time, dk and dv
    run backwards from the final state's gradient."""
    with torch.no_grad():
        q, k, v, state, got = _plain_attention_of(s)
        B, _, T, _ = q.shape
        dt = s['q'].dtype
        g = _heads_first(s['d_out']) * s['scale']
        dq, _ = _scan32(g, v, k, s['log_decay'], _clears32(s['resets'], B, T, False), None if state is None else state.transpose(2, 3).contiguous(), 1)
        back = [torch.flip(x, [2]) for x in (q, k, v, g)]
        clears = _clears32(s['resets'], B, T, True)
        dk, _ = _scan32(back[2], back[3], back[0], s['log_decay'], clears, s['d_final'].transpose(2, 3).contiguous(), 0)
        dv, d_state = _scan32(back[1], back[0], back[3], s['log_decay'], clears, s['d_final'], 0)
        grads = [x.transpose(1, 2).contiguous().to(dt) for x in (dq, torch.flip(dk, [2]), torch.flip(dv, [2]))]
        got['grads'] = grads + ([] if state is None else [d_state])
        return got


def _plain_attention_step(s):
    with torch.no_grad():
        q, k, v = (s[n].float() for n in ('q', 'k', 'v'))
        decay = torch.exp(s['log_decay'].double()).float().view(1, -1, 1, 1)
        if s['resets'] is not None:
            decay = decay * (~s['resets']).view(-1, 1, 1, 1)
        state = s['initial'] * decay + k[..., None] * v[..., None, :]
        s['initial'].copy_(state)
        return {'out': ((q * s['scale'])[..., None] * state).sum(dim=2).to(s['q'].dtype), 'state': s['initial']}


def _plain_norm_of(s):
    x = s['x'].detach().float()
    G, C = s['case']['groups'], x.shape[-1]
    xg = x.reshape(x.shape[0], -1, G, C // G)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    mid = xg - mean
    rstd = 1 / torch.sqrt((mid * mid).mean(dim=(1, 3), keepdim=True) + EPS)
    xhat = (mid * rstd).reshape(x.shape)
    z = xhat * s['weight'].detach().float() + s['bias'].detach().float()
    return xhat, rstd, z, {'out': _act32(z, s['case']['act']).to(s['x'].dtype)}


def _plain_norm(s):
    with torch.no_grad():
        return _plain_norm_of(s)[3]


def _plain_norm_train(s):
    with torch.no_grad():
        xhat, rstd, z, got = _plain_norm_of(s)
        dt, shape = s['x'].dtype, xhat.shape
        G, C = s['case']['groups'], shape[-1]
        dz = s['d_out'].float() * _act32_slope(z, s['case']['act'])
        rows = tuple(range(dz.dim() - 1))
        d_weight, d_bias = (dz * xhat).sum(dim=rows), dz.sum(dim=rows)
        dh = (dz * s['weight'].detach().float()).reshape(shape[0], -1, G, C // G)
        hg = xhat.reshape(dh.shape)
        dx = rstd * (dh - dh.mean(dim=(1, 3), keepdim=True) - hg * (dh * hg).mean(dim=(1, 3), keepdim=True))
        got['grads'] = [dx.reshape(shape).to(dt), d_weight.to(dt), d_bias.to(dt)]
        return got


def _plain_linear_of(s):
    x, w = s['x'].detach().float(), s['weight'].detach().float()
    z = torch.matmul(x, w.t()) + s['bias'].detach().float()
    y = _act32(z, s['case']['act'])
    if s['residual'] is not None:
        y = y + s['residual'].float()
    return x, w, z, {'out': y.to(s['x'].dtype)}


def _plain_linear(s):
    with torch.no_grad():
        return _plain_linear_of(s)[3]


def _plain_linear_train(s):
    with torch.no_grad():
        x, w, z, got = _plain_linear_of(s)
        dz = s['d_out'].float() * _act32_slope(z, s['case']['act'])
        dt = s['x'].dtype
        got['grads'] = [torch.matmul(dz, w).to(dt), torch.matmul(dz.t(), x).to(dt), dz.sum(dim=0).to(dt)]
        return got


# keyed by (operator, training, single step)
_plain = {('attention', False, False): _plain_attention, ('attention', True, False): _plain_attention_train, ('attention', False, True): _plain_attention_step,
          ('norm', False, False): _plain_norm, ('norm', True, False): _plain_norm_train, ('linear', False, False): _plain_linear,
          ('linear', True, False): _plain_linear_train}
_own = {('attention', False, False): _own_attention, ('attention', True, False): _own_attention_train, ('attention', False, True): _own_attention_step,
        ('norm', False, False): _own_norm, ('norm', True, False): _own_norm_train, ('linear', False, False): _own_linear,
        ('linear', True, False): _own_linear_train}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------
def work(case):
    e = torch.empty(0, dtype=DTYPES[case['dtype']]).element_size()
    train = case['mode'] == 'train'
    if case['op'] == 'attention':
        B, T, H, K, V = (case[k] for k in ('batch', 'steps', 'heads', 'dim_k', 'dim_v'))
        rows, state = B * T * H, B * H * K * V * 4
        nbytes = rows * (2 * K + 2 * V) * e + state * (2 if case['initial'] else 1) + (B * T if case['resets'] > 0 else 0) + H * 4
        flops = rows * 5 * K * V                   # decay, outer product and reading: the recurrent form
        if train:                                  # q, k, v and d_out again, three gradients, the states and their gradients
            nbytes += rows * (4 * K + 3 * V) * e + state * (3 if case['initial'] else 1)
            flops += rows * 13 * K * V
        return {'bytes': nbytes, 'flops': flops}
    if case['op'] == 'norm':
        n = case['batch'] * case['pixels'] * case['channels']
        return {'bytes': (5 if train else 2) * n * e + (4 if train else 2) * case['channels'] * e, 'flops': (30 if train else 10) * n}
    M, K, N = case['batch'], case['inputs'], case['outputs']
    nbytes = (M * K + N * K + N + M * N * (2 if case['residual'] else 1)) * e
    flops = 2 * M * N * K
    if train:                                      # x, weight and d_out again, three gradients
        nbytes += (M * N + 2 * M * K + 2 * N * K + N) * e
        flops *= 3
    return {'bytes': nbytes, 'flops': flops}


# ---- the same outputs in 64 bits, from the definitions ---------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {'attention': _exact_attention, 'norm': _exact_norm, 'linear': _exact_linear}[case['op']](case, s)


def _exact_attention(case, s):
    """The recurrence itself, one token after the other: S = decay * S (cleared where a token begins an episode) + k v^T, o = S^T q."""
    step = case['mode'] == 'step'
    q, k, v = (s[n].detach().double() for n in ('q', 'k', 'v'))
    if step:
        q, k, v = q[:, None], k[:, None], v[:, None]
    B, T, H, K = q.shape
    V = v.shape[-1]
    decay = torch.exp(s['log_decay'].double()).view(1, H, 1, 1)
    r = s['resets']
    stay = torch.ones(B, T, 1, 1, 1, dtype=torch.float64, device='cuda') if r is None else (~r).double().view(B, T, 1, 1, 1)
    S = torch.zeros(B, H, K, V, dtype=torch.float64, device='cuda') if s['initial'] is None else s['initial'].detach().double()
    train = case['mode'] == 'train'
    out, dq = torch.empty(B, T, H, V, dtype=torch.float64, device='cuda'), torch.empty_like(q)
    g = s['d_out'].double() * s['scale'] if train else None
    for t in range(T):
        S = S * (decay * stay[:, t]) + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = (S * q[:, t, :, :, None]).sum(dim=2) * s['scale']
        if train:
            dq[:, t] = (S * g[:, t, :, None, :]).sum(dim=3)
    if step:
        return {'out': out[:, 0], 'state': S}
    got = {'out': out, 'final': S}
    if train:
        D, dk, dv = s['d_final'].double(), torch.empty_like(k), torch.empty_like(v)
        for t in range(T - 1, -1, -1):
            D = D + q[:, t, :, :, None] * g[:, t, :, None, :]
            dk[:, t] = (D * v[:, t, :, None, :]).sum(dim=3)
            dv[:, t] = (D * k[:, t, :, :, None]).sum(dim=2)
            D = D * (decay * stay[:, t])
        got['grads'] = [dq, dk, dv] + ([D] if case['initial'] else [])
    return got


def _value_and_slope(z, name):
    """An activation and its derivative in 64 bits."""
    one = torch.ones_like(z)
    if name == 'SiLU':
        e = torch.exp(-z)
        return z / (1 + e), (1 + e + z * e) / (1 + e) ** 2
    if name == 'ELU':
        low = torch.exp(torch.minimum(z, 0 * z))
        return torch.where(z > 0, z, torch.expm1(torch.minimum(z, 0 * z))), torch.where(z > 0, one, low)
    if name == 'Tanh':
        t = torch.tanh(z)
        return t, 1 / torch.cosh(z) ** 2
    if name == 'ReLU':
        return torch.where(z > 0, z, 0 * z), torch.where(z > 0, one, 0 * z)
    return z, one


def _exact_norm(case, s):
    x = s['x'].detach().double()
    n, C, G = x.shape[0], case['channels'], case['groups']
    parts = x.reshape(n, -1, C).reshape(n, -1, G, C // G).permute(0, 2, 1, 3).reshape(n, G, -1)
    size = parts.shape[-1]
    mean = parts.sum(-1, keepdim=True) / size
    sd = torch.sqrt(((parts - mean) ** 2).sum(-1, keepdim=True) / size + EPS)

    def back(p):
        return p.reshape(n, G, -1, C // G).permute(0, 2, 1, 3).reshape(x.shape)
    unit = (parts - mean) / sd
    w, b = s['weight'].detach().double(), s['bias'].detach().double()
    y, slope = _value_and_slope(back(unit) * w + b, case['act'])
    got = {'out': y}
    if case['mode'] == 'train':
        dz = s['d_out'].double() * slope
        du = (dz * w).reshape(n, -1, G, C // G).permute(0, 2, 1, 3).reshape(n, G, -1)
        dx = (size * du - du.sum(-1, keepdim=True) - unit * (du * unit).sum(-1, keepdim=True)) / (size * sd)
        got['grads'] = [back(dx), (dz * back(unit)).reshape(-1, C).sum(0), dz.reshape(-1, C).sum(0)]
    return got


def _exact_linear(case, s):
    x, w = s['x'].detach().double(), s['weight'].detach().double()
    y, slope = _value_and_slope(x @ w.t() + s['bias'].detach().double(), case['act'])
    if s['residual'] is not None:
        y = y + s['residual'].double()
    got = {'out': y}
    if case['mode'] == 'train':
        dz = s['d_out'].double() * slope
        got['grads'] = [dz @ w, dz.t().contiguous() @ x, dz.sum(0)]
    return got

"""The operators of a sequence memory as PyTorch custom operators: `torch.ops.mineral.*` over include/mineral_memory.h.

    import mineral_amd.ops
    o, state = torch.ops.mineral.linear_attention(q, k, v, log_decay, resets, initial_state, scale)      # a rollout, a prompt
    o = torch.ops.mineral.linear_attention_step(q, k, v, log_decay, state, resets, scale)                # one token, acting
    y = torch.ops.mineral.group_norm_act(x, num_groups, weight, bias, eps, act_type)                     # channels last
    y = torch.ops.mineral.linear_act(x, weight, bias, residual, act_type)                                # act(x W^T + b) + residual

`act_type` is a name of the towers' configuration (None, 'SiLU', 'ELU', 'ReLU', 'Tanh') or 'GELU'.

Registered for the device key only, like the operators of ops.py: CPU tensors fail in the dispatcher.  Tensors keep their type
(float32, bfloat16 or float16); states are float32.  Calls run on the current stream of the tensors' device, whichever device is
current.  Operators are differentiable once unless their description says otherwise; a call that cannot be served raises.
"""

import ctypes as C

import torch

from . import _hip

_lib = torch.library.Library('mineral', 'FRAGMENT')

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_I3 = C.c_int64 * 3


class _on:
    """The tensors' device made current for the launch; nothing where it is already."""

    def __init__(self, t):
        self.guard = None if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


def _stream(t):
    return torch.cuda.current_stream(t.device).cuda_stream


def _require(ok, what, message):
    if not ok:
        raise ValueError(f'{what}: {message}')


def _same_device(what, t, *others):
    for o in others:
        if o is not None and o.device != t.device:
            raise ValueError(f'{what}: tensors on {t.device} and {o.device}')


def _rows(t):
    """`t` with its last dimension contiguous; every other stride stays."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _p(t):
    return None if t is None else t.data_ptr()


# ---- linear attention ----------------------------------------------------------------------------------------------------------
def _attention(what, q, k, v, log_decay, resets, state, scale, step):
    """Checks of the arguments, and their description; the second value keeps the tensors that it points into."""
    _require(q.dtype in _DTYPES, what, f'dtype {q.dtype} (float32, bfloat16 or float16)')
    _require(k.dtype == q.dtype and v.dtype == q.dtype, what, f'q, k and v of one type, got {q.dtype}, {k.dtype}, {v.dtype}')
    dims = 3 if step else 4
    _require(q.dim() == dims and k.shape == q.shape and v.dim() == dims and v.shape[:-1] == q.shape[:-1], what,
             f'q and k [batch, {"" if step else "steps, "}heads, dim_k], v [.., dim_v]; got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}')
    _same_device(what, q, k, v, log_decay, resets, state)
    B, H, K, V = q.shape[0], q.shape[-2], q.shape[-1], v.shape[-1]
    T = 1 if step else q.shape[1]
    _require(log_decay.dtype == torch.float32 and log_decay.shape == (H,), what, f'log_decay: float32 [{H}], got {log_decay.dtype} {tuple(log_decay.shape)}')
    if resets is not None:
        _require(resets.dtype in (torch.bool, torch.uint8) and resets.shape == ((B,) if step else (B, T)), what,
                 f'resets: bool or uint8 of {(B,) if step else (B, T)}, got {resets.dtype} {tuple(resets.shape)}')
        resets = resets.contiguous()
    if state is not None:
        _require(state.dtype == torch.float32 and state.shape == (B, H, K, V), what, f'state: float32 {(B, H, K, V)}, got {state.dtype} {tuple(state.shape)}')
        if not step:
            state = state.contiguous()
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    if step:
        strides = [_I3(t.stride(0), 0, t.stride(1)) for t in (q, k, v)]
    else:
        strides = [_I3(*t.stride()[:3]) for t in (q, k, v)]
    a = _hip.Attention(B, T, H, K, V, _DTYPES[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), *strides, log_decay.data_ptr(), _p(resets),
                       None if step else _p(state), scale)
    return a, (q, k, v, log_decay, resets, state)


def _workspace(what, a, backward, like):
    n = int(_hip.lib().mrl_linear_attention_workspace_bytes(a, backward))
    if n < 0:
        _hip.check(n, what)
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n else None, n


def _linear_attention(q, k, v, log_decay, resets=None, initial_state=None, scale=1.0):
    what = 'linear_attention'
    a, held = _attention(what, q, k, v, log_decay, resets, initial_state, scale, False)
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    final = torch.empty((a.batch, a.heads, a.dim_k, a.dim_v), dtype=torch.float32, device=v.device)
    ws, n = _workspace(what, a, 0, q)
    with _on(q):
        _hip.check(_hip.lib().mrl_linear_attention(a, out.data_ptr(), final.data_ptr(), _p(ws), n, _stream(q)), what)
    return out, final


def _linear_attention_backward(d_out, d_final, q, k, v, log_decay, resets, initial_state, scale, needs):
    what = 'linear_attention_backward'
    a, held = _attention(what, q, k, v, log_decay, resets, initial_state, scale, False)
    d_out = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if d_out is None else _rows(d_out)
    d_final = None if d_final is None else d_final.contiguous()
    need_q, need_k, need_v, need_s = needs
    new = lambda t, need: torch.empty(t.shape, dtype=t.dtype, device=t.device) if need else None  # noqa: E731
    dq, dk, dv = new(q, need_q), new(k, need_k), new(v, need_v or need_s)
    ds = torch.empty((a.batch, a.heads, a.dim_k, a.dim_v), dtype=torch.float32, device=v.device) if need_s else None
    ws, n = _workspace(what, a, 1, q)
    with _on(q):
        _hip.check(_hip.lib().mrl_linear_attention_backward(a, d_out.data_ptr(), _I3(*d_out.stride()[:3]), _p(d_final), _p(dq), _p(dk), _p(dv), _p(ds), _p(ws), n,
                                                            _stream(q)), what)
    return dq, dk, dv if need_v else None, ds


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, resets, initial_state, scale):
        ctx.set_materialize_grads(False)
        out, final = _linear_attention(q, k, v, log_decay, resets, initial_state, scale)
        ctx.save_for_backward(q, k, v, log_decay, resets, initial_state)
        ctx.scale = scale
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_final):
        if d_out is None and d_final is None:
            return (None,) * 7
        n = ctx.needs_input_grad
        dq, dk, dv, ds = _linear_attention_backward(d_out, d_final, *ctx.saved_tensors, ctx.scale, (n[0], n[1], n[2], n[5]))
        return dq, dk, dv, None, None, ds, None


def _linear_attention_autograd(q, k, v, log_decay, resets=None, initial_state=None, scale=1.0):
    if not _wants_grad(q, k, v, log_decay, initial_state):
        return _linear_attention(q, k, v, log_decay, resets, initial_state, scale)
    if log_decay.requires_grad:
        raise NotImplementedError('linear_attention: the decays are constants of the heads; log_decay has no gradient')
    return _LinearAttention.apply(q, k, v, log_decay, resets, initial_state, scale)


def _linear_attention_step(q, k, v, log_decay, state, resets=None, scale=1.0):
    what = 'linear_attention_step'
    if _wants_grad(q, k, v, log_decay, state):
        raise NotImplementedError(f'{what}: no gradient (linear_attention over the rollout has one); call it under torch.no_grad()')
    a, held = _attention(what, q, k, v, log_decay, resets, state, scale, True)
    _require(state.is_contiguous(), what, 'state is updated in place and has to be contiguous')
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    with _on(q):
        _hip.check(_hip.lib().mrl_linear_attention_step(a, state.data_ptr(), out.data_ptr(), _stream(q)), what)
    return out


def _act(what, act_type):
    if act_type not in _hip.ACT_TYPES:
        raise NotImplementedError(f'{what}: act_type={act_type!r} (built: {", ".join(str(n) for n in _hip.ACT_TYPES)})')
    return _hip.ACT_TYPES[act_type]


def _aligned(t):
    """Contiguous, on a 16-byte address."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


# ---- group norm ----------------------------------------------------------------------------------------------------------------
def _group_norm(what, x, num_groups, weight, bias, eps, act_type):
    """Checks of the arguments and their description."""
    _require(x.dtype in _DTYPES, what, f'dtype {x.dtype} (float32, bfloat16 or float16)')
    _require(x.dim() >= 2, what, f'x [batch, ..., channels], got {tuple(x.shape)}')
    C_ = x.shape[-1]
    _require(num_groups >= 1 and C_ >= 1 and C_ % num_groups == 0, what, f'{C_} channels are not {num_groups} groups')
    _require(eps >= 0.0, what, f'eps {eps}')
    _same_device(what, x, weight, bias)
    pdt = x.dtype
    for n, t in (('weight', weight), ('bias', bias)):
        if t is not None:
            _require(t.shape == (C_,) and t.dtype in (x.dtype, torch.float32), what, f'{n}: [{C_}] of {x.dtype} or float32, got {t.dtype} {tuple(t.shape)}')
            pdt = t.dtype
    _require(weight is None or bias is None or weight.dtype == bias.dtype, what, 'weight and bias of one type')
    pixels = 1
    for n in x.shape[1:-1]:
        pixels *= n
    return _hip.GroupNorm(x.shape[0], pixels, C_, num_groups, _DTYPES[x.dtype], _DTYPES[pdt], _act(what, act_type), eps), pdt


def _norm_workspace(what, a, backward, like):
    n = int(_hip.lib().mrl_group_norm_act_workspace_bytes(a, backward))
    if n < 0:
        _hip.check(n, what)
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n else None, n


def _group_norm_forward(x, num_groups, weight, bias, eps, act_type, keep):
    what = 'group_norm_act'
    a, _ = _group_norm(what, x, num_groups, weight, bias, eps, act_type)
    x = _aligned(x)
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, a.batch, num_groups), dtype=torch.float32, device=x.device) if keep else None
    ws, n = _norm_workspace(what, a, 0, x)
    with _on(x):
        _hip.check(_hip.lib().mrl_group_norm_act(a, x.data_ptr(), _p(weight), _p(bias), y.data_ptr(), _p(stats[0]) if keep else None, _p(stats[1]) if keep else None,
                                                 _p(ws), n, _stream(x)), what)
    return y, stats


def _group_norm_backward(dy, x, stats, num_groups, weight, bias, eps, act_type, need_params):
    what = 'group_norm_act_backward'
    a, pdt = _group_norm(what, x, num_groups, weight, bias, eps, act_type)
    x, dy = _aligned(x), _aligned(dy)
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel() == 0:
        return dx, *((torch.zeros(a.channels, dtype=pdt, device=x.device) for _ in range(2)) if need_params else (None, None))
    dw, db = (torch.empty(a.channels, dtype=pdt, device=x.device) if need_params else None for _ in range(2))
    ws, n = _norm_workspace(what, a, 1, x)
    with _on(x):
        _hip.check(_hip.lib().mrl_group_norm_act_backward(a, x.data_ptr(), dy.data_ptr(), _p(weight), _p(bias), stats[0].data_ptr(), stats[1].data_ptr(),
                                                          dx.data_ptr(), _p(dw), _p(db), _p(ws), n, _stream(x)), what)
    return dx, dw, db


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, num_groups, weight, bias, eps, act_type):
        y, stats = _group_norm_forward(x, num_groups, weight, bias, eps, act_type, True)
        ctx.save_for_backward(x, stats, weight, bias)
        ctx.args = (num_groups, eps, act_type)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, stats, weight, bias = ctx.saved_tensors
        num_groups, eps, act_type = ctx.args
        n = ctx.needs_input_grad
        dx, dw, db = _group_norm_backward(dy, x, stats, num_groups, weight, bias, eps, act_type, n[2] or n[3])
        return dx, None, dw if n[2] else None, db if n[3] else None, None, None


def _group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act_type=None):
    return _group_norm_forward(x, num_groups, weight, bias, eps, act_type, False)[0]


def _group_norm_act_autograd(x, num_groups, weight=None, bias=None, eps=1e-5, act_type=None):
    if _wants_grad(x, weight, bias):
        return _GroupNormAct.apply(x, num_groups, weight, bias, eps, act_type)
    return _group_norm_forward(x, num_groups, weight, bias, eps, act_type, False)[0]


# ---- linear layer ----------------------------------------------------------------------------------------------------------------
def _linear(what, x, weight, bias, residual, act_type):
    """Checks of the arguments; their description, and x as rows."""
    _require(x.dtype in _DTYPES, what, f'dtype {x.dtype} (float32, bfloat16 or float16)')
    _require(x.dim() >= 1 and weight.dim() == 2 and weight.shape[1] == x.shape[-1], what, f'x [.., inputs] and weight [outputs, inputs], got {tuple(x.shape)}, {tuple(weight.shape)}')
    K, N = x.shape[-1], weight.shape[0]
    _same_device(what, x, weight, bias, residual)
    for n, t in (('weight', weight), ('bias', bias), ('residual', residual)):
        _require(t is None or t.dtype == x.dtype, what, f'{n}: {x.dtype} like x, got {None if t is None else t.dtype}')
    _require(bias is None or bias.shape == (N,), what, f'bias: [{N}], got {None if bias is None else tuple(bias.shape)}')
    _require(residual is None or residual.shape == (*x.shape[:-1], N), what,
             f'residual: {(*x.shape[:-1], N)}, got {None if residual is None else tuple(residual.shape)}; expand a broadcast one')
    rows = 1
    for n in x.shape[:-1]:
        rows *= n
    x = x.reshape(rows, K)
    if K != 1 and x.stride(1) != 1 or rows > 1 and x.stride(0) < K:
        x = x.contiguous()
    return _hip.Linear(rows, x.stride(0) if rows > 1 else K, K, N, _DTYPES[x.dtype], _act(what, act_type)), x


def _linear_forward(x, weight, bias, residual, act_type, keep):
    what = 'linear_act'
    a, rows = _linear(what, x, weight, bias, residual, act_type)
    weight, bias, residual = (None if t is None else t.contiguous() for t in (weight, bias, residual))
    shape = (*x.shape[:-1], a.outputs)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    z = torch.empty(shape, dtype=x.dtype, device=x.device) if keep and act_type is not None else None
    with _on(x):
        _hip.check(_hip.lib().mrl_linear_act(a, rows.data_ptr(), weight.data_ptr(), _p(bias), _p(residual), y.data_ptr(), _p(z), _stream(x)), what)
    return y, z


def _linear_backward(dy, x, weight, z, act_type, needs):
    what = 'linear_act_backward'
    a, rows = _linear(what, x, weight, None, None, act_type)
    need_x, need_w, need_b = needs
    new = lambda shape, need: torch.empty(shape, dtype=x.dtype, device=x.device) if need else None  # noqa: E731
    dx, dw, db = new(x.shape, need_x), new(weight.shape, need_w), new((a.outputs,), need_b)
    if a.outputs == 0:
        return None if dx is None else dx.zero_(), dw, db
    weight, dy = weight.contiguous(), dy.contiguous()
    n = int(_hip.lib().mrl_linear_act_backward_workspace_bytes(a))
    if n < 0:
        _hip.check(n, what)
    ws = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
    with _on(x):
        _hip.check(_hip.lib().mrl_linear_act_backward(a, rows.data_ptr(), weight.data_ptr(), _p(z), dy.data_ptr(), _p(dx), _p(dw), _p(db), _p(ws), n, _stream(x)), what)
    return dx, dw, db


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act_type):
        y, z = _linear_forward(x, weight, bias, residual, act_type, True)
        ctx.save_for_backward(x, weight, z)
        ctx.act_type = act_type
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        n = ctx.needs_input_grad
        dx = dw = db = None
        if n[0] or n[1] or n[2]:
            dx, dw, db = _linear_backward(dy, x, weight, z, ctx.act_type, n[:3])
        return dx, dw, db, dy if n[3] else None, None


def _linear_act(x, weight, bias=None, residual=None, act_type=None):
    return _linear_forward(x, weight, bias, residual, act_type, False)[0]


def _linear_act_autograd(x, weight, bias=None, residual=None, act_type=None):
    if _wants_grad(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, act_type)
    return _linear_forward(x, weight, bias, residual, act_type, False)[0]


_lib.define('linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? resets=None, Tensor? initial_state=None, float scale=1.0) -> (Tensor, Tensor)')
_lib.define('linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, Tensor? resets=None, float scale=1.0) -> Tensor')
_lib.define('group_norm_act(Tensor x, int num_groups, Tensor? weight=None, Tensor? bias=None, float eps=1e-05, str? act_type=None) -> Tensor')
_lib.define('linear_act(Tensor x, Tensor weight, Tensor? bias=None, Tensor? residual=None, str? act_type=None) -> Tensor')

OPS = ('linear_attention', 'linear_attention_step', 'group_norm_act', 'linear_act')
for _name, _fn, _auto in (('linear_attention', _linear_attention, _linear_attention_autograd), ('linear_attention_step', _linear_attention_step, _linear_attention_step),
                          ('group_norm_act', _group_norm_act, _group_norm_act_autograd), ('linear_act', _linear_act, _linear_act_autograd)):
    _lib.impl(_name, _fn, 'CUDA')
    _lib.impl(_name, _auto, 'AutogradCUDA')

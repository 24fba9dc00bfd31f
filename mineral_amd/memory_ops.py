"""The operators of a sequence memory as PyTorch custom operators: `torch.ops.mineral.*` over include/mineral_memory.h.

    import mineral_amd.ops
    o, state = torch.ops.mineral.linear_attention(q, k, v, log_decay, resets, initial_state, scale)      # a rollout, a prompt
    o = torch.ops.mineral.linear_attention_step(q, k, v, log_decay, state, resets, scale)                # one token, acting

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


_lib.define('linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? resets=None, Tensor? initial_state=None, float scale=1.0) -> (Tensor, Tensor)')
_lib.define('linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, Tensor? resets=None, float scale=1.0) -> Tensor')

OPS = ('linear_attention', 'linear_attention_step')
for _name, _fn, _auto in (('linear_attention', _linear_attention, _linear_attention_autograd), ('linear_attention_step', _linear_attention_step, _linear_attention_step)):
    _lib.impl(_name, _fn, 'CUDA')
    _lib.impl(_name, _auto, 'AutogradCUDA')

"""The operators of a sequence memory as PyTorch custom operators: `torch.ops.mineral.*` over include/mineral_memory.h.

    import mineral_amd.ops
    o, state = torch.ops.mineral.linear_attention(q, k, v, log_decay, resets, initial_state, scale)      # a rollout, a prompt
    o = torch.ops.mineral.linear_attention_step(q, k, v, log_decay, state, resets, scale)                # one token, acting
    y = torch.ops.mineral.group_norm_act(x, num_groups, weight, bias, eps, act_type)                     # channels last
    y = torch.ops.mineral.linear_act(x, weight, bias, residual, act_type)                                # act(x W^T + b) + residual

`act_type` is a name of the towers' configuration (None, 'SiLU', 'ELU', 'ReLU', 'Tanh') or 'GELU'.  Tensors keep their type
(float32, bfloat16 or float16); states are float32 and linear_attention_step updates its state in place.  Calls run on the current
stream of the tensors' device, whichever device is current, and may be captured into a graph.  All but the step are differentiable
once (log_decay has no gradient).  A call that cannot be served raises: ValueError for arguments that do not fit, NotImplementedError
for what is not built, CPU tensors and forward-mode derivatives among it.  Tensors without data (device 'meta', and what tracers and
torch.compile put in a tensor's place) give the shapes and types of the results.

The operators are registered by libmineral_torch.so (csrc/torch_ops.cpp), host code over libmineral_ppo.so; this module loads it.
"""

import os

import torch

from . import _hip

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'libmineral_torch.so')

_hip.lib()
if not os.path.exists(LIB_PATH):
    raise _hip.HipLibraryError(f'{LIB_PATH} not found: build it with `make` at the repository root; there is no fallback')
torch.ops.load_library(LIB_PATH)

OPS = ('linear_attention', 'linear_attention_step', 'group_norm_act', 'linear_act')


# ---- shapes and types of the results, for tensors without data: sizes may be symbolic -------------------------------------------
def _need(ok, what, text):
    if not ok:
        raise ValueError(f'{what}: {text}')


def _known_type(what, t):
    _need(t.dtype in (torch.float32, torch.bfloat16, torch.float16), what, f'dtype {t.dtype} (float32, bfloat16 or float16)')


def _attention_state(what, q, k, v, log_decay, resets, state, dims):
    _known_type(what, q)
    _need(k.dtype == q.dtype and v.dtype == q.dtype, what, 'q, k and v of one type')
    _need(q.dim() == dims and v.dim() == dims and k.shape == q.shape and v.shape[:-1] == q.shape[:-1], what, f'q and k [.., heads, dim_k] and v [.., dim_v], got {q.shape}, {k.shape}, {v.shape}')
    batch, heads, dim_k, dim_v = q.shape[0], q.shape[-2], q.shape[-1], v.shape[-1]
    _need(log_decay.dtype == torch.float32 and log_decay.shape == (heads,), what, f'log_decay: float32 [{heads}]')
    _need(resets is None or (resets.dtype in (torch.bool, torch.uint8) and resets.shape == q.shape[:-2]), what, 'resets: bool or uint8 [batch, steps] (one step: [batch])')
    _need(state is None or (state.dtype == torch.float32 and state.shape == (batch, heads, dim_k, dim_v)), what, 'state: float32 [batch, heads, dim_k, dim_v]')
    return q.new_empty((batch, heads, dim_k, dim_v), dtype=torch.float32)


@torch.library.register_fake('mineral::linear_attention')
def _(q, k, v, log_decay, resets=None, initial_state=None, scale=1.0):
    final = _attention_state('linear_attention', q, k, v, log_decay, resets, initial_state, 4)
    return v.new_empty(v.shape), final


@torch.library.register_fake('mineral::linear_attention_step')
def _(q, k, v, log_decay, state, resets=None, scale=1.0):
    _attention_state('linear_attention_step', q, k, v, log_decay, resets, state, 3)
    return v.new_empty(v.shape)


def _asked(needs, *tensors):
    return [t.new_empty(t.shape) for i, t in enumerate(tensors) if needs >> i & 1]


@torch.library.register_fake('mineral::_linear_attention_backward')
def _(d_out, d_final, q, k, v, log_decay, resets, initial_state, scale, needs):
    return _asked(needs, q, k, v, initial_state)


def _norm(x, num_groups, weight, bias):
    what = 'group_norm_act'
    _known_type(what, x)
    _need(x.dim() >= 2 and num_groups >= 1 and x.shape[-1] % num_groups == 0, what, f'x [batch, ..., channels] in {num_groups} groups, got {x.shape}')
    for t in (weight, bias):
        _need(t is None or (t.shape == x.shape[-1:] and t.dtype in (x.dtype, torch.float32)), what, f'weight and bias: [channels] of {x.dtype} or float32')


@torch.library.register_fake('mineral::group_norm_act')
def _(x, num_groups, weight=None, bias=None, eps=1e-5, act_type=None):
    _norm(x, num_groups, weight, bias)
    return x.new_empty(x.shape)


@torch.library.register_fake('mineral::_group_norm_act_stats')
def _(x, num_groups, weight, bias, eps, act):
    _norm(x, num_groups, weight, bias)
    return x.new_empty(x.shape), x.new_empty((2, x.shape[0], num_groups), dtype=torch.float32)


@torch.library.register_fake('mineral::_group_norm_act_backward')
def _(dy, x, stats, weight, bias, num_groups, eps, act, needs):
    return _asked(needs, x, weight, bias)


def _linear(x, weight, bias, residual):
    what = 'linear_act'
    _known_type(what, x)
    _need(x.dim() >= 1 and weight.dim() == 2 and weight.shape[1] == x.shape[-1], what, f'x [.., inputs] and weight [outputs, inputs], got {x.shape}, {weight.shape}')
    _need(all(t is None or t.dtype == x.dtype for t in (weight, bias, residual)), what, f'weight, bias and residual of {x.dtype} like x')
    _need(bias is None or bias.shape == weight.shape[:1], what, 'bias: [outputs]')
    shape = (*x.shape[:-1], weight.shape[0])
    _need(residual is None or tuple(residual.shape) == shape, what, "residual: the output's shape")
    return x.new_empty(shape)


@torch.library.register_fake('mineral::linear_act')
def _(x, weight, bias=None, residual=None, act_type=None):
    return _linear(x, weight, bias, residual)


@torch.library.register_fake('mineral::_linear_act_slope')
def _(x, weight, bias, residual, act):
    return _linear(x, weight, bias, residual), _linear(x, weight, bias, residual)


@torch.library.register_fake('mineral::_linear_act_backward')
def _(dy, x, weight, slope, act, needs):
    return [t.new_empty(s) for i, (t, s) in enumerate(((x, x.shape), (weight, weight.shape), (x, weight.shape[:1]))) if needs >> i & 1]

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
for what is not built, CPU tensors among it.

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

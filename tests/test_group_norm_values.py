"""torch.ops.mineral.group_norm_act where a small error shows: saturated activations.

u = 2^-24."""

import pytest
import torch

import test_group_norm_act as gn

DEV = 'cuda:0'
DT = gn.DT
U = gn.U
EPS = 1e-5


def ops():
    import mineral_amd.ops  # noqa: F401
    return torch.ops.mineral


@pytest.mark.gpu
@pytest.mark.parametrize('shape,groups', [((4, 64), 2), ((3, 50, 24), 4)])
def test_slopes_in_the_tails_of_tanh(shape, groups):
    """fp32 gradients of units at |z| around 6 to 10, relative to themselves: with weights of zero, z is the bias, and d_bias the
    sum of dy times one slope.  The slope is off by (4|z| + 16) u of itself, a sum over at most 2^8 rows by 2^8 u."""
    x, _, _, dy = gn.make(shape, torch.float32, 32)
    C = shape[-1]
    b = torch.linspace(-10, 10, C)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, torch.zeros(C), b)]
    _, _, db = torch.autograd.grad(ops().group_norm_act(leaves[0], groups, leaves[1], leaves[2], EPS, 'Tanh'), leaves, dy.abs().to(DEV))
    want = dy.double().abs().sum(tuple(range(x.dim() - 1))) / torch.cosh(b.double()) ** 2
    err = (db.double().cpu() - want).abs() / want
    assert bool((err <= (4 * b.double().abs() + 16 + 256) * U).all()), err

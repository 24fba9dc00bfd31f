"""Linear attention held to the recurrence by a comparison that no NaN passes, and its gradients beside masked values by value.

The tests of test_linear_attention.py are run once more with that comparison: theirs asks whether an error lies above its bound,
which an error that is no number does not.  Bounds and inputs are the same."""

import pytest
import torch

import test_linear_attention as at
import test_memory_block as block

DEV = at.DEV
DT = at.DT


def check(got, ref, mag, dtype, T, K, what):
    """at.check, with everything in doubt refused."""
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps if got.dtype != torch.float32 else 1e-37
    err = (got.detach().double().cpu() - ref).abs()
    lim = half * ref.abs() * (1 + 2.0 ** -8) + at.unit(got.dtype, T, K) * mag + tiny
    assert bool(torch.isfinite(ref).all()) and bool(torch.isfinite(lim).all()), f'{what}: the reference is not finite'
    bad = ~(err <= lim)
    assert not bool(bad.any()), f'{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / lim).max()):.2f} of the bound'


@pytest.fixture
def strict(monkeypatch):
    monkeypatch.setattr(at, 'check', check)


def test_the_comparison_refuses_what_is_not_finite():
    ref, mag = torch.zeros(4, dtype=torch.float64), torch.ones(4, dtype=torch.float64)
    check(torch.zeros(4), ref, mag, torch.float32, 1, 1, 'equal')
    for bad in (float('nan'), float('inf'), -float('inf')):
        with pytest.raises(AssertionError, match='outside'):
            check(torch.tensor([0.0, bad, 0.0, 0.0]), ref, mag, torch.float32, 1, 1, 'bad')
        with pytest.raises(AssertionError, match='reference'):
            check(torch.zeros(4), ref + bad, mag, torch.float32, 1, 1, 'bad')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape', at.SHAPES)
@pytest.mark.parametrize('resets,initial', [(0.0, False), (0.1, True)])
def test_forward(strict, dtype, shape, resets, initial):
    at.test_forward_matches_the_recurrence(dtype, shape, resets, initial)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('shape', [(1, 1, 1, 1, 1), (2, 5, 3, 8, 12), (2, 32, 2, 64, 64), (1, 65, 2, 40, 72), (2, 130, 2, 128, 64), (1, 600, 2, 32, 32), (1, 700, 1, 17, 65)])
@pytest.mark.parametrize('resets,initial', [(0.0, False), (0.1, True)])
def test_gradients(strict, dtype, shape, resets, initial):
    at.test_gradients_match_the_recurrence(dtype, shape, resets, initial)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
def test_steps(strict, dtype):
    at.test_steps_equal_the_sequence(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('K,V', [(1, 1), (3, 5), (32, 32), (64, 64), (128, 128), (100, 36), (7, 128), (128, 2), (33, 65)])
@pytest.mark.parametrize('dtype', DT)
def test_step_widths(strict, dtype, K, V):
    at.test_step_widths(dtype, K, V)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T,at_,end', [(50, 10, 20), (60, 0, 20), (200, 70, 70), (200, 64, 127), (900, 300, 640)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_what_a_reset_drops(strict, dtype, T, at_, end, bad):
    at.test_what_a_reset_drops_leaks_nowhere(dtype, T, at_, end, bad)


@pytest.mark.gpu
def test_extreme_decays(strict):
    at.test_extreme_decays()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
def test_the_block(strict, dtype):
    block.test_a_rollout_and_its_gradient(dtype)
    block.test_acting_step_by_step(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', DT)
@pytest.mark.parametrize('T,bad_at,end', [(50, 10, 20), (60, 0, 20), (200, 70, 70), (200, 64, 127), (200, 65, 129), (900, 300, 640)])
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_gradients_beside_what_a_reset_drops(dtype, T, bad_at, end, bad):
    """Token `bad_at` holds `bad`; an episode begins at `end + 1`, and one at the start.  The gradients of the episode that follows are those
    of the clean inputs.  So is, inside the bad episode, every gradient that its formula keeps apart from the bad value: dq sees keys and
    values up to its own token and its own token's output gradient, dk and dv see queries and output gradients from their own token on
    and each other's operand at their own token."""
    B, H, K, V = 2, 2, 32, 48
    q, k, v, l, _, s = at.make(B, T, H, K, V, DT[dtype], 41, 0.0, True)
    resets = torch.zeros(B, T, dtype=torch.bool)
    resets[:, 0] = True
    resets[:, end + 1] = True
    g = torch.Generator().manual_seed(42)
    do, df = torch.randn(B, T, H, V, generator=g).to(DT[dtype]), torch.randn(B, H, K, V, generator=g)

    def grads(q, k, v, do, df):
        leaves = [t.double().requires_grad_(True) for t in (q, k, v)]
        o, f = at.recurrence(*leaves, l.double(), resets, None, 0.5)
        return torch.autograd.grad((o, f), leaves, (do.double(), df.double()))

    ref = grads(q, k, v, do, df)
    mag = grads(q.abs(), k.abs(), v.abs(), do.abs(), df.abs())
    token = torch.arange(T)
    later, before, after = token > end, token < bad_at, (token > bad_at)
    # tokens whose dq, dk, dv do not see token `bad_at`: at all; because they look only back, only ahead; or only at themselves
    every, back, ahead, own = torch.ones(T, dtype=torch.bool), later | before, later | after, token != bad_at
    clean = {'q': (every, ahead, ahead), 'k': (back, every, own), 'v': (back, own, every), 'd_out': (own, ahead, ahead)}
    for which in clean:
        xs = dict(q=q.clone(), k=k.clone(), v=v.clone(), d_out=do.clone())
        xs[which][:, bad_at, :, 0] = bad
        print(f'gradients beside a bad {which} {dtype} T={T} {bad}', flush=True)
        leaves = [xs[n].to(DEV).requires_grad_(True) for n in 'qkv'] + [s.to(DEV).requires_grad_(True)]
        o, f = at.ops().linear_attention(*leaves[:3], *at.dev(l, resets), leaves[3], 0.5)
        got = torch.autograd.grad((o, f), leaves, (xs['d_out'].to(DEV), df.to(DEV)))
        for n, a, r, m, keep in zip(('dq', 'dk', 'dv'), got, ref, mag, clean[which]):
            check(a[:, keep.to(DEV)], r[:, keep], m[:, keep], DT[dtype], T, max(K, V), f'{n} beside a bad {which}')
        assert torch.equal(got[3], torch.zeros_like(got[3]))


@pytest.mark.gpu
def test_more_than_2_to_the_31_outputs():
    """32769 rows of equal queries and keys: the last, whose outputs and gradients lie beyond 2^31, has the bits of a call of its own."""
    B, T, H, K = 2 ** 15 + 1, 64, 32, 32
    q, k, v, l, r, s = at.dev(*at.make(1, T, H, K, K, torch.bfloat16, 43))
    g = torch.Generator(device=DEV).manual_seed(44)
    big = torch.randn(B, T, H, K, generator=g, device=DEV, dtype=torch.bfloat16)
    do = torch.randn(B, T, H, K, generator=g, device=DEV, dtype=torch.bfloat16)
    big[0], big[-1], do[0], do[-1] = v[0], v[0], 1, 1

    def both(q, k, v, r, do):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o, f = at.ops().linear_attention(*leaves, l, r, None, 0.25)
        return (o.detach(), f.detach(), *torch.autograd.grad(o, leaves, do))

    got = both(q.expand(B, T, H, K), k.expand(B, T, H, K), big, r.expand(B, T), do)
    want = both(q, k, v, r, torch.ones_like(v))
    assert got[0].numel() > 2 ** 31
    for a, b in zip(got, want):
        assert torch.equal(a[-1], b[0]) and torch.equal(a[0], b[0])

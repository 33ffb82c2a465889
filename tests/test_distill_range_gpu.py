"""Distillation on logits whose magnitude is far above their differences: rows of one value (the type's lowest or largest), logits with a
common offset, temperatures near the least allowed one.  Against the definition in 64 bits on the same logits.

Tolerances: a logit enters as its difference from the row's largest, rounded once (2^-24 relative to the difference d), times 1 / T (two
roundings), so a probability is within ep = 2^-20 (2 + 2 max|d| / T + log V) + (V / 256 + 16) 2^-23 relative: exp2 and log contribute less than
2^-20 each, a sum over V terms in blocks of 64 to 256 threads the rest.  Row losses: T^2 ep (1 + log V).  The gradient is rounded once to its
type (u = half a step)."""
import math

import pytest
import torch

import lancet_b200 as LB

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FLOOR = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25, torch.float32: 1e-37}


def _check(x, values, idx, temperature, up=64.0):
    rows, vocab = x.shape
    x1 = x.detach().requires_grad_()
    mean = LB.distillation_loss(x1, values, idx, temperature)
    (dx,) = torch.autograd.grad(mean, (x1,), torch.tensor(up, device=DEV))
    got = LB.distill_fwd(x, values, idx, temperature)
    d = x.double() - x.double().max(dim=1, keepdim=True).values
    logp = d / temperature - torch.log(torch.exp(d / temperature).sum(dim=1, keepdim=True))
    q = torch.softmax(values.double() / temperature, dim=1)
    loss = temperature ** 2 * (torch.xlogy(q, q) - q * logp.gather(1, idx)).sum(dim=1)
    dz = torch.exp(logp).scatter_add(1, idx, -q) * (temperature * up / rows)
    spread = float(d.gather(1, idx).abs().max()) / temperature
    spread = max(spread, float(d[d > -1e4 * temperature].abs().max()) / temperature)
    ep = 2.0 ** -20 * (2 + 2 * spread + math.log(vocab)) + (vocab / 256 + 16) * 2.0 ** -23
    tol = temperature ** 2 * ep * (1 + math.log(vocab))
    assert bool(((got[0].double() - loss).abs() <= tol).all()), (got[0], loss)
    assert abs(float(mean.detach()) - float(loss.mean())) <= tol + 2.0 ** -22 * abs(float(loss.mean()))
    hit = torch.zeros_like(dz, dtype=torch.bool).scatter_(1, idx, True)
    err = U[x.dtype] * dz.abs() + torch.where(hit, ep * temperature * up / rows, ep * dz.abs()) + FLOOR[x.dtype]
    off = (dx.double() - dz).abs() - err
    assert bool((off <= 0).all()), "%g above the tolerance" % float(off.max())
    # a row's gradient sums to zero
    assert bool((dx.double().sum(dim=1).abs() <= err.sum(dim=1)).all())
    return got


def _teacher(rows, vocab, g, k=3):
    idx = torch.stack([torch.randperm(vocab, device=DEV, generator=g)[:k] for _ in range(rows)])
    return torch.randn((rows, k), device=DEV, generator=g), idx


@pytest.mark.parametrize("temperature", [0.001, 0.5, 0.7, 1.0, 2.0, 1000.0])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_of_one_value_are_uniform(dt, temperature):
    g = torch.Generator(device=DEV).manual_seed(1)
    fi = torch.finfo(dt)
    for rows, vocab in ((3, 300), (2, 40000)):                    # the second: several blocks per row
        values, idx = _teacher(rows, vocab, g)
        for value in (fi.min, fi.max, -1e4, 0.0):
            _check(torch.full((rows, vocab), value, dtype=dt, device=DEV), values, idx, temperature)


@pytest.mark.parametrize("temperature", [0.5, 1.0])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_neighbours_of_the_extreme_values(dt, temperature):
    """Half of the row a step of the type away from its extreme value: that half has no probability, the other half shares it."""
    g = torch.Generator(device=DEV).manual_seed(2)
    fi = torch.finfo(dt)
    for value, other in ((fi.max, fi.max * (1 - fi.eps)), (fi.min * (1 - fi.eps), fi.min)):
        x = torch.full((4, 300), value, dtype=dt, device=DEV)
        x[:, 1::2] = other
        assert bool((x[:, 0] > x[:, 1]).all())
        values, idx = _teacher(4, 150, g)
        _check(x, values, 2 * idx, temperature)


@pytest.mark.parametrize("offset,temperature", [(1e4, 1.0), (-1e4, 0.7), (1e6, 1.0), (-1e6, 3.0), (12.0, 0.001), (3e37, 0.5)])
def test_common_offset_of_float32_logits(offset, temperature):
    g = torch.Generator(device=DEV).manual_seed(3)
    for rows, vocab in ((5, 1000), (2, 30001)):
        x = torch.randn((rows, vocab), device=DEV, generator=g) * (3 if temperature > 0.01 else 0.003) + offset
        values, idx = _teacher(rows, vocab, g)
        _check(x, values, idx, temperature)


def test_saved_rows_name_the_live_ones():
    """`live_rows` is zero in ignored rows and only there, and the operators' forms give the gradient that the loss gives."""
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn((6, 70), device=DEV, generator=g) * 3 + 1e4
    x[1] = 0.0
    values, idx = _teacher(6, 70, g)
    idx[2] = -1
    loss_rows, lse, mean, inv_live, live, weights = LB.distill_fwd(x, values, idx, 2.0)
    assert live.dtype == torch.int32 and (live != 0).tolist() == [True, True, False, True, True, True]
    x1 = x.detach().requires_grad_()
    (want,) = torch.autograd.grad(LB.distillation_loss(x1, values, idx, 2.0), (x1,))
    assert torch.equal(LB.distill_bwd(x, idx, weights, live, lse, 2.0, inv_live=inv_live), want) and not bool(want[2].any())

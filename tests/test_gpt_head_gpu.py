"""The head's losses inside the GPT-MoE model: with `fused_head` the loss agrees with the one on kept logits up to the rounding of those logits,
the hidden rows get exactly the operator's gradient, and steps with a teacher run."""
import pytest
import torch

import lancet_b200 as LB
from lancet_b200.gpt_moe import GPTMoE, LansTrainer

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B, T, V, M = 2, 64, 500, 256


def _model(**kw):
    return GPTMoE(V, M, 4, 2, T, B, 512, 2, device=DEV, n_chunks=1, act="relu", fabric=LB.LocalFabric(1, 0, {}), **kw)


def _teacher(g, k=8):
    values, indices = torch.topk(torch.randn((B, T, V), device=DEV, generator=g), k, dim=-1)
    indices[:, -1] = -1                                          # the last position has no next token
    return values, indices


def test_fused_head_and_teacher():
    g = torch.Generator(device=DEV).manual_seed(1)
    ids = torch.randint(0, V, (B, T), device=DEV, generator=g)
    teacher = _teacher(g)
    out = {}
    for fused in (False, True):
        model = _model(fused_head=fused, distill_weight=0.25, distill_temperature=2.0)
        hidden = []
        model.ln.register_forward_hook(lambda mod, a, y: (y.retain_grad(), hidden.append(y))[0])
        plain, mixed = model(ids), model(ids, teacher)
        out[fused] = float(plain.detach()), float(mixed.detach())
        mixed.backward()
        rows = hidden[1].detach().reshape(-1, M)
        weight = model.emb.weight.detach().bfloat16()
        z = rows.float() @ weight.float().t()
        if fused:
            # the operators on the same rows, the same bits
            r = rows.requires_grad_()
            target = torch.full_like(ids, -1)
            target[:, :-1] = ids[:, 1:]
            loss = 0.75 * LB.linear_cross_entropy(r, weight, target, V) + 0.25 * LB.linear_distillation_loss(r, weight, *teacher, 2.0, V)
            (want,) = torch.autograd.grad(loss, (r,))
            assert torch.equal(loss.detach(), mixed.detach()) and torch.equal(hidden[1].grad.reshape(-1, M), want)
        assert all(bool(torch.isfinite(p.grad).all()) for p in model.parameters() if p.grad is not None)
        assert bool((model.emb.weight.grad[V:] == 0).all())
        model.close()
    # each logit is rounded once to bfloat16 where it is kept: a shift of at most 2^-8 |z|, in the loss twice (times the temperature squared
    # over itself for the soft part)
    tol = 2 * 2.0 ** -8 * float(z.abs().max()) + 1e-5
    assert abs(out[True][0] - out[False][0]) <= tol and abs(out[True][1] - out[False][1]) <= 0.75 * tol + 0.25 * 2.0 * tol


@pytest.mark.parametrize("fused", [False, True])
def test_trainer_steps_with_a_teacher(fused):
    g = torch.Generator(device=DEV).manual_seed(2)
    ids = torch.randint(0, V, (B, T), device=DEV, generator=g)
    model = _model(fused_head=fused)
    trainer = LansTrainer(model)
    before = model.emb.weight.detach().clone()
    for teacher in (None, _teacher(g)):
        assert bool(torch.isfinite(trainer.step(ids, teacher)))
    assert not torch.equal(before, model.emb.weight.detach())
    model.close()

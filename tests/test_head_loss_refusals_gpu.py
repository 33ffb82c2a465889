"""Calls of the head's losses that are refused: teachers whose values and indices do not belong together, sizes past 32 bits,
and saved tensors other than those of the forward call."""
import pytest
import torch

import lancet_b200 as LB

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_teacher_of_other_shapes():
    """Values and indices with as many entries in all, but other entries per row."""
    h, w = torch.zeros((6, 16), dtype=torch.bfloat16, device=DEV), torch.zeros((30, 16), dtype=torch.bfloat16, device=DEV)
    values, idx = torch.zeros((4, 3), device=DEV), torch.zeros((6, 2), dtype=torch.int64, device=DEV)
    for v, i in ((values, idx), (values.view(2, 6), idx.view(2, 3, 2)), (values.view(2, 2, 3), idx), (torch.zeros(12, device=DEV), idx),
                 (torch.tensor(0.0, device=DEV), torch.tensor(0, device=DEV))):
        with pytest.raises(ValueError):
            LB.linear_distillation_loss(h, w, v, i)
    want = LB.linear_distillation_loss(h, w, values.view(6, 2), idx)
    assert torch.equal(LB.linear_distillation_loss(h.view(2, 3, 16), w, values.view(2, 3, 2), idx), want)     # leading axes as they come


def test_sizes_past_32_bits():
    """More rows, classes or entries than 32 bits count (one element seen many times, so that it takes no memory) are not taken for the few that
    remain of their number in 32 bits."""
    one = torch.zeros((1, 1), dtype=torch.bfloat16, device=DEV)
    t, v, i = torch.zeros(1, dtype=torch.int64, device=DEV), torch.zeros((1, 1), device=DEV), torch.zeros((1, 1), dtype=torch.int64, device=DEV)
    for n in (2 ** 31, 2 ** 32 + 1):
        many = one.expand(n, 1)
        for bad in (lambda: LB.linear_cross_entropy(many, one, t.expand(n)), lambda: LB.linear_cross_entropy(one, many, t),
                    lambda: LB.linear_distillation_loss(many, one, v.expand(n, 1), i.expand(n, 1)),
                    lambda: LB.linear_distillation_loss(one, one, v.expand(1, n), i.expand(1, n)),
                    lambda: LB.distillation_loss(many, v.expand(n, 1), i.expand(n, 1)), lambda: LB.distillation_loss(one.expand(1, n), v, i),
                    lambda: LB.distillation_loss(one, v.expand(1, n), i.expand(1, n))):
            with pytest.raises(ValueError):
                bad()


def test_saved_tensors_of_another_shape_or_type():
    """What the operators' backward forms take back: each tensor in turn replaced by one of another shape, type, stride or place."""
    rows, classes, width, k = 6, 30, 16, 2
    h, w = torch.zeros((rows, width), dtype=torch.bfloat16, device=DEV), torch.zeros((classes, width), dtype=torch.bfloat16, device=DEV)
    t, x = torch.zeros(rows, dtype=torch.int64, device=DEV), torch.zeros((rows, classes), device=DEV)
    v, i = torch.zeros((rows, k), device=DEV), torch.zeros((rows, k), dtype=torch.int64, device=DEV)
    loss, lse, _, _, pos = LB.linear_xent_fwd(h, w, t)
    _, lse2, _, _, pos2, diff = LB.linear_distill_fwd(h, w, v, i)
    _, lse3, _, _, live, weights = LB.distill_fwd(x, v, i)
    for call, saved in ((lambda s: LB.linear_xent_bwd(h, w, t, *s), (loss, lse, pos)),
                        (lambda s: LB.linear_distill_bwd(h, w, i, *s), (diff, lse2, pos2)),
                        (lambda s: LB.distill_bwd(x, i, *s), (weights, live, lse3))):
        call(saved)
        for n, good in enumerate(saved):
            wide = torch.stack((good, good), dim=-1)
            for bad in (wide, wide[..., 0], good[:-1], good[0], good.cpu(), good.double(), good.to(torch.int64)):
                with pytest.raises((ValueError, TypeError)):
                    call(saved[:n] + (bad,) + saved[n + 1:])

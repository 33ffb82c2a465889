"""Calls of the head's losses that are refused: teachers whose values and indices do not belong together."""
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

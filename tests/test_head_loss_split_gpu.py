"""Gradients of the head on both sides of the sizes from which a reduction is cut: the sides meet their definition alike (see test_head_loss_gpu for
the tolerances)."""
import pytest
import torch

import test_head_loss_gpu as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("rows,vocab,width", [(2048, 256, 256), (2240, 256, 256),             # dW of one tile: 32 and 35 blocks of the reduction
                                              (3000, 2000, 512), (4800, 2000, 512),           # dW of 16 tiles
                                              (2264, 3500, 256), (2264, 4400, 256),           # dh of 9 tiles
                                              (300, 2100, 768), (300, 2300, 768)])            # dh of 6 tiles
def test_both_sides_of_the_limits(rows, vocab, width):
    h, w, g = T._operands(rows, vocab, width, torch.bfloat16, rows + vocab)
    target = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    live = torch.ones(rows, dtype=torch.bool, device=DEV)
    T._check_linear(h, w, target[:, None], torch.ones((rows, 1), dtype=torch.float64, device=DEV), live, 1.0, vocab, 1.0,
                    T._run_ce(h, w, target, vocab, 1.0), torch.bfloat16)

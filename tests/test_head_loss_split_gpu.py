"""The head on both sides of the sizes from which a reduction is cut, or blocks finish more rows: both meet the definition (see test_head_loss_gpu for
the tolerances)."""
import pytest
import torch

import lancet_b200 as LB
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


@pytest.mark.parametrize("rows,k", [(832, 16), (833, 16), (1100, 64), (1793, 64), (700, 200)])     # the last rows of one plan, the first of another
def test_rows_per_block_of_the_teachers(rows, k):
    vocab, width, dt, temperature = 900, 72, torch.bfloat16, 2.0
    h, w, g = T._operands(rows, vocab, width, dt, rows + k)
    values, idx = T._teacher_case(rows, vocab, k, torch.float32, g)
    q, at, live = T._teacher(values, idx, vocab, temperature)
    h1, w1 = h.detach().requires_grad_(), w.detach().requires_grad_()
    mean = LB.linear_distillation_loss(h1, w1, values, idx, temperature)
    dh, dw = torch.autograd.grad(mean, (h1, w1))
    T._check_linear(h, w, at, q, live, temperature, vocab, 1.0, (LB.linear_distill_fwd(h, w, values, idx, temperature)[0], mean.detach(), dh, dw), dt)

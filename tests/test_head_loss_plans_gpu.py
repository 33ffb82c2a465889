"""Plans of the head's losses that only certain sizes take: distillation over a vocabulary in several pieces, clusters of blocks per row with
16-bit logits, gradient rows aligned otherwise than the logits' with several blocks per row; and row losses where one class holds most of the
probability.  Definitions and tolerances are those of test_head_loss_gpu."""
import pytest
import torch

import lancet_b200 as LB
import test_head_loss_gpu as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dt,k,temperature", [(torch.bfloat16, 9, 2.0), (torch.float16, 33, 0.7)])
def test_linear_distillation_in_several_pieces(dt, k, temperature):
    """16384 rows x 40001 classes are two pieces of the backward pass; a tenth of the rows has a teacher, with entries in both pieces."""
    rows, vocab, width = 16384, 40001, 72
    h, w, g = T._operands(rows, vocab + 30, width, dt, 91)
    values, idx = T._teacher_case(rows, vocab, k, torch.float32, g)
    idx[:, 0] = vocab - 1 - torch.arange(rows, device=DEV) % 100             # the last classes
    idx[torch.rand(rows, device=DEV, generator=g) < 0.9] = -1
    q, at, live = T._teacher(values, idx, vocab, temperature)
    h[~live] = float("nan")
    w[vocab:] = float("nan")
    h1, w1 = h.detach().requires_grad_(), w.detach().requires_grad_()
    mean = LB.linear_distillation_loss(h1, w1, values, idx, temperature, vocab)
    dh, dw = torch.autograd.grad(mean, (h1, w1), torch.tensor(0.75, device=DEV))
    loss_rows = LB.linear_distill_fwd(h, w, values, idx, temperature, vocab)[0]
    h = torch.where(live[:, None], h, torch.zeros_like(h))
    w = torch.cat([w[:vocab], torch.zeros_like(w[vocab:])])
    T._check_linear(h, w, at, q, live, temperature, vocab, 0.75, (loss_rows, mean.detach(), dh, dw), dt)


@pytest.mark.parametrize("rows,vocab,cols", [(2, 50257, 50304), (40, 33001, 33001), (200, 20000, 20008)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_distillation_with_several_blocks_per_row(dt, rows, vocab, cols):
    g = T._gen(rows + vocab)
    values, idx = T._teacher_case(rows, vocab, 11, torch.float32, g)
    idx[:, 0] = vocab - 1
    x = (torch.randn((rows, cols), device=DEV, generator=g) * 3).to(dt)
    T._check_distill(x, values, idx, vocab, 1.5, dt)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_distillation_of_rows_aligned_otherwise_than_their_gradient(dt):
    """The first columns of a padded matrix: the gradient's rows follow each other without padding, so they start on other boundaries."""
    for rows, vocab, ld in ((9, 50257, 50304), (300, 20001, 20008), (700, 1001, 1024)):
        g = T._gen(rows + ld)
        values, idx = T._teacher_case(rows, vocab, 7, torch.float32, g)
        x = (torch.randn((rows, ld), device=DEV, generator=g) * 3).to(dt)[:, :vocab]
        T._check_distill(x, values, idx, vocab, 2.0, dt)


@pytest.mark.parametrize("dt,width", [(torch.bfloat16, 1024), (torch.float16, 1024), (torch.bfloat16, 2048)])
def test_losses_where_one_class_holds_the_probability(dt, width):
    """Rows that lean on their class's weight row up to a logit of about 12: the loss is the small difference of two large numbers.  The
    logit is a float32 dot product: a lane adds width / 32 products in order (partial sums of half its share on average), five more adds join
    the lanes, and log-sum-exp and the difference round four times: |error| <= B = (width / 64 + 9) 2^-24 z.  Those roundings go up as often as
    down, so the mean of the error over n independent rows stays within 5 B / sqrt(n) but for one time in 10^5 (Hoeffding); sums of products that are
    cut short instead move all rows the same way."""
    rows, vocab = 1024, 2000
    g = T._gen(width)
    w = (torch.randn((vocab, width), device=DEV, generator=g) * 0.02).to(dt)
    target = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    wt = w[target].float()
    # all products of a row with its class positive: sum |h| |w| is the logit itself
    h = (12.0 + torch.rand((rows, 1), device=DEV, generator=g)) / (wt * wt).sum(dim=1, keepdim=True) * wt
    h = h.to(dt)
    z = h.double() @ w.double().t()
    zt = z.gather(1, target[:, None])
    want = (torch.logsumexp(z - zt, dim=1))
    bound = (width / 64 + 9) * 2.0 ** -24 * float(zt.max())
    assert float(want.max()) < 0.2 and float(zt.min()) > 11.5
    values = torch.tensor([[9.0, -9.0]], device=DEV).expand(rows, 2).contiguous()
    idx = torch.stack([target, (target + 1) % vocab], dim=1)
    q = torch.softmax(values.double(), dim=1)
    logp = (z - zt).gather(1, idx) - want[:, None]
    soft = (q * (torch.log(q) - logp)).sum(dim=1)
    for got, ref in ((LB.linear_xent_fwd(h, w, target)[0], want), (LB.linear_distill_fwd(h, w, values, idx)[0], soft)):
        err = got.double() - ref
        assert float(err.abs().max()) <= bound
        assert abs(float(err.mean())) <= 5 * bound / rows ** 0.5, (float(err.mean()), bound)

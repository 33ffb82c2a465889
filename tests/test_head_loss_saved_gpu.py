"""What the head's losses save for their backward passes, taken through saved-tensor hooks: floating-point tensors stored in fewer bits, and
tensors moved to the host and back (other strides)."""
import pytest
import torch

import lancet_b200 as LB

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _inputs(classes=300, width=100, rows=70):
    g = torch.Generator(device=DEV).manual_seed(5)
    h = torch.randn((rows, width + 9), device=DEV, generator=g).bfloat16()[:, 3:3 + width]
    # rows on 16-byte boundaries of a wider matrix, the width itself no multiple of 8
    w = (torch.randn((classes, width + 4), device=DEV, generator=g) * 0.1).bfloat16()[:, :width]
    assert w.stride(0) % 8 == 0 and width % 8 != 0
    target = torch.randint(0, classes, (rows,), device=DEV, generator=g)
    target[::7] = -1
    values, idx = torch.randn((rows, 5), device=DEV, generator=g), torch.randint(0, classes, (rows, 5), device=DEV, generator=g)
    idx[::6] = -1
    return h.requires_grad_(), w.requires_grad_(), target, values, idx


def _losses(h, w, target, values, idx):
    x = (h.detach().float() @ w.detach().float().t()).requires_grad_()
    return ((LB.linear_cross_entropy(h, w, target), (h, w)), (LB.linear_distillation_loss(h, w, values, idx, 2.0), (h, w)),
            (LB.distillation_loss(x, values, idx, 2.0), (x,)))


def test_saved_floats_in_fewer_bits():
    """The row numbers are whole numbers and stay so: gradients move by the rounding of the saved sums only, ignored rows stay zero.
    float32 -> bfloat16 moves lse by 2^-8 |lse|, so a probability by a factor of exp(2^-8 |lse|) at most."""
    args = _inputs()
    want = [torch.autograd.grad(loss, leaves) for loss, leaves in _losses(*args)]
    pack = lambda t: t.bfloat16() if t.dtype == torch.float32 and t.dim() < 2 else t
    unpack = lambda t: t.float() if t.dtype == torch.bfloat16 and t.dim() < 2 else t
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        losses = _losses(*args)
    for (loss, leaves), ref in zip(losses, want):
        got = torch.autograd.grad(loss, leaves)
        assert bool((got[0][(ref[0] == 0).all(dim=1)] == 0).all())
        for a, b in zip(got, ref):
            assert bool(torch.isfinite(a).all())
            # |lse| is at most log 300 + 8 here; every gradient is a sum of probability differences times operands
            assert float((a.double() - b.double()).norm()) <= (2.0 ** -7 * 14 + 2.0 ** -7) * float(b.double().norm())


def test_saved_tensors_moved_to_the_host():
    """What comes back has the same values and no gaps between its rows."""
    args = _inputs()
    want = [torch.autograd.grad(loss, leaves) for loss, leaves in _losses(*args)]
    with torch.autograd.graph.save_on_cpu():
        losses = _losses(*args)
    for (loss, leaves), ref in zip(losses, want):
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, leaves), ref))

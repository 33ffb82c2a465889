"""Losses of the language-model head (linear cross entropy, distillation on logits and from hidden rows) against their definitions in 64
bits on the same 16-bit (or float32) inputs.

Tolerances, from the number formats alone.  u is half a step of the output type relative to the value (bfloat16 2^-8, float16 2^-11,
float32 2^-24).  A logit is a float32 sum of `width` products: |error| <= ez = width 2^-23 max sum|h||w|.  exp and log contribute at most
2^-20 relative.  So the row losses are within 2 ez / T T^2 + 2^-20 (1 + |lse|) T^2 of the definition, and probabilities within the relative
ep = 2 ez / T + 2^-20 (1 + max|z| / T).  The gradient of the logits is rounded once to the operands' type before the products (u + ep
relative, in float16 never below 2^-39 absolutely), a product of n terms in float32 adds n 2^-23 relative to the sum of magnitudes, the result is rounded once more
(u; float16 results are not finer than 2^-25)."""
import pytest
import torch

import lancet_b200 as LB

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FLOOR = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25, torch.float32: 1e-37}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _operands(rows, classes, width, dt, seed, std=0.1):
    g = _gen(seed)
    h = torch.randn((rows, width), device=DEV, generator=g).to(dt)
    w = (torch.randn((classes, width), device=DEV, generator=g) * std).to(dt)
    return h, w, g


def _soft(z, idx, q, temperature):
    """(loss rows, lse, dz of a row's own loss) of one block of live rows in 64 bits; q [rows, k] over idx [rows, k]."""
    lse = torch.logsumexp(z / temperature, dim=1)
    logp = z.gather(1, idx) / temperature - lse[:, None]
    loss = temperature ** 2 * (torch.xlogy(q, q) - q * logp).sum(dim=1)
    dz = torch.exp(z / temperature - lse[:, None]).scatter_add(1, idx, -q) * temperature
    return loss, lse, dz


def _teacher(values, idx, vocab, temperature):
    """(q, indices to read at, live rows) from the definition: entries that name no class do not count."""
    counts = (idx >= 0) & (idx < vocab)
    v = torch.where(counts, values.double() / temperature, -torch.inf)
    live = torch.isfinite(v.max(dim=1).values)
    q = torch.where(live[:, None], torch.softmax(torch.where(live[:, None], v, 0.0), dim=1), 0.0)
    return torch.where(counts, q, 0.0), torch.where(counts, idx, 0), live


def _check_linear(h, w, idx, q, live, temperature, vocab, up, got, dt):
    """got = (loss rows, mean, dh, dw)."""
    loss_rows, mean, dh, dw = got
    r = live.nonzero().flatten()
    n = max(1, r.numel())
    hd, wd = h.double(), w[:vocab].double()
    want_rows = torch.zeros(h.shape[0], dtype=torch.float64, device=DEV)
    want_dh = torch.zeros(h.shape, dtype=torch.float64, device=DEV)
    want_dw = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    tol_dh, tol_dw, tol_rows = torch.zeros_like(want_dh), torch.zeros_like(want_dw), 0.0
    if r.numel():
        hl = hd[r]
        z = hl @ wd.t()
        loss, lse, dz = _soft(z, idx[r], q[r], temperature)
        want_rows[r] = loss
        g = dz * (up / n)
        want_dh[r] = g @ wd
        want_dw[:vocab] = g.t() @ hl
        ez = h.shape[1] * 2.0 ** -23 * float((hl.abs() @ wd.abs().t()).max())
        tol_rows = temperature ** 2 * (2 * ez / temperature + 2.0 ** -20 * (1 + float(lse.abs().max())))
        ep = 2 * ez / temperature + 2.0 ** -20 * (1 + float(z.abs().max()) / temperature)
        # where dz is a difference at a teacher's class, its error is that of the probability
        err = U[dt] * g.abs() + ep * temperature * up / n + 2.0 ** -39
        err = torch.where(torch.zeros_like(z, dtype=torch.bool).scatter_(1, idx[r], True), err,
                          (U[dt] + ep) * g.abs() + 2.0 ** -39)
        tol_dh[r] = err @ wd.abs() + vocab * 2.0 ** -23 * (g.abs() @ wd.abs())
        tol_dw[:vocab] = err.t() @ hl.abs() + n * 2.0 ** -23 * (g.abs().t() @ hl.abs())
    assert bool(((loss_rows.double() - want_rows).abs() <= tol_rows).all())
    assert bool((loss_rows[~live] == 0).all())
    assert abs(float(mean) - float(want_rows.sum() / n)) <= tol_rows + 2.0 ** -22 * abs(float(want_rows.sum() / n))
    for name, a, b, tol in (("dhidden", dh, want_dh, tol_dh), ("dweight", dw, want_dw, tol_dw)):
        assert a.dtype == dt and a.shape == b.shape
        tol = tol + U[dt] * b.abs() + FLOOR[dt]
        off = (a.double() - b).abs() - tol
        assert bool((off <= 0).all()), "%s: %g above its tolerance (%g)" % (name, float(off.max()), float(tol.flatten()[off.argmax()]))
    assert bool((dh[~live] == 0).all()) and bool((dw[vocab:] == 0).all())


def _run_ce(h, w, target, vocab, up):
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    mean = LB.linear_cross_entropy(h, w, target, vocab)
    dh, dw = torch.autograd.grad(mean, (h, w), torch.tensor(up, device=DEV))
    loss_rows, lse, mean2 = LB.linear_xent_fwd(h.detach(), w.detach(), target, vocab)[:3]
    assert float(mean2) == float(mean.detach())
    return loss_rows, mean.detach(), dh, dw


@pytest.mark.parametrize("rows,vocab,pad,width,dt,ignored", [
    (1, 1, 1, 8, torch.bfloat16, 0.0), (1, 2, 5, 1, torch.float16, 0.0), (3, 50, 64, 100, torch.bfloat16, 0.0),
    (33, 1009, 1009, 128, torch.float16, 0.2), (127, 257, 300, 72, torch.bfloat16, 0.5), (128, 256, 256, 64, torch.float16, 0.0),
    (129, 255, 256, 65, torch.bfloat16, 0.1), (257, 2000, 2048, 200, torch.bfloat16, 0.9), (300, 777, 777, 513, torch.float16, 0.3),
    (1024, 4099, 4224, 512, torch.bfloat16, 0.02), (2500, 1000, 1000, 96, torch.bfloat16, 0.5), (40, 1009, 1024, 64, torch.bfloat16, 1.0),
    (513, 3, 3, 1027, torch.bfloat16, 0.0), (200, 700, 700, 240, torch.float16, 0.1), (700, 300, 333, 392, torch.bfloat16, 0.1),
    (2200, 520, 520, 371, torch.float16, 0.1), (64, 6000, 6000, 1040, torch.bfloat16, 0.0), (90, 3000, 3000, 257, torch.float16, 0.0),
    (20, 300, 300, 65, torch.float16, 1.0), (1, 1, 1, 13, torch.bfloat16, 0.0),
])
def test_linear_cross_entropy(rows, vocab, pad, width, dt, ignored):
    h, w, g = _operands(rows, pad, width, dt, rows + vocab)
    target = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    dead = torch.rand(rows, device=DEV, generator=g) < ignored
    target[dead] = -100
    if rows > 2 and not bool(dead.all()):
        target[1], dead[1] = vocab, True                      # names no class
    h[dead] = float("nan")                                    # what an ignored row holds does not matter
    w[vocab:] = float("nan")                                  # nor do rows behind the vocabulary
    got = _run_ce(h, w, target, vocab, 0.75)
    h = torch.where(dead[:, None], torch.zeros_like(h), h)
    w = torch.cat([w[:vocab], torch.zeros_like(w[vocab:])])
    _check_linear(h, w, target.clamp(0, vocab - 1)[:, None], torch.ones((rows, 1), dtype=torch.float64, device=DEV), ~dead, 1.0, vocab, 0.75, got, dt)


def test_linear_cross_entropy_in_several_pieces():
    """More rows x classes than one piece of the backward pass holds, at a narrow width."""
    rows, vocab, width, dt = 16384, 40001, 64, torch.bfloat16
    h, w, g = _operands(rows, vocab, width, dt, 5)
    target = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    target[::100] = -1
    got = _run_ce(h, w, target, vocab, 1.0)
    live = target >= 0
    # the definition a block of rows at a time; tolerances as in _check_linear, with sums over all live rows
    n, wd = int(live.sum()), w.double()
    want_dw, tol_dw = (torch.zeros(w.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    for r0 in range(0, rows, 2048):
        r = torch.arange(r0, r0 + 2048, device=DEV)
        r = r[live[r]]
        hl = h[r].double()
        z = hl @ wd.t()
        _, lse, dz = _soft(z, target[r][:, None], torch.ones((r.numel(), 1), dtype=torch.float64, device=DEV), 1.0)
        ez = width * 2.0 ** -23 * float((hl.abs() @ wd.abs().t()).max())
        assert bool(((got[0][r].double() - (lse - z.gather(1, target[r][:, None])[:, 0])).abs() <= 2 * ez + 2.0 ** -20 * (1 + lse)).all())
        gz = dz / n
        ep = 2 * ez + 2.0 ** -20 * (1 + float(z.abs().max()))
        err = (U[dt] + ep) * gz.abs()
        err.scatter_(1, target[r][:, None], (U[dt] * gz.abs() + ep / n).gather(1, target[r][:, None]))
        want = gz @ wd
        tol = err @ wd.abs() + vocab * 2.0 ** -23 * (gz.abs() @ wd.abs()) + U[dt] * want.abs() + 1e-37
        assert bool(((got[2][r].double() - want).abs() <= tol).all())
        want_dw += gz.t() @ hl
        tol_dw += err.t() @ hl.abs() + n * 2.0 ** -23 * (gz.abs().t() @ hl.abs())
    assert bool(((got[3].double() - want_dw).abs() <= tol_dw + U[dt] * want_dw.abs() + 1e-37).all())
    assert bool((got[2][~live] == 0).all())


@pytest.mark.parametrize("rows,vocab,pad,width,k,temperature,dt,vdt", [
    (1, 1, 1, 8, 1, 1.0, torch.bfloat16, torch.float32), (5, 60, 64, 100, 7, 2.0, torch.float16, torch.float16),
    (130, 1009, 1024, 128, 33, 0.7, torch.bfloat16, torch.bfloat16), (300, 2000, 2000, 260, 64, 3.0, torch.bfloat16, torch.float32),
    (2100, 300, 384, 64, 16, 1.5, torch.float16, torch.float32), (20, 600, 640, 64, 512, 1.0, torch.bfloat16, torch.float32),
])
def test_linear_distillation(rows, vocab, pad, width, k, temperature, dt, vdt):
    h, w, g = _operands(rows, pad, width, dt, rows * 7 + vocab)
    values, idx = _teacher_case(rows, vocab, k, vdt, g)
    q, at, live = _teacher(values, idx, vocab, temperature)
    h[~live] = float("inf")
    w[vocab:] = float("nan")
    h1, w1 = h.detach().requires_grad_(), w.detach().requires_grad_()
    mean = LB.linear_distillation_loss(h1, w1, values, idx, temperature, vocab)
    dh, dw = torch.autograd.grad(mean, (h1, w1), torch.tensor(0.75, device=DEV))
    loss_rows = LB.linear_distill_fwd(h, w, values, idx, temperature, vocab)[0]
    h = torch.where(live[:, None], h, torch.zeros_like(h))
    w = torch.cat([w[:vocab], torch.zeros_like(w[vocab:])])
    _check_linear(h, w, at, q, live, temperature, vocab, 0.75, (loss_rows, mean.detach(), dh, dw), dt)


def _teacher_case(rows, vocab, k, vdt, g):
    """Teacher rows with what can go wrong: padding entries with NaN values, an index behind the vocabulary, a class named twice,
    values of -inf and of the type's lowest, a row without entries and one whose values are all -inf."""
    values = (torch.randn((rows, k), device=DEV, generator=g) * 2).to(vdt)
    idx = torch.randint(0, vocab, (rows, k), device=DEV, generator=g)
    if k > 4:
        values[:, -1], idx[:, -1] = float("nan"), -1
        idx[::3, 1] = idx[::3, 0]
        values[::4, 2] = float("-inf")
        values[::5, 3] = torch.finfo(vdt).min
    if rows > 4:
        idx[2] = -1
        values[3] = float("-inf")
        idx[4, 0] = vocab
    return values, idx


@pytest.mark.parametrize("rows,vocab,cols,k,temperature,dt,vdt", [
    (1, 1, 1, 1, 1.0, torch.float32, torch.float32), (1, 9000, 9000, 3, 2.0, torch.bfloat16, torch.float32),
    (7, 50257, 50257, 8, 1.0, torch.float32, torch.float32), (9, 1001, 1024, 32, 0.5, torch.float16, torch.float16),
    (33, 777, 777, 7, 1.5, torch.bfloat16, torch.bfloat16), (600, 513, 520, 6, 4.0, torch.bfloat16, torch.float32),
    (12, 1003, 1003, 512, 1.0, torch.float16, torch.float32), (5, 7, 16, 5, 2.0, torch.float32, torch.bfloat16),
])
def test_distillation_on_logits(rows, vocab, cols, k, temperature, dt, vdt):
    g = _gen(rows + vocab + k)
    values, idx = _teacher_case(rows, vocab, k, vdt, g)
    x = (torch.randn((rows, cols), device=DEV, generator=g) * 3).to(dt)
    if vocab > 20:
        x[0, 5] = float("-inf")                                # a masked class
        x[0, 6] = torch.finfo(dt).min
        masked = (idx[0] == 5) | (idx[0] == 6)
        idx[0, masked] = 7                                     # that the teacher does not name: its loss would be infinite
    _check_distill(x, values, idx, vocab, temperature, dt)


def _check_distill(x, values, idx, vocab, temperature, dt, up=64.0):
    rows = x.shape[0]
    q, at, live = _teacher(values, idx, vocab, temperature)
    x[~live] = float("nan")
    x[:, vocab:] = float("nan")
    x1 = x.detach().requires_grad_()
    mean = LB.distillation_loss(x1, values, idx, temperature, vocab)
    (dx,) = torch.autograd.grad(mean, (x1,), torch.tensor(up, device=DEV))
    loss_rows = LB.distill_fwd(x, values, idx, temperature, vocab)[0]
    n = max(1, int(live.sum()))
    z = torch.where(live[:, None], x[:, :vocab].double(), 0.0)
    loss, lse, dz = _soft(z, at, q, temperature)
    loss, dz = torch.where(live, loss, 0.0), torch.where(live[:, None], dz, 0.0) * (up / n)
    big = float(z[z > -1e4].abs().max()) / temperature if bool((z > -1e4).any()) else 0.0
    # a difference (x - m) / T of magnitude d carries 2^-23 d; sums of up to `vocab` terms in blocks of 256 threads add vocab / 256 2^-23
    ep = 2.0 ** -20 * (2 + 2 * big) + (vocab / 256 + 16) * 2.0 ** -23
    tol = temperature ** 2 * (ep + 2.0 ** -20 * (1 + float(lse.abs().max())))
    assert bool(((loss_rows.double() - loss).abs() <= tol).all())
    assert abs(float(mean.detach()) - float(loss.sum() / n)) <= tol + 2.0 ** -22 * abs(float(loss.sum() / n))
    got = dx.double()
    assert dx.dtype == dt and bool((got[:, vocab:] == 0).all()) and bool((got[~live] == 0).all())
    hit = torch.zeros_like(z, dtype=torch.bool).scatter_(1, at, q > 0) | torch.zeros_like(z, dtype=torch.bool).scatter_(1, at, True)
    err = U[dt] * dz.abs() + torch.where(hit, ep * temperature * up / n, ep * dz.abs()) + FLOOR[dt]
    off = (got[:, :vocab] - dz).abs() - err
    assert bool((off <= 0).all()), "%g above the tolerance" % float(off.max())


def test_distillation_strided_and_unaligned_logits():
    """Rows of a wider matrix that start off 16-byte boundaries, the rows around them untouched."""
    g = _gen(3)
    for dt, lead, ld in ((torch.bfloat16, 3, 1031), (torch.float32, 1, 1030), (torch.float16, 8, 1040)):
        base = (torch.randn((40, ld), device=DEV, generator=g) * 3).to(dt)
        values, idx = _teacher_case(20, 1000, 9, torch.float32, g)
        x = base[::2, lead:lead + 1010]
        _check_distill(x.clone(), values, idx, 1000, 1.5, dt)
        want = LB.distill_fwd(x.clone(), values, idx, 1.5, 1000)[:2]
        got = LB.distill_fwd(x, values, idx, 1.5, 1000)[:2]
        for a, b in zip(got, want):
            assert bool(((a - b).abs() <= 2.0 ** -18 * (1 + b.abs())).all())
        xt = x.t().contiguous().t()                            # columns not adjacent
        assert torch.equal(LB.distill_fwd(xt, values, idx, 1.5, 1000)[1], want[1])


def test_all_masked_by_the_lowest_value():
    """A row of nothing but the type's lowest value is uniform, as in the definition (differences before the scale)."""
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.full((2, 300), torch.finfo(dt).min, dtype=dt, device=DEV).requires_grad_()
        values = torch.zeros((2, 1), device=DEV)
        idx = torch.tensor([[3], [299]], device=DEV)
        (dx,) = torch.autograd.grad(LB.distillation_loss(x, values, idx, 1.0), (x,))
        # float32 log-sum-exp of such a row rounds to the maximum itself: every probability comes out as 1 (as in float32 arithmetic
        # of the definition), float16's lowest is small enough for the logarithm to count
        want = 0.5 / 300 if dt == torch.float16 else 0.5
        other = dx[0, 4].item()
        assert abs(other - want) <= want * 2.0 ** -7


def test_strides_of_hidden_and_weight():
    rows, vocab, width, dt = 70, 300, 96, torch.bfloat16
    g = _gen(11)
    base = torch.randn((2 * rows, width + 11), device=DEV, generator=g).to(dt)
    wbase = (torch.randn((vocab, width + 5), device=DEV, generator=g) * 0.1).to(dt)
    target = torch.randint(0, vocab, (2 * rows,), device=DEV, generator=g)[::2]
    plain = None
    for h, w in ((base[::2, 3:3 + width], wbase[:, 1:1 + width]),                       # rows off 16-byte boundaries
                 (base[::2, 3:3 + width].contiguous(), wbase[:, 1:1 + width].contiguous()),
                 (base[::2, 3:3 + width].t().contiguous().t(), wbase[:, 1:1 + width].t().contiguous().t())):
        got = _run_ce(h, w, target, vocab, 1.0)
        if plain is None:
            plain = got
        assert all(torch.equal(a, b) for a, b in zip(got, plain))
    one = base[:1, :width].expand(rows, width)                                            # one row, broadcast
    h1 = base[:1, :width].detach().requires_grad_()
    w1 = wbase[:, :width].detach()
    (d1,) = torch.autograd.grad(LB.linear_cross_entropy(h1.expand(rows, width), w1, target, vocab), (h1,))
    d = _run_ce(one, w1, target, vocab, 1.0)[2]
    assert torch.equal(d1, d.sum(dim=0, keepdim=True))


def test_leading_axes_autocast_and_frozen_operands():
    B, T, vocab, width = 3, 17, 130, 64
    g = _gen(21)
    h = torch.randn((B, T, width), device=DEV, generator=g).requires_grad_()
    w = (torch.randn((256, width), device=DEV, generator=g) * 0.1).requires_grad_()
    target = torch.randint(0, vocab, (B, T), device=DEV, generator=g)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = LB.linear_cross_entropy(h, w, target, vocab)
    dh, dw = torch.autograd.grad(loss, (h, w))
    assert dh.shape == h.shape and dh.dtype == torch.float32 and dw.dtype == torch.float32
    hb, wb = h.detach().bfloat16().reshape(-1, width), w.detach().bfloat16()
    got = _run_ce(hb, wb, target.reshape(-1), vocab, 1.0)
    assert torch.equal(got[1], loss.detach()) and torch.equal(got[2].float().reshape(h.shape), dh) and torch.equal(got[3].float(), dw)
    h1, w1 = hb.clone().requires_grad_(), wb.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(LB.linear_cross_entropy(h1, wb, target, vocab), (h1,))[0], got[2])
    assert torch.equal(torch.autograd.grad(LB.linear_cross_entropy(hb, w1, target, vocab), (w1,))[0], got[3])
    with torch.no_grad():
        assert not LB.linear_cross_entropy(hb, wb, target, vocab).requires_grad
    loss = LB.linear_cross_entropy(h1, w1, target, vocab)       # the same graph twice, the loss changed in between
    first = torch.autograd.grad(loss, (h1, w1), retain_graph=True)
    loss.detach().mul_(2)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, (h1, w1)), first))


def test_capped_grids_and_plain_launches():
    """The process-wide knobs of the grouped GEMM hold for the head's products too: fewer workers cut the reductions differently, plain
    launches give the same bits."""
    L = LB._capi.lib()
    for rows, vocab, width in ((300, 3000, 300), (40, 5000, 192)):
        h, w, g = _operands(rows, vocab, width, torch.bfloat16, rows)
        target = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
        live = torch.ones(rows, dtype=torch.bool, device=DEV)
        want = _run_ce(h, w, target, vocab, 1.0)
        try:
            assert L.lancet_set_chained_launch(0) == 0
            assert all(torch.equal(a, b) for a, b in zip(_run_ce(h, w, target, vocab, 1.0), want))
            for ctas in (1, 3, 10, 147):
                assert L.lancet_set_cta_limits(0, ctas) == 0
                _check_linear(h, w, target[:, None], torch.ones((rows, 1), dtype=torch.float64, device=DEV), live, 1.0, vocab, 1.0,
                              _run_ce(h, w, target, vocab, 1.0), torch.bfloat16)
        finally:
            L.lancet_set_chained_launch(1)
            L.lancet_set_cta_limits(0, 0)


def test_matrices_of_one_row():
    """One class or one row taken out of a wider matrix: the stride of an axis of length 1 means nothing."""
    g = _gen(71)
    base = torch.randn((9, 29), device=DEV, generator=g).bfloat16()
    target = torch.zeros(4, dtype=torch.int64, device=DEV)
    for h, w, t in ((base[:4, :8], base[8:9, :8], target), (base[8:9, :8], base[:4, :8], target[:1])):
        got = _run_ce(h, w, t, None, 1.0)
        want = _run_ce(h.clone(memory_format=torch.contiguous_format).reshape(h.shape), w.contiguous().clone().reshape(w.shape), t, None, 1.0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x, v, i = base[8:9, 3:20], torch.randn((1, 2), device=DEV, generator=g), torch.tensor([[1, 4]], device=DEV)
    assert torch.equal(LB.distill_fwd(x, v, i)[1], LB.distill_fwd(x.contiguous().clone(), v, i)[1])
    _check_distill(x.clone(), v, i, 17, 1.0, torch.bfloat16)


def test_offsets_past_32_bits():
    """More than 2^31 elements of weight, gradient and logits: the last rows against the definition."""
    rows, classes, width, dt = 2, 140000, 16384, torch.bfloat16
    g = _gen(81)
    h = torch.randn((rows, width), device=DEV, generator=g).to(dt).requires_grad_()
    w = torch.zeros((classes, width), dtype=dt, device=DEV)
    w[-300:] = (torch.randn((300, width), device=DEV, generator=g) * 0.02).to(dt)      # the others have logits of 0
    w.requires_grad_()
    target = torch.tensor([classes - 1, classes - 5], device=DEV)
    loss = LB.linear_cross_entropy(h, w, target)
    dh, dw = torch.autograd.grad(loss, (h, w))
    z = h.detach().double() @ w.detach()[-300:].double().t()
    lse = torch.log(torch.exp(z).sum(dim=1) + (classes - 300))
    dz = torch.exp(z - lse[:, None])
    dz[0, -1] -= 1
    dz[1, -5] -= 1
    dz /= rows
    ez = width * 2.0 ** -23 * float((h.detach().double().abs() @ w.detach()[-300:].double().abs().t()).max())
    assert abs(float(loss.detach()) - float((lse - z[torch.arange(2), target - (classes - 300)]).mean())) <= 2 * ez + 2.0 ** -20 * 20
    ep = 2 * ez + 2.0 ** -20 * (1 + float(z.abs().max()))
    err = (U[dt] + ep) * dz.abs() + ep / rows
    want = dz.t() @ h.detach().double()
    assert bool(((dw[-300:].double() - want).abs() <= err.t() @ h.detach().double().abs() + U[dt] * want.abs() + 1e-37).all())
    # dh: the 139700 zero rows add nothing
    want = dz @ w.detach()[-300:].double()
    tol = (err + classes * 2.0 ** -23 * dz.abs()) @ w.detach()[-300:].double().abs() + U[dt] * want.abs() + 1e-37
    assert bool(((dh.double() - want).abs() <= tol).all())
    del w, dw, dh
    rows, classes = 43000, 50304
    x = torch.zeros((rows, classes), dtype=dt, device=DEV)
    x[-2:] = (torch.randn((2, classes), device=DEV, generator=g) * 3).to(dt)
    idx = torch.full((rows, 1), -1, device=DEV)
    idx[-2:] = torch.tensor([[50000], [7]], device=DEV)
    values = torch.zeros((rows, 1), device=DEV)
    loss_rows, lse, mean, inv_live, live, weights = LB.distill_fwd(x, values, idx)
    dx = LB.distill_bwd(x, idx, weights, live, lse, inv_live=inv_live)
    loss, lse64, dz = _soft(x[-2:].double(), idx[-2:], torch.ones((2, 1), dtype=torch.float64, device=DEV), 1.0)
    ep = 2.0 ** -20 * (2 + 2 * 20) + (classes / 256 + 16) * 2.0 ** -23
    assert bool(((loss_rows[-2:].double() - loss).abs() <= ep + 2.0 ** -20 * 20).all()) and float(inv_live) == 0.5
    assert bool(((dx[-2:].double() - dz / 2).abs() <= (U[dt] + ep) * dz.abs() + ep * (dz < 0) + 1e-37).all())
    assert not bool(dx[:-2].any())


def test_differences_of_the_loss():
    """Central differences of the losses along directions that 16-bit inputs can take: |D - <g, d>| <= e^2 S^3 / 6 (the third derivative of a
    log-sum-exp along a line is at most the cube of the spread S of the logits' slopes) + 2^-18 (1 + loss) / e + the gradient's rounding."""
    rows, vocab, width, k, dt = 6, 40, 64, 3, torch.bfloat16
    h, w, g = _operands(rows, vocab, width, dt, 31)
    target = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    values, idx = torch.randn((rows, k), device=DEV, generator=g), torch.randint(0, vocab, (rows, k), device=DEV, generator=g)
    losses = (lambda a, b: LB.linear_cross_entropy(a, b, target), lambda a, b: LB.linear_distillation_loss(a, b, values, idx, 2.0))
    e = 2.0 ** -5
    for f in losses:
        h1, w1 = h.clone().requires_grad_(), w.clone().requires_grad_()
        dh, dw = torch.autograd.grad(f(h1, w1), (h1, w1))
        for which, grad in ((0, dh), (1, dw)):
            # a direction of whole multiples of the inputs' spacing at their largest magnitude, so that the shifted inputs are exact
            x = (h, w)[which].double()
            step = 2.0 ** -4 if which == 0 else 2.0 ** -6
            grid = (x / step).round() * step
            d = torch.sign(grad.double())
            args = [h, w]
            def at(s):
                args[which] = (grid + s * step * d).to(dt)
                assert torch.equal(args[which].double(), grid + s * step * d)
                return float(f(*args))
            args[which] = grid.to(dt)
            hh, ww = [a.clone().requires_grad_() for a in args]
            gr = torch.autograd.grad(f(hh, ww), (hh, ww))[which].double()
            diff = (at(1) - at(-1)) / 2
            slope = float((gr * d).sum()) * step
            z1 = (step * d) @ w.double().t() if which == 0 else h.double() @ (step * d).t()
            spread = float((z1.max(dim=1).values - z1.min(dim=1).values).max())
            tol = spread ** 3 / 6 + 2.0 ** -18 * (1 + abs(at(1))) + U[dt] * float(gr.abs().sum()) * step * 4
            assert abs(diff - slope) <= tol, (which, diff, slope, tol)


def test_repeated_streams_and_capture():
    """Same bits again, on two streams at once, and from a captured graph replayed on new inputs while eager calls run between."""
    rows, vocab, width, dt = 200, 2003, 256, torch.bfloat16
    h, w, g = _operands(rows, vocab, width, dt, 41)
    h2 = torch.randn((rows, width), device=DEV, generator=g).to(dt)
    target = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    target[::9] = -1
    values, idx = torch.randn((rows, 5), device=DEV, generator=g), torch.randint(0, vocab, (rows, 5), device=DEV, generator=g)

    def both(a, b):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        l1 = LB.linear_cross_entropy(a, b, target)
        l2 = LB.linear_distillation_loss(a, b, values, idx, 2.0)
        x = (a.detach() @ b.detach().t()).requires_grad_()
        l3 = LB.distillation_loss(x, values, idx, 2.0)
        return [l1.detach(), l2.detach(), l3.detach(), *torch.autograd.grad(l1, (a, b)), *torch.autograd.grad(l2, (a, b)),
                *torch.autograd.grad(l3, (x,))]

    want, want2 = both(h, w), both(h2, w)
    assert all(torch.equal(a, b) for a, b in zip(both(h, w), want))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, x in ((s1, h), (s2, h2)):
            with torch.cuda.stream(s):
                got.append(both(x, w))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want if i % 2 == 0 else want2))
    static = h.clone()
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):                                          # two graphs that hold the operators
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both(static, w))
        graphs.append(graph)
    for x, ref in ((h2, want2), (h, want), (h2, want2)):
        static.copy_(x)
        for graph in graphs:
            graph.replay()
        mid = both(h, w)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(mid, want))
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, ref))
    assert int(LB.gemm_status(torch.device(DEV))) == 0


def test_together_as_a_mixed_loss():
    """A student's step on targets and a teacher at once: the gradients of the sum are the sums of the gradients, and the linear forms agree
    with the forms on logits (whose logits are rounded to 16 bits: exp of a logit z moves by u |z| relative)."""
    rows, vocab, pad, width, k, dt = 96, 500, 512, 128, 8, torch.bfloat16
    h, w, g = _operands(rows, pad, width, dt, 51, std=0.05)
    target = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    teacher = torch.randn((rows, vocab), device=DEV, generator=g)
    values, idx = torch.topk(teacher, k, dim=1)
    h1, w1 = h.clone().requires_grad_(), w.clone().requires_grad_()
    linear = 0.25 * LB.linear_cross_entropy(h1, w1, target, vocab) + 0.75 * LB.linear_distillation_loss(h1, w1, values, idx, 2.0, vocab)
    got = torch.autograd.grad(linear, (h1, w1))
    h2, w2 = h.clone().requires_grad_(), w.clone().requires_grad_()
    logits = torch.nn.functional.linear(h2, w2)
    plain = 0.25 * LB.softmax_cross_entropy(logits, target, vocab) + 0.75 * LB.distillation_loss(logits, values, idx, 2.0, vocab)
    want = torch.autograd.grad(plain, (h2, w2))
    zmax = float(logits.detach().float().abs().max())
    assert abs(float(linear.detach()) - float(plain.detach())) <= 4 * U[dt] * zmax
    # both sides round dz and the results (u each) and the plain side the logits; relative to the sums of magnitudes
    mags = ((0.25 + 0.75 * 2.0) * 2 / rows)                     # sum of |dz| over a row is at most this
    tol = (6 * U[dt] + 4 * U[dt] * zmax) * mags * float(w.float().abs().max())
    assert bool(((got[0].float() - want[0].float()).abs() <= tol).all())
    col = mags * rows * float(h.float().abs().max())
    assert bool(((got[1].float() - want[1].float()).abs() <= (6 * U[dt] + 4 * U[dt] * zmax) * col).all())


def test_no_rows_and_refusals():
    dt = torch.bfloat16
    h, w, g = _operands(4, 32, 16, dt, 61)
    t = torch.zeros(4, dtype=torch.int64, device=DEV)
    v, i = torch.zeros((4, 2), device=DEV), torch.zeros((4, 2), dtype=torch.int64, device=DEV)
    h0, w0 = h[:0].clone().requires_grad_(), w.clone().requires_grad_()
    loss = LB.linear_cross_entropy(h0, w0, t[:0])
    dh, dw = torch.autograd.grad(loss, (h0, w0))
    assert float(loss.detach()) == 0.0 and dh.shape == (0, 16) and bool((dw == 0).all())
    x0 = torch.zeros((0, 32), device=DEV).requires_grad_()
    assert torch.autograd.grad(LB.distillation_loss(x0, v[:0], i[:0]), (x0,))[0].shape == (0, 32)
    for bad in (lambda: LB.linear_cross_entropy(h.float(), w.float(), t), lambda: LB.linear_cross_entropy(h, w.half(), t),
                lambda: LB.linear_cross_entropy(h, w, t.int()), lambda: LB.linear_cross_entropy(h, w, t[:3]),
                lambda: LB.linear_distillation_loss(h, w, v, i.int()), lambda: LB.linear_distillation_loss(h, w, v.double(), i),
                lambda: LB.distillation_loss(h.double(), v, i)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: LB.linear_cross_entropy(h.cpu(), w, t), lambda: LB.linear_cross_entropy(h, w[:, :8], t),
                lambda: LB.linear_cross_entropy(h, w, t, 33), lambda: LB.linear_cross_entropy(h, w, t, 0),
                lambda: LB.linear_distillation_loss(h, w, v[:, :1], i), lambda: LB.linear_distillation_loss(h, w, v[:3], i[:3]),
                lambda: LB.distillation_loss(h, v, i, 1.0, 17), lambda: LB.distillation_loss(h[0], v, i)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: LB.linear_distillation_loss(h, w, v, i, 0.0), lambda: LB.distillation_loss(h, v, i, -1.0),
                lambda: LB.distillation_loss(h, v[:, :0], i[:, :0]), lambda: LB.distillation_loss(h, v, i, float("nan")),
                lambda: LB.linear_distillation_loss(h, w, torch.zeros((4, 513), device=DEV), torch.zeros((4, 513), dtype=torch.int64, device=DEV))):
        with pytest.raises(LB.LancetError):
            bad()

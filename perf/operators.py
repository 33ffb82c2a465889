"""Measured cases of the language-model head's losses: cross entropy and distillation from a teacher's top logits.

Three operators, each as a training step calls it (loss and gradients) and the first also as scoring calls it (row losses only):

  linear_ce       loss of `hidden @ weight.T` against target tokens, gradients of hidden and weight; the logits are not kept
  distill         loss of given logits against a teacher's top-k logits, gradient of the logits
  linear_distill  as `distill`, from hidden rows and the head's weight; the logits are not kept

With `own` false `run` computes them in their plain form; with `own` true it makes the calls of the package."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_MACS = 16384 * 50257 * 2048          # rows x vocabulary x width of the largest listed case
MOST_LOGITS = 8192 * 50304


def listed():
    return [
        # a test-sized model's head: one launch's work, latency counts
        dict(name="ce_tiny", op="linear_ce", rows=33, vocab=1009, pad=1009, width=128, dtype="fp16", ignored=0.1, grad=True),
        # a single token's loss and gradients: the head's weight is what moves
        dict(name="ce_one_row", op="linear_ce", rows=1, vocab=50257, pad=50304, width=1024, dtype="bf16", ignored=0.0, grad=True),
        # scoring one sequence: row losses only
        dict(name="ce_score", op="linear_ce", rows=511, vocab=50257, pad=50304, width=1024, dtype="bf16", ignored=0.0, grad=False),
        # the training step of the 12-layer model: 16 sequences of 512 tokens, the last position of each without a target
        dict(name="ce_train", op="linear_ce", rows=8192, vocab=50257, pad=50304, width=1024, dtype="bf16", ignored=1 / 512, grad=True),
        # fine-tuning on answers: about half of the rows are prompt tokens without a target; ragged sizes
        dict(name="ce_answers", op="linear_ce", rows=4095, vocab=32003, pad=32003, width=2048, dtype="fp16", ignored=0.5, grad=True),
        # the largest head: the tokens and the width of the dispatch workload
        dict(name="ce_large", op="linear_ce", rows=16384, vocab=50257, pad=50304, width=2048, dtype="bf16", ignored=0.0, grad=True),
        # a few rows of float32 logits
        dict(name="distill_few", op="distill", rows=7, vocab=50257, pad=50257, k=8, temperature=1.0, dtype="fp32", ignored=0.0, grad=True),
        # ragged half-precision logits with an odd row length, a fifth of the rows without a teacher
        dict(name="distill_ragged", op="distill", rows=1023, vocab=32003, pad=32003, k=17, temperature=1.5, dtype="fp16", ignored=0.2, grad=True),
        # the training step's logits
        dict(name="distill_train", op="distill", rows=8192, vocab=50257, pad=50304, k=32, temperature=2.0, dtype="bf16", ignored=1 / 512, grad=True),
        # a short batch
        dict(name="lin_distill_few", op="linear_distill", rows=64, vocab=50257, pad=50304, width=512, k=16, temperature=1.0, dtype="bf16", ignored=0.0, grad=True),
        # the training step
        dict(name="lin_distill_train", op="linear_distill", rows=8192, vocab=50257, pad=50304, width=1024, k=32, temperature=2.0, dtype="bf16", ignored=1 / 512, grad=True),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("linear_ce", "linear_ce", "distill", "linear_distill"))
    case = dict(op=op, dtype=rng.choice(("bf16", "fp16") if op != "distill" else ("bf16", "fp16", "fp32")),
                ignored=rng.choice((0.0, 0.0, 0.1, 0.5)), grad=op != "linear_ce" or rng.random() < 0.8)
    vocab = _spread(rng, 300, 130000)
    if op == "distill":
        rows = _spread(rng, 1, max(1, min(16384, MOST_LOGITS // (2 * vocab))))
    else:
        width = _spread(rng, 64, 4096)
        if rng.random() < 0.8:
            width = (width + 63) // 64 * 64
        case["width"] = width
        rows = _spread(rng, 1, max(1, min(16384, MOST_MACS // (2 * vocab * width))))
    case.update(rows=rows, vocab=vocab, pad=vocab if rng.random() < 0.3 else (vocab + 127) // 128 * 128)
    if op != "linear_ce":
        case.update(k=_spread(rng, 1, 128), temperature=round(rng.uniform(0.5, 4.0), 2))
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab, pad, dt = case["rows"], case["vocab"], case["pad"], DTYPES[case["dtype"]]
    op = case["op"]

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=g)

    dead = rand(rows) < case["ignored"]
    # upstream factor of the loss: an accumulated step's, in half precision with the loss scale that keeps the gradient of a
    # mean over many rows out of the type's subnormals
    s = {"case": case, "up": (0.25 + rand(1)[0]) * (4.0 * rows if dt == torch.float16 else 1.0)}
    if op == "linear_ce":
        idx = torch.randint(0, vocab, (rows, 1), device="cuda", generator=g)
        s["target"] = idx[:, 0].masked_fill(dead, -1)
    else:
        k = case["k"]
        idx = torch.randint(0, vocab, (rows, k), device="cuda", generator=g)
        s["top_indices"] = idx.masked_fill(dead[:, None], -1)
        s["top_values"] = (8.0 + 2.0 * randn(rows, k)).sort(dim=1, descending=True).values      # as a top-k gives them
    if op == "distill":
        x = randn(rows, pad)
        x.scatter_add_(1, idx, 0.5 * s["top_values"] + randn(rows, k))                          # a student on its way
        s["logits"] = x.to(dt).requires_grad_(case["grad"])
    else:
        width = case["width"]
        w = (0.02 * randn(pad, width)).to(dt)
        # normalised rows that lean towards their token: its logit stands 0 to 12 above the others
        lean = 12.0 * rand(rows, 1) / (0.0004 * width)
        h = randn(rows, width) + lean * w[idx[:, 0]].float()
        s["hidden"] = h.to(dt).requires_grad_(case["grad"])
        s["weight"] = w.requires_grad_(case["grad"])
    return s


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        if case["op"] == "linear_ce":
            return _plain_linear_ce(state, case)
        if case["op"] == "distill":
            return _plain_distill(state, case)
        return _plain_linear_distill(state, case)


def _run_own(state, case):
    import lancet_b200 as LB
    vocab = case["vocab"]
    if case["op"] == "linear_ce":
        if not case["grad"]:
            loss_rows, lse_rows = LB.linear_xent_fwd(state["hidden"], state["weight"], state["target"], vocab)[:2]
            return {"loss_rows": loss_rows, "lse_rows": lse_rows}
        loss = LB.linear_cross_entropy(state["hidden"], state["weight"], state["target"], vocab)
        dh, dw = torch.autograd.grad(loss, (state["hidden"], state["weight"]), state["up"])
        return {"loss": loss.detach(), "dhidden": dh, "dweight": dw}
    if case["op"] == "distill":
        loss = LB.distillation_loss(state["logits"], state["top_values"], state["top_indices"], case["temperature"], vocab)
        (dx,) = torch.autograd.grad(loss, (state["logits"],), state["up"])
        return {"loss": loss.detach(), "dlogits": dx}
    loss = LB.linear_distillation_loss(state["hidden"], state["weight"], state["top_values"], state["top_indices"],
                                       case["temperature"], vocab)
    dh, dw = torch.autograd.grad(loss, (state["hidden"], state["weight"]), state["up"])
    return {"loss": loss.detach(), "dhidden": dh, "dweight": dw}


def _log_sum_exp(z):
    m = z.max(dim=1).values
    return m + torch.log(torch.exp(z - m[:, None]).sum(dim=1))


def _head_gradients(state, dz, vocab):
    h, w = state["hidden"], state["weight"]
    dw = torch.zeros(w.shape, dtype=w.dtype, device=w.device)
    dw[:vocab] = (dz.t() @ h.float()).to(w.dtype)
    return (dz @ w[:vocab].float()).to(h.dtype), dw


def _plain_linear_ce(state, case):
    vocab, target = case["vocab"], state["target"]
    z = state["hidden"].float() @ state["weight"][:vocab].float().t()
    live = target >= 0
    at = target.clamp(min=0)[:, None]
    lse = _log_sum_exp(z)
    loss_rows = torch.where(live, lse - z.gather(1, at)[:, 0], 0.0)
    if not case["grad"]:
        return {"loss_rows": loss_rows, "lse_rows": torch.where(live, lse, 0.0)}
    n = live.sum().clamp(min=1)
    p = torch.exp(z - lse[:, None])
    p.scatter_add_(1, at, -torch.ones_like(loss_rows)[:, None])
    p *= (live * (state["up"] / n))[:, None]
    dh, dw = _head_gradients(state, p, vocab)
    return {"loss": loss_rows.sum() / n, "dhidden": dh, "dweight": dw}


def _plain_teacher(state, temperature):
    """Teacher probabilities over its top entries, their logarithms, the indices to read at and the live rows."""
    idx, v = state["top_indices"], state["top_values"].float() / temperature
    live = (idx >= 0).any(dim=1)
    logq = v - _log_sum_exp(v)[:, None]
    return torch.exp(logq) * live[:, None], logq, idx.clamp(min=0), live


def _plain_distill_of(z, state, case):
    """(loss rows, gradient of the mean with respect to the logits z, live rows counted)"""
    t = case["temperature"]
    q, logq, at, live = _plain_teacher(state, t)
    zt = z / t
    lse = _log_sum_exp(zt)
    logp = zt.gather(1, at) - lse[:, None]
    n = live.sum().clamp(min=1)
    loss_rows = t * t * (q * (logq - logp)).sum(dim=1)
    p = torch.exp(zt - lse[:, None])
    p.scatter_add_(1, at, -q)
    p *= (live * (t * state["up"] / n))[:, None]
    return loss_rows.sum() / n, p


def _plain_distill(state, case):
    x, vocab = state["logits"], case["vocab"]
    loss, dz = _plain_distill_of(x[:, :vocab].float(), state, case)
    dx = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
    dx[:, :vocab] = dz.to(x.dtype)
    return {"loss": loss, "dlogits": dx}


def _plain_linear_distill(state, case):
    vocab = case["vocab"]
    z = state["hidden"].float() @ state["weight"][:vocab].float().t()
    loss, dz = _plain_distill_of(z, state, case)
    dh, dw = _head_gradients(state, dz, vocab)
    return {"loss": loss, "dhidden": dh, "dweight": dw}


def _live_rows(case):
    return max(1, round(case["rows"] * (1 - case["ignored"])))


def work(case):
    """Rows without a target or teacher need no arithmetic.  The head's gradients need three products of rows x vocabulary x
    width (the logits once, each gradient once); scoring needs one."""
    rows, live, vocab, pad = case["rows"], _live_rows(case), case["vocab"], case["pad"]
    size = 4 if case["dtype"] == "fp32" else 2
    teacher = 0 if case["op"] == "linear_ce" else rows * case["k"] * (4 + 8)
    if case["op"] == "distill":
        return {"bytes": live * vocab * size + rows * pad * size + teacher, "flops": 8 * live * vocab}
    width = case["width"]
    operands = (live + vocab) * width * size
    if not case["grad"]:
        return {"bytes": operands + rows * 16, "flops": 2 * live * vocab * width}
    return {"bytes": operands + (rows + pad) * width * size + rows * 8 + teacher, "flops": 6 * live * vocab * width}


def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time: for target t, loss = -log softmax(z)_t; for teacher entries (i, v),
    q = softmax(v / T) and loss = T^2 sum_i q_i (log q_i - log softmax(z / T)_i).  Gradients are those of the mean over live rows."""
    s = prepare(case, seed)
    rows, vocab, t = case["rows"], case["vocab"], float(case.get("temperature", 1.0))
    up = s["up"].double()
    with torch.no_grad():
        if case["op"] == "linear_ce":
            idx = s["target"][:, None]
            q_all = torch.ones((rows, 1), dtype=torch.float64, device="cuda")
        else:
            idx = s["top_indices"]
            q_all = torch.softmax(s["top_values"].double() / t, dim=1)
        live = idx[:, 0] >= 0
        n = max(1, int(live.sum()))
        linear = case["op"] != "distill"
        if linear:
            h, w = s["hidden"].double(), s["weight"][:vocab].double()
            dh = torch.zeros_like(h)
            dw = torch.zeros(s["weight"].shape, dtype=torch.float64, device="cuda")
        else:
            dx = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
        loss_rows = torch.zeros(rows, dtype=torch.float64, device="cuda")
        lse_rows = torch.zeros(rows, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 28) // vocab)
        for r0 in range(0, rows, step):
            r = torch.arange(r0, min(rows, r0 + step), device="cuda")
            r = r[live[r]]
            if r.numel() == 0:
                continue
            z = (h[r] @ w.t() if linear else s["logits"][r, :vocab].double()) / t
            lse = torch.logsumexp(z, dim=1)
            q = q_all[r]
            # x log x is 0 at 0
            loss_rows[r] = t * t * (torch.xlogy(q, q) - q * (z.gather(1, idx[r]) - lse[:, None])).sum(dim=1)
            lse_rows[r] = lse
            if not case["grad"]:
                continue
            dz = torch.zeros_like(z).scatter_add_(1, idx[r], q).neg_().add_(torch.exp(z - lse[:, None])).mul_(t * up / n)
            if linear:
                dh[r] = dz @ w
                dw[:vocab] += dz.t() @ h[r]
            else:
                dx[r, :vocab] = dz
        if not case["grad"]:
            return {"loss_rows": loss_rows, "lse_rows": lse_rows}
        loss = loss_rows.sum() / n
        return {"loss": loss, "dhidden": dh, "dweight": dw} if linear else {"loss": loss, "dlogits": dx}

"""Entry points of the head's losses without a GPU: invalid calls are refused before the device is touched, and the Python operators refuse CPU
tensors and wrong types."""
import ctypes

import pytest
import torch

import lancet_b200 as LB
from lancet_b200 import _capi

ONE = ctypes.c_void_p(256)
BF16, F32 = 2, 0


@pytest.fixture(scope="module")
def L():
    LB.build.build()
    return _capi.lib()


def _xent_fwd(L, hidden=ONE, ldh=64, weight=ONE, ldw=64, target=ONE, rows=4, vocab=100, width=64, dtype=BF16, loss=ONE, lse=ONE, pos=ONE,
              mean=ONE, inv=ONE, ws=ONE, nws=1 << 40, status=ONE):
    return L.lancet_linear_xent_fwd(hidden, ldh, weight, ldw, target, rows, vocab, width, dtype, loss, lse, pos, mean, inv, ws, nws, status, None)


def _distill_fwd(L, k=4, temperature=1.0, values_dtype=F32, **kw):
    a = dict(hidden=ONE, ldh=64, weight=ONE, ldw=64, rows=4, vocab=100, width=64, dtype=BF16, values=ONE, indices=ONE, ws=ONE, nws=1 << 40)
    a.update(kw)
    return L.lancet_linear_distill_fwd(a["hidden"], a["ldh"], a["weight"], a["ldw"], a["values"], values_dtype, a["indices"], k, temperature,
                                       a["rows"], a["vocab"], a["width"], a["dtype"], ONE, ONE, ONE, ONE, ONE, ONE, a["ws"], a["nws"], ONE, None)


def test_linear_losses_refuse_bad_sizes_types_and_pointers(L):
    assert _xent_fwd(L, dtype=F32) == 6 and b"bfloat16 or float16" in L.lancet_last_error()
    for kw in (dict(rows=-1), dict(vocab=0), dict(width=0), dict(ldh=63), dict(ldw=56), dict(ldw=68), dict(weight=ctypes.c_void_p(8)),
               dict(hidden=ctypes.c_void_p(257)), dict(rows=(1 << 26) + 1), dict(nws=64), dict(ws=ctypes.c_void_p(16)), dict(ws=None)):
        assert _xent_fwd(L, **kw) == 1, kw
    for kw in (dict(hidden=None), dict(weight=None), dict(target=None), dict(loss=None), dict(lse=None), dict(pos=None), dict(mean=None),
               dict(inv=None), dict(status=None)):
        assert _xent_fwd(L, **kw) == 2, kw
    for kw in (dict(k=0), dict(k=513), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
               dict(temperature=float("inf")), dict(values_dtype=9), dict(nws=64)):
        assert _distill_fwd(L, **kw) == 1, kw
    assert _distill_fwd(L, values=None) == 2 and _distill_fwd(L, indices=None) == 2
    args = [ONE, 64, ONE, 64, ONE, ONE, ONE, ONE, 4, 100, 99, 64, BF16, None, None, 1.0, ONE, ONE, ONE, 1 << 40, ONE, None]
    assert L.lancet_linear_xent_bwd(*args) == 1 and b"weight rows" in L.lancet_last_error()
    args[10], args[19] = 100, 64
    assert L.lancet_linear_xent_bwd(*args) == 1 and b"workspace" in L.lancet_last_error()
    args[19], args[7] = 1 << 40, None
    assert L.lancet_linear_xent_bwd(*args) == 2
    args[7], args[16], args[17] = ONE, None, None       # no gradient wanted: nothing to do
    assert L.lancet_linear_xent_bwd(*args) == 0


def test_distillation_refuses(L):
    f = lambda **kw: L.lancet_distill_fwd(*[{**dict(x=ONE, ld=64, v=ONE, vd=F32, i=ONE, k=4, t=1.0, rows=4, vocab=60, dt=F32, a=ONE, b=ONE, c=ONE,
                                                    d=ONE, m=ONE, n=ONE, st=None), **kw}[n] for n in
                                            ("x", "ld", "v", "vd", "i", "k", "t", "rows", "vocab", "dt", "a", "b", "c", "d", "m", "n", "st")])
    for kw in (dict(ld=59), dict(vocab=0), dict(rows=-1), dict(dt=3), dict(vd=-1), dict(k=0), dict(k=513), dict(t=0.0), dict(t=2e3)):
        assert f(**kw) == 1, kw
    for kw in (dict(x=None), dict(v=None), dict(i=None), dict(a=None), dict(b=None), dict(c=None), dict(d=None), dict(m=None), dict(n=None)):
        assert f(**kw) == 2, kw
    g = lambda **kw: L.lancet_distill_bwd(*[{**dict(x=ONE, ld=64, i=ONE, w=ONE, l=ONE, k=4, t=1.0, rows=4, vocab=60, cols=64, dt=F32, lse=ONE, go=None,
                                                    inv=None, s=1.0, dx=ONE, ldd=64, st=None), **kw}[n] for n in
                                            ("x", "ld", "i", "w", "l", "k", "t", "rows", "vocab", "cols", "dt", "lse", "go", "inv", "s", "dx", "ldd", "st")])
    for kw in (dict(cols=59), dict(ldd=63), dict(ld=59), dict(k=0), dict(t=-1.0), dict(dt=7)):
        assert g(**kw) == 1, kw
    for kw in (dict(x=None), dict(i=None), dict(w=None), dict(l=None), dict(lse=None), dict(dx=None)):
        assert g(**kw) == 2, kw
    assert g(rows=0, x=None) == 0


def test_copy_rows_and_workspace_queries(L):
    assert L.lancet_copy_rows(ONE, 5, ONE, 7, 2, 5, None) == 1 and L.lancet_copy_rows(ONE, 4, ONE, 8, 2, 5, None) == 1
    assert L.lancet_copy_rows(None, 5, ONE, 8, 2, 5, None) == 2 and L.lancet_copy_rows(ONE, 5, ctypes.c_void_p(8), 8, 2, 5, None) == 1
    assert L.lancet_copy_rows(None, 5, None, 8, 0, 5, None) == 0
    f, b = L.lancet_linear_loss_fwd_workspace_bytes, L.lancet_linear_loss_bwd_workspace_bytes
    assert f(-1, 10, 8, 0) == 0 and f(1, 0, 8, 0) == 0 and b(1, 10, 0) == 0
    assert f(0, 10, 8, 0) > 0 and b(0, 10, 8) > 0
    assert f(8192, 50257, 1024, 32) > f(8192, 50257, 1024, 0) > 8192 * 1024 * 2
    # dz of a piece takes at most 1 GiB unless that were fewer than 4096 classes
    assert b(8192, 50257, 1024) < (1 << 30) + (128 << 20)
    assert b(65536, 200000, 64) < (1 << 30) + (256 << 20)
    assert 262144 * 4096 * 2 <= b(262144, 50257, 64) < 262144 * 4096 * 2 + (512 << 20)


def test_operators_refuse_cpu_tensors():
    h, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(9, 8, dtype=torch.bfloat16)
    t, v, i = torch.zeros(4, dtype=torch.int64), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64)
    for f in (lambda: LB.linear_cross_entropy(h, w, t), lambda: LB.linear_distillation_loss(h, w, v, i), lambda: LB.distillation_loss(h, v, i),
              lambda: LB.linear_xent_fwd(h, w, t), lambda: LB.distill_fwd(h, v, i)):
        with pytest.raises(ValueError):
            f()

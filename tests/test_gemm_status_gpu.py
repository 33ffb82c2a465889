"""The status word of the bounded waits where the first call on a device runs under stream capture."""
import pytest
import torch

import lancet_b200 as LB
from lancet_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_word_first_made_under_capture(monkeypatch):
    g = torch.Generator(device=DEV).manual_seed(6)
    h, w = torch.randn((40, 64), device=DEV, generator=g).bfloat16(), torch.randn((300, 64), device=DEV, generator=g).bfloat16()
    target = torch.randint(0, 300, (40,), device=DEV, generator=g)
    want = LB.linear_xent_fwd(h, w, target)[0]
    monkeypatch.setattr(ops, "_gemm_status", {})
    monkeypatch.setattr(ops, "_filling", {}, raising=False)
    seen, launch = [], ops._launch
    monkeypatch.setattr(ops, "_launch", lambda fn, like, *args: (seen.append(args[-1]), launch(fn, like, *args)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = LB.linear_xent_fwd(h, w, target)[0]
        out = LB.linear_xent_fwd(h, w, target)[0]
        more = [torch.full((1,), 7, dtype=torch.int32, device=DEV) for _ in range(64)]     # would take over a word that no one holds
    graph.replay()
    word = LB.gemm_status(torch.device(DEV))
    assert torch.equal(out, want) and all(int(t) == 7 for t in more)
    assert seen == 2 * [word.data_ptr()] and int(word) == 0
    # the word is the same under every name of the device, for every operator, and is not the graph's to fill
    assert LB.gemm_status(DEV) is word and LB.gemm_status(torch.device("cuda", torch.cuda.current_device())) is word
    word.fill_(3)
    graph.replay()
    assert int(word) == 3
    word.zero_()
    del graph, out, more
    torch.cuda.empty_cache()
    assert torch.equal(LB.linear_xent_fwd(h, w, target)[0], want) and seen[2] == word.data_ptr() and int(word) == 0

"""Scratch of captured calls: owned by their graph, shared by the calls of a capture,
handed on when the graph is gone."""
import gc

import pytest
import torch

from tests.paged_util import Pool

pytestmark = pytest.mark.gpu


def _capture(call, times=1):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [call() for _ in range(times)]
    return graph, outs


def test_blocks_belong_to_their_graph(gpu):
    import rdnattention as ra

    pool = Pool([900, 1500], 2, 64, 16, torch.float16, seed=1)
    k, v, table, lens, _ = pool.on(gpu)
    q = torch.randn(2, 8, 64, device=gpu).half()

    def call():
        return ra.paged_attention(q, k, v, table, lens)

    want = call()
    torch.cuda.synchronize()
    ra.trim_scratch()
    start = ra.scratch_stats()["allocations"]
    first, outs = _capture(call, 3)  # one after the other: one block
    assert ra.scratch_stats()["allocations"] == start + 1
    second, more = _capture(call)  # another graph: another block
    assert ra.scratch_stats()["allocations"] == start + 2
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for o in outs + more:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip((first, second), streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs + more)
    del first
    gc.collect()
    third, last = _capture(call)  # the first graph's block
    assert ra.scratch_stats()["allocations"] == start + 2
    third.replay()
    second.replay()
    torch.cuda.synchronize()
    assert torch.equal(last[0], want) and torch.equal(more[0], want)
    del second, third
    gc.collect()
    ra.trim_scratch()
    assert torch.equal(call(), want)


def test_graphs_of_other_sizes(gpu):
    """A block handed on to a call that needs less; one too small is not."""
    import rdnattention as ra

    made = []
    for n in (1500, 300, 4000):
        q, k, v = (torch.randn(1, 8, n, 64, device=gpu).half() for _ in range(3))
        cos = torch.rand(n, 32, device=gpu)
        want = ra.flash_attn(q, k, v, is_causal=True, rot_cos=cos, rot_sin=cos)
        torch.cuda.synchronize()
        graph, outs = _capture(lambda: ra.flash_attn(q, k, v, is_causal=True, rot_cos=cos, rot_sin=cos))
        for _ in range(3):
            outs[0].zero_()
            graph.replay()
            ra.flash_attn(q, k, v, rot_cos=cos, rot_sin=cos)
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want)
        if n == 1500:
            del graph
            gc.collect()
        else:
            made.append((graph, outs, want, q, k, v, cos))
    for graph, outs, want, *_ in made:
        outs[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want)

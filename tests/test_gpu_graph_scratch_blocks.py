"""Blocks of captured calls: counted, handed on to calls of about their size alone, given
back where the device has no memory left, and by trim_scratch()."""
import gc

import pytest
import torch

from tests.paged_util import Pool

pytestmark = pytest.mark.gpu

MB = 1 << 20


def _capture(call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


def _gone():
    gc.collect()
    torch.cuda.synchronize()


def _graphs():
    import rdnattention as ra

    st = ra.scratch_stats()
    return st["graph_blocks"], st["graph_bytes"]


@pytest.fixture
def calls(gpu):
    """Calls of 24 MiB of scratch (a rotated copy of the keys), and of two."""
    import rdnattention as ra

    q, k, v = (torch.randn(4, 8, 3000, 128, device=gpu).half() for _ in range(3))
    cos = torch.rand(3000, 64, device=gpu)
    pool = Pool([900, 1500], 2, 64, 16, torch.float16, seed=1)
    pk, pv, table, lens, _ = pool.on(gpu)
    pq = torch.randn(2, 8, 64, device=gpu).half()

    def large():
        return ra.flash_attn(q, k, v, is_causal=True, rot_cos=cos, rot_sin=cos)

    def small():
        return ra.paged_attention(pq, pk, pv, table, lens)

    _gone()
    ra.trim_scratch()
    return large, small


def test_large_blocks_are_not_for_small_calls(calls):
    import rdnattention as ra

    large, small = calls
    want, want_small = large(), small()
    n, held = _graphs()
    graph, out = _capture(large)
    assert _graphs()[0] == n + 1 and _graphs()[1] >= held + 23 * MB
    del graph, out
    _gone()
    assert _graphs()[0] == n + 1  # to be handed on
    graph, out = _capture(small)
    assert _graphs()[0] == n + 2  # not to this one
    again, same = _capture(large)
    assert _graphs()[0] == n + 2  # but to this one
    for _ in range(3):
        out.zero_()
        same.zero_()
        graph.replay()
        again.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_small) and torch.equal(same, want)
    ra.trim_scratch()
    assert _graphs()[0] == n + 2  # both have their graphs
    graph.replay()
    again.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want_small) and torch.equal(same, want)
    del graph, again
    _gone()
    ra.trim_scratch()
    assert _graphs() == (n, held)


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_no_memory_for_a_captured_call(gpu, calls):
    """A call whose scratch no device holds (2^24 rows of 32 heads of 256 in 32 bits, all one
    row of the query): an error, after the blocks that no graph owns were given back, and
    the next capture works."""
    import rdnattention as ra

    large, small = calls
    want = small()
    n, held = _graphs()
    graph, out = _capture(large)
    del graph, out
    _gone()
    assert _graphs()[0] == n + 1
    pool = Pool([64, 64], 32, 256, 16, torch.float16, seed=2)
    k, v, table, lens, _ = pool.on(gpu)
    row = torch.zeros(1, 32, 256, device=gpu).half()
    rows = row.expand(1 << 24, 32, 256)
    with pytest.raises(ra.RDNAttentionError, match="scratch allocation failed"):
        _capture(lambda: ra.paged_prefix_attention(rows, k, v, table[1:], lens[1:].contiguous(), table[:1],
                                                   lens[:1].contiguous(), out=rows))
    torch.cuda.synchronize()
    assert _graphs() == (n, held)
    graph, out = _capture(small)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)

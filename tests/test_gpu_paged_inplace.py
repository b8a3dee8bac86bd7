"""rdna_paged_append with query_out == query (the C ABI; the Python call always
makes a new tensor): the bits of the call out of place."""
import pytest
import torch

from tests.paged_util import Pool, rope_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("part", [False, True])
def test_queries_rotated_in_place(gpu, d, pairs, part):
    """Many rows, so that the chunks of a head fall into several workgroups; a view
    into a wider tensor; padding rows and, with part, channels behind the rotated."""
    import rdnattention as ra
    from rdnattention import paged

    hq, hkv, rows, pad = 5, 1, 700, 3
    pool = Pool([400, 300], hkv, d, 16, torch.float16, seed=d)
    k, v, table, lens, _ = pool.on(gpu)
    cos, sin = (t.to(gpu) for t in rope_tables(500, 16 if part and d > 32 else d // 2))
    cu = torch.tensor([0, 400, 700], dtype=torch.int32, device=gpu)
    wide = torch.randn(rows + pad, hq + 2, d, device=gpu).half()
    q = wide[:, 1:1 + hq]
    x = torch.randn(rows + pad, hkv, d, device=gpu).half()
    want = ra.paged_append(x, x, k, v, table, lens, cu_seqlens_q=cu, query=q, rot_cos=cos, rot_sin=sin,
                           rot_interleaved=pairs)
    beside = wide.clone()
    c = paged._cache(k, v, table, lens, "seq_lens", cu, None, None, rows + pad)[0]
    stream = torch.cuda.current_stream().cuda_stream
    rc = paged._lib.rdna_paged_append(c, x.data_ptr(), x.data_ptr(), *x.stride()[:2], *x.stride()[:2], rows + pad, 0,
                                      q.data_ptr(), q.data_ptr(), *q.stride()[:2], *q.stride()[:2], hq, None,
                                      cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1],
                                      1 if pairs else 0, stream)
    torch.cuda.synchronize()
    assert rc == 0, ra.last_error()
    assert torch.equal(q, want)
    assert torch.equal(wide[:, 0], beside[:, 0]) and torch.equal(wide[:, -1], beside[:, -1])

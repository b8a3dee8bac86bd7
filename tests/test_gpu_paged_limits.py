"""Ragged calls near the largest sizes."""
import pytest
import torch

from tests.paged_util import Pool

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ns", [[1, 300, 0, 33], [1, 1, 1, 1]])
def test_many_rows_and_a_wide_table(gpu, ns):
    """65536 rows (padding, but the host does not know) and tables of 2^20 keys: more than
    2^31 tiles of 32 rows and 32 keys, of which the kernel of few rows has four sequences'."""
    import rdnattention as ra

    page, width, rows = 1024, 1024, 65536
    assert (rows * 4 // 32 + 4) * 8 * (width * page // 32 + 1) > 2 ** 31
    pool = Pool([700, 900, 40, 2000], 8, 32, page, torch.float16, seed=1)
    k, v, table, lens, _ = pool.on(gpu)
    wide = torch.full((4, width), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    live = sum(ns)
    torch.manual_seed(0)
    q = torch.zeros(rows, 32, 32, dtype=torch.float16, device=gpu)
    q[:live] = torch.randn(live, 32, 32, device=gpu).half()
    cu = torch.tensor([sum(ns[:i]) for i in range(5)], dtype=torch.int32, device=gpu)
    out = torch.full_like(q, 7.0)
    got = ra.paged_attention(q, k, v, wide, lens, cu_seqlens_q=cu, out=out)
    want = ra.paged_attention(q[:live], k, v, table, lens, cu_seqlens_q=cu)
    # the same keys in shares of other sizes.  All values are below 8: in each call the weights
    # (which sum to 1) are rounded to fp16, 2^-11 * 8, and the output once, 2^-9 there; twice both
    assert v.abs().max() < 8
    assert (got[:live].float() - want.float()).abs().max() <= 2.0 ** -7 + 2.0 ** -8
    assert (got[live:] == 7).all()

"""Rows that see no key are zeros, whatever the keys hold that other rows see."""
import pytest
import torch

from tests.paged_util import Pool

pytestmark = pytest.mark.gpu

TYPES = [(torch.float16, False, 64), (torch.bfloat16, False, 160), (torch.float16, True, 128)]


def spoil(pool, b, key):
    at = pool.where(b, [key])
    if pool.i8:
        pool.vs[at] = float("inf")
    else:
        pool.v[at] = float("nan")


@pytest.mark.parametrize("dtype,i8,d", TYPES)
@pytest.mark.parametrize("n,length", [(5, 3), (90, 60), (300, 100), (700, 650)])
def test_rows_before_the_first_key(gpu, dtype, i8, d, n, length):
    import rdnattention as ra

    pool = Pool([length, 500], 2, d, 16, dtype, i8, seed=n)
    spoil(pool, 0, 0)
    k, v, table, lens, scales = pool.on(gpu)
    q = torch.randn(n + 1, 8, d, device=gpu).to(dtype)
    cu = torch.tensor([0, n, n + 1], dtype=torch.int32, device=gpu)
    got = ra.paged_attention(q, k, v, table, lens, cu_seqlens_q=cu, **scales)
    assert (got[:n - length] == 0).all()
    assert not torch.isfinite(got[n - length:n]).any()  # key 0 is seen by all the others
    assert torch.isfinite(got[n:]).all()


@pytest.mark.parametrize("dtype,i8,d", TYPES)
@pytest.mark.parametrize("n", [6, 40, 80])
def test_drafts_that_see_nothing(gpu, dtype, i8, d, n):
    import rdnattention as ra

    pool = Pool([n], 2, d, 16, dtype, i8, seed=n)
    spoil(pool, 0, 1)
    k, v, table, lens, scales = pool.on(gpu)
    tree = torch.ones(1, n, n, dtype=torch.bool, device=gpu).tril()
    tree[0, 3:5] = False
    q = torch.randn(n, 8, d, device=gpu).to(dtype)
    got = ra.paged_tree_attention(q, k, v, table, lens, tree, **scales)
    assert (got[3:5] == 0).all()

"""The output beside a log-sum-exp or behind a prefix is as exact as the plain call's: where
all keys have the same values, O is those values whatever the weights round to."""
import pytest
import torch

from tests.paged_util import Pool

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _pool(lens, hkv, d, page, dtype, seed):
    pool = Pool(lens, hkv, d, page, dtype, seed=seed)
    g = torch.Generator().manual_seed(seed)
    value = torch.randn(hkv, d, generator=g).to(dtype)
    pool.v[:] = value
    return pool, value


# sum p v / sum p with the p that the products take: sums in 32 bits, at most 700 terms in
# four chains of each of two lanes and the merge of parts, stay within 2^-16 of v, a tenth of
# half a step of either type at the least: the nearest number is v itself.
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 128, 160, 256])
@pytest.mark.parametrize("lens,ns", [([40, 64, 200], [40, 33, 65]), ([700, 300], [260, 300])])
def test_values_all_alike(gpu, dtype, d, lens, ns):
    import rdnattention as ra

    pool, value = _pool(list(lens) + [5, 130], 2, d, 16, dtype, d)
    k, v, table, dl, _ = pool.on(gpu)
    b = len(lens)
    q = (2 * torch.randn(sum(ns), 8, d, generator=torch.Generator().manual_seed(3))).to(dtype).to(gpu)
    cu = torch.tensor([sum(ns[:i]) for i in range(b + 1)], dtype=torch.int32, device=gpu)
    want = value.repeat_interleave(4, 0).to(gpu).expand(sum(ns), -1, -1)
    kw = dict(cu_seqlens_q=cu, is_causal=False)
    own = (table[:b], dl[:b].contiguous())
    assert torch.equal(ra.paged_attention(q, k, v, *own, **kw), want)
    out, _ = ra.paged_attention(q, k, v, *own, return_lse=True, **kw)
    assert torch.equal(out, want)
    for i in (b, b + 1):
        out = ra.paged_prefix_attention(q, k, v, table[i:i + 1], dl[i:i + 1].contiguous(), *own, **kw)
        assert torch.equal(out, want)

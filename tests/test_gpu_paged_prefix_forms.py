"""paged_prefix_attention of single tokens on both sides of the rule that has prefixes and
sequences in one launch: many sequences, long prefixes, wide tables over short ones."""
import pytest
import torch

from tests.paged_util import Pool
from tests.test_gpu_paged_prefix import BF16, F16, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,hq,hkv,prefix,d,dtype,i8", [
    (100, 8, 8, [70], 64, F16, False), (140, 8, 8, [70], 64, F16, False),  # 800 and 1120 sequences x kv heads
    (120, 64, 1, [100], 64, BF16, False), (140, 64, 1, [100], 64, BF16, True),  # 7680 and 8960 rows x heads
    # as many key tiles of all row tiles as are read in one launch, of 256 channels, and more
    (4, 2, 2, [60000, 10, 0, 7], 256, F16, False), (4, 2, 2, [66000, 10, 0, 7], 256, F16, False),
    (8, 4, 2, [120000, 900], 128, F16, True), (8, 4, 2, [190000, 900, 3], 128, BF16, False)])
def test_both_forms(gpu, b, hq, hkv, prefix, d, dtype, i8):
    lens = [1 + (37 * i) % 90 for i in range(b)]
    seqs = [b * i // len(prefix) for i in range(len(prefix) + 1)]
    run(gpu, lens, [1] * b, prefix, seqs, hq, hkv, d, dtype, i8, page=64, uniform=True,
        name=f"forms {b} {hq}/{hkv} {prefix} {d}")


@pytest.mark.parametrize("ns", [[1] * 24, [1, 2, 0, 3] * 6])
def test_the_same_rows_in_both_forms(gpu, ns):
    """A table of prefixes that covers far more keys than they have takes the other form: the
    same up to two roundings of P and the output's (bf16 2^-8 each, of values up to 4)."""
    import rdnattention as ra

    pool = Pool([30 + b for b in range(24)] + [400, 90], 2, 64, 16, BF16, seed=8)
    k, v, table, lens, _ = pool.on(gpu)
    cu = torch.tensor([sum(ns[:i]) for i in range(25)], dtype=torch.int32, device=gpu)
    q = torch.randn(sum(ns), 8, 64, device=gpu).to(BF16)
    wide = torch.full((2, 40000), -1, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table[24:]
    args = dict(prefix_seqs=torch.tensor([0, 13, 24], dtype=torch.int32, device=gpu), cu_seqlens_q=cu,
                max_seqlen_q=3, return_lse=True)
    own = (lens[24:].contiguous(), table[:24], lens[:24].contiguous())
    one, lse = ra.paged_prefix_attention(q, k, v, table[24:], *own, **args)
    other, lse_other = ra.paged_prefix_attention(q, k, v, wide, *own, **args)
    assert not torch.equal(one, other)  # the other kernels
    assert ((one.float() - other.float()).abs() <= 3 * 2.0 ** -8 * 4).all()
    assert torch.allclose(lse, lse_other, rtol=0, atol=2.0 ** -16)

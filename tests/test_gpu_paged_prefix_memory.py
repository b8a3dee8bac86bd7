"""paged_prefix_attention where the device has no memory for the prefixes' part of the rows."""
import pytest
import torch

from tests.paged_util import Pool
from tests.test_gpu_scratch import _small_pool

pytestmark = pytest.mark.gpu


def test_no_memory_for_scratch(gpu):
    """An error, nothing written, and the same result as before once there is memory."""
    import rdnattention as ra

    pool = Pool([900, 700, 2000], 2, 128, 16, torch.float16, seed=6)
    k, v, table, lens, _ = pool.on(gpu)
    q = torch.randn(1400, 16, 128, device=gpu).half()  # 11.6 MB of scratch

    def call(out=None):
        return ra.paged_prefix_attention(q, k, v, table[2:], lens[2:].contiguous(), table[:2], lens[:2].contiguous(),
                                         out=out)

    want = call()
    out = torch.full_like(q, 7.0)
    with _small_pool(4 << 20):
        with pytest.raises(ra.RDNAttentionError, match="scratch allocation failed"):
            call(out)
        torch.cuda.synchronize()
    assert (out == 7).all()
    assert torch.equal(call(out), want) and out is not want

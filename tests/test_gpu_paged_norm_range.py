"""Norms of rows whose squares leave fp32's range: bf16 holds values from 1e-40 to 3e38."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-6])
@pytest.mark.parametrize("rope", [False, True])
def test_rows_of_any_size(gpu, d, eps, rope):
    """x w / sqrt(mean(x^2) + eps) in 64 bits: the result is off by half a step of bf16 (2^-8
    of the value) and, before that, by the fp32 operations: norm, weight and rotation 2^-20 of
    the pair's size; results below 2^-126 by 2^-133, half of bf16's smallest step there, and
    2^-149 of fp32."""
    import rdnattention as ra

    g = torch.Generator().manual_seed(d)
    sizes = [1.0, 1e-15, 1e-17, 1e-18, 1e-19, 1e-20, 1e-30, 3e-39, 1e17, 1e18, 1e19, 1e25, 1e38]
    rows, heads = len(sizes), 3
    x = (torch.rand(rows, heads, d, generator=g) * 2 - 1) * torch.tensor(sizes)[:, None, None]
    x[2, 1] = x[0, 1]  # heads of one wave of both kinds
    x = x.to(BF16)
    w = torch.rand(d, generator=g) + 0.5
    ang = torch.rand(4, d // 2, generator=g)
    cos, sin = ang.cos(), ang.sin()
    kw = {"rot_cos": cos.to(gpu), "rot_sin": sin.to(gpu)} if rope else {}
    kc = torch.zeros(rows, 4, heads, d, dtype=BF16, device=gpu)
    vc = torch.zeros_like(kc)
    table = torch.arange(rows, dtype=torch.int32, device=gpu)[:, None].contiguous()
    lens = torch.full((rows,), 2, dtype=torch.int32, device=gpu)
    q = ra.paged_append(x.to(gpu), x.to(gpu), kc, vc, table, lens, query=x.to(gpu), query_norm=w.to(gpu),
                        key_norm=w.to(gpu), norm_eps=eps, **kw)
    xd = x.double()
    least = float(torch.tensor(eps, dtype=torch.float32))
    want = xd / (xd.square().mean(-1, keepdim=True) + least).sqrt() * w.double()
    size = want.abs()
    if rope:
        a, b = want[..., 0::2], want[..., 1::2]
        c, s = cos[1].double(), sin[1].double()
        want, size = torch.empty_like(want), torch.empty_like(want)
        want[..., 0::2], want[..., 1::2] = a * c - b * s, a * s + b * c
        size[..., 0::2] = size[..., 1::2] = a.abs() + b.abs()
    tol = want.abs() * 2.0 ** -8 + size * 2.0 ** -20 + 2.0 ** -133 + 2.0 ** -149
    for name, got in (("queries", q), ("keys", kc[:, 1])):
        off = (got.cpu().double() - want).abs() / tol
        assert off.max() <= 1.0, (name, float(off.max()), int(off.amax((1, 2)).argmax()))
    assert torch.equal(vc[:, 1].cpu(), x)


@pytest.mark.parametrize("eps", [1e-40, 1e-6])
@pytest.mark.parametrize("dtype", [torch.float16, BF16])
def test_rows_of_zeros_infinities_and_nan(gpu, dtype, eps):
    import rdnattention as ra

    d = 64
    x = torch.ones(4, 2, d).to(dtype)
    x[0] = 0.0
    x[1, 0, 5] = float("inf")
    x[2, 1, 7] = float("nan")
    kc = torch.zeros(4, 4, 2, d, dtype=dtype, device=gpu)
    table = torch.arange(4, dtype=torch.int32, device=gpu)[:, None].contiguous()
    lens = torch.ones(4, dtype=torch.int32, device=gpu)
    w = torch.ones(d, device=gpu)
    q = ra.paged_append(x.to(gpu), x.to(gpu), kc, torch.zeros_like(kc), table, lens, query=x.to(gpu), query_norm=w,
                        key_norm=w, norm_eps=eps).cpu().float()
    assert (q[0] == 0).all() and (q[3] == 1).all() and (q[1, 1] == 1).all() and (q[2, 0] == 1).all()
    # the definition: every finite x / inf is 0, inf / inf and all of a row with NaN are NaN
    assert torch.isnan(q[1, 0, 5]) and (q[1, 0, torch.arange(d) != 5] == 0).all() and torch.isnan(q[2, 1]).all()
    assert torch.equal(q.isnan(), kc[:, 0].cpu().isnan())

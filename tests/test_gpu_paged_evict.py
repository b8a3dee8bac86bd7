"""paged_evict: every byte of the caches against the plain form, ties, values that are no
numbers, long and short sequences, graphs."""
import pytest
import torch

from tests.gpu_util import log
from tests.paged_util import Pool

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def chosen(w, budget, first, recent):
    """Kept indices of one head's weights [n], in order."""
    n = len(w)
    if n <= budget:
        return list(range(n))
    x = [(-float("inf"), 0) if v != v else (v + 0.0, 1) for v in w.tolist()]
    between = sorted(range(first, n - recent), key=lambda i: (-x[i][0], -x[i][1], i))[:budget - first - recent]
    return sorted(list(range(first)) + between + list(range(n - recent, n)))


def run(gpu, lens, hkv, d, dtype, i8, budget, first=0, recent=0, page=16, layout="nhd", seed=1, weights=None, name=""):
    import rdnattention as ra

    pool = Pool(lens, hkv, d, page, dtype, i8, seed=seed, layout=layout)
    g = torch.Generator().manual_seed(seed)
    w = torch.rand(pool.pages, page, hkv, generator=g) if weights is None else weights(pool, g)
    k, v, table, dl, scales = pool.on(gpu)
    dw = w.to(gpu)
    if layout != "nhd":
        dw = dw.transpose(1, 2).contiguous().transpose(1, 2)
    got_lens, kept = ra.paged_evict(k, v, table, dl, dw, budget, first=first, recent=recent, **scales)
    torch.cuda.synchronize()
    assert got_lens.dtype == torch.int32 and kept.shape == (len(lens), hkv, budget)
    parts = {"k": (k, pool.k), "v": (v, pool.v), "w": (dw, w)}
    if i8:
        parts.update(ks=(scales["key_scale"], pool.ks), vs=(scales["value_scale"], pool.vs))
    want = {n: x[1].clone() for n, x in parts.items()}
    free = torch.zeros(pool.pages, page, dtype=torch.bool)  # behind the new lengths
    for b, n in enumerate(lens):
        n = max(0, n)
        m = min(n, budget)
        assert int(got_lens[b]) == m
        for h in range(hkv):
            pg, off = pool.where(b, torch.arange(n))
            keep = chosen(w[pg, off, h], budget, first, recent)
            assert kept[b, h].tolist() == keep + [-1] * (budget - m), f"{name} sequence {b} head {h}"
            src, dst = pool.where(b, keep), pool.where(b, torch.arange(m))
            for part in want.values():
                part[dst[0], dst[1], h] = part[src[0], src[1], h].clone()
        if n > m:
            free[pool.where(b, torch.arange(m, n))] = True
    for n, (got, _) in parts.items():
        a, z = got.cpu()[~free], want[n][~free]
        assert torch.equal(a.nan_to_num(nan=7.5) if a.is_floating_point() else a,
                           z.nan_to_num(nan=7.5) if z.is_floating_point() else z), f"{name}: {n}"
    log(f"[paged evict] {name}")


@pytest.mark.parametrize("dtype,i8,d", [(F16, False, 128), (BF16, False, 64), (F16, False, 32), (BF16, False, 96),
                                        (F16, False, 256), (F16, True, 128), (BF16, True, 64)])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "kv"])
def test_types(gpu, dtype, i8, d, layout):
    run(gpu, [5, 130, 0, 64, 65, 400], 3, d, dtype, i8, 64, first=4, recent=16, layout=layout, name=f"{dtype} {i8} {d}")


@pytest.mark.parametrize("budget,first,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (10, 4, 6), (10, 10, 0), (10, 0, 10),
                                                 (63, 0, 0), (64, 3, 0), (199, 7, 100), (200, 0, 5), (201, 0, 0), (300, 1, 1)])
@pytest.mark.parametrize("page", [1, 16, 128])
def test_budgets(gpu, budget, first, recent, page):
    run(gpu, [200, 7, 201, 64], 2, 32, F16, False, budget, first, recent, page=page, name=f"{budget} {first} {recent}")


@pytest.mark.parametrize("kind", ["equal", "few values", "specials", "signs", "falling", "rising", "one bit"])
def test_ties_and_specials(gpu, kind):
    """Equal weights: those in front.  NaN is below -inf, -0 is 0."""

    def weights(pool, g):
        shape = (pool.pages, 16, 2)
        if kind == "equal":
            return torch.full(shape, 0.25)
        if kind == "few values":
            return torch.randint(0, 3, shape, generator=g).float()
        if kind == "specials":
            x = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-42, -1e-42, 3.4e38, -float("nan")])
            return x[torch.randint(0, 9, shape, generator=g)]
        if kind == "signs":
            return torch.randn(shape, generator=g)
        if kind == "one bit":  # in the lowest
            return (torch.randint(0, 2, shape, generator=g) + 0x3f800000).int().view(torch.float32)
        w = torch.zeros(shape)
        for b, n in enumerate(pool.lens):
            up = torch.arange(n).float()[:, None].expand(n, 2)
            w[pool.where(b, torch.arange(n))] = up if kind == "rising" else -up
        return w

    for budget, first, recent in ((50, 0, 0), (100, 10, 20), (299, 0, 0)):
        run(gpu, [300, 90, 1000], 2, 32, F16, False, budget, first, recent, weights=weights, name=kind)


@pytest.mark.parametrize("n,budget", [(9000, 3000), (34816, 1025), (40000, 20001)])
def test_long(gpu, n, budget):
    """Past the weights that fit the LDS, and more rows than are moved at once."""
    run(gpu, [n, 700], 1, 32, F16, False, budget, 4, 300, page=64, name=f"long {n} {budget}")


def test_many_sequences_and_heads(gpu):
    run(gpu, [(53 * b) % 300 for b in range(150)], 5, 32, BF16, False, 100, 2, 30, page=8, name="many")


@pytest.mark.parametrize("i8", [False, True])
def test_pages_outside_the_cache(gpu, i8):
    """Nothing moves from or to places without a page, and no other sequence is touched."""
    import rdnattention as ra

    pool = Pool([130, 200], 2, 64, 16, F16, i8, seed=3, extra_width=0)
    k, v, table, lens, scales = pool.on(gpu)
    table[0, 0], table[0, 3] = 2 ** 31 - 1, -1
    lens[0] = 2 ** 31 - 1  # taken as the table's
    w = torch.rand(pool.pages, 16, 2, device=gpu)
    got, kept = ra.paged_evict(k, v, table, lens, w, 100, first=4, recent=8, **scales)
    torch.cuda.synchronize()
    assert got.tolist() == [100, 100] and int(kept[0].max()) < table.shape[1] * 16
    other = pool.unused()
    assert torch.equal(k.cpu()[other], pool.k[other]) and torch.equal(v.cpu()[other], pool.v[other])


def test_again_and_graph(gpu):
    """Captured with the lengths, replayed; the second eviction goes on from the first."""
    import rdnattention as ra

    pool = Pool([500, 40, 301], 2, 64, 16, F16, seed=5)
    k, v, table, lens, _ = pool.on(gpu)
    w = torch.rand(pool.pages, 16, 2, device=gpu)
    start = k.clone(), v.clone(), w.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, kept = ra.paged_evict(k, v, table, lens, w, 128, first=4, recent=32)
        got2, kept2 = ra.paged_evict(k, v, table, got, w, 100, first=4, recent=32)
    for rep in range(3):
        lens.sub_(rep)
        for x, y in zip((k, v, w), start):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        ek, ev, ew = (x.clone() for x in start)
        a, b = ra.paged_evict(ek, ev, table, lens, ew, 128, first=4, recent=32)
        c, d = ra.paged_evict(ek, ev, table, a, ew, 100, first=4, recent=32)
        torch.cuda.synchronize()
        for x, y in ((got, a), (kept, b), (got2, c), (kept2, d), (k, ek), (v, ev), (w, ew)):
            assert torch.equal(x, y), f"replay {rep}"
        # the same as keeping 100 at once, where the budget is what differs
        fk, fv, fw = (x.clone() for x in start)
        e, f = ra.paged_evict(fk, fv, table, lens, fw, 100, first=4, recent=32)
        assert torch.equal(e, c) and torch.equal(b.gather(2, d.clamp(min=0).long()).where(d >= 0, d), f)


def test_offsets_past_32_bits(gpu):
    import rdnattention as ra

    pages, page, hkv, d = 140000, 16, 8, 128  # 4.6 GB each
    pool = Pool([200], hkv, d, page, F16, seed=17)
    k, v, table, lens, _ = pool.on(gpu)
    w = torch.rand(pool.pages, page, hkv, device=gpu)
    big_k, big_v = (torch.empty(pages, page, hkv, d, dtype=F16, device=gpu) for _ in range(2))
    big_w = torch.empty(pages, page, hkv, device=gpu)
    n = (200 + page - 1) // page
    far = torch.arange(pages - 1, pages - 1 - n, -1, dtype=torch.int32, device=gpu)[None]
    near = pool.table[0, :n].to(gpu).long()
    big_k[far[0].long()], big_v[far[0].long()], big_w[far[0].long()] = k[near], v[near], w[near]
    a = ra.paged_evict(k, v, table, lens, w, 90, recent=10)
    b = ra.paged_evict(big_k, big_v, far, lens, big_w, 90, recent=10)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    use = slice(0, 5)  # whole pages of the 90
    assert torch.equal(big_k[far[0, use].long()], k[near[use]]) and torch.equal(big_v[far[0, use].long()], v[near[use]])
    assert torch.equal(big_w[far[0, use].long()], w[near[use]])

"""paged_key_weights against its formula in 64 bits: every type and head dim, ragged rows,
masks, rows that see nothing, what the pages and old weights hold, graphs."""
import math

import pytest
import torch

from tests.gpu_util import log
from tests.paged_util import Pool, visible

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
TYPES = [(F16, False), (BF16, False), (F16, True), (BF16, True)]


def reference(q, lse, k, ok, scale, i8):
    """(sum over rows and heads of exp(score - lse) [len, hkv], its bound) in 64 bits.  A
    weight is off, relative to itself, by its score's error ((d + 2) 2^-24 of the sum of the
    products' magnitudes, and 2^-22 of that in the exponent; int8 2^-23 more) and by 2^-21
    each of the exponential and of the factor that holds the rest of lse; n of them are
    summed in 32 bits in four chains for each of 16 rows, at worst n / 16 + 8 roundings."""
    n, hq, d = q.shape
    length, hkv, _ = k.shape
    out = torch.zeros(length, hkv, dtype=torch.float64)
    tol = torch.full((length, hkv), 1e-30, dtype=torch.float64)
    for h in range(hq):
        kv = h // (hq // hkv)
        kh = k[:, kv]
        s = q[:, h].double() @ kh.t() * scale
        mag = q[:, h].double().abs() @ kh.abs().t() * abs(scale)
        p = torch.exp(s - lse[:, h, None].double()).masked_fill(~ok | (lse[:, h, None] == -math.inf), 0.0)
        out[:, kv] += p.sum(0)
        ds = mag * ((d + 2) * 2.0 ** -24 + 2.0 ** -22 + (2.0 ** -23 if i8 else 0.0)) + 2.0 ** -20
        tol[:, kv] += (p * ds).sum(0)
    return out, tol + out * (n * (hq // hkv) / 16 + 8) * 2.0 ** -24


def run(gpu, lens, ns, hq, hkv, d, dtype, i8=False, page=16, causal=True, window=-1, scale=None, decay=1.0, seed=1,
        pad=0, uniform=False, max_q=None, layout="nhd", spoil=False, lse=None, old=None, name=""):
    import rdnattention as ra

    pool = Pool(lens, hkv, d, page, dtype, i8, seed=seed, layout=layout)
    if spoil:
        unused = pool.unused()
        if i8:
            pool.ks[unused] = float("nan")
        else:
            pool.k[unused] = float("nan")
    g = torch.Generator().manual_seed(seed)
    rows = sum(ns) + pad
    q = torch.randn(rows, hq + 2, d, generator=g).to(dtype)[:, 1:1 + hq]  # a view
    k, _, table, dl, scales = pool.on(gpu)
    sc = d ** -0.5 if scale is None else scale
    if lse is None:
        lse = torch.zeros(rows, hq)
        at = 0
        for b, n in enumerate(ns):
            length = max(0, lens[b])
            kk = pool.rows(b, length)[0]
            ok = visible(n, length, causal, window)
            for h in range(hq):
                s = (q[at:at + n, h].double() @ kk[:, h // (hq // hkv)].t() * sc).masked_fill(~ok, -math.inf)
                lse[at:at + n, h] = torch.logsumexp(s, -1).float()
            at += n
    w = torch.rand(pool.pages, page, hkv, generator=g) if old is None else old(pool)
    dw = w.to(gpu)
    if layout == "hnd":
        dw = dw.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "kv":
        dw = torch.stack((dw, dw), 1)[:, 1]
    kw = {}
    if not uniform:
        kw["cu_seqlens_q"] = torch.tensor([sum(ns[:i]) for i in range(len(ns) + 1)], dtype=torch.int32, device=gpu)
        kw["max_seqlen_q"] = max_q
    assert ra.paged_key_weights(q.to(gpu), lse.to(gpu), k, table, dl, dw, is_causal=causal, window_size=window,
                                scale=scale, key_scale=scales.get("key_scale"), decay=decay, **kw) is None
    torch.cuda.synchronize()
    got = dw.cpu()
    rest = torch.ones(pool.pages, page, dtype=torch.bool)
    at, worst = 0, 0.0
    for b, n in enumerate(ns):
        length = max(0, lens[b])
        if n and length:
            want, tol = reference(q[at:at + n], lse[at:at + n], pool.rows(b, length)[0], visible(n, length, causal, window),
                                  sc, i8)
            pg, off = pool.where(b, torch.arange(length))
            rest[pg, off] = False
            before = torch.where((torch.arange(length) < length - n)[:, None] & (decay != 0.0),
                                 w[pg, off].double() * decay, torch.zeros_like(want))
            want, tol = want + before, tol + 2.0 ** -23 * before.abs()
            x = got[pg, off].double()
            assert torch.isfinite(x).all(), f"{name} sequence {b}"
            worst = max(worst, float(((x - want).abs() / tol).max()))
            assert worst <= 1.0, f"{name} sequence {b}: {worst:.3f} of the bound"
        at += n
    assert torch.equal(got[rest].nan_to_num(), w[rest].nan_to_num())
    log(f"[paged weights] {name}: {worst:.3f} of the bound")
    return got


@pytest.mark.parametrize("dtype,i8", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_decode(gpu, dtype, i8, d):
    run(gpu, [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 700, 1111], [1] * 13, 8, 2, d, dtype, i8, uniform=True, seed=d,
        name=f"decode {dtype} {i8} {d}")


@pytest.mark.parametrize("dtype,i8", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_prompts(gpu, dtype, i8, d):
    lens = [1, 40, 64, 65, 333, 600]
    run(gpu, lens, lens, 8, 2, d, dtype, i8, seed=d + 1, name=f"prompts {dtype} {i8} {d}")
    run(gpu, [900, 300, 97], [64, 64, 64], 8, 2, d, dtype, i8, uniform=True, decay=0.5, seed=d + 2, name="last rows")


@pytest.mark.parametrize("d", [32, 96, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_head_dims(gpu, d, dtype):
    run(gpu, [5, 130, 400], [1] * 3, 6, 2, d, dtype, page=32, uniform=True, seed=d, name=f"decode {d}")
    run(gpu, [5, 130, 400], [5, 100, 150], 6, 2, d, dtype, page=32, seed=d, name=f"chunks {d}")


@pytest.mark.parametrize("page", [1, 4, 8, 64, 1024])
@pytest.mark.parametrize("i8", [False, True])
def test_pages(gpu, page, i8):
    run(gpu, [7, 90, 261], [1] * 3, 4, 2, 64, F16, i8, page=page, uniform=True, spoil=True, name=f"page {page}")
    run(gpu, [7, 90, 261], [7, 50, 200], 4, 2, 64, F16, i8, page=page, spoil=True, name=f"chunks, page {page}")


@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (32, 1), (40, 1), (64, 2), (24, 8)])
@pytest.mark.parametrize("layout", ["hnd", "kv"])
def test_heads_and_layouts(gpu, hq, hkv, layout):
    run(gpu, [200, 77], [1, 1], hq, hkv, 64, F16, uniform=True, layout=layout, name=f"heads {hq}/{hkv}")
    run(gpu, [200, 77], [9, 77], hq, hkv, 64, F16, layout=layout, name=f"chunks {hq}/{hkv}")


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [-1, 1, 17, 100, 5000, 2 ** 31 - 1])
def test_mixed_batches_and_masks(gpu, i8, causal, window):
    """Single tokens, chunks and prompts, sequences without rows and without keys, more rows
    than keys, padding."""
    lens = [700, 0, 1, 300, 64, 512, 129, 3, 33]
    ns = [1, 0, 1, 300, 3, 0, 100, 5, 33]
    for most in (None, 300):
        run(gpu, lens, ns, 8, 2, 64, F16, i8, causal=causal, window=window, pad=5, max_q=most, decay=0.25,
            name=f"mixed {causal} {window}")
    run(gpu, [300, 129, 64, 3], [1] * 4, 4, 2, 64, F16, i8, causal=causal, window=window, uniform=True, name="decode")


@pytest.mark.parametrize("max_q", [0, 1, 8])
def test_more_rows_than_max_seqlen_q(gpu, max_q):
    run(gpu, [300, 9, 700, 64] + [200] * 30, [150, 3, 40, 64] + [33] * 30, 8, 2, 64, F16, max_q=max_q, name="more rows")


def test_many_sequences(gpu):
    lens = [(37 * b) % 150 for b in range(200)]
    ns = [0 if b % 7 == 3 else min(1, lens[b]) for b in range(200)]
    run(gpu, lens, ns, 4, 1, 32, F16, page=8, pad=2, name="200 sequences")
    ns = [min(lens[b], 40) if b % 5 == 0 else n for b, n in enumerate(ns)]
    run(gpu, lens, ns, 4, 1, 32, F16, page=8, name="200 sequences, chunks among them")


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
def test_scales(gpu, scale):
    run(gpu, [90, 200], [1, 1], 4, 2, 64, F16, scale=scale, uniform=True, name=f"scale {scale}")
    run(gpu, [90, 200], [90, 60], 4, 2, 64, F16, scale=scale, name=f"scale {scale}")


@pytest.mark.parametrize("ns", [[1, 1, 1], [30, 70, 64]])
def test_old_weights(gpu, ns):
    """New keys' old weights are not read, with decay 0 none: NaN there leaves no trace."""

    def new_are_nan(pool):
        w = torch.rand(pool.pages, 16, 2)
        for b, n in enumerate(ns):
            w[pool.where(b, torch.arange(pool.lens[b] - n, pool.lens[b]))] = float("nan")
        return w

    lens = [200, 70, 300]
    run(gpu, lens, ns, 8, 2, 64, F16, old=new_are_nan, decay=0.9, name="new keys")
    run(gpu, lens, ns, 8, 2, 64, F16, old=lambda p: torch.full((p.pages, 16, 2), float("nan")), decay=0.0, name="decay 0")


@pytest.mark.parametrize("ns", [[1, 1], [40, 66]])
def test_rows_that_add_nothing(gpu, ns):
    """lse of -inf (the row sees nothing) and of +inf."""
    for x in (-math.inf, math.inf):
        lse = torch.full((sum(ns), 8), x)
        run(gpu, [100, 90], ns, 8, 2, 64, F16, lse=lse, decay=0.5, name=f"lse {x}")
    lse = torch.randn(sum(ns), 8) + 4
    lse[0, 3], lse[-1, 0] = -math.inf, math.inf
    run(gpu, [100, 90], ns, 8, 2, 64, F16, lse=lse, name="lse of some")


@pytest.mark.parametrize("ns", [[1, 1, 1], [70, 64, 70]])
@pytest.mark.parametrize("i8", [False, True])
def test_pages_outside_the_cache(gpu, ns, i8):
    """A table entry that is no page leads nowhere, and touches no other sequence."""
    import rdnattention as ra

    pool = Pool([70, 64, 130], 2, 64, 16, F16, i8, seed=14, extra_width=0)
    k, _, table, lens, scales = pool.on(gpu)
    cu = torch.tensor([0, ns[0], ns[0] + ns[1], sum(ns)], dtype=torch.int32, device=gpu)
    q = torch.randn(sum(ns), 4, 64, device=gpu).half()
    lse = torch.full((sum(ns), 4), 4.0, device=gpu)
    kw = dict(cu_seqlens_q=cu, key_scale=scales.get("key_scale"))
    good = torch.rand(pool.pages, 16, 2, device=gpu)
    bad = good.clone()
    before = good.clone()
    ra.paged_key_weights(q, lse, k, table, lens, good, **kw)
    table[1, 0], table[1, 2] = 2 ** 31 - 1, -1
    far = lens.clone()
    far[1] = 2 ** 31 - 1
    ra.paged_key_weights(q, lse, k, table, far, bad, **kw)
    torch.cuda.synchronize()
    for b in range(3):
        pg, off = (i.to(gpu) for i in pool.where(b, torch.arange(pool.lens[b])))
        if b != 1:
            # other lengths are other shares: the same weights, none negative, summed in another
            # order, each order off by at most (rows x heads / 16 + 8) 2^-24 (see reference)
            off_by = 2 * (ns[b] * 2 / 16 + 8) * 2.0 ** -24 * good[pg, off]
            assert ((bad[pg, off] - good[pg, off]).abs() <= off_by).all()
        else:
            gone = (torch.arange(64, device=gpu) // 16 == 0) | (torch.arange(64, device=gpu) // 16 == 2)
            assert torch.equal(bad[pg, off][gone], before[pg, off][gone])
    other = pool.unused().to(gpu)
    assert torch.equal(bad[other], before[other])


def test_a_key_that_is_not_finite_reaches_no_other(gpu):
    import rdnattention as ra

    pool = Pool([300], 2, 64, 16, F16, seed=15)
    pg, off = pool.where(0, [77])
    pool.k[pg, off, 1] = float("inf")
    k, _, table, lens, _ = pool.on(gpu)
    for n in (1, 40):
        q = torch.randn(n, 8, 64, device=gpu).half()
        w = torch.zeros(pool.pages, 16, 2, device=gpu)
        ra.paged_key_weights(q, torch.full((n, 8), 4.0, device=gpu), k, table, lens, w)
        bad = torch.zeros_like(w, dtype=torch.bool)
        bad[pg.to(gpu), off.to(gpu), 1] = True
        assert torch.isfinite(w[~bad]).all()


def test_with_the_attention(gpu):
    """With paged_attention's lse every row's weights sum to 1: of all keys rows x heads.  Each
    weight is good to 2^-14 relative here (scores below 2^6 in 32 bits, 2^-18 of the lse)."""
    import rdnattention as ra

    lens, ns = [900, 40, 333], [1, 40, 70]
    pool = Pool(lens, 2, 128, 16, BF16, seed=16)
    k, v, table, dl, _ = pool.on(gpu)
    q = torch.randn(sum(ns), 8, 128, device=gpu).bfloat16()
    cu = torch.tensor([0, 1, 41, 111], dtype=torch.int32, device=gpu)
    _, lse = ra.paged_attention(q, k, v, table, dl, cu_seqlens_q=cu, return_lse=True)
    w = torch.full((pool.pages, 16, 2), 5.0, device=gpu)
    ra.paged_key_weights(q, lse, k, table, dl, w, cu_seqlens_q=cu, decay=0.0)
    for b, n in enumerate(ns):
        pg, off = (i.to(gpu) for i in pool.where(b, torch.arange(lens[b])))
        total = w[pg, off].double().sum(0)
        assert ((total - n * 4).abs() <= n * 4 * 2.0 ** -14).all()


@pytest.mark.parametrize("ns", [[1] * 4, [1, 500, 1, 40]])
def test_graph_and_same_bits(gpu, ns):
    import rdnattention as ra

    pool = Pool([900, 600, 64, 333], 2, 64, 16, F16, seed=20)
    k, _, table, lens, _ = pool.on(gpu)
    q = torch.randn(sum(ns), 8, 64, device=gpu).half()
    lse = torch.full((sum(ns), 8), 6.0, device=gpu)
    cu = torch.tensor([sum(ns[:i]) for i in range(5)], dtype=torch.int32, device=gpu)
    start = torch.rand(pool.pages, 16, 2, device=gpu)
    w = start.clone()

    def call(x):
        ra.paged_key_weights(q, lse, k, table, lens, x, cu_seqlens_q=cu, max_seqlen_q=max(ns), decay=0.5)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(w)
    for rep in range(4):
        q.copy_(torch.randn(q.shape, device=gpu))
        lens.copy_(torch.tensor([900 - 100 * rep, 600, 64 - rep, 333], dtype=torch.int32))
        w.copy_(start)
        torch.cuda.synchronize()
        graph.replay()
        eager = start.clone()
        call(eager)
        torch.cuda.synchronize()
        assert torch.equal(w, eager), f"replay {rep}"
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = start.clone()
        call(again)
    side.synchronize()
    assert torch.equal(again, eager)


def test_offsets_past_32_bits(gpu):
    import rdnattention as ra

    pages, page, hkv, d = 140000, 16, 8, 128  # 4.6 GB
    pool = Pool([200], hkv, d, page, F16, seed=17)
    k, _, _, lens, _ = pool.on(gpu)
    big = torch.empty(pages, page, hkv, d, dtype=F16, device=gpu)
    n = (200 + page - 1) // page
    table = torch.arange(pages - 1, pages - 1 - n, -1, dtype=torch.int32, device=gpu)[None]
    for i in range(n):
        big[pages - 1 - i] = k[pool.table[0, i]]
    for rows in (1, 40):
        q = torch.randn(rows, 32, d, device=gpu).half()
        lse = torch.full((rows, 32), 5.0, device=gpu)
        a, b = torch.zeros(pool.pages, page, hkv, device=gpu), torch.zeros(pages, page, hkv, device=gpu)
        ra.paged_key_weights(q, lse, k, pool.table.to(gpu), lens, a)
        ra.paged_key_weights(q, lse, big, table, lens, b)
        assert torch.equal(b[table[0].long()], a[pool.table[0, :n].to(gpu).long()])


@pytest.mark.parametrize("dtype,i8", TYPES)
@pytest.mark.parametrize("window", [-1, 50])
def test_between_one_row_tile_and_many(gpu, dtype, i8, window):
    ns = [8, 9, 16, 17, 31, 32, 33, 40]  # with 4 heads of a kv head: 32 to 160 rows
    lens = [300, 9, 700, 64, 31, 1000, 333, 50]
    run(gpu, lens, ns, 8, 2, 64, dtype, i8, window=window, name=f"mixed rows {dtype} {i8}")
    for n in (9, 32, 33):
        run(gpu, lens, [n] * len(lens), 8, 2, 64, dtype, i8, window=window, uniform=True, name=f"{n} rows {dtype} {i8}")

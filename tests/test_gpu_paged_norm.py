"""paged_append with norms and positions of several axes, against the formulas in
64 bits: every head dim and type, partial rotations, ragged and strided rows, rows
without a place, int8 pages bit for bit, graphs and streams."""
import pytest
import torch

from tests.gpu_util import log
from tests.paged_util import Pool, rope_tables

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def normed(x, w, eps):
    x = x.double()
    if w is None:
        return x
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def turned(x, cos, sin, pairs):
    """x [rows, heads, d] rotated by cos and sin [rows, c], and the size of the two
    products that each channel is a sum of."""
    y, size, m = x.clone(), x.abs(), cos.shape[-1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = (slice(0, 2 * m, 2), slice(1, 2 * m, 2)) if pairs else (slice(0, m), slice(m, 2 * m))
    u, v = x[..., a], x[..., b]
    y[..., a], size[..., a] = u * c - v * s, (u * c).abs() + (v * s).abs()
    y[..., b], size[..., b] = u * s + v * c, (u * s).abs() + (v * c).abs()
    return y, size


def check_near(got, want, size, dtype, name=""):
    """In 32 bits: a sum of d squares in a tree of at most 14 roundings of 2^-24 each
    (halved by the root), the division by d, eps, root and reciprocal at most 2^-23 each,
    the products with r and w 2^-24 each: 7 + 8 + 2 = 17 of 2^-24 before the rotation,
    whose two products and sum add 3 of each product; then half a step of the type
    (fp16's subnormals: 2^-25)."""
    got = got.cpu().double()
    tol = torch.finfo(dtype).eps / 2 * 1.001 * want.abs() + 20 * 2.0 ** -24 * size + 2.0 ** -25
    over = ((got - want).abs() / tol).max() if want.numel() else torch.zeros(())
    assert torch.isfinite(got).all() and over <= 1.0, f"{name}: {float(over):.3f} of the bound"


def rounded(x, dtype):
    """64-bit values rounded once to dtype.  (torch rounds them to 32 bits first, which
    moves a value just beside the middle between two of dtype's onto it, and then to the
    even one: of bf16 about one in 2^17.)"""
    y = x.to(dtype)
    bits = y.view(torch.int16)
    best, gap = y, (y.double() - x).abs()
    for step in (-1, 1):
        z = (bits + step).view(dtype)
        far = (z.double() - x).abs()
        nearer = torch.isfinite(z) & ((far < gap) | (far == gap) & (bits % 2 != 0))
        best, gap = torch.where(nearer, z, best), torch.where(nearer, far, gap)
    return best


def whole(x, dtype):
    """(int8 rows, scales) of rows that were rounded to dtype."""
    x = rounded(x.double(), dtype).float()
    s = x.abs().amax(-1) * torch.tensor(1.0 / 127.0)
    s = torch.where(s == 0, torch.ones_like(s), s)
    return torch.clamp(torch.round(x / s[..., None]), -127, 127).to(torch.int8), s


def run(gpu, lens, ns, hq, hkv, d, dtype, i8=False, pairs=True, cols=None, axes=0, norms="qk", wtype=torch.float32,
        eps=1e-6, pad=0, seed=0, rot_rows=None, layout="nhd", name=""):
    import rdnattention as ra

    g = torch.Generator().manual_seed(seed)
    ragged = pad > 0 or len(set(ns)) > 1
    pool = Pool(lens, hkv, d, 16, dtype, i8, seed=seed, layout=layout)
    rows = sum(ns) + pad
    scale = torch.rand(rows, hq + 2 * hkv, 1, generator=g) * 3 + 0.05
    fused = (torch.randn(rows, hq + 2 * hkv, d, generator=g) * scale).to(dtype)  # one projection's output
    if rows > 1:
        fused[1, 0] = 0  # a head of zeros
    q, k, v = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]
    qw, kw_ = ((1 + 0.5 * torch.randn(d, generator=g)).to(wtype) for _ in range(2))
    qw, kw_ = (qw if "q" in norms else None), (kw_ if "k" in norms else None)
    seq = [b for b, n in enumerate(ns) for _ in range(n)]
    idx = torch.tensor([lens[b] - n + i for b, n in enumerate(ns) for i in range(n)] + [-1] * pad)
    cols = d // 2 if cols is None else cols
    rot_rows = rot_rows or max(lens) + 40
    cos, sin = rope_tables(rot_rows, max(cols, 1))
    df = fused.to(gpu)
    kc, vc, table, dl, kw = pool.on(gpu)
    kw = dict(kw, query=df[:, :hq] if "q" in norms or cols else None, norm_eps=eps,
              query_norm=None if qw is None else qw.to(gpu), key_norm=None if kw_ is None else kw_.to(gpu))
    if ragged:
        kw["cu_seqlens_q"] = torch.tensor([sum(ns[:i]) for i in range(len(ns) + 1)], dtype=torch.int32, device=gpu)
    pos = None
    if cols:
        kw.update(rot_cos=cos.to(gpu), rot_sin=sin.to(gpu), rot_interleaved=pairs)
        if axes:
            # some outside the tables and the axes
            pos = torch.randint(-2, rot_rows + 2, (rows, axes), generator=g, dtype=torch.int32)
            axis = torch.randint(-1, axes + 1, (cols,), generator=g, dtype=torch.int32)
            kw.update(positions=pos.to(gpu), rot_axes=axis.to(gpu))
    got = ra.paged_append(df[:, hq:hq + hkv], df[:, hq + hkv:], kc, vc, table, dl, **kw)
    torch.cuda.synchronize()

    live = torch.arange(rows) < sum(ns)
    placed = live & (idx >= 0)
    turns = live if pos is not None else placed

    def want(x, w):
        y = x.double().clone()
        y[live] = normed(x[live], w, eps)
        size = y.abs()
        if cols:
            at = (pos.long()[:, axis.long().clamp(0, axes - 1)] if pos is not None else idx[:, None].expand(-1, cols))
            at = at.clamp(0, rot_rows - 1)
            z, zs = turned(y, cos.gather(0, at), sin.gather(0, at), pairs)
            y[turns], size[turns] = z[turns], zs[turns]
        return y, size

    wq, sq = want(q, qw)
    if kw["query"] is not None:
        check_near(got, wq, sq, dtype, name + " queries")
        assert torch.equal(got[~live.to(gpu)].cpu(), q[~live])  # padding comes out as it is
    else:
        assert got is None
    wk, sk = want(k, kw_)
    rest = torch.ones(pool.pages, 16, dtype=torch.bool)
    kc, vc = kc.cpu(), vc.cpu()
    at = [pool.where(seq[r], [int(idx[r])]) for r in torch.nonzero(placed).flatten().tolist()]
    pg, off = (torch.cat(x) for x in zip(*at)) if at else (torch.zeros(0, dtype=torch.long),) * 2
    rest[pg, off] = False
    assert torch.equal(kc[rest], pool.k[rest]) and torch.equal(vc[rest], pool.v[rest])
    if i8:
        ks, vs = kw["key_scale"].cpu(), kw["value_scale"].cpu()
        assert torch.equal(ks[rest], pool.ks[rest]) and torch.equal(vs[rest], pool.vs[rest])
        for cache, sc, w in ((kc, ks, wk), (vc, vs, v)):
            ints, s = whole(w[placed], dtype)
            assert torch.equal(sc[pg, off], s) and torch.equal(cache[pg, off], ints)
    else:
        check_near(kc[pg, off], wk[placed], sk[placed], dtype, name + " keys")
        assert torch.equal(vc[pg, off], v[placed])
    log(f"[paged norm] {name} {dtype} {i8} {d}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("pairs", [True, False])
def test_head_dims(gpu, dtype, d, pairs):
    run(gpu, [5, 40, 17], [2, 2, 2], 6, 3, d, dtype, pairs=pairs, seed=d, name="uniform")
    run(gpu, [5, 40, 0, 17, 100, 3], [5, 1, 0, 17, 33, 4], 5, 1, d, dtype, pairs=pairs, pad=3, axes=3, seed=d + 1,
        name="ragged, three axes, a row without a place")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("axes", [0, 1, 4])
def test_int8_pages(gpu, dtype, d, pairs, axes):
    run(gpu, [5, 40, 0, 17, 100, 3], [5, 1, 0, 17, 33, 4], 6, 3, d, dtype, True, pairs=pairs, axes=axes, pad=4, seed=d,
        name="int8")


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("pairs", [True, False])
def test_many_rows(gpu, i8, pairs):
    """Calls large enough for several heads per group of lanes, an odd number of heads."""
    run(gpu, [700, 900, 1, 400], [700, 333, 1, 400], 33, 3, 128, F16, i8, pairs=pairs, axes=2, pad=1, seed=3, name="many")
    run(gpu, [1500], [1500], 40, 5, 64, BF16, i8, pairs=pairs, seed=4, name="many, one sequence")


@pytest.mark.parametrize("norms", ["q", "k", "qk"])
@pytest.mark.parametrize("cols", [0, 8, 32])
@pytest.mark.parametrize("pairs", [True, False])
def test_parts(gpu, norms, cols, pairs):
    """Norms of one of the two, no or a partial rotation, weights of the rows' type."""
    run(gpu, [40, 7], [3, 3], 4, 2, 96, F16, cols=cols, norms=norms, pairs=pairs, wtype=F16, name=f"{norms} {cols}")
    run(gpu, [40, 7], [3, 3], 4, 2, 128, BF16, cols=cols, norms=norms, pairs=pairs, wtype=BF16, axes=2 if cols else 0,
        eps=0.5, seed=1, name=f"{norms} {cols}")


@pytest.mark.parametrize("layout", ["hnd", "kv"])
def test_layouts(gpu, layout):
    run(gpu, [40, 7], [3, 3], 4, 2, 64, F16, layout=layout, name=layout)
    run(gpu, [40, 7], [3, 3], 4, 2, 64, F16, True, layout=layout, name=layout)


def test_axes_without_norms(gpu):
    """rot_axes alone; with the same position on all axes it is the plain rotation."""
    import rdnattention as ra

    run(gpu, [40, 7], [3, 3], 4, 2, 64, F16, axes=3, norms="", name="axes alone")
    pool = Pool([60], 2, 128, 16, F16, seed=1)
    q, k = torch.randn(50, 4, 128, device=gpu).half(), torch.randn(50, 2, 128, device=gpu).half()
    cos, sin = (t.to(gpu) for t in rope_tables(99, 64))
    pos = torch.randint(0, 99, (50,), dtype=torch.int32, device=gpu)
    axis = torch.randint(0, 3, (64,), dtype=torch.int32, device=gpu)
    out = []
    for kw in (dict(positions=pos), dict(positions=pos[:, None].expand(50, 3).contiguous(), rot_axes=axis),
               dict(positions=pos[:, None].expand(50, 1), rot_axes=torch.zeros_like(axis))):
        kc, vc, table, lens, _ = pool.on(gpu)
        x = ra.paged_append(k, k, kc, vc, table, lens, query=q, rot_cos=cos, rot_sin=sin, **kw)
        out.append((x.float(), kc.float()))
    # two products and a sum in 32 bits each, of values below 8, rounded to fp16 below 8
    for a in out[1:]:
        for x, y in zip(a, out[0]):
            assert y.abs().max() < 8 and (x - y).abs().max() <= 2.0 ** -8
    assert torch.equal(out[1][0], out[2][0])


def test_zero_rows_and_extreme_values(gpu):
    """A head of zeros stays zeros with eps > 0; a scaled head has the same norm; an
    infinite channel leaves the others of its head zero and is NaN itself."""
    import rdnattention as ra

    pool = Pool([4], 1, 64, 16, BF16, seed=1)
    kc, vc, table, lens, _ = pool.on(gpu)
    x = torch.randn(4, 1, 64, device=gpu).bfloat16()
    x[1] = 0
    x[2] = x[0] * 2.0 ** 40
    x[3, 0, 5] = float("inf")
    w = torch.ones(64, device=gpu)
    q = ra.paged_append(x, x, kc, vc, table, lens, query=x, query_norm=w, key_norm=w, norm_eps=1e-20).cpu()
    assert (q[1] == 0).all()
    # the same but for eps: r is off by 1e-20 / mean / 2 and 2^-23, which may move one rounding
    assert ((q[2].double() - q[0].double()).abs() <= 2.0 ** -7 * q[0].double().abs()).all()
    assert q[3, 0, 5].isnan() and (q[3, 0, :5] == 0).all() and (q[3, 0, 6:] == 0).all()
    pg, off = (i.to(gpu) for i in pool.where(0, torch.arange(4)))
    assert torch.equal(torch.nan_to_num(kc[pg, off]).cpu(), torch.nan_to_num(q))


def test_graph_and_stream(gpu):
    """A captured append, replayed with other rows, lengths and positions."""
    import rdnattention as ra

    pool = Pool([50, 60], 2, 128, 16, F16, seed=1)
    kc, vc, table, lens, _ = pool.on(gpu)
    cos, sin = (t.to(gpu) for t in rope_tables(200, 64))
    x = torch.randn(2, 8, 128, device=gpu).half()
    pos = torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    kw = dict(query=x[:, :4], rot_cos=cos, rot_sin=sin, rot_interleaved=False, positions=pos,
              rot_axes=torch.arange(64, dtype=torch.int32, device=gpu) % 3, query_norm=torch.rand(128, device=gpu),
              key_norm=torch.rand(128, device=gpu))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = ra.paged_append(x[:, 4:6], x[:, 6:], kc, vc, table, lens, **kw)
    for i in range(3):
        x.copy_(torch.randn(2, 8, 128, device=gpu))
        pos.copy_(torch.randint(0, 200, (2, 3), device=gpu))
        lens.sub_(1)
        before = kc.clone(), vc.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = ra.paged_append(x[:, 4:6], x[:, 6:], *before, table, lens, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = ra.paged_append(x[:, 4:6], x[:, 6:], kc, vc, table, lens, **kw)
    other.synchronize()
    assert torch.equal(again, want)


def test_queries_normed_in_place(gpu):
    """The C ABI with query_out == query."""
    import rdnattention as ra
    from rdnattention import paged

    for d in (64, 96, 256):
        pool = Pool([400], 1, d, 16, F16, seed=d)
        kc, vc, table, lens, _ = pool.on(gpu)
        cos, sin = (t.to(gpu) for t in rope_tables(500, d // 2))
        q = torch.randn(400, 7, d, device=gpu).half()
        x = torch.randn(400, 1, d, device=gpu).half()
        w = torch.rand(d, device=gpu)
        want = ra.paged_append(x, x, kc, vc, table, lens, query=q, rot_cos=cos, rot_sin=sin, rot_interleaved=False,
                               query_norm=w)
        c = paged._cache(kc, vc, table, lens, "seq_lens", None, None, None, 400)[0]
        norm = paged._NORM.pack(w.data_ptr(), 0, 0, 1, 0, 1e-6, 3)
        rc = paged._lib.rdna_paged_append_norm(
            c, norm, x.data_ptr(), x.data_ptr(), *x.stride()[:2], *x.stride()[:2], 400, 0, q.data_ptr(), q.data_ptr(),
            *q.stride()[:2], *q.stride()[:2], 7, None, cos.data_ptr(), sin.data_ptr(), 500, d, 0,
            torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0, ra.last_error()
        assert torch.equal(q, want)

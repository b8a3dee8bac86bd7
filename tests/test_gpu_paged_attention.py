"""paged_attention and paged_tree_attention against their definitions in 64
bits: every type and head dim, ragged and empty sequences, pages that end
inside tiles, windows, trees, what the pages hold where no key is, views and
far offsets, streams and graphs."""
import pytest
import torch

from tests.gpu_util import log
from tests.paged_util import Pool, check, reference, visible

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def run(gpu, pool, ns, hq, *, causal=True, window=-1, tree=None, scale=None, seed=1, pad=0, uniform=False, qview=False,
        out=None, max_q=None, name=""):
    """The call and its reference on `pool`, with ns[b] new rows per sequence.
    Returns the output."""
    import rdnattention as ra

    g = torch.Generator().manual_seed(seed)
    rows = sum(ns) + pad
    q = torch.randn(rows, hq, pool.d, generator=g).to(pool.dtype)
    if qview:  # a slice of a fused projection
        wide = torch.randn(rows, hq + 4, pool.d, generator=g).to(pool.dtype)
        wide[:, 2:2 + hq] = q
        dq = wide.to(gpu)[:, 2:2 + hq]
    else:
        dq = q.to(gpu)
    k, v, table, lens, scales = pool.on(gpu)
    kw = dict(scales, scale=scale, out=out)
    if not uniform:
        cu = [0]
        for n in ns:
            cu.append(cu[-1] + n)
        kw["cu_seqlens_q"] = torch.tensor(cu, dtype=torch.int32, device=gpu)
        if max_q is not None:
            kw["max_seqlen_q"] = max_q
    if tree is not None:
        got = ra.paged_tree_attention(dq, k, v, table, lens, tree.to(gpu), **kw)
    else:
        got = ra.paged_attention(dq, k, v, table, lens, is_causal=causal, window_size=window, **kw)
    torch.cuda.synchronize()
    at = 0
    worst = 0.0
    for b, n in enumerate(ns):
        length = max(0, pool.lens[b])
        kk, vv = pool.rows(b, length)
        ok = visible(n, length, causal, window, None if tree is None else tree[b])
        want, tol = reference(q[at:at + n], kk, vv, ok, pool.d ** -0.5 if scale is None else scale, pool.dtype, pool.i8)
        worst = max(worst, check(got[at:at + n], want, tol, f"{name} sequence {b}") if n else 0.0)
        at += n
    if pad and out is None:
        assert (got[at:] == 0).all()
    log(f"[paged attention] {name}: {worst:.3f} of the bound")
    return got


TYPES = [(F16, False), (BF16, False), (F16, True), (BF16, True)]


@pytest.mark.parametrize("dtype,i8", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_decode(gpu, dtype, i8, d):
    pool = Pool([1, 2, 31, 32, 33, 63, 64, 65, 255, 256, 257, 700, 1111], 2, d, 16, dtype, i8, seed=d)
    run(gpu, pool, [1] * 13, 8, uniform=True, name=f"decode {dtype} {i8} {d}")


@pytest.mark.parametrize("dtype,i8", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_prompts(gpu, dtype, i8, d):
    lens = [1, 40, 64, 65, 333, 600]
    pool = Pool(lens, 2, d, 16, dtype, i8, seed=d + 1)
    run(gpu, pool, lens, 8, name=f"prompts {dtype} {i8} {d}")


@pytest.mark.parametrize("d", [32, 96, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_head_dims(gpu, d, dtype):
    pool = Pool([5, 130, 400], 2, d, 32, dtype, seed=d)
    run(gpu, pool, [1, 1, 1], 6, uniform=True, name=f"decode {d} {dtype}")
    run(gpu, pool, [5, 100, 150], 6, name=f"chunks {d} {dtype}")


@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 64, 128, 1024])
@pytest.mark.parametrize("i8", [False, True])
def test_page_sizes(gpu, page, i8):
    pool = Pool([7, 90, 261], 2, 64, page, F16, i8, seed=page)
    run(gpu, pool, [1, 1, 1], 4, uniform=True, name=f"decode page {page}")
    run(gpu, pool, [7, 50, 200], 4, name=f"chunks page {page}")


@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 5), (7, 1), (24, 8), (32, 1), (40, 1), (64, 2)])
def test_heads(gpu, hq, hkv):
    pool = Pool([200, 77], hkv, 64, 16, F16, seed=hq)
    run(gpu, pool, [1, 1], hq, uniform=True, name=f"decode heads {hq}/{hkv}")
    run(gpu, pool, [9, 77], hq, name=f"chunks heads {hq}/{hkv}")


@pytest.mark.parametrize("i8", [False, True])
def test_mixed_batch(gpu, i8):
    """Single tokens, chunks and whole prompts in one call, sequences without
    rows and without keys between them, padding behind them."""
    lens = [700, 0, 1, 300, 64, 512, 129, 2000, 33]
    ns = [1, 0, 1, 300, 3, 0, 100, 1, 33]
    pool = Pool(lens, 2, 64, 16, F16, i8, seed=5)
    run(gpu, pool, ns, 8, pad=5, name="mixed")
    run(gpu, pool, ns, 8, pad=5, max_q=300, name="mixed, longest known")


def test_many_sequences(gpu):
    """More sequences than lanes of a wave, some without rows."""
    lens = [(37 * b) % 150 for b in range(200)]
    ns = [0 if b % 7 == 3 else min(1, lens[b]) for b in range(200)]
    pool = Pool(lens, 1, 32, 8, F16, seed=6)
    run(gpu, pool, ns, 4, pad=2, name="200 sequences")
    ns = [min(lens[b], 20) if b % 5 == 0 else n for b, n in enumerate(ns)]
    run(gpu, pool, ns, 4, name="200 sequences, chunks among them")


@pytest.mark.parametrize("dtype,i8,d", [(F16, False, 128), (BF16, False, 96), (F16, False, 32), (BF16, False, 160),
                                        (F16, True, 128), (BF16, True, 64)])
@pytest.mark.parametrize("window", [-1, 40])
def test_many_row_tiles_per_worker(gpu, dtype, i8, d, window):
    lens = [1 + (37 * b) % 131 for b in range(150)]
    pool = Pool(lens, 8, d, 16, dtype, i8, seed=d)
    run(gpu, pool, lens, 32, window=window, name=f"many prompts {dtype} {i8} {d} {window}")


@pytest.mark.parametrize("dtype,i8", [(F16, False), (F16, True)])
@pytest.mark.parametrize("max_q", [0, 1, 8])
def test_more_rows_than_max_seqlen_q(gpu, dtype, i8, max_q):
    lens = [300, 9, 700, 64] + [200] * 30
    pool = Pool(lens, 2, 64, 16, dtype, i8, seed=6)
    run(gpu, pool, [150, 3, 40, 64] + [33] * 30, 8, max_q=max_q, name=f"max_seqlen_q {max_q} {dtype} {i8}")


@pytest.mark.parametrize("causal", [True, False])
def test_more_row_tiles_than_lanes(gpu, causal):
    lens = [30, 1150, 700]
    pool = Pool(lens, 1, 32, 64, F16, seed=5)
    run(gpu, pool, [1, 1150, 300], 16, causal=causal, name=f"long prompt {causal}")
    run(gpu, pool, [30, 1150, 700], 16, causal=causal, window=90, name=f"long prompt, window {causal}")


@pytest.mark.parametrize("dtype,i8,d", [(F16, False, 128), (BF16, False, 96), (F16, True, 128)])
def test_many_heads(gpu, dtype, i8, d):
    """512 kv heads and more of all sequences: workgroups of four waves, most of
    them with several whole heads."""
    lens = [(53 * b) % 400 + 1 for b in range(130)]
    lens[7], lens[100] = 3000, 0
    pool = Pool(lens, 4, d, 16, dtype, i8, seed=30)
    run(gpu, pool, [1] * 130, 8, uniform=True, name="many heads")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [-1, 1, 2, 17, 64, 100, 5000, 2 ** 31 - 1])
def test_masks(gpu, causal, window):
    pool = Pool([300, 129, 64, 3], 2, 64, 16, F16, seed=7)
    run(gpu, pool, [1, 1, 1, 1], 4, causal=causal, window=window, uniform=True, name=f"decode {causal} {window}")
    run(gpu, pool, [200, 129, 5, 3], 4, causal=causal, window=window, name=f"chunks {causal} {window}")


def test_rows_without_keys(gpu):
    """More rows than keys: the first rows see nothing and come out as zeros;
    sequences of no key and negative lengths likewise."""
    pool = Pool([3, 0, -5, 70], 2, 64, 16, F16, seed=8)
    got = run(gpu, pool, [5, 2, 2, 100], 8, name="rows without keys")
    assert (got[:2] == 0).all() and (got[5:9] == 0).all() and (got[9:39] == 0).all()
    run(gpu, Pool([0, 0], 2, 128, 16, BF16, seed=9), [1, 1], 8, uniform=True, name="empty caches")


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0, 3.0e-20])
def test_scales(gpu, scale):
    pool = Pool([90, 200], 2, 64, 16, F16, seed=10)
    run(gpu, pool, [1, 1], 4, scale=scale, uniform=True, name=f"decode scale {scale}")
    run(gpu, pool, [90, 60], 4, scale=scale, name=f"chunks scale {scale}")


@pytest.mark.parametrize("layout", ["hnd", "kv"])
@pytest.mark.parametrize("dtype,i8", [(BF16, False), (F16, True)])
def test_layouts(gpu, layout, dtype, i8):
    pool = Pool([90, 333], 4, 128, 16, dtype, i8, seed=11, layout=layout)
    run(gpu, pool, [1, 1], 8, uniform=True, qview=True, name=f"decode {layout}")
    run(gpu, pool, [90, 100], 8, qview=True, name=f"chunks {layout}")


@pytest.mark.parametrize("ns", [[1, 1, 1], [40, 3, 90]])
@pytest.mark.parametrize("dtype,i8", [(F16, False), (BF16, False), (F16, True)])
def test_places_without_keys_may_hold_anything(gpu, ns, dtype, i8):
    """NaN and infinities behind a sequence's last key, in pages of no sequence
    and in the scales there leave no trace."""
    pool = Pool([41, 8, 200], 2, 64, 16, dtype, i8, seed=12)
    unused = pool.unused()
    if i8:
        pool.ks[unused] = float("nan")
        pool.vs[unused] = float("inf")
    else:
        pool.k[unused] = float("nan")
        pool.v[unused] = float("inf")
    run(gpu, pool, ns, 4, name="junk in unused places")


@pytest.mark.parametrize("ns", [[1, 1], [1, 90]])
def test_window_ends_inside_pages_of_junk(gpu, ns):
    """Keys that a window has left behind may be overwritten: their pages are
    handed out again, or hold nothing finite."""
    pool = Pool([150, 300], 2, 64, 16, F16, seed=13)
    run(gpu, pool, ns, 4, window=20, name="window")
    for b, n in enumerate(pool.lens):
        first = n - ns[b] - 20 + 1  # before every row's window
        if first > 0:
            at = pool.where(b, torch.arange(first))
            pool.k[at] = float("inf")
            pool.v[at] = float("nan")
    kk = Pool.rows

    def rows(b, n):  # the reference multiplies hidden values by zero
        k, v = kk(pool, b, n)
        return k.nan_to_num(0.0, 0.0, 0.0), v.nan_to_num(0.0, 0.0, 0.0)

    pool.rows = rows
    run(gpu, pool, ns, 4, window=20, name="window over junk")


@pytest.mark.parametrize("ns", [[1, 1, 1], [70, 64, 70]])
@pytest.mark.parametrize("i8", [False, True])
def test_pages_outside_the_cache(gpu, ns, i8):
    """A table entry that is no page leads nowhere, and touches no other
    sequence; so do lengths beyond the table."""
    import rdnattention as ra

    pool = Pool([70, 64, 130], 2, 64, 16, F16, i8, seed=14, extra_width=0)
    good = run(gpu, pool, ns, 4, name="before")
    k, v, table, lens, scales = pool.on(gpu)
    table[1, 0], table[1, 2] = 2 ** 31 - 1, -1
    cu = torch.tensor([0, ns[0], ns[0] + ns[1], sum(ns)], dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(sum(ns), 4, 64, generator=g).half().to(gpu)
    got = ra.paged_attention(q, k, v, table, lens, cu_seqlens_q=cu, **scales)
    a, z = ns[0], ns[0] + ns[1]
    assert torch.equal(got[:a], good[:a]) and torch.equal(got[z:], good[z:])
    assert torch.isfinite(got.float()).all()
    # the last sequence's length is past its table: taken as the table's 144 keys
    far = lens.clone()
    far[2] = 2 ** 31 - 1
    want = lens.clone()
    want[2] = table.shape[1] * 16
    table[2] = torch.arange(table.shape[1], dtype=torch.int32, device=gpu)
    assert torch.equal(ra.paged_attention(q, k, v, table, far, cu_seqlens_q=cu, **scales),
                       ra.paged_attention(q, k, v, table, want, cu_seqlens_q=cu, **scales))


@pytest.mark.parametrize("cu", [[0, 90, 20, 130], [-5, 30, 60, 4000], [50, 50, 50, 50], [130, 0, 0, 0]])
def test_row_ranges_out_of_order(gpu, cu):
    """Row ranges that make no sense stay inside the row tensors."""
    import rdnattention as ra

    pool = Pool([70, 64, 130], 2, 64, 16, F16, seed=15)
    k, v, table, lens, _ = pool.on(gpu)
    buf = torch.full((140, 4, 64), 7.0, dtype=F16, device=gpu)
    q = torch.randn(130, 4, 64, device=gpu).half()
    ra.paged_attention(q, k, v, table, lens, cu_seqlens_q=torch.tensor(cu, dtype=torch.int32, device=gpu),
                       out=buf[5:135])
    torch.cuda.synchronize()
    assert (buf[:5] == 7).all() and (buf[135:] == 7).all()


def test_padding_rows_of_a_given_output(gpu):
    pool = Pool([30, 100], 2, 64, 16, F16, seed=16)
    for ns in ([1, 1], [1, 60]):
        out = torch.full((sum(ns) + 3, 4, 64), 5.0, dtype=F16, device=gpu)
        got = run(gpu, pool, ns, 4, pad=3, out=out, name="given output")
        assert got is out and (out[sum(ns):] == 5).all()


@pytest.mark.parametrize("ns", [[1], [130]])
def test_offsets_past_32_bits(gpu, ns):
    """A cache of more than 2^32 bytes, the sequence in its last pages."""
    import rdnattention as ra

    pages, page, hkv, d = 140000, 16, 8, 128  # 4.6 GB each
    pool = Pool([200], hkv, d, page, F16, seed=17)
    k, v, _, lens, _ = pool.on(gpu)
    big_k = torch.empty(pages, page, hkv, d, dtype=F16, device=gpu)
    big_v = torch.empty(pages, page, hkv, d, dtype=F16, device=gpu)
    n = (200 + page - 1) // page
    table = torch.arange(pages - 1, pages - 1 - n, -1, dtype=torch.int32, device=gpu)[None]
    for i in range(n):
        big_k[pages - 1 - i] = k[pool.table[0, i]]
        big_v[pages - 1 - i] = v[pool.table[0, i]]
    q = torch.randn(ns[0], 32, d, device=gpu).half()
    want = ra.paged_attention(q, k, v, pool.table.to(gpu), lens)
    assert torch.equal(ra.paged_attention(q, big_k, big_v, table, lens), want)


@pytest.mark.parametrize("n", [1, 2, 8, 9, 17, 64, 70, 150])
@pytest.mark.parametrize("dtype,i8", [(F16, False), (BF16, False), (F16, True)])
def test_trees(gpu, n, dtype, i8):
    g = torch.Generator().manual_seed(n)
    lens = [n, n + 1, n + 40, n + 300]
    pool = Pool(lens, 2, 64, 16, dtype, i8, seed=n)
    tree = torch.rand(4, n, n, generator=g) < 0.5
    tree[0, 0] = False  # a row that sees nothing at all: no prefix either
    got = run(gpu, pool, [n] * 4, 8, tree=tree, uniform=True, name=f"tree {n}")
    assert (got[0] == 0).all()


def test_ragged_trees(gpu):
    """Fewer drafts than the mask, none, more than the mask, more than keys."""
    g = torch.Generator().manual_seed(3)
    pool = Pool([50, 20, 30, 7, 100], 2, 64, 16, F16, seed=18)
    tree = torch.rand(5, 12, 12, generator=g) < 0.4
    run(gpu, pool, [5, 0, 12, 10, 15], 4, tree=tree, pad=2, name="ragged trees")
    run(gpu, pool, [5, 0, 12, 10, 15], 4, tree=tree.expand(5, 12, 12), name="ragged trees, one mask")
    one = tree[:1].expand(5, 12, 12)  # a mask shared by all sequences
    run(gpu, pool, [5, 0, 12, 10, 15], 4, tree=one, name="shared mask")


def test_causal_tree_is_causal_attention(gpu):
    import rdnattention as ra

    pool = Pool([90, 200], 2, 128, 16, F16, seed=19)
    k, v, table, lens, _ = pool.on(gpu)
    q = torch.randn(2 * 20, 8, 128, device=gpu).half()
    tree = torch.ones(20, 20, dtype=torch.bool, device=gpu).tril()[None].expand(2, 20, 20)
    a = ra.paged_tree_attention(q, k, v, table, lens, tree)
    b = ra.paged_attention(q, k, v, table, lens)
    assert torch.equal(a, b)


@pytest.mark.parametrize("ns", [[1] * 4, [1, 500, 1, 30]])
@pytest.mark.parametrize("i8", [False, True])
def test_graph_replays(gpu, ns, i8):
    """Captured once, replayed with other lengths, pages and queries in the same
    tensors, eager calls on the same stream in between."""
    import rdnattention as ra

    pool = Pool([900, 600, 64, 333], 2, 64, 16, F16, i8, seed=20)
    k, v, table, lens, scales = pool.on(gpu)
    q = torch.randn(sum(ns), 8, 64, device=gpu).half()
    cu = torch.tensor([sum(ns[:i]) for i in range(5)], dtype=torch.int32, device=gpu)

    def call():
        return ra.paged_attention(q, k, v, table, lens, cu_seqlens_q=cu, max_seqlen_q=max(ns), **scales)

    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for rep in range(4):
        q.copy_(torch.randn(q.shape, device=gpu))
        lens.copy_(torch.tensor([900 - 100 * rep, 600, 64 - rep, 333], dtype=torch.int32))
        out.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), f"replay {rep}"


def test_two_graphs_and_two_streams(gpu):
    """Calls side by side have scratch of their own."""
    import rdnattention as ra

    pools = [Pool([2000, 1500], 2, 128, 16, F16, seed=s) for s in (21, 22)]
    dev = [p.on(gpu) for p in pools]
    qs = [torch.randn(2, 8, 128, device=gpu).half() for _ in pools]

    def call(i):
        k, v, table, lens, _ = dev[i]
        return ra.paged_attention(qs[i], k, v, table, lens)

    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pools]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(i))
        graphs.append(graph)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i]) for i in range(2))


@pytest.mark.parametrize("ns,max_q", [([1] * 40, 1), ([1, 300, 5, 40] * 10, 300)])
def test_output_over_the_query(gpu, ns, max_q):
    import rdnattention as ra

    lens = [n + 13 * (b % 40) for b, n in enumerate(ns)]
    for dtype, d in ((F16, 128), (BF16, 160)):
        pool = Pool(lens, 2, d, 16, dtype, seed=24)
        k, v, table, lens_t, _ = pool.on(gpu)
        q = torch.randn(sum(ns), 16, d, device=gpu).to(dtype)
        cu = torch.tensor([sum(ns[:i]) for i in range(len(ns) + 1)], dtype=torch.int32, device=gpu)
        want = ra.paged_attention(q, k, v, table, lens_t, cu_seqlens_q=cu, max_seqlen_q=max_q)
        got = q.clone()
        assert ra.paged_attention(got, k, v, table, lens_t, cu_seqlens_q=cu, max_seqlen_q=max_q, out=got) is got
        assert torch.equal(got, want)


@pytest.mark.parametrize("own_streams", [True, False])
def test_two_host_threads(gpu, own_streams):
    import threading

    import rdnattention as ra

    jobs, failed = [], []
    for i, ns in enumerate(([1, 1], [1, 200])):
        pool = Pool([900, 1500], 2, 64, 16, F16, seed=30 + i)
        k, v, table, lens, _ = pool.on(gpu)
        q = torch.randn(sum(ns), 8, 64, device=gpu).half()
        cu = torch.tensor([0, ns[0], sum(ns)], dtype=torch.int32, device=gpu)
        jobs.append(lambda q=q, k=k, v=v, t=table, n=lens, cu=cu, m=max(ns): ra.paged_attention(
            q, k, v, t, n, cu_seqlens_q=cu, max_seqlen_q=m))
    want = [job() for job in jobs]
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream() if own_streams else torch.cuda.default_stream()):
                got = [jobs[i]() for _ in range(30)]
                torch.cuda.current_stream().synchronize()
            assert all(torch.equal(x, want[i]) for x in got)
        except BaseException as e:  # reported by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_same_bits_every_time(gpu):
    import rdnattention as ra

    pool = Pool([3000, 77, 1024], 4, 128, 16, BF16, seed=23)
    k, v, table, lens, _ = pool.on(gpu)
    for n in (1, 33):
        q = torch.randn(3 * n, 16, 128, device=gpu).to(BF16)
        first = ra.paged_attention(q, k, v, table, lens)
        for _ in range(5):
            assert torch.equal(ra.paged_attention(q, k, v, table, lens), first)


@pytest.mark.parametrize("ns", [[1, 1, 1], [70, 64, 90]])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_int8_scales_of_any_size(gpu, ns, dtype):
    """Scales from 2^-40 to 2^6, growing and falling along the keys, zeros and
    negative ones among them: the weights they meet stay in fp16's range."""
    pool = Pool([600, 64, 90], 2, 64, 16, dtype, True, seed=26)
    for b, lo, hi in ((0, -40, 6), (1, -30, -10), (2, 6, -40)):
        n = pool.lens[b]
        at = pool.where(b, torch.arange(n))
        pool.vs[at] = torch.exp2(torch.linspace(lo, hi, n))[:, None].expand(n, 2)
    at = pool.where(0, torch.arange(0, 600, 7))
    pool.vs[at] = 0.0
    at = pool.where(0, torch.arange(3, 600, 11))
    pool.vs[at] = -pool.vs[at]
    at = pool.where(2, torch.arange(0, 90, 5))
    pool.ks[at] = -pool.ks[at]
    run(gpu, pool, ns, 4, name="scales")


def test_large_scores(gpu):
    """Scores of hundreds of log2 units: the running maximum moves often, most
    weights vanish."""
    for ns in ([1, 1], [100, 128]):
        pool = Pool([700, 128], 2, 64, 16, F16, seed=24, std=4.0)
        run(gpu, pool, ns, 4, scale=2.0, name="large scores")


def test_a_nan_score_reaches_its_row_only(gpu):
    import rdnattention as ra

    pool = Pool([700], 2, 64, 16, F16, seed=25)
    k, v, table, lens, _ = pool.on(gpu)
    for n in (1, 40):
        q = torch.randn(n, 8, 64, device=gpu).half()
        q[0, 3] = float("nan")
        got = ra.paged_attention(q, k, v, table, lens)
        bad = torch.zeros(n, 8, dtype=torch.bool, device=gpu)
        bad[0, 3] = True
        assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()

"""paged_prefix_attention and the log-sum-exp of paged_attention against their
definitions in 64 bits: every type and head dim, prefixes of any length, groups of
sequences, ragged rows, what the pages hold where no key is, streams and graphs."""
import math

import pytest
import torch

from tests.gpu_util import log
from tests.paged_util import Pool, check, reference, visible

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
TYPES = [(F16, False), (BF16, False), (F16, True), (BF16, True)]


def lse_reference(q, k, ok, scale, i8):
    """(log-sum-exp, bound) in 64 bits.  The scores are off by (d + 2) 2^-24 of the sum of
    their products' magnitudes, and by 2^-22 of their own size in the exponent (int8:
    2^-23 more, the scales), the exponential by 2^-21, sums and the joining of parts by
    2^-18 in all, and the logarithm, taken in steps of log2 units that are as large as the
    result, by 2^-22 of it."""
    n, hq, d = q.shape
    g = hq // k.shape[1]
    out = torch.full((n, hq), -math.inf, dtype=torch.float64)
    tol = torch.full((n, hq), 1e-30, dtype=torch.float64)
    if k.shape[0] == 0 or n == 0:
        return out, tol
    seen = ok.any(-1)
    for h in range(hq):
        kh = k[:, h // g]
        s = (q[:, h].double() @ kh.t() * scale).masked_fill(~ok, -math.inf)
        mag = (q[:, h].double().abs() @ kh.abs().t() * abs(scale)).masked_fill(~ok, 0.0)
        out[:, h] = torch.logsumexp(s, -1)
        tol[:, h] = mag.amax(-1) * ((d + 2) * 2.0 ** -24 + 2.0 ** -22 + (2.0 ** -23 if i8 else 0.0)) + 2.0 ** -21 + \
            2.0 ** -18 + out[:, h].nan_to_num(0.0, 0.0, 0.0).abs() * 2.0 ** -22
    out[~seen] = -math.inf
    return out, tol


def check_lse(got, want, tol, name):
    got = got.cpu().double()
    empty = want == -math.inf
    assert (got[empty] == -math.inf).all(), name
    if (~empty).any():
        over = float(((got - want)[~empty].abs() / tol[~empty]).max())
        assert over <= 1.0, f"{name}: lse off by {over:.3f} of its bound"


def run(gpu, lens, ns, prefix, seqs, hq, hkv, d, dtype, i8=False, page=16, causal=True, scale=None, seed=1, pad=0,
        uniform=False, max_q=None, out=None, layout="nhd", spoil=False, given=True, name=""):
    """The call and its reference: own keys lens[b], rows ns[b], prefixes of prefix[i]
    keys, the sequences seqs[i] .. seqs[i + 1] - 1 behind each."""
    import rdnattention as ra

    b = len(lens)
    pool = Pool(list(lens) + list(prefix), hkv, d, page, dtype, i8, seed=seed, layout=layout)
    if spoil:
        unused = pool.unused()
        if i8:
            pool.ks[unused], pool.vs[unused] = float("nan"), float("inf")
        else:
            pool.k[unused], pool.v[unused] = float("nan"), float("inf")
    g = torch.Generator().manual_seed(seed)
    rows = sum(ns) + pad
    q = torch.randn(rows, hq, d, generator=g).to(dtype)
    k, v, table, all_lens, scales = pool.on(gpu)
    kw = dict(scales, scale=scale, out=out, is_causal=causal, return_lse=True)
    if not uniform:
        kw["cu_seqlens_q"] = torch.tensor([sum(ns[:i]) for i in range(b + 1)], dtype=torch.int32, device=gpu)
        kw["max_seqlen_q"] = max_q
    if given:
        kw["prefix_seqs"] = torch.tensor(seqs, dtype=torch.int32, device=gpu)
    got, lse = ra.paged_prefix_attention(q.to(gpu), k, v, table[b:], all_lens[b:].contiguous(), table[:b],
                                         all_lens[:b].contiguous(), **kw)
    torch.cuda.synchronize()
    at, worst = 0, 0.0
    of = [i for i in range(len(prefix)) for _ in range(seqs[i + 1] - seqs[i])]
    sc = d ** -0.5 if scale is None else scale
    for s, n in enumerate(ns):
        own, shared = max(0, lens[s]), max(0, prefix[of[s]])
        ok_, ov = pool.rows(s, own)
        pk, pv = pool.rows(b + of[s], shared)
        ok = torch.cat((torch.ones(n, shared, dtype=torch.bool), visible(n, own, causal)), 1)
        kk, vv = torch.cat((pk, ok_)), torch.cat((pv, ov))
        want, tol = reference(q[at:at + n], kk, vv, ok, sc, dtype, i8)
        if n:
            worst = max(worst, check(got[at:at + n], want, tol, f"{name} sequence {s}"))
            check_lse(lse[at:at + n], *lse_reference(q[at:at + n], kk, ok, sc, i8), f"{name} sequence {s}")
        at += n
    if pad:
        assert (lse[at:] == -math.inf).all()
        if out is None:
            assert (got[at:] == 0).all()
    log(f"[paged prefix] {name}: {worst:.3f} of the bound")
    return got, lse


@pytest.mark.parametrize("dtype,i8", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 700])
def test_decode(gpu, dtype, i8, d, prefix):
    lens = [1, 2, 31, 32, 33, 64, 65, 257, 400, 5]
    run(gpu, lens, [1] * 10, [prefix], [0, 10], 8, 2, d, dtype, i8, uniform=True, seed=d, given=False,
        name=f"decode {dtype} {i8} {d} {prefix}")


@pytest.mark.parametrize("d", [32, 96, 160, 192, 224, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_head_dims(gpu, d, dtype):
    run(gpu, [5, 130, 40] * 4, [1] * 12, [300], [0, 12], 6, 2, d, dtype, uniform=True, page=32, seed=d, name=f"decode {d}")
    run(gpu, [5, 130, 40], [5, 100, 1], [300], [0, 3], 6, 2, d, dtype, page=32, seed=d, name=f"chunks {d}")
    run(gpu, [5, 130], [1, 1], [300], [0, 2], 6, 2, d, dtype, uniform=True, page=32, seed=d, name=f"few rows {d}")


@pytest.mark.parametrize("dtype,i8", TYPES)
def test_few_rows(gpu, dtype, i8):
    """So few rows in all that the prefix is streamed too."""
    for b, hq in ((1, 1), (1, 32), (3, 8), (8, 4)):
        run(gpu, [40 + 3 * i for i in range(b)], [1] * b, [2000], [0, b], hq, 1, 64, dtype, i8, uniform=True,
            name=f"few {b} {hq}")


@pytest.mark.parametrize("dtype,i8", TYPES)
def test_groups(gpu, dtype, i8):
    """Several prefixes, an empty one, one without sequences, one of a single one."""
    lens = [3, 70, 20, 1, 300, 41, 64, 8, 9]
    for ns in ([1] * 9, [3, 40, 1, 1, 200, 0, 64, 8, 1]):
        run(gpu, lens, ns, [257, 0, 90, 64, 500], [0, 4, 5, 5, 6, 9], 8, 2, 64, dtype, i8, uniform=ns == [1] * 9,
            pad=0 if ns == [1] * 9 else 3, name=f"groups {dtype} {i8}")


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("causal", [True, False])
def test_mixed_batch(gpu, i8, causal):
    """Single tokens, chunks and prompts behind one prefix, rows without own keys and
    sequences without rows, padding behind them."""
    lens = [700, 0, 1, 300, 64, 512, 129, 3, 33]
    ns = [1, 0, 1, 300, 3, 0, 100, 5, 33]
    for most in (None, 300):
        run(gpu, lens, ns, [333], [0, 9], 8, 2, 64, F16, i8, causal=causal, pad=5, max_q=most, name="mixed")


def test_without_keys(gpu):
    """Rows that see nothing: zeros and -inf."""
    got, lse = run(gpu, [0, 3, -4], [1, 5, 2], [0], [0, 3], 4, 2, 64, F16, name="no keys")
    assert (got[:3] == 0).all() and (lse[:3] == -math.inf).all() and (got[6:] == 0).all()
    run(gpu, [0, 3, -4], [1, 5, 2], [50], [0, 3], 4, 2, 64, F16, name="prefix alone")
    run(gpu, [0, 0], [1, 1], [-3, 70], [0, 1, 2], 4, 2, 128, BF16, True, uniform=True, name="negative length")


@pytest.mark.parametrize("dtype,i8,d", [(F16, False, 128), (BF16, False, 64), (F16, True, 128), (BF16, False, 256)])
def test_many_whole_items(gpu, dtype, i8, d):
    """More row tiles than workgroups: whole items in both parts."""
    lens = [1 + (37 * b) % 131 for b in range(150)]
    run(gpu, lens, lens, [70] * 30, list(range(0, 151, 5)), 16, 8, d, dtype, i8, name=f"many prompts {d}")


def test_long_prefix_and_many_rows(gpu):
    run(gpu, [20 + b for b in range(70)], [1] * 70, [9001], [0, 70], 32, 4, 128, BF16, page=64, uniform=True, name="long")
    run(gpu, [400, 390], [400, 10], [5000], [0, 2], 8, 2, 128, F16, name="long, chunks")


@pytest.mark.parametrize("page", [1, 4, 16, 128, 1024])
@pytest.mark.parametrize("i8", [False, True])
def test_pages(gpu, page, i8):
    run(gpu, [7, 90, 61] * 5, [1] * 15, [301], [0, 15], 4, 2, 64, F16, i8, page=page, uniform=True, spoil=True,
        name=f"page {page}")
    run(gpu, [7, 90, 61], [7, 50, 20], [301], [0, 3], 4, 2, 64, F16, i8, page=page, spoil=True, name=f"page {page}, chunks")


@pytest.mark.parametrize("layout", ["hnd", "kv"])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (40, 8), (64, 2)])
def test_heads_and_layouts(gpu, layout, hq, hkv):
    run(gpu, [20, 77, 5], [1] * 3, [200], [0, 3], hq, hkv, 64, F16, uniform=True, layout=layout, name=f"heads {hq}/{hkv}")
    run(gpu, [20, 77, 5], [9, 77, 1], [200], [0, 3], hq, hkv, 64, F16, layout=layout, name=f"chunks {hq}/{hkv}")


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
def test_scales(gpu, scale):
    run(gpu, [90, 20], [1, 1], [200], [0, 2], 32, 2, 64, F16, scale=scale, uniform=True, name=f"scale {scale}")
    run(gpu, [90, 20], [90, 6], [200], [0, 2], 4, 2, 64, F16, scale=scale, name=f"scale {scale}")


def test_given_output_and_over_the_query(gpu):
    import rdnattention as ra

    for ns in ([1, 1], [1, 60]):
        out = torch.full((sum(ns) + 3, 4, 64), 5.0, dtype=F16, device=gpu)
        got, _ = run(gpu, [30, 100], ns, [80], [0, 2], 4, 2, 64, F16, pad=3, out=out, name="given output")
        assert got is out and (out[sum(ns):] == 5).all()
    pool = Pool([200, 300, 700], 2, 128, 16, F16, seed=3)
    k, v, table, lens, _ = pool.on(gpu)
    cu = torch.tensor([0, 1, 200], dtype=torch.int32, device=gpu)
    q = torch.randn(200, 8, 128, device=gpu).half()
    args = (k, v, table[2:], lens[2:].contiguous(), table[:2], lens[:2].contiguous())
    want = ra.paged_prefix_attention(q, *args, cu_seqlens_q=cu)
    mine = q.clone()
    assert ra.paged_prefix_attention(mine, *args, cu_seqlens_q=cu, out=mine) is mine
    assert torch.equal(mine, want)


@pytest.mark.parametrize("dtype,i8", TYPES)
@pytest.mark.parametrize("ns", [[1] * 4, [1, 300, 5, 70]])
@pytest.mark.parametrize("window", [-1, 50])
def test_lse_of_paged_attention(gpu, dtype, i8, ns, window):
    """return_lse: the output that the call gives without, but for the rounding of the
    weights' sum, and the log-sum-exp."""
    import rdnattention as ra

    lens = [900, 400, 5, 3000 if ns[1] == 1 else 100]
    pool = Pool(lens, 2, 64, 16, dtype, i8, seed=4)
    k, v, table, dl, scales = pool.on(gpu)
    q = torch.randn(sum(ns) + 2, 8, 64, generator=torch.Generator().manual_seed(1)).to(dtype)
    cu = torch.tensor([sum(ns[:i]) for i in range(5)], dtype=torch.int32, device=gpu)
    kw = dict(scales, cu_seqlens_q=cu, window_size=window)
    out, lse = ra.paged_attention(q.to(gpu), k, v, table, dl, return_lse=True, **kw)
    assert (out[sum(ns):] == 0).all() and (lse[sum(ns):] == -math.inf).all()
    at = 0
    for b, n in enumerate(ns):
        kk, vv = pool.rows(b, lens[b])
        ok = visible(n, lens[b], True, window)
        want, tol = reference(q[at:at + n], kk, vv, ok, 0.125, dtype, i8)
        check(out[at:at + n], want, tol, f"sequence {b}")
        check_lse(lse[at:at + n], *lse_reference(q[at:at + n], kk, ok, 0.125, i8), f"sequence {b}")
        at += n


def test_nan_reaches_its_row_only(gpu):
    import rdnattention as ra

    pool = Pool([60, 50, 700], 2, 64, 16, F16, seed=25)
    k, v, table, lens, _ = pool.on(gpu)
    for n in (1, 40):
        q = torch.randn(2 * n, 8, 64, device=gpu).half()
        q[0, 3] = float("nan")
        got, lse = ra.paged_prefix_attention(q, k, v, table[2:], lens[2:].contiguous(), table[:2], lens[:2].contiguous(),
                                             return_lse=True)
        bad = torch.zeros(2 * n, 8, dtype=torch.bool, device=gpu)
        bad[0, 3] = True
        assert torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()
        assert torch.isnan(lse[bad]).all() and torch.isfinite(lse[~bad]).all()


def test_pages_and_groups_that_make_no_sense(gpu):
    """Table entries that are no page, lengths past the table, sequence ranges out of
    order: nothing outside the tensors is read or written."""
    import rdnattention as ra

    pool = Pool([40, 64, 30, 130], 2, 64, 16, F16, seed=14)
    k, v, table, lens, _ = pool.on(gpu)
    buf = torch.full((130, 4, 64), 7.0, dtype=F16, device=gpu)
    q = torch.randn(120, 4, 64, device=gpu).half()
    for seqs in ([0, 5, -1, 3], [3, 0, 3, 0], [-9, 1, 1, 90], [2 ** 31 - 1] * 4):
        prefix = table[3:].expand(3, -1).contiguous()
        prefix[0, 0], prefix[1, 1] = 2 ** 31 - 1, -1
        far = torch.tensor([2 ** 31 - 1, 60, -2 ** 31], dtype=torch.int32, device=gpu)
        ra.paged_prefix_attention(q, k, v, prefix, far, table[:3], lens[:3].contiguous(), out=buf[5:125],
                                  prefix_seqs=torch.tensor(seqs, dtype=torch.int32, device=gpu))
        torch.cuda.synchronize()
        assert (buf[:5] == 7).all() and (buf[125:] == 7).all()


@pytest.mark.parametrize("ns", [[1] * 12, [1, 200, 1, 30] * 3])
def test_graphs_and_streams(gpu, ns):
    """Two captured calls, replayed side by side with other lengths and queries, eager calls in
    between; the same bits every time."""
    import rdnattention as ra

    calls, tensors, outs, graphs = [], [], [], []
    for i in range(2):
        pool = Pool([220 + 7 * b for b in range(12)] + [1500, 60], 2, 64, 16, F16, seed=20 + i)
        k, v, table, lens, _ = pool.on(gpu)
        q = torch.randn(sum(ns), 8, 64, device=gpu).half()
        cu = torch.tensor([sum(ns[:j]) for j in range(13)], dtype=torch.int32, device=gpu)
        seqs = torch.tensor([0, 8, 12], dtype=torch.int32, device=gpu)
        own, shared = lens[:12].contiguous(), lens[12:].contiguous()
        calls.append(lambda q=q, k=k, v=v, t=table, own=own, shared=shared, cu=cu, seqs=seqs: ra.paged_prefix_attention(
            q, k, v, t[12:], shared, t[:12], own, prefix_seqs=seqs, cu_seqlens_q=cu, max_seqlen_q=max(ns),
            return_lse=True))
        tensors.append((q, own, shared))
        calls[i]()
    torch.cuda.synchronize()
    for call in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in calls]
    for rep in range(4):
        for (q, own, shared), o in zip(tensors, outs):
            q.copy_(torch.randn(q.shape, device=gpu))
            own.sub_(1)
            shared.sub_(9)
            o[0].fill_(9.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for call, o in zip(calls, outs):
            eager, lse = call()
            assert torch.equal(o[0], eager) and torch.equal(o[1], lse), f"replay {rep}"


def test_offsets_past_32_bits(gpu):
    """A cache of more than 2^32 bytes, the prefix in its last pages."""
    import rdnattention as ra

    pages, page, hkv, d = 140000, 16, 8, 128  # 4.6 GB each
    pool = Pool([30, 200], hkv, d, page, F16, seed=17)
    k, v, table, lens, _ = pool.on(gpu)
    big_k = torch.empty(pages, page, hkv, d, dtype=F16, device=gpu)
    big_v = torch.empty(pages, page, hkv, d, dtype=F16, device=gpu)
    far = table.clone()
    for b in range(2):
        for i in range((pool.lens[b] + page - 1) // page):
            p = int(pool.table[b, i])
            far[b, i] = pages - 1 - p
            big_k[pages - 1 - p], big_v[pages - 1 - p] = k[p], v[p]
    q = torch.randn(20, 32, d, device=gpu).half()
    args = lens[1:].contiguous(), lens[:1].contiguous()
    want = ra.paged_prefix_attention(q, k, v, table[1:], args[0], table[:1], args[1])
    assert torch.equal(ra.paged_prefix_attention(q, big_k, big_v, far[1:], args[0], far[:1], args[1]), want)

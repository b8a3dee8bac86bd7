"""The cache operators together, as a server uses them over several steps: normed appends at
the positions of the text, attention behind a shared prefix, the keys' weights, eviction."""
import pytest
import torch

from tests.gpu_util import log
from tests.paged_util import check, reference, rope_tables, visible
from tests.test_gpu_paged_evict import chosen
from tests.test_gpu_paged_norm import check_near, normed, turned
from tests.test_gpu_paged_prefix import check_lse, lse_reference
from tests.test_gpu_paged_weights import reference as weights_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,i8", [(torch.float16, False), (torch.bfloat16, False), (torch.float16, True)])
@pytest.mark.parametrize("captured", [False, True])
def test_serving(gpu, dtype, i8, captured):
    """Three sequences behind a prefix of 150 tokens begin with prompts of 70, 33 and 1
    tokens, then decode; when a cache has more than 48 own keys it is cut to 32.  Every
    call's results are checked against its formula on the cache that it was given."""
    import rdnattention as ra

    hq, hkv, d, page, seqs, shared = 8, 2, 64, 16, 3, 150
    g = torch.Generator().manual_seed(7)
    pages, width = 40, 6
    order = torch.randperm(pages, generator=g).int()
    prefix_table, table = order[:10][None].contiguous(), order[10:10 + seqs * width].reshape(seqs, width).contiguous()
    kind = torch.int8 if i8 else dtype
    kc, vc = (torch.zeros(pages, page, hkv, d, dtype=kind, device=gpu) for _ in range(2))
    scales = {n: torch.ones(pages, page, hkv, device=gpu) for n in ("key_scale", "value_scale")} if i8 else {}
    weights = torch.full((pages, page, hkv), float("nan"), device=gpu)
    cos, sin = rope_tables(400, d // 2)
    axis = torch.arange(d // 2, dtype=torch.int32) % 3
    qw, kw = (1 + 0.3 * torch.randn(d, generator=g) for _ in range(2))
    norm = dict(rot_cos=cos.to(gpu), rot_sin=sin.to(gpu), rot_interleaved=False, rot_axes=axis.to(gpu),
                query_norm=qw.to(gpu), key_norm=kw.to(gpu))
    dt, dp, plen = table.to(gpu), prefix_table.to(gpu), torch.tensor([shared], dtype=torch.int32, device=gpu)

    def rows_of(n):
        return torch.randn(n, hq + 2 * hkv, d, generator=g).to(dtype)

    # the prefix, once
    x = rows_of(shared).to(gpu)
    at = torch.arange(shared, dtype=torch.int32, device=gpu)[:, None].expand(-1, 3).contiguous()
    ra.paged_append(x[:, hq:hq + hkv], x[:, hq + hkv:], kc, vc, dp, plen, query=x[:, :hq], positions=at, **norm, **scales)

    lens = torch.zeros(seqs, dtype=torch.int32, device=gpu)
    text = [shared] * seqs  # positions
    graph, static = None, {}
    evictions = 0
    for step in range(24):
        ns = [70, 33, 1] if step == 0 else [1] * seqs
        cu = torch.tensor([0, ns[0], ns[0] + ns[1], sum(ns)], dtype=torch.int32, device=gpu)
        x = rows_of(sum(ns))
        pos = torch.cat([torch.arange(text[b], text[b] + n) for b, n in enumerate(ns)]).int()[:, None].expand(-1, 3).contiguous()
        pos[:, 2] += 1
        text = [t + n for t, n in zip(text, ns)]
        lens += torch.tensor(ns, dtype=torch.int32, device=gpu)
        before = weights.clone()

        def work(x, pos):
            q = ra.paged_append(x[:, hq:hq + hkv], x[:, hq + hkv:], kc, vc, dt, lens, cu_seqlens_q=cu, query=x[:, :hq],
                                positions=pos, **norm, **scales)
            out, lse = ra.paged_prefix_attention(q, kc, vc, dp, plen, dt, lens, cu_seqlens_q=cu, max_seqlen_q=max(ns),
                                                 return_lse=True, **scales)
            ra.paged_key_weights(q, lse, kc, dt, lens, weights, cu_seqlens_q=cu, max_seqlen_q=max(ns), decay=0.9,
                                 key_scale=scales.get("key_scale"))
            return q, out, lse

        if captured and step >= 1:
            if graph is None:
                static = {"x": x.to(gpu), "pos": pos.to(gpu), "cu": cu}
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    static["outs"] = work(static["x"], static["pos"])
            static["x"].copy_(x)
            static["pos"].copy_(pos)
            graph.replay()
            q, out, lse = static["outs"]
        else:
            q, out, lse = work(x.to(gpu), pos.to(gpu))
        torch.cuda.synchronize()

        sel = pos.long()[:, axis.long()]
        c, s = cos.gather(0, sel), sin.gather(0, sel)
        wq, size = turned(normed(x[:, :hq], qw, 1e-6), c, s, False)
        check_near(q, wq, size, dtype, f"step {step} queries")

        def cached(rows, n):
            i = torch.arange(n)
            pg, off = rows.long()[i // page], i % page
            k, v = kc.cpu()[pg, off].double(), vc.cpu()[pg, off].double()
            if i8:
                k = k * scales["key_scale"].cpu()[pg, off].double()[..., None]
                v = v * scales["value_scale"].cpu()[pg, off].double()[..., None]
            return k, v

        pk, pv = cached(prefix_table[0], shared)
        r = 0
        for b, n in enumerate(ns):
            length = int(lens[b])
            ok_, ov = cached(table[b], length)
            seen = visible(n, length)
            ok = torch.cat((torch.ones(n, shared, dtype=torch.bool), seen), 1)
            kk, vv = torch.cat((pk, ok_)), torch.cat((pv, ov))
            mine = slice(r, r + n)
            if not i8:  # the appended rows (int8 ones bit for bit elsewhere)
                wk, size = turned(normed(x[mine, hq:hq + hkv], kw, 1e-6), c[mine], s[mine], False)
                check_near(ok_[length - n:], wk, size, dtype, f"step {step} keys")
            want, tol = reference(q[mine].cpu(), kk, vv, ok, d ** -0.5, dtype, i8)
            check(out[mine], want, tol, f"step {step} sequence {b}")
            check_lse(lse[mine], *lse_reference(q[mine].cpu(), kk, ok, d ** -0.5, i8), f"step {step} sequence {b}")
            want, tol = weights_reference(q[mine].cpu(), lse[mine].cpu(), ok_, seen, d ** -0.5, i8)
            i = torch.arange(length)
            pg, off = table[b].long()[i // page], i % page
            was = torch.where((i < length - n)[:, None], before.cpu()[pg, off].double() * 0.9, torch.zeros_like(want))
            got = weights.cpu()[pg, off].double()
            assert ((got - want - was).abs() <= tol + 2.0 ** -22 * was.abs()).all(), f"step {step} sequence {b}: weights"
            r += n
        if int(lens.max()) > 48:
            evictions += 1
            full = [cached(table[b], int(lens[b])) for b in range(seqs)]
            heard = weights.cpu()
            new, kept = ra.paged_evict(kc, vc, dt, lens, weights, 32, first=2, recent=8, **scales)
            torch.cuda.synchronize()
            for b in range(seqs):
                n, m = int(lens[b]), int(new[b])
                assert m == min(n, 32)
                i = torch.arange(n)
                pg, off = table[b].long()[i // page], i % page
                k, v = cached(table[b], m)
                for h in range(hkv):
                    keep = chosen(heard[pg, off, h], 32, 2, 8)
                    assert kept[b, h, :m].tolist() == keep
                    assert torch.equal(k[:, h], full[b][0][keep, h]) and torch.equal(v[:, h], full[b][1][keep, h])
            lens.copy_(new)
    assert evictions >= 2
    log(f"[paged serving] {dtype} {i8} {captured}: {evictions} evictions")

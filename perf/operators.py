"""The operators of a paged key/value cache whose speed is tracked.

A server keeps the keys and values of its sequences in pages of a few tokens;
a table lists each sequence's pages.  The operators, as a server calls them:

  append   paged_append: one step's new keys and values go to their places in
           the pages, the position rotation applied to keys and queries
  attn     paged_attention: the newest rows of each sequence against its pages
           (single tokens, chunks, whole prompts, all three in one batch)
  tree     paged_tree_attention: drafted tokens that form a tree, each of which
           sees the prefix and its own ancestors
  commit   paged_commit: after the drafts are verified, the accepted ones move
           up behind the prefix

listed() holds the fixed cases, draw() gives others of the same ranges.  A case
is a dict of plain values:
  op      the operator
  dtype   "f16" or "bf16", of the queries and of new keys and values
  i8      whether the cache holds int8 with a scale per token and head
  b       sequences
  hq, hkv, d, page
  klo, khi   the sequences' lengths in the cache, new rows among them
  qlo, qhi   new rows per sequence (commit: accepted drafts per sequence)
  n       tree, commit: drafts per sequence
  rope    append: "none", "pairs" (channels 2i, 2i + 1) or "halves" (i, i + d/2)
  causal, window   attn
Where lo < hi the sequences are ragged; their lengths follow from the case
alone.
"""
import math
import random

import torch

own = False

KEYS = ("op", "dtype", "i8", "b", "hq", "hkv", "d", "page", "klo", "khi", "qlo", "qhi", "n", "rope", "causal",
        "window")

# a drawn case asks for at most this much (below the largest listed ones)
MAX_FLOPS = 2.5e11
MAX_BYTES = 1.5e9
# the caches that append and commit return whole stay below this many elements
MAX_POOL = 60_000_000


def _case(name, *values):
    case = dict(zip(KEYS, values))
    return dict(case, name=name) if name else case


def listed():
    return [
        # one sequence, one new token of an 8B-class grouped-query layer: the smallest call
        _case("append_b1", "append", "f16", False, 1, 32, 8, 128, 16, 500, 500, 1, 1, 0, "pairs", True, -1),
        # a served batch, one new token each
        _case("append_b128_bf16", "append", "bf16", False, 128, 32, 8, 128, 16, 20, 400, 1, 1, 0, "halves", True, -1),
        # prompts of ragged lengths into an int8 cache
        _case("append_prompts_i8", "append", "f16", True, 5, 16, 4, 64, 32, 200, 900, 150, 900, 0, "pairs", True, -1),
        # one sequence, one new token, a short cache: latency counts
        _case("attn_decode_b1_k2048", "attn", "f16", False, 1, 32, 8, 128, 16, 2048, 2048, 1, 1, 0, "none", True, -1),
        # a served batch with long, ragged caches: memory bound
        _case("attn_decode_b16_bf16", "attn", "bf16", False, 16, 32, 8, 128, 64, 4000, 32768, 1, 1, 0, "none", True,
              -1),
        # an int8 cache is kept because decode is memory bound
        _case("attn_decode_b32_i8", "attn", "f16", True, 32, 32, 8, 128, 16, 8192, 8192, 1, 1, 0, "none", True, -1),
        # a step that continues decoding and works through chunks of prompts
        _case("attn_mixed_d64", "attn", "f16", False, 24, 16, 8, 64, 16, 700, 6001, 1, 512, 0, "none", True, -1),
        # whole prompts of a grouped-query layer: matrix products
        _case("attn_prompts_b4", "attn", "f16", False, 4, 32, 8, 128, 32, 4096, 4096, 4096, 4096, 0, "none", True,
              -1),
        # one sequence with a small tree of drafts
        _case("tree_b1_n16", "tree", "f16", False, 1, 32, 8, 128, 16, 2065, 2065, 16, 16, 16, "none", True, -1),
        # a batch with wide trees and ragged caches
        _case("tree_b8_n60_bf16", "tree", "bf16", False, 8, 32, 8, 128, 64, 1237, 16384, 60, 60, 60, "none", True,
              -1),
        # accepted drafts of one step
        _case("commit_b64_bf16", "commit", "bf16", False, 64, 32, 8, 128, 16, 70, 300, 1, 8, 60, "none", True, -1),
        # the same of an int8 cache
        _case("commit_b8_i8", "commit", "f16", True, 8, 16, 4, 64, 16, 40, 200, 1, 5, 17, "none", True, -1),
    ]


HEADS = ((8, 8), (16, 16), (32, 8), (32, 8), (16, 4), (16, 8), (24, 8), (40, 8), (32, 1))


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(("append", "attn", "attn", "attn", "tree", "commit"))
    hq, hkv = rng.choice(HEADS)
    i8 = rng.random() < 0.3
    dtype = rng.choice(("f16", "bf16"))
    d = rng.choice((64, 128)) if i8 else rng.choice((64, 128, 128, 32 * rng.randint(1, 8)))
    page = rng.choice((16, 16, 32, 64, 128, 256))
    b = _log_int(rng, 1, 128)
    n, rope, causal, window = 0, "none", True, -1
    qlo = qhi = 1
    if op == "append":
        if rng.random() < 0.5:  # prompts
            qhi = _log_int(rng, 8, 4096)
            qlo = rng.randint(1, qhi)
        khi = qhi + _log_int(rng, 1, 512)
        klo = rng.randint(qhi, khi)
        rope = rng.choice(("none", "pairs", "halves"))
    elif op == "attn":
        kind = rng.choice(("decode", "decode", "chunk", "prompt", "mixed"))
        khi = _log_int(rng, 16, 32768 if kind == "decode" else 8192)
        klo = rng.choice((khi, rng.randint(1, khi)))
        if kind == "decode":
            qlo = qhi = rng.choice((1, 1, 1, 2, 4))
        elif kind == "prompt":
            qlo = qhi = klo = khi
        else:
            qhi = _log_int(rng, 2, 2048)
            qlo = qhi if kind == "chunk" else 1
        klo, khi = max(klo, qhi), max(khi, qhi)
        causal = rng.random() < 0.9
        if rng.random() < 0.2:
            window = _log_int(rng, 16, 4096)
    elif op == "tree":
        n = qlo = qhi = _log_int(rng, 2, 128)
        khi = n + _log_int(rng, 1, 16384)
        klo = rng.choice((khi, rng.randint(n, khi)))
    else:
        n = _log_int(rng, 2, 128)
        qlo, qhi = rng.choice(((0, n), (1, min(n, 8)), (n, n)))
        khi = n + _log_int(rng, 1, 512)
        klo = rng.randint(n, khi)
    case = _case(None, op, dtype, i8, b, hq, hkv, d, page, klo, khi, qlo, qhi, n, rope, causal, window)
    while True:
        w = work(case)
        pool = case["b"] * (case["khi"] + page) * hkv * d if op in ("append", "commit") else 0
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES and pool <= MAX_POOL:
            return case
        if case["b"] > 1:
            case["b"] //= 2
            continue
        if case["qlo"] == case["khi"]:  # a prompt
            case["qlo"] = case["qhi"] = case["klo"] = case["khi"] = int(case["khi"] * 0.7)
        else:
            case["khi"] = max(case["qhi"], case["n"], int(case["khi"] * 0.7))
            case["klo"] = min(case["klo"], case["khi"])


def lengths(case):
    """(keys, new rows) of each sequence, from the case alone."""
    rng = random.Random(" ".join(str(case[k]) for k in KEYS))
    out = []
    for i in range(case["b"]):
        k = rng.randint(case["klo"], case["khi"])
        q = rng.randint(case["qlo"], case["qhi"])
        if case["op"] == "attn" and case["qlo"] == 1 and case["qhi"] > 4 and i % 4:
            q = 1  # a mixed batch: most sequences decode
        if case["op"] != "commit":
            k = max(k, q)
        if case["op"] == "attn" and case["qlo"] == case["klo"] == case["khi"]:
            q = k
        out.append((k, q))
    return out


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _tree(n, rng):
    """Ancestors (and self) of n drafts, parents before children."""
    seen = []
    for i in range(n):
        row = [False] * n
        if i > 0:
            row = list(seen[rng.randint(max(0, i - 8), i - 1)])
        row[i] = True
        seen.append(row)
    return seen


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    rng = random.Random(int(seed))
    dt = torch.float16 if case["dtype"] == "f16" else torch.bfloat16
    b, hq, hkv, d, page, n = (case[k] for k in ("b", "hq", "hkv", "d", "page", "n"))
    lens = lengths(case)
    width = max((k + page - 1) // page for k, _ in lens)
    need = [(k + page - 1) // page for k, _ in lens]
    pages = sum(need)
    order = list(range(pages))
    rng.shuffle(order)  # pages are handed out as they become free
    table, at = [], 0
    for m in need:
        table.append(order[at:at + m] + [0] * (width - m))
        at += m

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    st = {"case": case, "lens": lens, "table": ints(table), "seq_lens": ints([k for k, _ in lens])}
    if case["i8"]:
        for c in ("k", "v"):
            st[c + "_cache"] = torch.randint(-127, 128, (pages, page, hkv, d), generator=g, device=dev,
                                             dtype=torch.int8)
            # a row's scale is its largest magnitude / 127
            st[c + "_scale"] = (2.0 + torch.rand(pages, page, hkv, generator=g, device=dev)) / 127.0
    else:
        st["k_cache"], st["v_cache"] = randn(pages, page, hkv, d), randn(pages, page, hkv, d)
        st["k_scale"] = st["v_scale"] = None
    if case["op"] == "commit":
        st["prefix"] = ints([k - n for k, _ in lens])
        paths = []
        for _, q in lens:
            # the first drafts of the path were also the first of the tree, the others are behind
            # the places that the path moves to
            m = max(2 * q - n, rng.randint(0, min(q, 2)))
            path = list(range(m)) + sorted(rng.sample(range(q, n), q - m))
            paths.append(path + [-1] * (n - q))
        st["path"], st["accepted"] = ints(paths), ints([q for _, q in lens])
        return st
    rows = sum(q for _, q in lens)
    cu = [0]
    for _, q in lens:
        cu.append(cu[-1] + q)
    st["cu"] = ints(cu)
    st["uniform"] = len(set(q for _, q in lens)) == 1
    st["max_q"] = max(q for _, q in lens)
    st["q"] = randn(rows, hq, d)
    if case["op"] == "append":
        st["k"], st["v"] = randn(rows, hkv, d), randn(rows, hkv, d)
        if case["rope"] != "none":
            inv = 10000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
            ang = torch.arange(max(k for k, _ in lens), device=dev, dtype=torch.float64)[:, None] * inv
            st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
    if case["op"] == "tree":
        st["mask"] = torch.tensor([_tree(n, rng) for _ in range(b)], dtype=torch.bool, device=dev)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _dequantised(st):
    """What the int8 caches stand for, in the type of the rows they come from."""
    dt = torch.float16 if st["case"]["dtype"] == "f16" else torch.bfloat16
    return ((st["k_cache"].float() * st["k_scale"][..., None]).to(dt),
            (st["v_cache"].float() * st["v_scale"][..., None]).to(dt))


def _run_own(st):
    import rdnattention

    case = st["case"]
    scales = {"key_scale": st["k_scale"], "value_scale": st["v_scale"]} if case["i8"] else {}
    caches = (st["k_cache"], st["v_cache"])
    if case["op"] == "commit":
        rdnattention.paged_commit(*caches, st["table"], st["prefix"], st["path"], st["accepted"], **scales)
        return _dequantised(st) if case["i8"] else caches
    rows = {} if st["uniform"] else {"cu_seqlens_q": st["cu"]}
    if case["op"] == "append":
        rope = {}
        if case["rope"] != "none":
            rope = {"query": st["q"], "rot_cos": st["cos"], "rot_sin": st["sin"],
                    "rot_interleaved": case["rope"] == "pairs"}
        q = rdnattention.paged_append(st["k"], st["v"], *caches, st["table"], st["seq_lens"], **rows, **rope, **scales)
        out = _dequantised(st) if case["i8"] else caches
        return (q,) + out if rope else out
    if case["op"] == "tree":
        return rdnattention.paged_tree_attention(st["q"], *caches, st["table"], st["seq_lens"], st["mask"], **rows,
                                                 **scales)
    if rows:
        rows["max_seqlen_q"] = st["max_q"]
    return rdnattention.paged_attention(st["q"], *caches, st["table"], st["seq_lens"], is_causal=case["causal"],
                                        window_size=case["window"], **rows, **scales)


def _rotated(x, cos, sin, rope, wide):
    """x [rows, heads, d], cos / sin [rows, d / 2]: rotated, in x's type (in 64
    bits before that where the result is quantised: next to a border the last
    bit decides)."""
    xf = x.double() if wide else x.float()
    c, s = cos[:, None].to(xf.dtype), sin[:, None].to(xf.dtype)
    out = torch.empty_like(xf)
    half = x.shape[-1] // 2
    first, second = (slice(0, None, 2), slice(1, None, 2)) if rope == "pairs" else (slice(0, half), slice(half, None))
    a, b = xf[..., first], xf[..., second]
    out[..., first] = a * c - b * s
    out[..., second] = a * s + b * c
    return out.to(x.dtype)


def _to_int8(x):
    """(int8, scale per row): the per-token scheme of quantize_int8_qk_pertoken."""
    x = x.float()
    s = x.abs().amax(-1, keepdim=True) * (1.0 / 127.0)
    s = torch.where(s == 0, torch.ones_like(s), s)
    return torch.clamp(torch.round(x / s), -127, 127).to(torch.int8), s.squeeze(-1)


def _plain_append(st):
    case, page = st["case"], st["case"]["page"]
    cu, lens = st["cu"], st["seq_lens"]
    t = torch.arange(st["k"].shape[0], device=cu.device, dtype=torch.int32)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = (lens - cu[1:])[seq] + t  # the last new row is the sequence's last key
    q, k, v = st["q"], st["k"], st["v"]
    rope = case["rope"]
    if rope != "none":
        cos, sin = st["cos"][pos], st["sin"][pos]
        q, k = _rotated(q, cos, sin, rope, False), _rotated(k, cos, sin, rope, case["i8"])
    pg, off = st["table"][seq, pos // page].long(), (pos % page).long()
    if case["i8"]:
        k, ks = _to_int8(k)
        v, vs = _to_int8(v)
        st["k_scale"][pg, off] = ks
        st["v_scale"][pg, off] = vs
    st["k_cache"][pg, off] = k
    st["v_cache"][pg, off] = v
    out = _dequantised(st) if case["i8"] else (st["k_cache"], st["v_cache"])
    return (q,) + out if rope != "none" else out


def _visible(case, keys, rows, device):
    """Which keys each of a sequence's rows sees (causal rows end at the last
    key, a causal window counts back from there, a two-sided one spans
    window / 2 keys each way)."""
    at = torch.arange(keys - rows, keys, device=device)[:, None]
    key = torch.arange(keys, device=device)[None]
    ok = torch.ones(rows, keys, dtype=torch.bool, device=device)
    w = case["window"]
    if case["causal"]:
        ok &= key <= at
        if w > 0:
            ok &= at - key < w
    elif w > 0:
        ok &= (at - key).abs() <= w // 2
    return ok


def _plain_attention(st):
    case, page = st["case"], st["case"]["page"]
    hq, hkv, d, n = case["hq"], case["hkv"], case["d"], case["n"]
    ratio = hq // hkv
    out = torch.empty_like(st["q"])
    at = 0
    for i, (keys, rows) in enumerate(st["lens"]):
        pages = st["table"][i, :(keys + page - 1) // page].long()
        k = st["k_cache"][pages].flatten(0, 1)[:keys].float()
        v = st["v_cache"][pages].flatten(0, 1)[:keys].float()
        if case["i8"]:
            k = k * st["k_scale"][pages].flatten(0, 1)[:keys, :, None]
            v = v * st["v_scale"][pages].flatten(0, 1)[:keys, :, None]
        k, v = k.permute(1, 2, 0).contiguous(), v.transpose(0, 1).contiguous()
        if case["op"] == "tree":
            ok = torch.ones(rows, keys, dtype=torch.bool, device=k.device)
            ok[:, keys - rows:] = st["mask"][i, :rows, :rows]
        else:
            ok = _visible(case, keys, rows, k.device)
        q = st["q"][at:at + rows].float().reshape(rows, hkv, ratio, d).permute(1, 2, 0, 3).contiguous()
        step = max(1, (1 << 29) // max(1, ratio * rows * keys))  # kv heads at a time: 2 GB of scores
        for h in range(0, hkv, step):
            qh = q[h:h + step].flatten(1, 2)
            s = torch.matmul(qh, k[h:h + step]) * d ** -0.5
            s = s.reshape(-1, ratio, rows, keys).masked_fill_(~ok, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p.reshape(-1, ratio * rows, keys), v[h:h + step]).reshape(-1, ratio, rows, d)
            o = o / torch.where(total == 0, torch.ones_like(total), total)
            out[at:at + rows, h * ratio:(h + step) * ratio] = o.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
        at += rows
    return out


def _plain_commit(st):
    case, page = st["case"], st["case"]["page"]
    path, prefix, table = st["path"], st["prefix"], st["table"]
    i = torch.arange(path.shape[1], device=path.device, dtype=torch.int32)[None]
    src = prefix[:, None] + torch.where(i < st["accepted"][:, None], path, i)
    dst = prefix[:, None] + i
    spg, dpg = (table.gather(1, (x // page).long()).long() for x in (src, dst))
    so, do = (src % page).long(), (dst % page).long()
    parts = ("k_cache", "v_cache") + (("k_scale", "v_scale") if case["i8"] else ())
    for name in parts:
        st[name][dpg, do] = st[name][spg, so]
    return _dequantised(st) if case["i8"] else (st["k_cache"], st["v_cache"])


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _plain_append(state) if op == "append" else _plain_commit(state) if op == "commit" else \
        _plain_attention(state)


# ---------------------------------------------------------------------------
# work and accuracy
# ---------------------------------------------------------------------------
def work(case):
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    lens = lengths(case)
    row = hkv * (d * (1 if case["i8"] else 2) + (4 if case["i8"] else 0))  # a cached token's keys, or its values
    rows = sum(q for _, q in lens)
    tables = 4 * (2 * b + sum((k + case["page"] - 1) // case["page"] for k, _ in lens))
    if case["op"] == "commit":
        # the whole caches of int8 are also returned in 16 bits
        pool = sum((k + case["page"] - 1) // case["page"] * case["page"] for k, _ in lens)
        extra = 2 * pool * (row + hkv * d * 2) if case["i8"] else 0
        return {"bytes": rows * 4 * row + 4 * b * case["n"] + tables + extra, "flops": rows}
    if case["op"] == "append":
        size = rows * (2 * hkv * d * 2 + 2 * row)
        flops = 0
        if case["rope"] != "none":
            size += rows * 2 * hq * d * 2 + max(k for k, _ in lens) * d * 4
            flops += rows * (hq + hkv) * d * 3
        if case["i8"]:
            pool = sum((k + case["page"] - 1) // case["page"] * case["page"] for k, _ in lens)
            size += 2 * pool * (row + hkv * d * 2)
            flops += rows * hkv * d * 6
        return {"bytes": size + tables, "flops": max(flops, rows)}
    pairs = keys = 0
    for k, q in lens:
        lo, hi = 0, k - 1  # keys that some row sees
        w = case["window"]
        if case["op"] == "tree":
            pairs += q * k
        else:
            first, last = k - q, k - 1
            if w > 0:
                lo = max(0, first - (w - 1 if case["causal"] else w // 2))
            if not case["causal"] and w <= 0:
                pairs += q * k
            else:
                for at in (first, last) if q > 64 else range(first, last + 1):
                    a = max(0, at - (w - 1 if case["causal"] else w // 2)) if w > 0 else 0
                    z = at if case["causal"] else min(k - 1, at + w // 2)
                    pairs += (z - a + 1) * (q / 2 if q > 64 else 1)
        keys += hi - lo + 1
    return {"bytes": rows * hq * d * 4 + 2 * keys * row + tables, "flops": int(4 * hq * pairs * d)}


def _exact_rows(st, i):
    """Sequence i's cached keys and values in 64 bits, [hkv, keys, d]."""
    case, page = st["case"], st["case"]["page"]
    keys = st["lens"][i][0]
    at = torch.arange(keys, device=st["table"].device)
    pg, off = st["table"][i].long()[at // page], at % page
    k, v = st["k_cache"][pg, off].double(), st["v_cache"][pg, off].double()
    if case["i8"]:
        k, v = k * st["k_scale"][pg, off].double()[..., None], v * st["v_scale"][pg, off].double()[..., None]
    return k.transpose(0, 1), v.transpose(0, 1)


def _exact_attention(st):
    case = st["case"]
    ratio = case["hq"] // case["hkv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    at = 0
    for i, (keys, rows) in enumerate(st["lens"]):
        k, v = _exact_rows(st, i)
        for h in range(case["hq"]):
            kt, vh = k[h // ratio].t().contiguous(), v[h // ratio].contiguous()
            block = max(1, (1 << 27) // (8 * keys))
            for r in range(0, rows, block):
                n = min(block, rows - r)
                s = st["q"][at + r:at + r + n, h].double() @ kt / math.sqrt(case["d"])
                row = torch.arange(r, r + n, device=s.device)[:, None]
                key = torch.arange(keys, device=s.device)[None]
                pos = keys - rows + row
                if case["op"] == "tree":
                    draft = (key - (keys - rows)).clamp(min=0)
                    hide = (key >= keys - rows) & ~st["mask"][i][row, draft]
                elif case["causal"]:
                    hide = key > pos
                    if case["window"] > 0:
                        hide = hide | (key <= pos - case["window"])
                else:
                    hide = torch.zeros_like(key > pos)
                    if case["window"] > 0:
                        hide = (key > pos + case["window"] // 2) | (key < pos - case["window"] // 2)
                s = s.masked_fill(hide, -math.inf)
                p = torch.softmax(s, -1).nan_to_num(0.0)
                out[at + r:at + r + n, h] = p @ vh
        at += rows
    return out


def _exact_append(st):
    case, page = st["case"], st["case"]["page"]
    d, rope = case["d"], case["rope"]
    k_all, v_all = st["k_cache"].double(), st["v_cache"].double()
    if case["i8"]:
        k_all, v_all = k_all * st["k_scale"].double()[..., None], v_all * st["v_scale"].double()[..., None]
    q_all = st["q"].double()

    def turned(x, pos):
        c, s = st["cos"][pos].double()[:, None], st["sin"][pos].double()[:, None]
        z = torch.complex(c.expand(-1, x.shape[1], -1).contiguous(), s.expand(-1, x.shape[1], -1).contiguous())
        if rope == "pairs":
            w = torch.view_as_complex(x.double().reshape(*x.shape[:-1], d // 2, 2).contiguous()) * z
            return torch.view_as_real(w).flatten(-2)
        w = torch.complex(x[..., :d // 2].double().contiguous(), x[..., d // 2:].double().contiguous()) * z
        return torch.cat((w.real, w.imag), -1)

    def stored(x):
        if not case["i8"]:
            return x
        x = x.to(st["k"].dtype).double()  # rotated rows have the new keys' type before they are quantised
        # scales are 32-bit numbers: the largest magnitude times the 32-bit 1 / 127
        s = (x.abs().amax(-1, keepdim=True) * torch.tensor(1 / 127, dtype=torch.float32).item()).float().double()
        s = torch.where(s == 0, torch.ones_like(s), s)
        # and so are the quotients that are rounded to whole numbers
        return (x / s).float().double().round().clamp(-127, 127) * s

    at = 0
    for i, (keys, rows) in enumerate(st["lens"]):
        pos = torch.arange(keys - rows, keys, device=st["table"].device)
        pg, off = st["table"][i].long()[pos // page], pos % page
        k, v = st["k"][at:at + rows].double(), st["v"][at:at + rows].double()
        if rope != "none":
            k = turned(st["k"][at:at + rows], pos)
            q_all[at:at + rows] = turned(st["q"][at:at + rows], pos)
        k_all[pg, off] = stored(k)
        v_all[pg, off] = stored(v)
        at += rows
    return (q_all, k_all, v_all) if rope != "none" else (k_all, v_all)


def _exact_commit(st):
    case, page = st["case"], st["case"]["page"]
    caches = [st[c + "_cache"].double() * (st[c + "_scale"].double()[..., None] if case["i8"] else 1) for c in "kv"]
    for i, (keys, accepted) in enumerate(st["lens"]):
        src = keys - case["n"] + st["path"][i, :accepted].long()
        dst = keys - case["n"] + torch.arange(accepted, device=src.device)
        table = st["table"][i].long()
        for x in caches:
            x[table[dst // page], dst % page] = x[table[src // page], src % page].clone()
    return tuple(caches)


def exact(case, seed):
    """The operators' definitions in 64 bits on the same inputs."""
    st = prepare(case, seed)
    op = case["op"]
    return _exact_append(st) if op == "append" else _exact_commit(st) if op == "commit" else _exact_attention(st)

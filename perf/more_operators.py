"""More operators of the paged key/value cache whose speed is tracked.

A server that keeps keys and values in pages (see paged_attention) also calls:

  norm     paged_append with norm weights: each head of a step's queries and
           keys is divided by its root mean square and rotated on the way into
           the cache, by one position per row or by several (time, height and
           width of image and video tokens), each for its own frequencies
  prefix   paged_prefix_attention: sequences whose own keys follow a prefix that
           a group of them shares
  weights  paged_key_weights: the attention that each cached key has received
           from a step's rows, added to its weight
  evict    paged_evict: of each head, the keys of the largest weights move up to
           the front, the first and the newest ones among them

listed() holds the fixed cases, draw() gives others of the same ranges.  A case
is a dict of plain values:
  op      the operator
  dtype   "f16" or "bf16", of the rows
  i8      whether the cache holds int8 with a scale per token and head
  b       sequences
  hq, hkv, d, page
  klo, khi   the sequences' own keys, new rows among them
  qlo, qhi   new rows per sequence
  rope    norm: "none", "pairs" (channels 2i, 2i + 1) or "halves" (i, i + d/2)
  axes    norm: positions per row; 0: the row's index in its sequence
  plo, phi, groups   prefix: the prefixes' lengths, and how many there are
  budget, first, recent   evict: keys kept of each sequence, of which the first
          and the newest in any case
Where lo < hi the sequences are ragged; their lengths follow from the case
alone.
"""
import math
import random

import numpy as np
import torch

own = False

KEYS = ("op", "dtype", "i8", "b", "hq", "hkv", "d", "page", "klo", "khi", "qlo", "qhi", "rope", "axes", "plo", "phi",
        "groups", "budget", "first", "recent")

# a drawn case asks for at most this much (below the largest listed ones)
MAX_FLOPS = 1.2e11
MAX_BYTES = 5.5e8
# the caches that are returned whole stay below this many elements
MAX_POOL = 24_000_000
# ... and the plain form's scores of padded rows and keys
MAX_SCORES = 2_000_000_000


def _case(name, *values):
    case = dict(zip(KEYS, values))
    return dict(case, name=name) if name else case


def listed():
    return [
        # one sequence, one new token of an 8B-class grouped-query layer: the smallest call
        _case("norm_b1", "norm", "f16", False, 1, 32, 8, 128, 16, 500, 500, 1, 1, "halves", 0, 0, 0, 0, 0, 0, 0),
        # ragged prompts of text and images, positions of three axes: memory bound
        _case("norm_axes_prompts_bf16", "norm", "bf16", False, 4, 32, 8, 128, 16, 1, 1, 600, 2200, "halves", 3, 0, 0, 0,
              0, 0, 0),
        # chunks of prompts into an int8 cache, behind keys of earlier chunks
        _case("norm_chunks_i8", "norm", "f16", True, 5, 16, 4, 64, 32, 1, 1000, 150, 900, "pairs", 1, 0, 0, 0, 0, 0, 0),
        # a few sequences that have just begun behind one instruction text: latency counts
        _case("prefix_b8_p1000", "prefix", "f16", False, 8, 32, 8, 128, 16, 1, 60, 1, 1, "none", 0, 1000, 1000, 1, 0, 0,
              0),
        # a served batch, one new token each, behind one long document
        _case("prefix_b64_p8192_bf16", "prefix", "bf16", False, 64, 32, 8, 128, 16, 20, 500, 1, 1, "none", 0, 8192,
              8192, 1, 0, 0, 0),
        # four documents, each with its own readers, in an int8 cache
        _case("prefix_b40_g4_i8", "prefix", "f16", True, 40, 32, 8, 128, 16, 10, 300, 1, 1, "none", 0, 500, 6000, 4, 0,
              0, 0),
        # chunks of questions about one document, some sequences already decoding: matrix products
        _case("prefix_chunks_p8192", "prefix", "f16", False, 6, 32, 8, 128, 32, 300, 900, 1, 300, "none", 0, 8192, 8192,
              1, 0, 0, 0),
        # one sequence, one new token: latency counts
        _case("weights_b1_k2000", "weights", "f16", False, 1, 32, 8, 128, 16, 2000, 2000, 1, 1, "none", 0, 0, 0, 0, 0,
              0, 0),
        # a served batch with long, ragged caches: memory bound
        _case("weights_b16_bf16", "weights", "bf16", False, 16, 32, 8, 128, 64, 4000, 32768, 1, 1, "none", 0, 0, 0, 0,
              0, 0, 0),
        # whole prompts: matrix products
        _case("weights_prompts_b2", "weights", "f16", False, 2, 32, 8, 128, 32, 4096, 4096, 4096, 4096, "none", 0, 0, 0,
              0, 0, 0, 0),
        # short caches cut to their budget
        _case("evict_b4_k600", "evict", "f16", False, 4, 32, 8, 128, 16, 600, 600, 1, 1, "none", 0, 0, 0, 0, 512, 4,
              128),
        # ragged long ones, some of them short of the budget
        _case("evict_b6_k3900_bf16", "evict", "bf16", False, 6, 32, 8, 128, 64, 900, 3900, 1, 1, "none", 0, 0, 0, 0,
              1024, 4, 256),
    ]


HEADS = ((8, 8), (16, 16), (32, 8), (32, 8), (16, 4), (16, 8), (40, 8), (32, 1))


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(("norm", "norm", "prefix", "prefix", "prefix", "weights", "weights", "evict"))
    hq, hkv = rng.choice(HEADS)
    i8 = rng.random() < 0.25
    dtype = rng.choice(("f16", "bf16"))
    d = rng.choice((64, 128)) if i8 else rng.choice((64, 128, 128, 32 * rng.randint(1, 8)))
    page = rng.choice((16, 16, 32, 64, 128))
    b = _log_int(rng, 1, 64)
    rope, axes, plo, phi, groups, budget, first, recent = "none", 0, 0, 0, 0, 0, 0, 0
    qlo = qhi = 1
    if op == "norm":
        if rng.random() < 0.5:  # prompts
            qhi = _log_int(rng, 8, 2000)
            qlo = rng.randint(1, qhi)
        khi = qhi + _log_int(rng, 1, 300)
        klo = rng.randint(qhi, khi)
        rope = rng.choice(("none", "pairs", "halves", "halves"))
        axes = 0 if rope == "none" else rng.choice((0, 1, 2, 3))
    elif op == "prefix":
        phi = _log_int(rng, 50, 16384)
        plo = rng.choice((phi, rng.randint(1, phi)))
        groups = rng.choice((1, 1, rng.randint(1, min(b, 6))))
        if rng.random() < 0.3:
            qhi = _log_int(rng, 2, 400)
            qlo = rng.choice((1, qhi))
        khi = qhi + _log_int(rng, 1, 1000)
        klo = rng.randint(qhi, khi)
    elif op == "weights":
        khi = _log_int(rng, 16, 32768)
        klo = rng.choice((khi, rng.randint(1, khi)))
        kind = rng.choice(("decode", "decode", "last", "prompt"))
        if kind == "last":  # the last rows of each prompt
            qlo = qhi = min(klo, rng.choice((16, 32, 64)))
        elif kind == "prompt":
            khi = klo = qlo = qhi = _log_int(rng, 16, 4000)
    else:
        khi = _log_int(rng, 64, 16384)
        klo = rng.choice((khi, rng.randint(1, khi)))
        budget = max(1, int(khi * rng.uniform(0.1, 0.9)))
        first = min(4, budget // 4)
        recent = int(budget * rng.uniform(0.0, 0.5))
    case = _case(None, op, dtype, i8, b, hq, hkv, d, page, klo, khi, qlo, qhi, rope, axes, plo, phi, groups, budget,
                 first, recent)
    while True:
        w = work(case)
        pool = case["b"] * (case["khi"] + page) * hkv * d if op in ("norm", "evict") else 0
        scores = case["b"] * hq * case["qhi"] * (case["khi"] + case["phi"] * case["groups"])
        scores = 0 if op in ("norm", "evict") else scores
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES and pool <= MAX_POOL and scores <= MAX_SCORES:
            return case
        if case["b"] > 1:
            case["b"] //= 2
            case["groups"] = min(case["groups"], case["b"])
            continue
        if case["qlo"] == case["khi"]:  # a prompt
            case["qlo"] = case["qhi"] = case["klo"] = case["khi"] = int(case["khi"] * 0.7)
        else:
            case["phi"] = int(case["phi"] * 0.7)
            case["plo"] = min(case["plo"], case["phi"])
            case["khi"] = max(case["qhi"], case["budget"], int(case["khi"] * 0.7))
            case["klo"] = min(case["klo"], case["khi"])
            if case["khi"] == case["budget"]:
                case["budget"] = max(case["first"] + case["recent"], int(case["budget"] * 0.7), 1)


def lengths(case):
    """(own keys, new rows) of each sequence, from the case alone."""
    rng = random.Random(" ".join(str(case[k]) for k in KEYS))
    out = []
    for i in range(case["b"]):
        k = rng.randint(case["klo"], case["khi"])
        q = rng.randint(case["qlo"], case["qhi"])
        if case["op"] == "prefix" and case["qlo"] == 1 and case["qhi"] > 4 and i % 3 == 2:
            q = 1  # a mixed batch: some sequences decode
        k = max(k, q)
        if case["op"] == "weights" and case["qlo"] == case["klo"] == case["khi"]:
            q = k
        out.append((k, q))
    return out


def prefixes(case):
    """(keys, sequences) of each prefix, from the case alone."""
    rng = random.Random("prefixes " + " ".join(str(case[k]) for k in KEYS))
    cuts = sorted(rng.sample(range(1, case["b"]), case["groups"] - 1)) if case["groups"] > 1 else []
    ends = [0] + cuts + [case["b"]]
    return [(rng.randint(case["plo"], case["phi"]), z - a) for a, z in zip(ends, ends[1:])]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _positions(n, first, axes, rng):
    """Positions of n rows from index `first` on: text counts on all axes alike, an
    image's patches share the time and count rows and columns from there."""
    out, at, i = [], first, 0
    while i < n:
        text = rng.randint(1, 60)
        out += [[at + j] * axes for j in range(min(text, n - i))]
        i, at = i + text, at + text
        high, wide = rng.randint(4, 24), rng.randint(4, 24)
        out += [[at, at + j // wide, at + j % wide][:axes] for j in range(max(0, min(high * wide, n - i)))]
        i, at = i + high * wide, at + max(high, wide)
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    rng = random.Random(int(seed))
    dt = torch.float16 if case["dtype"] == "f16" else torch.bfloat16
    hq, hkv, d, page = (case[k] for k in ("hq", "hkv", "d", "page"))
    lens = lengths(case)
    shared = prefixes(case) if case["op"] == "prefix" else []
    need = [(k + page - 1) // page for k, _ in lens + shared]
    pages = sum(need)
    order = list(range(pages))
    rng.shuffle(order)  # pages are handed out as they become free
    rows_of, at = [], 0
    for m in need:
        rows_of.append(order[at:at + m])
        at += m

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    def table(lists):
        width = max(len(x) for x in lists)
        return ints([x + [0] * (width - len(x)) for x in lists])

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    st = {"case": case, "table": table(rows_of[:len(lens)]), "seq_lens": ints([k for k, _ in lens]),
          "max_k": max(k for k, _ in lens), "max_q": max(q for _, q in lens), "uniform": len({q for _, q in lens}) == 1}
    for c in "k" if case["op"] == "weights" else "kv":
        st[c + "_scale"] = None
        if case["i8"]:
            st[c + "_cache"] = torch.randint(-127, 128, (pages, page, hkv, d), generator=g, device=dev,
                                             dtype=torch.int8)
            # a row's scale is its largest magnitude / 127
            st[c + "_scale"] = (2.0 + torch.rand(pages, page, hkv, generator=g, device=dev)) / 127.0
        else:
            st[c + "_cache"] = randn(pages, page, hkv, d)
    if case["op"] == "evict":
        # some keys are looked at by most rows, most by few
        w = torch.rand(pages, page, hkv, generator=g, device=dev)
        st["weights"] = 0.02 * (1.0 / (w + 1e-3) - 0.99)
        st["key_weights"] = torch.empty_like(st["weights"])
        return st
    rows = sum(q for _, q in lens)
    cu = [0]
    for _, q in lens:
        cu.append(cu[-1] + q)
    st["cu"] = ints(cu)
    st["q"] = randn(rows, hq, d)
    if case["op"] == "norm":
        st["k"], st["v"] = randn(rows, hkv, d), randn(rows, hkv, d)
        st["q_norm"], st["k_norm"] = (1.0 + 0.3 * randn(d, dtype=torch.float32) for _ in range(2))
        if case["rope"] != "none":
            inv = 1000000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
            ang = torch.arange(2 * max(k for k, _ in lens) + 64, device=dev, dtype=torch.float64)[:, None] * inv
            st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        if case["axes"]:
            st["positions"] = ints([p for k, q in lens for p in _positions(q, k - q, case["axes"], rng)])
            # the frequencies' axes in turn, or one axis after the other
            cols = range(d // 2)
            st["rot_axes"] = ints([c % case["axes"] if case["rope"] == "halves" else c * case["axes"] // (d // 2)
                                   for c in cols])
    if case["op"] == "prefix":
        st["prefix_table"], st["prefix_lens"] = table(rows_of[len(lens):]), ints([k for k, _ in shared])
        st["max_p"] = max(k for k, _ in shared)
        seqs = [0]
        for _, n in shared:
            seqs.append(seqs[-1] + n)
        st["prefix_seqs"] = ints(seqs)
    if case["op"] == "weights":
        st["key_weights"] = torch.rand(pages, page, hkv, generator=g, device=dev)
        st["lse"] = _attend(st, st["q"], st["cu"], st["max_q"], st["table"], st["seq_lens"], st["max_k"], True,
                            False)[1]
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _dequantised(st):
    """What the int8 caches stand for, in the type of the rows they come from."""
    dt = torch.float16 if st["case"]["dtype"] == "f16" else torch.bfloat16
    return ((st["k_cache"].float() * st["k_scale"][..., None]).to(dt),
            (st["v_cache"].float() * st["v_scale"][..., None]).to(dt))


def _caches(st):
    return _dequantised(st) if st["case"]["i8"] else (st["k_cache"], st["v_cache"])


def _run_own(st):
    import rdnattention

    case = st["case"]
    scales = {}
    if case["i8"] and case["op"] != "weights":
        scales = {"key_scale": st["k_scale"], "value_scale": st["v_scale"]}
    rows = {} if st["uniform"] else {"cu_seqlens_q": st.get("cu")}
    if case["op"] == "norm":
        rope = {}
        if case["rope"] != "none":
            rope = {"rot_cos": st["cos"], "rot_sin": st["sin"], "rot_interleaved": case["rope"] == "pairs"}
        if case["axes"]:
            rope.update(positions=st["positions"], rot_axes=st["rot_axes"])
        q = rdnattention.paged_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"], st["seq_lens"],
                                      query=st["q"], query_norm=st["q_norm"], key_norm=st["k_norm"], norm_eps=1e-6,
                                      **rows, **rope, **scales)
        return (q,) + _caches(st)
    if case["op"] == "prefix":
        if rows:
            rows["max_seqlen_q"] = st["max_q"]
        return rdnattention.paged_prefix_attention(st["q"], st["k_cache"], st["v_cache"], st["prefix_table"],
                                                   st["prefix_lens"], st["table"], st["seq_lens"],
                                                   prefix_seqs=st["prefix_seqs"], return_lse=True, **rows, **scales)
    if case["op"] == "weights":
        rdnattention.paged_key_weights(st["q"], st["lse"], st["k_cache"], st["table"], st["seq_lens"],
                                       st["key_weights"], key_scale=st["k_scale"], decay=0.75, **rows)
        return st["key_weights"]
    st["key_weights"].copy_(st["weights"])  # as the steps before left them
    lens, kept = rdnattention.paged_evict(st["k_cache"], st["v_cache"], st["table"], st["seq_lens"], st["key_weights"],
                                          case["budget"], first=case["first"], recent=case["recent"], **scales)
    return (lens, kept, st["key_weights"]) + _caches(st)


def _plain_norm(st):
    case, page = st["case"], st["case"]["page"]
    cu, lens = st["cu"], st["seq_lens"]
    t = torch.arange(st["k"].shape[0], device=cu.device, dtype=torch.int32)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = (lens - cu[1:])[seq] + t  # the last new row is the sequence's last key
    if case["rope"] != "none":
        if case["axes"]:
            at = st["positions"].long()[:, st["rot_axes"].long()]
            cos, sin = st["cos"].gather(0, at), st["sin"].gather(0, at)
        else:
            cos, sin = st["cos"][pos], st["sin"][pos]

    def turned(x, weight, wide):
        """Normed and rotated, in x's type (in 64 bits before that where the result is
        quantised: next to a border the last bit decides)."""
        xf = x.double() if wide else x.float()
        xf = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + 1e-6) * weight.to(xf.dtype)
        if case["rope"] == "none":
            return xf.to(x.dtype)
        c, s = cos[:, None].to(xf.dtype), sin[:, None].to(xf.dtype)
        out, half = torch.empty_like(xf), case["d"] // 2
        first, second = (slice(0, None, 2), slice(1, None, 2)) if case["rope"] == "pairs" else \
            (slice(0, half), slice(half, None))
        a, b = xf[..., first], xf[..., second]
        out[..., first] = a * c - b * s
        out[..., second] = a * s + b * c
        return out.to(x.dtype)

    def to_int8(x):
        x = x.float()
        s = x.abs().amax(-1, keepdim=True) * (1.0 / 127.0)
        s = torch.where(s == 0, torch.ones_like(s), s)
        return torch.clamp(torch.round(x / s), -127, 127).to(torch.int8), s.squeeze(-1)

    q, k, v = turned(st["q"], st["q_norm"], False), turned(st["k"], st["k_norm"], case["i8"]), st["v"]
    pg, off = st["table"][seq, pos // page].long(), (pos % page).long()
    if case["i8"]:
        k, st["k_scale"][pg, off] = to_int8(k)
        v, st["v_scale"][pg, off] = to_int8(v)
    st["k_cache"][pg, off] = k
    st["v_cache"][pg, off] = v
    return (q,) + _caches(st)


def _padded(st, cache, scale, table, n):
    """The first n keys (or values) of each of the table's rows, [rows, hkv, n, d] in
    32 bits, int8 ones times their scales."""
    page = st["case"]["page"]
    table = table[:, :(n + page - 1) // page].long()
    x = cache[table].flatten(1, 2)[:, :n].float()
    if scale is not None:
        x = x * scale[table].flatten(1, 2)[:, :n, :, None]
    return x.transpose(1, 2).contiguous()


def _row_places(cu, rows):
    t = torch.arange(rows, device=cu.device, dtype=torch.int32)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    return seq, (t - cu[seq]).long()


def _scores(st, q, cu, max_q, table, lens, max_k, causal):
    """Scores of padded rows and keys, [sequences, hkv, max_q, ratio, max_k], -inf
    where a row does not see a key, and the rows' places in them."""
    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    seq, i = _row_places(cu, q.shape[0])
    b = table.shape[0]
    qp = torch.zeros(b, max_q, hq, d, device=q.device)
    qp[seq, i] = q.float()
    qp = qp.reshape(b, max_q, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(b * hkv, -1, d).contiguous()
    k = _padded(st, st["k_cache"], st["k_scale"], table, max_k)
    s = torch.bmm(qp, k.flatten(0, 1).transpose(1, 2).contiguous()) * d ** -0.5
    s = s.reshape(b, hkv, max_q, hq // hkv, max_k)
    key = torch.arange(max_k, device=q.device)
    hide = (key >= lens[:, None])[:, None]
    if causal:
        at = (lens - (cu[1:] - cu[:-1]))[:, None] + torch.arange(max_q, device=q.device)
        hide = hide | (key > at[..., None])
    return s.masked_fill_(hide[:, None, :, None], -math.inf), seq, i


def _attend(st, q, cu, max_q, table, lens, max_k, causal, values):
    """Attention of the rows over one of their parts: (output or None, log-sum-exp)."""
    case = st["case"]
    s, seq, i = _scores(st, q, cu, max_q, table, lens, max_k, causal)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).squeeze(-1).permute(0, 2, 1, 3).flatten(2)[seq, i]
    if not values:
        return None, lse
    v = _padded(st, st["v_cache"], st["v_scale"], table, max_k)
    o = torch.bmm(p.flatten(0, 1).flatten(1, 2), v.flatten(0, 1)).reshape(*p.shape[:-1], case["d"])
    o = o / torch.where(total == 0, torch.ones_like(total), total)
    return o.permute(0, 2, 1, 3, 4).flatten(2, 3)[seq, i], lse


def _plain_prefix(st):
    mine, a = _attend(st, st["q"], st["cu"], st["max_q"], st["table"], st["seq_lens"], st["max_k"], True, True)
    cu = st["cu"][st["prefix_seqs"].long()]  # a prefix's rows are those of its sequences
    theirs, b = _attend(st, st["q"], cu, st["q"].shape[0], st["prefix_table"], st["prefix_lens"], st["max_p"], False,
                        True)
    m = torch.maximum(a, b)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    x, y = (a - m).exp(), (b - m).exp()
    total = x + y
    out = mine * x[..., None] + theirs * y[..., None]
    out = out / torch.where(total == 0, torch.ones_like(total), total)[..., None]
    return out.to(st["q"].dtype), m + total.log()


def _plain_weights(st):
    case, page, lens = st["case"], st["case"]["page"], st["seq_lens"]
    s, seq, i = _scores(st, st["q"], st["cu"], st["max_q"], st["table"], lens, st["max_k"], True)
    lse = torch.full((case["b"], st["max_q"], case["hq"]), math.inf, device=s.device)
    lse[seq, i] = st["lse"]
    lse = lse.reshape(case["b"], st["max_q"], case["hkv"], -1).permute(0, 2, 1, 3)[..., None]
    w = s.sub_(lse).exp_().flatten(2, 3).sum(2).transpose(1, 2)  # [sequences, max_k, hkv]
    key = torch.arange(st["max_k"], device=s.device)
    b, j = (key < lens[:, None]).nonzero(as_tuple=True)
    pg, off = st["table"][b, j // page].long(), j % page
    old = j < (lens - (st["cu"][1:] - st["cu"][:-1]))[b]
    was = torch.where(old[:, None], st["key_weights"][pg, off] * 0.75, torch.zeros_like(w[b, j]))
    st["key_weights"][pg, off] = was + w[b, j]
    return st["key_weights"]


def _plain_evict(st):
    case, page, lens, table = st["case"], st["case"]["page"], st["seq_lens"], st["table"].long()
    st["key_weights"].copy_(st["weights"])  # as the steps before left them
    n, dev = table.shape[1] * page, table.device
    w = st["key_weights"][table].flatten(1, 2).transpose(1, 2)  # [sequences, hkv, n]
    key = torch.arange(n, device=dev)
    length = lens[:, None, None]
    held = (key < case["first"]) | (key >= length - case["recent"]) | (length <= case["budget"])
    w = torch.where(held, torch.full_like(w, math.inf), w).masked_fill(key >= length, -math.inf)
    width = min(n, case["budget"])
    best = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :width]
    count = torch.clamp(lens, max=case["budget"])
    used = (torch.arange(width, device=dev) < count[:, None, None]).expand(best.shape)
    best = torch.where(used, best, torch.full_like(best, n)).sort(-1).values
    kept = torch.full((case["b"], case["hkv"], case["budget"]), -1, dtype=torch.int32, device=dev)
    kept[..., :width] = torch.where(used, best, torch.full_like(best, -1)).int()
    b, h, j = used.nonzero(as_tuple=True)
    src = best[b, h, j]
    there, here = (table[b, src // page], src % page, h), (table[b, j // page], j % page, h)
    st["key_weights"][here] = st["key_weights"][there]
    st["k_cache"][here] = st["k_cache"][there]
    st["v_cache"][here] = st["v_cache"][there]
    if case["i8"]:
        st["k_scale"][here] = st["k_scale"][there]
        st["v_scale"][here] = st["v_scale"][there]
    return (count, kept, st["key_weights"]) + _caches(st)


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _plain_norm(state) if op == "norm" else _plain_prefix(state) if op == "prefix" else \
        _plain_weights(state) if op == "weights" else _plain_evict(state)


# ---------------------------------------------------------------------------
# work and accuracy
# ---------------------------------------------------------------------------
def work(case):
    b, hq, hkv, d, page = (case[k] for k in ("b", "hq", "hkv", "d", "page"))
    lens = lengths(case)
    row = hkv * (d * (1 if case["i8"] else 2) + (4 if case["i8"] else 0))  # a cached token's keys, or its values
    rows = sum(q for _, q in lens)
    tables = 4 * (2 * b + sum((k + page - 1) // page for k, _ in lens))
    # the whole caches of int8 are also returned in 16 bits
    pool = sum((k + page - 1) // page * page for k, _ in lens)
    extra = 2 * pool * (row + hkv * d * 2) if case["i8"] else 0
    if case["op"] == "norm":
        size = rows * (2 * hkv * d * 2 + 2 * row + 2 * hq * d * 2) + 8 * d
        flops = rows * (hq + hkv) * d * 4
        if case["rope"] != "none":
            size += max(k for k, _ in lens) * d * 4 + 4 * rows * case["axes"]
            flops += rows * (hq + hkv) * d * 3
        if case["i8"]:
            flops += rows * hkv * d * 6
        return {"bytes": size + tables + extra, "flops": flops}
    if case["op"] == "evict":
        kept = sum(min(k, case["budget"]) for k, _ in lens)
        moved = sum(case["budget"] - case["first"] for k, _ in lens if k > case["budget"])
        size = sum(k for k, _ in lens) * hkv * 4 + moved * (4 * row + 4 * hkv) + 4 * kept * hkv
        return {"bytes": size + tables + extra + 8 * pool * hkv, "flops": sum(k for k, _ in lens) * hkv * 4}
    causal = sum(q * (k - q) + q * (q + 1) // 2 for k, q in lens)
    if case["op"] == "weights":
        size = rows * hq * (2 * d + 4) + sum(k for k, _ in lens) * (row + 8 * hkv)
        return {"bytes": size + tables, "flops": 2 * hq * d * causal}
    shared = prefixes(case)
    at, pairs = 0, causal
    for k, n in shared:
        pairs += k * sum(q for _, q in lens[at:at + n])
        at += n
    keys = sum(k for k, _ in lens + shared)
    return {"bytes": rows * hq * (4 * d + 4) + 2 * keys * row + tables, "flops": 4 * hq * d * pairs}


def _exact_rows(st, cache, scale, table, n):
    """The first n keys (or values) of one sequence in 64 bits, [n, hkv, d]."""
    at = torch.arange(n, device=table.device)
    pg, off = table.long()[at // st["case"]["page"]], at % st["case"]["page"]
    x = cache[pg, off].double()
    return x if scale is None else x * scale[pg, off].double()[..., None]


def _exact_norm(st, case):
    page, d, rope = case["page"], case["d"], case["rope"]
    k_all, v_all = st["k_cache"].double(), st["v_cache"].double()
    if case["i8"]:
        k_all, v_all = k_all * st["k_scale"].double()[..., None], v_all * st["v_scale"].double()[..., None]

    def turned(x, weight, pos):
        x = x.double()
        x = x / (x.square().sum(-1, keepdim=True) / d + 1e-6).sqrt() * weight.double()
        if rope == "none":
            return x
        col = torch.arange(d // 2, device=x.device)
        c, s = st["cos"][pos, col].double()[:, None], st["sin"][pos, col].double()[:, None]
        z = torch.complex(c.expand(-1, x.shape[1], -1).contiguous(), s.expand(-1, x.shape[1], -1).contiguous())
        if rope == "pairs":
            w = torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * z
            return torch.view_as_real(w).flatten(-2)
        w = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * z
        return torch.cat((w.real, w.imag), -1)

    def stored(x):
        if not case["i8"]:
            return x
        x = x.to(st["k"].dtype).double()  # rows have the new keys' type before they are quantised
        # scales are 32-bit numbers: the largest magnitude times the 32-bit 1 / 127
        s = (x.abs().amax(-1, keepdim=True) * torch.tensor(1 / 127, dtype=torch.float32).item()).float().double()
        s = torch.where(s == 0, torch.ones_like(s), s)
        # and so are the quotients that are rounded to whole numbers
        return (x / s).float().double().round().clamp(-127, 127) * s

    q_all, at = st["q"].double(), 0
    for i, (keys, rows) in enumerate(lengths(case)):
        pos = torch.arange(keys - rows, keys, device=st["table"].device)
        pg, off = st["table"][i].long()[pos // page], pos % page
        mine = slice(at, at + rows)
        where = st["positions"][mine].long()[:, st["rot_axes"].long()] if case["axes"] else pos[:, None]
        q_all[mine] = turned(st["q"][mine], st["q_norm"], where)
        k_all[pg, off] = stored(turned(st["k"][mine], st["k_norm"], where))
        v_all[pg, off] = stored(st["v"][mine].double())
        at += rows
    return q_all, k_all, v_all


def _exact_prefix(st, case):
    shared, lens = prefixes(case), lengths(case)
    ratio = case["hq"] // case["hkv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    lse = torch.zeros(st["q"].shape[:2], dtype=torch.float64, device=st["q"].device)
    at = i = 0
    for g, (common, seqs) in enumerate(shared):
        pk, pv = (_exact_rows(st, st[c + "_cache"], st[c + "_scale"], st["prefix_table"][g], common) for c in "kv")
        for _ in range(seqs):
            keys, rows = lens[i]
            ok, ov = (_exact_rows(st, st[c + "_cache"], st[c + "_scale"], st["table"][i], keys) for c in "kv")
            hide = torch.ones(rows, common + keys, dtype=torch.bool, device=out.device).triu(common + keys - rows + 1)
            for h in range(case["hkv"]):
                k, v = torch.cat((pk[:, h], ok[:, h])), torch.cat((pv[:, h], ov[:, h]))
                for x in range(h * ratio, (h + 1) * ratio):
                    s = st["q"][at:at + rows, x].double() @ k.t().contiguous() / math.sqrt(case["d"])
                    s = s.masked_fill(hide, -math.inf)
                    out[at:at + rows, x] = torch.softmax(s, -1) @ v
                    lse[at:at + rows, x] = torch.logsumexp(s, -1)
            at, i = at + rows, i + 1
    return out, lse


def _exact_weights(st, case):
    page, ratio = case["page"], case["hq"] // case["hkv"]
    out = st["key_weights"].double()
    at = 0
    for i, (keys, rows) in enumerate(lengths(case)):
        k = _exact_rows(st, st["k_cache"], st["k_scale"], st["table"][i], keys)
        j = torch.arange(keys, device=out.device)
        pg, off = st["table"][i].long()[j // page], j % page
        hide = torch.ones(rows, keys, dtype=torch.bool, device=out.device).triu(keys - rows + 1)
        for h in range(case["hkv"]):
            got = torch.zeros(keys, dtype=torch.float64, device=out.device)
            for x in range(h * ratio, (h + 1) * ratio):
                s = st["q"][at:at + rows, x].double() @ k[:, h].t().contiguous() / math.sqrt(case["d"])
                got += torch.exp(s - st["lse"][at:at + rows, x, None].double()).masked_fill(hide, 0.0).sum(0)
            out[pg, off, h] = torch.where(j < keys - rows, 0.75 * out[pg, off, h], torch.zeros_like(got)) + got
        at += rows
    return out


def _exact_evict(st, case):
    page = case["page"]
    out = {c: st[c + "_cache"].double() for c in "kv"}
    if case["i8"]:
        out = {c: x * st[c + "_scale"].double()[..., None] for c, x in out.items()}
    weights, table = st["weights"].double(), st["table"].long()
    heard = st["weights"].cpu().numpy()
    kept = np.full((case["b"], case["hkv"], case["budget"]), -1, dtype=np.int32)
    count = []
    for i, (keys, _) in enumerate(lengths(case)):
        n = min(keys, case["budget"])
        count.append(n)
        at = np.arange(keys)
        pages = st["table"][i].cpu().numpy()
        for h in range(case["hkv"]):
            w = heard[pages[at // page], at % page, h].astype(np.float64)
            if keys > n:
                w[:case["first"]] = np.inf
                w[keys - case["recent"]:] = np.inf
            kept[i, h, :n] = np.sort(np.lexsort((at, -w))[:n])
            src = torch.from_numpy(kept[i, h, :n].astype(np.int64)).to(table.device)
            dst = torch.arange(n, device=table.device)
            for x in (weights, out["k"], out["v"]):
                x[table[i][dst // page], dst % page, h] = x[table[i][src // page], src % page, h].clone()
    dev = table.device
    return (torch.tensor(count, dtype=torch.int32, device=dev), torch.from_numpy(kept).to(dev), weights, out["k"],
            out["v"])


def exact(case, seed):
    """The operators' definitions in 64 bits on the same inputs."""
    st = prepare(case, seed)
    op = case["op"]
    return _exact_norm(st, case) if op == "norm" else _exact_prefix(st, case) if op == "prefix" else \
        _exact_weights(st, case) if op == "weights" else _exact_evict(st, case)

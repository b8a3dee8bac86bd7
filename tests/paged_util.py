"""Paged caches for the tests: random pools and tables, the operators' plain
forms in 64 bits, and the bounds that their outputs are held to."""
from __future__ import annotations

import random

import torch


def _round_unit(dtype):
    """Half a step, relative to the value."""
    return torch.finfo(dtype).eps / 2


class Pool:
    """Pages of `lens` keys per sequence, in shuffled order, as CPU tensors.

    layout "nhd": [pages, page, heads, d]; "hnd": a view of [pages, heads, page,
    d]; "kv": keys and values views of one [pages, 2, page, heads, d]."""

    def __init__(self, lens, hkv, d, page, dtype, i8=False, seed=0, layout="nhd", spare=3, extra_width=1, std=1.0):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.lens, self.hkv, self.d, self.page, self.dtype, self.i8 = list(lens), hkv, d, page, dtype, i8
        need = [(max(0, n) + page - 1) // page for n in lens]
        self.pages = sum(need) + spare
        order = list(range(self.pages))
        rng.shuffle(order)
        width = max(need + [0]) + extra_width
        self.table = torch.full((len(lens), width), -7, dtype=torch.int32)  # unused entries are no pages
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = torch.tensor(order[at:at + m], dtype=torch.int32)
            at += m

        def pool():
            if i8:
                return torch.randint(-127, 128, (self.pages, page, hkv, d), generator=g, dtype=torch.int8)
            return (torch.randn(self.pages, page, hkv, d, generator=g) * std).to(dtype)

        k, v = pool(), pool()
        if layout == "hnd":
            k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
        elif layout == "kv":
            both = torch.stack((k, v), 1)
            k, v = both[:, 0], both[:, 1]
        self.layout = layout
        self.k, self.v = k, v
        self.ks = self.vs = None
        if i8:
            self.ks = (0.5 + torch.rand(self.pages, page, hkv, generator=g)) * 3.0 / 127.0
            self.vs = (0.5 + torch.rand(self.pages, page, hkv, generator=g)) * 3.0 / 127.0

    def seq_lens(self, dev="cpu"):
        return torch.tensor(self.lens, dtype=torch.int32, device=dev)

    def where(self, b, idx):
        """(page, token) of keys idx of sequence b."""
        idx = torch.as_tensor(idx, dtype=torch.long)
        return self.table[b].long()[idx // self.page], idx % self.page

    def unused(self):
        """Mask [pages, page] of the places that hold no key of any sequence."""
        m = torch.ones(self.pages, self.page, dtype=torch.bool)
        for b, n in enumerate(self.lens):
            if n > 0:
                m[self.where(b, torch.arange(n))] = False
        return m

    def rows(self, b, n):
        """The first n keys and values of sequence b in 64 bits, [n, hkv, d]."""
        pg, off = self.where(b, torch.arange(n))
        k, v = self.k[pg, off].double(), self.v[pg, off].double()
        if self.i8:
            k, v = k * self.ks[pg, off].double()[..., None], v * self.vs[pg, off].double()[..., None]
        return k, v

    def on(self, dev):
        """Device copies with the same strides: (key_cache, value_cache,
        block_tables, seq_lens, scales)."""

        def move(x):
            y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=dev)
            return y.copy_(x)

        if self.layout == "kv":
            both = torch.stack((self.k, self.v), 1).to(dev)
            k, v = both[:, 0], both[:, 1]
        else:
            k, v = move(self.k), move(self.v)
        scales = {"key_scale": self.ks.to(dev), "value_scale": self.vs.to(dev)} if self.i8 else {}
        return k, v, self.table.to(dev), self.seq_lens(dev), scales


def visible(n, length, causal=True, window=-1, tree=None):
    """bool [n, length]: which keys each of the n newest rows sees."""
    row = torch.arange(n)[:, None]
    key = torch.arange(length)[None]
    at = length - n + row
    if tree is not None:
        m = tree.shape[0]
        ok = (key < length - n).expand(n, length).clone()
        for i in range(n):
            for j in range(n):
                c = length - n + j
                if c >= 0 and i < m and j < m and bool(tree[i, j]):
                    ok[i, c] = True
        return ok
    ok = torch.ones(n, length, dtype=torch.bool)
    if causal:
        ok &= key <= at
        if window > 0:
            ok &= at - key < window
    elif window > 0:
        ok &= (at - key).abs() <= window // 2
    return ok


def reference(q, k, v, ok, scale, dtype, i8):
    """softmax(scale q k^T) v over the keys that ok allows, in 64 bits, and the
    bound of a kernel's error.  q [n, hq, d], k and v [len, hkv, d].

    With u half a step of `dtype`: the weights p are rounded to it (u A, A = sum
    p |v|; below fp16's normal range by at most 2^-25 each, relative to a largest
    weight of at least 1 before the division by the sum), the scores are sums of d
    products in 32 bits ((d + 2) 2^-24 of the sum of magnitudes, and their own size
    times 2^-22 in the exponent, whose function is good to 2^-21; sums and the merge
    of parts 2^-18 of A in all), a change ds of the scores changes the output by at
    most 2 ds A, and the output is rounded once (u |out|; 2^-25 in fp16's subnormal
    range).  int8 keys and values are exact, their scales meet the scores and the
    weights in 32 bits (2^-23 more), and the weights are fp16's, within 2^-31 of the
    largest value each where they are small."""
    u = _round_unit(dtype)
    w = _round_unit(torch.float16) if i8 else u
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    n, hq, d = q.shape
    length, hkv, _ = k.shape
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    tol = torch.full((n, hq, d), max(sub, 1e-30), dtype=torch.float64)
    if length == 0 or n == 0:
        return out, tol
    g = hq // hkv
    for h in range(hq):
        qh, kh, vh = q[:, h].double(), k[:, h // g], v[:, h // g]
        s = qh @ kh.t() * scale
        mag = qh.abs() @ kh.abs().t() * abs(scale)
        s = s.masked_fill(~ok, float("-inf"))
        seen = ok.any(-1)
        p = torch.zeros_like(s)
        p[seen] = torch.softmax(s[seen], -1)
        o = p @ vh
        a = p @ vh.abs()
        ds = (mag * ((d + 2) * 2.0 ** -24 + 2.0 ** -22 + (2.0 ** -23 if i8 else 0.0))).masked_fill(~ok, 0.0).amax(-1, keepdim=True)
        ds = ds + 2.0 ** -21
        vsum = ok.double() @ (torch.full_like(vh, float(vh.abs().max()) * 2.0 ** -31) if i8 else vh.abs() * sub)
        out[:, h] = o
        tol[:, h] += w * a + 2 * ds * a + 2.0 ** -18 * a + u * o.abs() * 1.01 + vsum
    return out, tol


def check(got, want, tol, name=""):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), f"{name}: non-finite output"
    over = (got - want).abs() / tol
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{name}: error {worst:.3f} of its bound at {int(over.argmax())}"
    return worst


def rope_tables(rows, cols, base=10000.0):
    inv = base ** (-torch.arange(cols, dtype=torch.float64) / cols)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def rotate(x, cos, sin, interleaved):
    """x [rows, heads, d] rotated in 64 bits by the rows' cos and sin [rows, c]."""
    y = x.double().clone()
    c, s = cos.double()[:, None], sin.double()[:, None]
    m = cos.shape[-1]
    a, b = (slice(0, 2 * m, 2), slice(1, 2 * m, 2)) if interleaved else (slice(0, m), slice(m, 2 * m))
    u, w = x[..., a].double(), x[..., b].double()
    y[..., a] = u * c - w * s
    y[..., b] = u * s + w * c
    return y

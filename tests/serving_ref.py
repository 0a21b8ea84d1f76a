"""Plain 64-bit forms of the serving operators, and the bounds their f32 / 16-bit
results are held to. One sequence, one head, one row at a time: no batching, no
tiles, no splitting."""
from __future__ import annotations

import numpy as np
import torch

U32 = 2.0**-24  # half a step of f32, relative


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


class Geometry:
    """Sequences with their page tables over a pool whose other pages and slots hold garbage."""

    def __init__(self, seed, heads, kv_heads, head_size, page, lens, rows, shared=0, pad_rows=0, spare_pages=3,
                 spare_slots=2):
        rng = np.random.default_rng(seed)
        self.rng, self.heads, self.kv, self.hd, self.page = rng, heads, kv_heads, head_size, page
        self.lens, self.rows, self.shared = list(lens), list(rows), shared
        first = shared // page
        need = [max(0, -(-n // page) - first) for n in lens]
        self.n_pages = first + sum(need) + spare_pages
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), first + max(need + [0]) + spare_slots), 0xFFFFFFFF, np.uint32)
        self.table[:, :first] = order[:first]
        at = first
        for i, n in enumerate(need):
            self.table[i, first : first + n] = order[at : at + n]
            at += n
        self.row_start = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
        self.n_rows = int(self.row_start[-1]) + pad_rows

    def device(self, yl, status=None, shared=None, n_rows=None):
        t = [torch.from_numpy(a.view(np.int32).copy()).cuda()
             for a in (self.row_start, np.asarray(self.lens, np.uint32), self.table)]
        return yl.SeqBatch(*t, self.n_rows if n_rows is None else n_rows,
                           shared_len=self.shared if shared is None else shared, status=status)

    def pool(self, dtype, std=1.0):
        shape = (self.n_pages, self.page, self.kv, self.hd)
        return tuple(torch.from_numpy(self.rng.standard_normal(shape) * std).to(dtype) for _ in range(2))

    def positions(self, i):
        """Positions of sequence i's rows (negative: the row has none)."""
        return self.lens[i] - self.rows[i] + np.arange(self.rows[i])

    def gather(self, i, pool):
        """Sequence i's keys or values in order; zeros where the table names no page."""
        pos = np.arange(self.lens[i])
        ids = self.table[i, pos // self.page].astype(np.int64)
        good = ids < self.n_pages
        rows = pool[torch.from_numpy(np.where(good, ids, 0)), torch.from_numpy(pos % self.page)].double()
        return torch.where(torch.from_numpy(good)[:, None, None], rows, 0.0)


def attention(g: Geometry, q, k, v, scale, limit=1 << 31, only=None):
    """(out, lse, out_bound, lse_bound) in 64 bits. The bounds count, for scores of |terms| sum A: products and sums of
    hd terms, each off by at most two half steps of f32 (a tensor core may truncate) in chains of hd/4 + 16; for the
    softmax: exp of an f32 argument (its rounding: |s| * 2 U32; exp itself: 4 U32) and sums in chains of n/4 + 64; for a
    16-bit type one half step on every weight. Output rounding is added by the caller. only: the rows to compute."""
    n, group = g.n_rows, g.heads // g.kv
    out = torch.zeros(n, g.heads, g.hd, dtype=torch.float64)
    lse = torch.full((n, g.heads), -torch.inf, dtype=torch.float64)
    ob, lb = torch.zeros_like(out), torch.zeros_like(lse)
    p_round = 0.0 if q.dtype == torch.float32 else half_step(q.dtype)
    for i in range(len(g.lens)):
        if not g.rows[i]:
            continue
        ks, vs = g.gather(i, k), g.gather(i, v)
        for t, pos in enumerate(g.positions(i)):
            if pos < 0:
                continue
            r, m = int(g.row_start[i]) + t, min(int(pos) + 1, limit)
            if only is not None and r not in only:
                continue
            for h in range(g.heads):
                qq, kk, vv = q[r, h].double(), ks[:m, h // group], vs[:m, h // group]
                s = kk @ qq * scale
                p = torch.softmax(s, 0)
                out[r, h], lse[r, h] = p @ vv, torch.logsumexp(s, 0)
                terms = float((kk.abs() @ qq.abs() * abs(scale)).max())
                ds = terms * (g.hd / 4 + 16) * 2 * U32 + float(s.abs().max()) * 4 * U32
                chain = (m / 4 + 64) * 2 * U32 + 4 * U32
                ob[r, h] = (p @ vv.abs()) * (2 * ds + 2 * chain + 2 * p_round)
                lb[r, h] = ds + chain + abs(float(lse[r, h])) * 2 * U32
    return out, lse, ob, lb


def append(g: Geometry, qkv, k, v, cs, half):
    """(q, k, v, bounds of each) in 64 bits: the pools with the new rows written, q of the new rows."""
    n, hd = g.n_rows, g.hd
    x = qkv.double().view(n, g.heads + 2 * g.kv, hd).clone()
    bound = torch.zeros_like(x)
    kk, vv = k.double().clone(), v.double().clone()
    kb, vb = torch.zeros_like(kk), torch.zeros_like(vv)
    for i in range(len(g.lens)):
        for t, pos in enumerate(g.positions(i)):
            r = int(g.row_start[i]) + t
            if cs is not None:
                c, s = cs[pos, :, 0].double(), cs[pos, :, 1].double()
                rot = x[r, : g.heads + g.kv]
                ia = torch.arange(hd // 2) if half else torch.arange(0, hd, 2)
                ib = ia + hd // 2 if half else ia + 1
                a, b = rot[:, ia].clone(), rot[:, ib].clone()
                rot[:, ia], rot[:, ib] = a * c - b * s, a * s + b * c
                bound[r, : g.heads + g.kv, ia] = 2 * U32 * ((a * c).abs() + (b * s).abs())
                bound[r, : g.heads + g.kv, ib] = 2 * U32 * ((a * s).abs() + (b * c).abs())
            page, at = int(g.table[i, pos // g.page]), int(pos % g.page)
            kk[page, at], kb[page, at] = x[r, g.heads : g.heads + g.kv], bound[r, g.heads : g.heads + g.kv]
            vv[page, at] = x[r, g.heads + g.kv :]
    return x[:, : g.heads], kk, vv, bound[:, : g.heads], kb, vb


def rope_cs(n, hd):
    angle = np.arange(n)[:, None] * 10000.0 ** (-np.arange(hd // 2) / (hd // 2))
    return torch.from_numpy(np.stack([np.cos(angle), np.sin(angle)], -1)).float()


def logprobs(x, tokens, k):
    """(logprobs, entropy, ids, top_logprobs, bound of the first two and of the last) in 64 bits, rows with a
    distribution only. The bounds count: sums in chains of V/512 + 64 (two half steps each, for the joining), exp of an
    f32 difference d (|d| * 4 half steps weighted by its share, exp itself 8), log1p and the last subtractions."""
    n, vocab = x.shape
    x = x.double()
    m = x.max(1, keepdim=True)[0]
    d = x - m
    e = d.exp()
    total = e.sum(1)
    weighted = torch.where(e > 0, e * d, 0.0).sum(1)
    lse = total.log()
    entropy = lse - weighted / total
    rel = (vocab / 512 + 64) * 2 * U32 + 8 * U32 + 4 * U32 * (weighted.abs() / total)
    ids = np.stack([np.lexsort((np.arange(vocab), -(row + 0.0)))[:k] for row in x.numpy()]) if k else np.zeros((n, 0))
    top = d.gather(1, torch.from_numpy(ids.astype(np.int64))) - lse[:, None] if k else torch.zeros(n, 0).double()
    lp = d.gather(1, tokens.long()[:, None])[:, 0] - lse
    finite = lambda t: torch.where(t.isfinite(), t.abs(), 0.0)  # noqa: E731
    return (lp, entropy, ids, top, rel + 4 * U32 * (finite(lp) + lse.abs()),
            # W is off by rel of itself and by 4 half steps of |d| more in each of its terms
            rel * (1 + (weighted.abs() / total)) + 8 * U32 * (torch.where(e > 0, e * d * d, 0.0).sum(1) / total)
            + 4 * U32 * (entropy + lse),
            rel[:, None] + 4 * U32 * (finite(top) + lse[:, None].abs()))

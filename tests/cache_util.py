"""Plain 64-bit forms of the bounded paged cache's operators, for its tests."""
from __future__ import annotations

import numpy as np

HD, PAGE = 128, 64


def torch():
    import torch as t

    return t


class Setup:
    """A PagedCache over a shuffled page pool: random K/V everywhere, NaN-free weights, positions -1."""

    def __init__(self, rows, kvh, max_len, seed=0, extra_pages=2, weights=True, slot_stride=None, device="cuda"):
        t = torch()
        g = t.Generator(device=device)
        g.manual_seed(seed)
        self.g, self.rows, self.kvh, self.max_len = g, rows, kvh, max_len
        pages = -(-max_len // PAGE)
        pool = rows * pages + extra_pages
        self.k = t.randn(pool, kvh, PAGE, HD, generator=g, device=device, dtype=t.bfloat16)
        self.v = t.randn(pool, kvh, PAGE, HD, generator=g, device=device, dtype=t.bfloat16)
        order = t.randperm(pool, generator=g, device=device)[: rows * pages]
        self.tables = order.view(rows, pages).to(t.int32)
        self.w = self.pos = None
        if weights:
            stride = slot_stride or max_len
            self.w = t.rand(rows, kvh, stride, generator=g, device=device)[:, :, :max_len]
            self.pos = t.full((rows, kvh, stride), -1, dtype=t.int32, device=device)[:, :, :max_len]

    def cache(self, **kw):
        from inference_b200 import PagedCache

        return PagedCache(self.k, self.v, self.tables, self.w, self.pos, **kw)

    def randn(self, *shape):
        t = torch()
        return t.randn(*shape, generator=self.g, device=self.k.device, dtype=t.bfloat16)

    def slots(self, pages, row, head, n):
        """Slots 0 .. n - 1 of a sequence and kv head in 64 bits."""
        need = -(-n // PAGE)
        return pages[self.tables[row, :need].long(), head].reshape(-1, HD)[:n].double()

    def behind(self, pages, lens, value):
        """Fills every slot at or behind a sequence's length, and every unused page, with `value`."""
        t = torch()
        keep = t.zeros(pages.shape[0], PAGE, dtype=t.bool, device=pages.device)
        for r, n in enumerate(lens):
            for p in range(-(-n // PAGE)):
                keep[int(self.tables[r, p]), : min(PAGE, n - p * PAGE)] = True
        pages.masked_fill_(~keep[:, None, :, None], value)


def ints(values, device="cuda"):
    t = torch()
    return t.tensor(values, dtype=t.int32, device=device)


def attention(s: Setup, q, lens):
    """64-bit attention: (out, slot weights of this query, the tolerance of each).

    Tolerances.  A score is a sum of 128 exact products, added in 32 bits: off by at most 128 roundings
    (2^-23 each where the adder truncates) of the sum of the products' sizes; that and the scaling
    (2^-23 of the score) give every score an error of at most d.  Numerator and denominator of a probability are each off by
    exp(d) - 1, and by 2^-20 for exp2 (2 units of 2^-23), the sum over slots (a tree of at most 2^-23 a level, and 64 terms
    in line) and the division.  The output adds 2^-15 of sum p |v| (the sums' roundings, 2^-23 each where the adder
    truncates), and its one rounding to BF16, 2^-8."""
    t = torch()
    rows, qh = q.shape[0], q.shape[1]
    G = qh // s.kvh
    out = t.zeros(rows, qh, HD, dtype=t.float64, device=q.device)
    out_tol = t.zeros_like(out)
    dw = t.zeros(rows, s.kvh, s.max_len, dtype=t.float64, device=q.device)
    dw_tol = t.zeros_like(dw)
    for r, n in enumerate(lens):
        if n == 0:
            continue
        for h in range(s.kvh):
            k, v = s.slots(s.k, r, h, n), s.slots(s.v, r, h, n)
            x = q[r, h * G:(h + 1) * G].double()
            score = k @ x.T / HD ** 0.5
            d = ((k.abs() @ x.abs().T) * (128 * 2.0 ** -23) / HD ** 0.5 + score.abs() * 2.0 ** -22).nan_to_num(0.0, 0.0).amax(dim=0)
            p = t.softmax(score, dim=0)
            rel = 2 * (t.exp(d) - 1) + 2.0 ** -19
            o = p.T @ v
            out[r, h * G:(h + 1) * G] = o
            out_tol[r, h * G:(h + 1) * G] = o.abs() * 2.0 ** -8 + (p.T @ v.abs()) * (rel + 2.0 ** -15)[:, None]
            dw[r, h, :n] = p.sum(dim=1)
            dw_tol[r, h, :n] = (p * rel).sum(dim=1)
    return out, out_tol, dw, dw_tol


def close(got, want, tol, what=""):
    t = torch()
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    both_nan = t.isnan(got) & t.isnan(want)
    bad &= ~both_nan
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at "
                                 f"{bad.nonzero()[0].tolist()}: {got[bad][:3].tolist()} for {want[bad][:3].tolist()}, "
                                 f"tolerance {tol[bad][:3].tolist()}")


def turn(x, w, cos, sin, eps):
    """RMSNorm with weights then rotate-half RoPE in 64 bits, and its tolerance: 16 roundings of 2^-24 of the head's
    largest rotated size (sum of squares, root, division, products), then one to BF16."""
    t = torch()
    x = x.double()
    y = x * w.double() / ((x * x).mean(dim=-1, keepdim=True) + eps).sqrt()
    a, b = y[..., :64], y[..., 64:]
    c, d = cos.double()[:, None], sin.double()[:, None]
    z = t.cat([a * c - b * d, b * c + a * d], dim=-1)
    size = t.cat([a.abs() + b.abs()] * 2, dim=-1)
    return z, z.abs() * 2.0 ** -8 + size * 2.0 ** -20


def evict(lens, next_pos, keep, recent, weights, positions):
    """Per (row, head): the slots holding what, after an eviction, as (lens_out, {(row, head): (holes, movers)})."""
    moves = {}
    for r, n in enumerate(lens):
        for h in range(weights.shape[1]):
            if n <= keep:
                moves[r, h] = ([], [])
                continue
            w, p = weights[r, h, :n], positions[r, h, :n]
            rank = [(0 if int(p[i]) >= next_pos[r] - recent else 1,
                     (1, 0.0) if np.isnan(w[i]) else (0, -float(w[i])), i) for i in range(n)]
            kept = {i for _, _, i in sorted((a, b if a else (0, 0.0), i) for a, b, i in rank)[:keep]}
            moves[r, h] = ([i for i in range(keep) if i not in kept], [i for i in range(keep, n) if i in kept])
    return [min(n, keep) for n in lens], moves


def apply_moves(s: Setup, moves, k, v, w, p):
    """The moves on copies of K, V, weights and positions."""
    k, v, w, p = k.clone(), v.clone(), w.clone(), p.clone()
    for (r, h), (holes, movers) in moves.items():
        assert len(holes) == len(movers)
        if not holes:
            continue
        a, b = ints(holes, k.device).long(), ints(movers, k.device).long()
        ta, tb = s.tables[r][a // PAGE].long(), s.tables[r][b // PAGE].long()
        k[ta, h, a % PAGE] = k[tb, h, b % PAGE]
        v[ta, h, a % PAGE] = v[tb, h, b % PAGE]
        w[r, h, a] = w[r, h, b]
        p[r, h, a] = p[r, h, b]
    return k, v, w, p

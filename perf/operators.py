"""Timed cases of the bounded paged KV cache's operators: append, attention of
one new token per sequence with accumulated attention weights, and eviction by
those weights.

``own`` chooses the side: False computes each operator from elementary torch
operations in fp32, True makes the calls a user makes of inference_b200
(PagedCache and the B200Backend cache_* methods).
"""
from __future__ import annotations

import math

import torch

own = False

HD = 128  # head dimension
PAGE = 64  # slots per page
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # one sequence, the smallest model's heads, a short chat turn: latency
        {"name": "attend-1x300", "op": "attend", "rows": 1, "q_heads": 16, "kv_heads": 8, "len": 300,
         "ragged": False, "accumulate": True},
        # one sequence at the end of a 4096-token window
        {"name": "attend-1x4095", "op": "attend", "rows": 1, "q_heads": 32, "kv_heads": 8, "len": 4095,
         "ragged": False, "accumulate": True},
        # one sequence with a very long history, the largest model's heads, no weights kept
        {"name": "attend-1x100001", "op": "attend", "rows": 1, "q_heads": 64, "kv_heads": 8, "len": 100001,
         "ragged": False, "accumulate": False},
        # a serving batch of sixteen sequences of different lengths
        {"name": "attend-16x4096", "op": "attend", "rows": 16, "q_heads": 32, "kv_heads": 8, "len": 4096,
         "ragged": True, "accumulate": True},
        # many short sequences on one rank of a model sharded over eight GPUs
        {"name": "attend-200x500-shard", "op": "attend", "rows": 200, "q_heads": 8, "kv_heads": 1, "len": 500,
         "ragged": True, "accumulate": True},
        # a full server: many long sequences
        {"name": "attend-64x8192", "op": "attend", "rows": 64, "q_heads": 32, "kv_heads": 8, "len": 8192,
         "ragged": True, "accumulate": True},
        # one page's worth of new tokens evicted again from every sequence of a batch
        {"name": "evict-16x2112", "op": "evict", "rows": 16, "kv_heads": 8, "len": 2112, "keep": 2048, "recent": 256,
         "ragged": False},
        # one long prompt cut to the budget
        {"name": "evict-1x32768", "op": "evict", "rows": 1, "kv_heads": 8, "len": 32768, "keep": 4096,
         "recent": 1024, "ragged": False},
        # a batch of prompts of different lengths cut to the budget
        {"name": "evict-32x8000", "op": "evict", "rows": 32, "kv_heads": 8, "len": 8000, "keep": 2000, "recent": 500,
         "ragged": True},
        # one decode token
        {"name": "append-1", "op": "append", "rows": 1, "q_heads": 32, "kv_heads": 8, "len": 512, "prompt": False},
        # a decode step of a full server
        {"name": "append-256", "op": "append", "rows": 256, "q_heads": 32, "kv_heads": 8, "len": 512,
         "prompt": False},
        # the tokens of one long prompt at once
        {"name": "append-prompt-4001", "op": "append", "rows": 4001, "q_heads": 64, "kv_heads": 8, "len": 4096,
         "prompt": True},
    ]


HEADS = [(16, 8), (32, 8), (64, 8), (8, 8), (16, 4), (8, 2), (16, 2), (4, 1), (8, 1), (16, 1), (40, 8), (24, 8), (12, 4)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "evict", "evict", "append"])
    qh, kvh = rng.choice(HEADS)
    if op == "attend":
        rows = _log(rng, 1, 256)
        length = _log(rng, 1, min(100000, max(2, 2_200_000 // (rows * kvh))))
        return {"op": op, "rows": rows, "q_heads": qh, "kv_heads": kvh, "len": length,
                "ragged": rng.random() < 0.7, "accumulate": rng.random() < 0.8}
    if op == "evict":
        rows = _log(rng, 1, 64)
        length = _log(rng, 65, min(32768, 1_600_000 // (rows * kvh)))
        keep = max(1, int(length * rng.uniform(0.1, 0.99)))
        return {"op": op, "rows": rows, "kv_heads": kvh, "len": length, "keep": keep,
                "recent": int(keep * rng.uniform(0.0, 0.7)), "ragged": rng.random() < 0.5}
    prompt = rng.random() < 0.5
    rows = _log(rng, 1, 4000 if prompt else 300)
    return {"op": op, "rows": rows, "q_heads": qh, "kv_heads": kvh, "len": rows + 60 if prompt else 512,
            "prompt": prompt}


# ---------------------------------------------------------------- inputs


def _lens(case):
    """The sequences' lengths: all `len`, or spread over [len / 8, len] in a fixed scattered order."""
    n, top = case["rows"], case["len"]
    if not case.get("ragged"):
        return [top] * n
    low = max(1, top // 8)
    return [top if r == 0 else low + int((top - low) * ((r * 0.6180339887498949) % 1.0)) for r in range(n)]


def _prompt(case):
    return case["op"] == "append" and case["prompt"]


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(shape, generator=g, dtype=dtype, device=dev)

    seqs = 1 if _prompt(case) else case["rows"]
    kvh, cap = case["kv_heads"], case["len"]
    pages = -(-cap // PAGE)
    pool = seqs * pages + 3
    s = {"case": dict(case), "seqs": seqs, "max_len": cap}
    s["k_pages"] = normal(pool, kvh, PAGE, HD)
    s["v_pages"] = normal(pool, kvh, PAGE, HD)
    order = torch.randperm(pool, generator=g, device=dev)[: seqs * pages]
    s["tables"] = order.view(seqs, pages).to(torch.int32)
    s["weights"] = torch.zeros(seqs, kvh, cap, dtype=torch.float32, device=dev)
    s["positions"] = torch.zeros(seqs, kvh, cap, dtype=torch.int32, device=dev)

    if case["op"] == "attend":
        # normalised queries and keys, as after the per-head RMSNorm with weights near one
        s["q"] = normal(seqs, case["q_heads"], HD)
        s["out"] = torch.empty_like(s["q"])
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=dev)
        s["weights"] = torch.rand(seqs, kvh, cap, generator=g, dtype=torch.float32, device=dev)
    elif case["op"] == "evict":
        lens = torch.tensor(_lens(case), dtype=torch.int32, device=dev)
        # heavy-tailed accumulated weights, some slots never attended
        w = torch.exp(2.0 * torch.randn(seqs, kvh, cap, generator=g, device=dev)) * 0.01
        u = torch.rand(seqs, kvh, cap, generator=g, device=dev)
        s["weights"] = torch.where(u < 0.05, torch.zeros_like(w), w)
        # slots hold the sequence's positions in an order that earlier evictions have scattered
        u = torch.rand(seqs, kvh, cap, generator=g, device=dev)
        behind = torch.arange(cap, device=dev) >= lens.view(-1, 1, 1)
        rank = torch.argsort(torch.argsort(u + 2.0 * behind, dim=-1), dim=-1).to(torch.int32)
        gone = torch.randint(0, 1000, (seqs,), generator=g, device=dev, dtype=torch.int32)
        s["positions"] = rank + gone.view(-1, 1, 1)
        s["next_pos"] = lens + gone
        s["lens"] = lens
        s["lens_out"] = torch.zeros_like(lens)
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["positions_out"] = torch.zeros_like(s["positions"])
    else:
        n, qh = case["rows"], case["q_heads"]
        s["qkv"] = normal(n, qh + 2 * kvh, HD)  # the rows of one QKV product
        s["q_out"] = torch.empty(n, qh, HD, dtype=torch.bfloat16, device=dev)
        s["q_norm"] = (1.0 + 0.1 * normal(HD, dtype=torch.float32)).to(torch.bfloat16)
        s["k_norm"] = (1.0 + 0.1 * normal(HD, dtype=torch.float32)).to(torch.bfloat16)
        limit = 8192
        inv = THETA ** (-torch.arange(0, HD, 2, dtype=torch.float64, device=dev) / HD)
        angle = torch.arange(limit, dtype=torch.float64, device=dev)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["prompt"]:
            first = int(torch.randint(0, min(limit, cap) - n + 1, (1,), generator=g, device=dev))
            s["slots"] = torch.arange(first, first + n, dtype=torch.int32, device=dev)
            s["token_pos"] = s["slots"].clone()
            s["row_seq"] = torch.zeros(n, dtype=torch.int32, device=dev)
            s["lens_out"] = None
        else:
            s["slots"] = torch.randint(0, cap, (n,), generator=g, device=dev, dtype=torch.int32)
            s["token_pos"] = s["slots"] + torch.randint(0, limit - cap, (n,), generator=g, device=dev,
                                                        dtype=torch.int32)
            s["row_seq"] = None
            s["lens_out"] = torch.zeros_like(s["slots"])
    if own:
        from inference_b200 import B200Backend, PagedCache, RopeCache

        s["be"] = B200Backend(0)
        s["cache"] = PagedCache(s["k_pages"], s["v_pages"], s["tables"], s["weights"], s["positions"])
        if case["op"] == "append":
            s["rope"] = RopeCache(s["cos"], s["sin"])
    return s


# ---------------------------------------------------------------- the plain forms


def _gather(s, pages):
    """[seqs, kv_heads, slots, 128] of the pool, in fp32."""
    t = pages[s["tables"].long()].transpose(1, 2)
    return t.reshape(t.shape[0], t.shape[1], -1, HD)[:, :, : s["max_len"]].float()


def _attend(s):
    c = s["case"]
    n, qh, kvh, cap = c["rows"], c["q_heads"], c["kv_heads"], s["max_len"]
    valid = (torch.arange(cap, device=s["q"].device) < s["lens"].view(-1, 1)).view(n, 1, 1, cap)
    q = s["q"].float().view(n, kvh, qh // kvh, HD)
    score = torch.matmul(q, _gather(s, s["k_pages"]).transpose(2, 3)) / math.sqrt(HD)
    score = score.masked_fill(~valid, -math.inf)
    top = score.max(dim=-1, keepdim=True).values
    p = torch.exp(score - top)
    p = p / p.sum(dim=-1, keepdim=True)
    s["out"].copy_(torch.matmul(p, _gather(s, s["v_pages"])).view(n, qh, HD))
    if not c["accumulate"]:
        return {"out": s["out"]}
    s["weights"] += p.sum(dim=2)
    return {"out": s["out"], "weights": s["weights"]}


def _evict(s):
    c = s["case"]
    keep, cap = c["keep"], s["max_len"]
    dev = s["lens"].device
    slot = torch.arange(cap, device=dev)
    lens = s["lens"].view(-1, 1, 1)
    kept_n = lens.clamp(max=keep)
    protect = s["positions"] >= (s["next_pos"].view(-1, 1, 1) - c["recent"])
    key = torch.where(protect, torch.full_like(s["weights"], math.inf), s["weights"])
    key = torch.where(slot < lens, key, torch.full_like(key, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(protect).scatter_(-1, order, (slot < kept_n).expand_as(order))
    hole = (~kept & (slot < kept_n)).nonzero(as_tuple=True)
    move = (kept & (slot >= kept_n)).nonzero(as_tuple=True)  # as many as holes in every row and head
    to, of = [(s["tables"][r, j // PAGE].long(), h, j % PAGE) for r, h, j in (hole, move)]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[to] = pages[of]
    inside = slot < kept_n
    for name in ("weights", "positions"):
        v = s[name].clone()
        v[hole] = s[name][move]
        s[name + "_out"].copy_(torch.where(inside, v, s[name + "_out"]))
    s["lens_out"].copy_(kept_n.view(-1))
    return {k: s[k] for k in ("k_pages", "v_pages", "weights_out", "positions_out", "lens_out")}


def _turn(x, w, cos, sin):
    x = x.float()
    y = x * w.float() * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    a, b = y[..., : HD // 2], y[..., HD // 2:]
    c, d = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * d, b * c + a * d], dim=-1).to(torch.bfloat16)


def _append(s):
    c = s["case"]
    n, qh, kvh = c["rows"], c["q_heads"], c["kv_heads"]
    q, k, v = s["qkv"].split([qh, kvh, kvh], dim=1)
    at = s["token_pos"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    s["q_out"].copy_(_turn(q, s["q_norm"], cos, sin))
    slot = s["slots"].long()
    seq = torch.arange(n, device=slot.device) if s["row_seq"] is None else s["row_seq"].long()
    page = s["tables"][seq, slot // PAGE].long()
    s["k_pages"][page, :, slot % PAGE] = _turn(k, s["k_norm"], cos, sin)
    s["v_pages"][page, :, slot % PAGE] = v
    s["weights"][seq, :, slot] = 0.0
    s["positions"][seq, :, slot] = s["token_pos"][:, None]
    got = {k: s[k] for k in ("q_out", "k_pages", "v_pages", "weights", "positions")}
    if s["lens_out"] is not None:
        s["lens_out"].copy_(s["slots"] + 1)
        got["lens_out"] = s["lens_out"]
    return got


def run(s):
    c = s["case"]
    if not own:
        return {"attend": _attend, "evict": _evict, "append": _append}[c["op"]](s)
    be, cache = s["be"], s["cache"]
    if c["op"] == "attend":
        be.cache_attention(cache, s["q"], s["lens"], s["out"], accumulate=c["accumulate"])
        return {"out": s["out"], "weights": s["weights"]} if c["accumulate"] else {"out": s["out"]}
    if c["op"] == "evict":
        be.cache_evict(cache, s["lens"], s["next_pos"], c["keep"], c["recent"], s["lens_out"],
                       weights_out=s["weights_out"], positions_out=s["positions_out"])
        return {k: s[k] for k in ("k_pages", "v_pages", "weights_out", "positions_out", "lens_out")}
    qh, kvh = c["q_heads"], c["kv_heads"]
    q, k, v = s["qkv"].split([qh, kvh, kvh], dim=1)
    be.cache_append(cache, q, k, v, s["q_norm"], s["k_norm"], s["rope"], s["token_pos"], s["slots"], s["q_out"], EPS,
                    lens_out=s["lens_out"], row_seq=s["row_seq"])
    got = {k: s[k] for k in ("q_out", "k_pages", "v_pages", "weights", "positions")}
    if s["lens_out"] is not None:
        got["lens_out"] = s["lens_out"]
    return got


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    lens = _lens(case)
    kvh = case["kv_heads"]
    if case["op"] == "attend":
        slots = sum(lens) * kvh
        b = slots * (2 * HD * 2 + (8 if case["accumulate"] else 0)) + case["rows"] * case["q_heads"] * HD * 4
        return {"bytes": b, "flops": slots * (case["q_heads"] // kvh) * 4 * HD}
    if case["op"] == "evict":
        # weights and positions read, the kept ones written; of `keep` slots the share that falls
        # behind `keep` moves (the slots' order says nothing of their weight)
        b = 0.0
        for n in lens:
            kept = min(n, case["keep"])
            b += kvh * (n * 8 + kept * 8 + kept * (1 - kept / n) * 2 * 2 * HD * 2)
        return {"bytes": b, "flops": 0}
    rows, qh = case["rows"], case["q_heads"]
    return {"bytes": rows * ((qh + 2 * kvh) * HD * 4 + HD * 4 + kvh * 8), "flops": rows * (qh + kvh) * HD * 8}


# ---------------------------------------------------------------- from the definition, in 64 bits


def _exact_attend(s):
    c = s["case"]
    group = c["q_heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    weights = s["weights"].double()
    for r, length in enumerate(_lens(c)):
        pages = s["tables"][r, : -(-length // PAGE)].long()
        for h in range(c["kv_heads"]):
            k = s["k_pages"][pages, h].reshape(-1, HD)[:length].double()
            v = s["v_pages"][pages, h].reshape(-1, HD)[:length].double()
            heads = slice(h * group, (h + 1) * group)
            p = torch.softmax(k @ s["q"][r, heads].double().T * HD ** -0.5, dim=0)
            out[r, heads] = p.T @ v
            weights[r, h, :length] += p.sum(dim=1)
    return {"out": out, "weights": weights} if c["accumulate"] else {"out": out}


def _exact_evict(s):
    c = s["case"]
    weights, positions = s["weights"].cpu(), s["positions"].cpu()
    wo, po = torch.zeros_like(weights), torch.zeros_like(positions)
    lo = torch.tensor([min(n, c["keep"]) for n in _lens(c)], dtype=torch.int32)
    k, v = s["k_pages"].clone(), s["v_pages"].clone()
    for r, length in enumerate(_lens(c)):
        stay = int(lo[r])
        first = int(s["next_pos"][r]) - c["recent"]
        for h in range(c["kv_heads"]):
            w, p = weights[r, h, :length], positions[r, h, :length]
            # heaviest first; among equals the lower slot; protected slots before all others
            score = torch.where(p >= first, torch.tensor(math.inf, dtype=torch.float64), w.double())
            chosen = torch.argsort(-score, stable=True)[:stay].sort().values
            tail = chosen[chosen >= stay]
            present = torch.zeros(stay, dtype=torch.bool)
            present[chosen[chosen < stay]] = True
            holes = (~present).nonzero().view(-1)
            source = torch.arange(stay)
            source[holes] = tail
            wo[r, h, :stay], po[r, h, :stay] = w[source], p[source]
            a, b = holes.to(k.device), tail.to(k.device)
            pa, pb = s["tables"][r][a // PAGE].long(), s["tables"][r][b // PAGE].long()
            k[pa, h, a % PAGE] = s["k_pages"][pb, h, b % PAGE]
            v[pa, h, a % PAGE] = s["v_pages"][pb, h, b % PAGE]
    return {"k_pages": k, "v_pages": v, "weights_out": wo, "positions_out": po, "lens_out": lo}


def _exact_append(s):
    c = s["case"]
    qh, kvh = c["q_heads"], c["kv_heads"]
    x = s["qkv"].double()
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    cos, sin = s["cos"].double()[s["token_pos"].long()], s["sin"].double()[s["token_pos"].long()]
    turned = []
    for part, w in ((x[:, :qh], s["q_norm"]), (x[:, qh:qh + kvh], s["k_norm"])):
        y = part * w.double() / ((part ** 2).sum(-1, keepdim=True) / HD + EPS).sqrt()
        z = torch.complex(y[..., :64], y[..., 64:]) * torch.complex(cos, sin)[:, None]
        turned.append(torch.cat([z.real, z.imag], -1))
    weights, positions = s["weights"].clone(), s["positions"].clone()
    slots, at = s["slots"].tolist(), s["token_pos"].tolist()
    tables = s["tables"].tolist()
    seqs = [0] * len(slots) if c["prompt"] else list(range(len(slots)))
    page = torch.tensor([tables[a][b // PAGE] for a, b in zip(seqs, slots)], device=x.device)
    where = torch.tensor([b % PAGE for b in slots], device=x.device)
    for h in range(kvh):
        k_pages[page, h, where] = turned[1][:, h]
        v_pages[page, h, where] = x[:, qh + kvh + h]
        weights[seqs, h, slots] = 0.0
        positions[seqs, h, slots] = torch.tensor(at, dtype=torch.int32, device=x.device)
    got = {"q_out": turned[0], "k_pages": k_pages, "v_pages": v_pages, "weights": weights, "positions": positions}
    if s["lens_out"] is not None:
        got["lens_out"] = torch.tensor([b + 1 for b in slots], dtype=torch.int32)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "evict": _exact_evict, "append": _exact_append}[case["op"]](s)

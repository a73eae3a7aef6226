"""The bounded paged KV cache on the GPU: append, attention with accumulated
weights and eviction, each against a plain form in 64 bits (cache_util.py), and
a decode loop of the three together."""
import math

import numpy as np
import pytest

import cache_util as cu
from cache_util import HD, PAGE, Setup, close, ints

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def be():
    from inference_b200 import B200Backend

    return B200Backend(0)


def bits(t):
    import torch

    return t.view(torch.int16 if t.dtype == torch.bfloat16 else torch.int32)


def same(a, b):
    import torch

    return torch.equal(bits(a), bits(b))


def check_attention(be, s, cache, q, lens, accumulate=True, out=None):
    import torch

    want, tol, dw, dw_tol = cu.attention(s, q, lens)
    before = s.w.clone() if s.w is not None else None
    out = torch.full_like(q, 7.0) if out is None else out
    be.cache_attention(cache, q, ints(lens), out, accumulate=accumulate)
    cache.sync()
    close(out, want, tol, "out")
    if accumulate:
        full = before.double() + dw
        # one more rounding: the addition to the weight
        close(s.w, full, dw_tol + full.abs() * 2.0 ** -23, "weights")
        for r, n in enumerate(lens):  # slots behind the length keep their weights bit for bit
            assert same(s.w[r, :, n:], before[r, :, n:])
    elif before is not None:
        assert same(s.w, before)
    return out


LENS = [[1], [0], [2, 0, 1, 64, 63, 65, 128, 127, 129, 15, 16, 17, 33, 300], [1000], [4095], [20000, 3, 700]]


@pytest.mark.parametrize("qh,kvh", [(8, 8), (16, 8), (32, 8), (64, 8), (8, 1), (16, 1), (12, 4), (5, 1), (22, 2), (7, 7)])
@pytest.mark.parametrize("lens", LENS, ids=lambda v: "x".join(map(str, v)))
def test_attention(be, qh, kvh, lens):
    """Every head-group size and lengths around page and fragment borders, on a shuffled pool whose unused slots hold NaN
    and infinity (they must not reach any output)."""
    s = Setup(len(lens), kvh, max(max(lens), 1), seed=qh * 100 + len(lens))
    s.behind(s.k, lens, math.nan)
    s.behind(s.v, lens, math.inf if qh % 2 else math.nan)
    q = s.randn(len(lens), qh, HD)
    with s.cache() as cache:
        check_attention(be, s, cache, q, lens)


@pytest.mark.parametrize("accumulate", [True, False])
def test_attention_many_rows(be, accumulate):
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(0, 700, 300)]
    s = Setup(300, 2, 700, seed=1)
    q = s.randn(300, 8, HD)
    with s.cache() as cache:
        check_attention(be, s, cache, q, lens, accumulate)


@pytest.mark.parametrize("rows", [31, 32, 33, 100, 255, 256, 257])
@pytest.mark.parametrize("most", [40, 400])
def test_attention_row_counts(be, rows, most):
    """Row counts around those at which the scan of the lengths changes form, idle rows among them; short and long runs."""
    rng = np.random.default_rng(rows)
    lens = [0 if r % 5 == 3 else int(x) for r, x in enumerate(rng.integers(0, most, rows))]
    s = Setup(rows, 1, most, seed=rows)
    q = s.randn(rows, 4, HD)
    with s.cache() as cache:
        check_attention(be, s, cache, q, lens)


def test_attention_most_rows(be):
    """The largest number of sequences, most of them idle."""
    lens = [0] * 4096
    lens[0], lens[1000], lens[4095] = 70, 1, 130
    s = Setup(4096, 1, 130, seed=2)
    q = s.randn(4096, 2, HD)
    with s.cache() as cache:
        check_attention(be, s, cache, q, lens)


def test_attention_strided_rows_padded_slots_and_alias(be):
    """Queries as a slice of a wider row, weights with padding behind the slots, the output over the query; max_len below
    what the buffers cover."""
    import torch

    lens = [100, 1, 77]
    s = Setup(3, 4, 130, seed=3, slot_stride=150)
    wide = s.randn(3, 8 + 4 + 4, HD)
    q = wide[:, :8]
    rest = wide[:, 8:].clone()
    want = q.clone()
    with s.cache(max_len=101) as cache:
        first = check_attention(be, s, cache, want, lens, False)
        be.cache_attention(cache, q, ints(lens), q, accumulate=False)
        cache.sync()
        assert same(q.contiguous(), first) and same(wide[:, 8:].contiguous(), rest)
        strided = torch.zeros(3, 11, HD, dtype=torch.bfloat16, device="cuda")
        check_attention(be, s, cache, want, lens, True, out=strided[:, 2:10])
        assert not strided[:, :2].any() and not strided[:, 10:].any()


def test_attention_of_sharp_and_extreme_scores(be):
    """Scores far apart (one slot takes all), equal everywhere, and so large that exp overflows without the maximum."""
    s = Setup(3, 1, 200, seed=4)
    lens = [200, 200, 190]
    q = s.randn(3, 4, HD)
    q[0] *= 40.0
    q[1] = 0.0
    s.k[s.tables[2, 1].long(), 0, 5] = q[2, 1] * 30.0
    with s.cache() as cache:
        check_attention(be, s, cache, q, lens)


def test_attention_of_nan_and_infinity_in_live_slots(be):
    """What lives in a used slot counts, as in the formula: NaN in a key or value reaches its own sequence and head and no
    other; an infinite value makes its dimension infinite or NaN (the probabilities are multiplied in two parts); a key
    that makes a score -inf drops its slot."""
    import torch

    lens = [70, 70, 70, 70, 10]
    s = Setup(5, 2, 70, seed=6)
    q = s.randn(5, 4, HD).abs() + 0.1
    s.k[s.tables[0, 1].long(), 0, 3, 7] = math.nan
    s.v[s.tables[1, 0].long(), 1, 9, 100] = math.nan
    s.v[s.tables[2, 0].long(), 0, 9, 4] = math.inf
    s.k[s.tables[3, 0].long(), 1, 20, 0] = -math.inf
    before = s.w.clone()
    out = torch.empty_like(q)
    with s.cache() as cache:
        be.cache_attention(cache, q, ints(lens), out)
        cache.sync()
    want, tol, dw, _ = cu.attention(s, q, lens)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), fine)
    assert bool(torch.isnan(out)[torch.isnan(want)].all())
    close(out[fine], want[fine], tol[fine])
    assert torch.equal(torch.isnan(s.w), torch.isnan(before.double() + dw))
    assert float(s.w[3, 1, 20]) == float(before[3, 1, 20])


def test_attention_keeps_the_probabilities_bits(be):
    """Outputs that cancel down to the last bits of a probability.  Three slots with p = 1, p1 = 2^x of -1 < x < 0 and
    p2 near 2^-7 (the division by their sum L comes last), values -c0, 1 and -c2 with c0 = p1 rounded to BF16 and
    c2 = (p1 - c0) / p2 rounded to BF16: what is left is below 2^-17.

    Tolerance: times L, the exponential's 2^-22 of p1 <= 1, the scaling's roundings 2^-24 of |x| < 1 twice, and the sum:
    three parts' products of three slots, each term cut below 2^-23 of the largest, 1: 9 * 2^-23; together below
    12 * 2^-23 (1.4e-6; a probability held in 16 bits is off by up to 2^-18, 3.8e-6).  What p2 is off by is multiplied
    by c2 < 2^-2 and falls inside of it.  Then one rounding to BF16."""
    import torch

    rows, kvh = 64, 8
    s = Setup(rows, kvh, 3, seed=71)
    q = torch.zeros(rows, kvh, HD, dtype=torch.bfloat16, device="cuda")
    q[:, :, 0] = 1.0
    s.k.zero_()
    first = s.tables[:, 0].long()
    s.k[first, :, 1, 0] = -torch.linspace(0.1, 7.8, rows * kvh, device="cuda").view(rows, kvh).bfloat16()
    s.k[first, :, 2, 0] = -55.0
    p = torch.exp(s.k[first, :, :3, 0].double() / HD ** 0.5)  # [rows, kvh, 3]
    p1, p2 = p[..., 1], p[..., 2]
    c0 = p1.bfloat16()
    c2 = ((p1 - c0.double()) / p2).bfloat16()
    s.v[first, :, 0] = -c0[..., None]
    s.v[first, :, 1] = 1.0
    s.v[first, :, 2] = -c2[..., None]
    total = p.sum(dim=-1)
    want = (p1 - c0.double() - p2 * c2.double()) / total
    assert float((want * total).abs().max()) < 2.0 ** -17 and float(c2.double().abs().max()) <= 0.26
    out = torch.empty_like(q)
    with s.cache() as cache:
        be.cache_attention(cache, q, ints([3] * rows), out)
        cache.sync()
    close(out, want[..., None].expand_as(out), (12 * 2.0 ** -23 / total + want.abs() * 2.0 ** -8)[..., None].expand_as(out))


def infinite_values(s, lens):
    """Infinite values in live slots, in dimensions of their own: one of either sign in a sequence's first, middle and last
    slot; both signs in one dimension (NaN by the formula); NaN beside infinity."""
    tables = s.tables.tolist()
    for r, n in enumerate(lens):
        for h in range(s.kvh):
            for dim, marks in ((3, [(0, math.inf)]), (64, [(n // 2, -math.inf)]), (127, [(n - 1, math.inf)]),
                               (50, [(0, math.inf), (n - 1, -math.inf)]), (51, [(0, math.nan), (n // 2, math.inf)]),
                               (52, [(j, math.inf) for j in range(0, n, 50)])):
                if len(marks) == 1 or n > 1:
                    for j, value in marks:
                        s.v[tables[r][j // PAGE], h, j % PAGE, dim] = value


@pytest.mark.parametrize("qh,kvh", [(4, 2), (3, 1), (32, 4), (16, 1)])
@pytest.mark.parametrize("lens", [[1, 64, 70, 16], [2000, 130], [400] * 150, [20000, 3]], ids=lambda v: f"{len(v)}x{v[0]}")
@pytest.mark.parametrize("even", [True, False])
def test_attention_of_infinite_values(be, qh, kvh, lens, even):
    """An infinite value in a live slot makes its dimension infinite, as in the formula: whole runs and cut ones, joined from
    few parts and many, with probabilities that are exact in BF16 (all scores equal) and that are not."""
    import torch

    s = Setup(len(lens), kvh, max(lens), seed=qh + len(lens))
    infinite_values(s, lens)
    q = torch.zeros(len(lens), qh, HD, dtype=torch.bfloat16, device="cuda") if even else s.randn(len(lens), qh, HD)
    want, tol, dw, dw_tol = cu.attention(s, q, lens)
    before, out = s.w.clone(), torch.empty_like(q)
    with s.cache() as cache:
        be.cache_attention(cache, q, ints(lens), out)
        cache.sync()
    fine, got = torch.isfinite(want), out.double()
    assert bool(torch.isinf(want).any())
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    close(got[fine], want[fine], tol[fine], "out")
    full = before.double() + dw
    close(s.w, full, dw_tol + full.abs() * 2.0 ** -23, "weights")


@pytest.mark.parametrize("bad", ["page_high", "page_negative", "length_high", "length_negative"])
def test_attention_refuses_bad_device_values(be, bad):
    """A page outside the pool or a length outside the cache poisons its own row (NaN) and no other, leaves that row's
    weights, and is reported once."""
    import torch

    from inference_b200 import Q3Error

    lens = [100, 150, 64]
    s = Setup(3, 2, 150, seed=7)
    q = s.randn(3, 4, HD)
    want, tol, dw, dw_tol = cu.attention(s, q, lens)
    before = s.w.clone()
    given = list(lens)
    if bad == "page_high":
        s.tables[1, 2] = s.k.shape[0]
    elif bad == "page_negative":
        s.tables[1, 0] = -1
    else:
        given[1] = 151 if bad == "length_high" else -5
    out = torch.zeros_like(q)
    with s.cache() as cache:
        be.cache_attention(cache, q, ints(given), out)
        with pytest.raises(Q3Error) as e:
            cache.sync()
        assert e.value.status == 5 and ("page" if bad.startswith("page") else "length") in str(e.value)
        cache.sync()  # reported and cleared
    assert torch.isnan(out[1]).all()
    close(out[[0, 2]], want[[0, 2]], tol[[0, 2]])
    full = before.double() + dw
    close(s.w[[0, 2]], full[[0, 2]], (dw_tol + full.abs() * 2.0 ** -23)[[0, 2]])
    assert same(s.w[1], before[1])


def test_bad_pages_in_runs_of_one_worker(be):
    """Enough tiles that runs are finished where they were begun, and long ones that are cut: bad pages in the first, a
    middle and the last tile of short and long runs.  Their rows become NaN and keep their weights, all others (bad entries
    behind the length among them) are those of the 64-bit form."""
    import torch

    from inference_b200 import Q3Error

    rng = np.random.default_rng(73)
    lens = [int(x) for x in rng.integers(200, 351, 300)]
    lens[7], lens[100], lens[299] = 2000, 1999, 2000
    s = Setup(300, 2, 2000, seed=74)
    q = s.randn(300, 8, HD)
    want, tol, dw, dw_tol = cu.attention(s, q, lens)
    before = s.w.clone()
    pool = s.k.shape[0]
    for r, page, value in ((0, 0, pool), (3, 1, -1), (4, (lens[4] - 1) // PAGE, 1 << 30), (7, 0, pool), (100, 17, -7),
                           (299, 31, pool + 3), (298, 0, -1), (298, 1, -1), (50, 2, -1 << 31)):
        s.tables[r, page] = value
    bad = [0, 3, 4, 7, 50, 100, 298, 299]
    s.tables[1, (lens[1] + PAGE - 1) // PAGE:] = -1  # no slot lies there
    out = torch.zeros_like(q)
    with s.cache() as cache:
        for accumulate in (True, False):
            be.cache_attention(cache, q, ints(lens), out, accumulate=accumulate)
            with pytest.raises(Q3Error, match="page"):
                cache.sync()
            assert bool(torch.isnan(out[bad]).all())
            good = [r for r in range(300) if r not in bad]
            close(out[good], want[good], tol[good], "out")
            full = before.double() + dw
            close(s.w[good], full[good], (dw_tol + full.abs() * 2.0 ** -23)[good], "weights")
            assert same(s.w[bad], before[bad])
            out.zero_()


def test_attention_of_a_full_gpu(be):
    """Enough tiles that chunks are taken dynamically, in several tiers, and runs are cut into many parts; twice, for the
    same bits whoever takes what."""
    import torch

    lens = [20000, 19999, 1, 20000, 64, 17000, 20000, 8001]
    s = Setup(8, 8, 20000, seed=9)
    q = s.randn(8, 32, HD)
    start = s.w.clone()
    with s.cache() as cache:
        first = check_attention(be, s, cache, q, lens)
        after = s.w.clone()
        for _ in range(2):
            s.w.copy_(start)
            out = torch.empty_like(q)
            be.cache_attention(cache, q, ints(lens), out)
            cache.sync()
            assert same(out, first) and same(s.w, after)


def test_one_very_long_sequence(be):
    """One kv head of sixteen query heads over 150000 slots: every SM has a part of the one run."""
    s = Setup(1, 1, 150000, seed=10)
    q = s.randn(1, 16, HD)
    with s.cache() as cache:
        check_attention(be, s, cache, q, [149999])


def test_far_offsets(be):
    """Pages and slot state whose element offsets pass 32 bits, in all three operators."""
    import torch

    pool, kvh, rows, stride = 34000, 8, 3, 400_000_000  # 2.2e9 elements of K, 9.6e9 of weights
    free = torch.cuda.mem_get_info()[0]
    if free < 120 << 30:
        pytest.skip("needs 100 GB of device memory")
    s = Setup(rows, kvh, 200, seed=13)
    small_k, small_v, small_tables = s.k, s.v, s.tables
    s.k = torch.empty(pool, kvh, PAGE, HD, dtype=torch.bfloat16, device="cuda")
    s.v = torch.empty_like(s.k)
    s.tables = (pool - 1 - torch.arange(12, device="cuda").view(3, 4)).to(torch.int32)
    s.k[s.tables.long().view(-1)] = small_k[small_tables.long().view(-1)]
    s.v[s.tables.long().view(-1)] = small_v[small_tables.long().view(-1)]
    w = torch.empty(rows, kvh, stride, dtype=torch.float32, device="cuda")[:, :, :200]
    p = torch.empty(rows, kvh, stride, dtype=torch.int32, device="cuda")[:, :, :200]
    w.copy_(s.w)
    s.w, s.pos = w, p
    lens = [199, 150, 1]
    weights, positions, next_pos = fill_state(s, lens, seed=2, ties=False)
    q = s.randn(rows, 32, HD)
    rope = tables(be)
    with s.cache() as cache:
        check_attention(be, s, cache, q, lens)
        weights = s.w.cpu().numpy()
        _, moves = cu.evict(lens, next_pos, 100, 20, weights, positions)
        lens_t, held = ints(lens), s.slots(s.k, 0, 7, 199).clone()
        be.cache_evict(cache, lens_t, ints(next_pos), 100, 20, lens_t)
        cache.sync()
        now = s.slots(s.k, 0, 7, 100)
        for a, b in zip(*moves[0, 7]):
            held[a] = held[b]
        assert torch.equal(now, held[:100]) and lens_t.tolist() == [100, 100, 1]
        kv = s.randn(2, rows, kvh, HD)
        out = torch.empty_like(q)
        be.cache_append(cache, q, kv[0], kv[1], s.randn(HD), s.randn(HD), rope, ints([5, 6, 7]), lens_t, out, EPS,
                        lens_out=lens_t)
        cache.sync()
        page = int(s.tables[2, 0])
        assert same(s.v[page, :, 1], kv[1][2]) and int(s.pos[2, 7, 1]) == 7 and lens_t.tolist() == [101, 101, 2]
    del s, w, p
    torch.cuda.empty_cache()


def test_attention_is_deterministic(be):
    import torch

    lens = [5000, 17, 900, 64]
    s = Setup(4, 8, 5000, seed=8)
    q = s.randn(4, 32, HD)
    start = s.w.clone()
    got = []
    with s.cache() as cache:
        for _ in range(3):
            s.w.copy_(start)
            out = torch.empty_like(q)
            be.cache_attention(cache, q, ints(lens), out)
            cache.sync()
            got.append((out, s.w.clone()))
    assert all(same(a, got[0][0]) and same(b, got[0][1]) for a, b in got)


def tables(be, limit=600):
    return be.make_rope_cache(limit, HD, 1e6)


def check_append(be, s, qh, slots, token_pos, row_seq=None, aliases=False):
    """One append against the plain form; everything it does not name stays bit for bit."""
    import torch

    n, kvh = len(slots), s.kvh
    rope = tables(be)
    wide = s.randn(n, qh + 2 * kvh, HD)
    q, k, v = wide.split([qh, kvh, kvh], dim=1)
    qn, kn = s.randn(HD), s.randn(HD)
    pos = ints(token_pos).long().clamp(0, 599)
    zq, tq = cu.turn(q, qn, rope.cosine[pos], rope.sine[pos], EPS)
    zk, tk = cu.turn(k, kn, rope.cosine[pos], rope.sine[pos], EPS)
    before = [x.clone() for x in (s.k, s.v, s.w, s.pos, wide)]
    slot_t = ints(slots)
    q_out = q if aliases else torch.full((n, qh, HD), 5.0, dtype=torch.bfloat16, device="cuda")
    lens_out = slot_t if aliases else torch.full((n,), 99, dtype=torch.int32, device="cuda")
    with s.cache() as cache:
        be.cache_append(cache, q, k, v, qn, kn, rope, ints(token_pos), slot_t, q_out, EPS, lens_out=lens_out,
                        row_seq=None if row_seq is None else ints(row_seq))
        cache.sync()
    wk, wv, ww, wp, ww_ = before
    live = [i for i in range(n) if slots[i] >= 0]
    for i in live:
        seq = i if row_seq is None else row_seq[i]
        page = int(s.tables[seq, slots[i] // PAGE])
        at = slots[i] % PAGE
        close(q_out[i], zq[i], tq[i], "query")
        close(s.k[page, :, at], zk[i], tk[i], "key")
        wk[page, :, at] = s.k[page, :, at]
        wv[page, :, at] = v[i]
        ww[seq, :, slots[i]] = 0.0
        wp[seq, :, slots[i]] = token_pos[i]
        assert int(lens_out[i]) == slots[i] + 1
    for i in set(range(n)) - set(live):
        assert int(lens_out[i]) == (slots[i] if aliases else 99)
        if not aliases:
            assert (q_out[i] == 5.0).all()
    assert same(s.k, wk) and same(s.v, wv) and same(s.w, ww) and same(s.pos, wp)
    if not aliases:
        assert same(wide, ww_)


@pytest.mark.parametrize("aliases", [False, True])
@pytest.mark.parametrize("qh,kvh", [(8, 8), (32, 8), (64, 8), (4, 1), (15, 5), (1, 1)])
def test_append(be, qh, kvh, aliases):
    s = Setup(6, kvh, 200, seed=qh)
    check_append(be, s, qh, [0, 199, 63, 64, -1, 130], [0, 599, 64, 63, 7, 1], aliases=aliases)


def test_append_of_a_prompt(be):
    """Many rows of few sequences, in any order."""
    s = Setup(3, 2, 500, seed=11)
    rng = np.random.default_rng(3)
    seqs = rng.permutation([0] * 400 + [2] * 77).tolist()
    order = {0: rng.permutation(500)[:400].tolist(), 2: rng.permutation(500)[:77].tolist()}
    check_append(be, s, 4, [order[r].pop() for r in seqs], rng.integers(0, 600, 477).tolist(), row_seq=seqs)


@pytest.mark.parametrize("qh,kvh", [(64, 8), (42, 7), (45, 1), (6, 3), (1, 1), (400, 2)])
def test_append_of_many_rows(be, qh, kvh):
    """Enough rows for the streaming form (and, with few heads, rows too short for it, with 400 query heads too long): rows
    left out, rows with bad values among them, every other row as in the plain form."""
    import torch

    from inference_b200 import Q3Error

    n = 1300
    s = Setup(3, kvh, 700, seed=qh)
    rng = np.random.default_rng(qh)
    order = {r: rng.permutation(700).tolist() for r in range(3)}
    seqs = [int(x) for x in rng.integers(0, 3, n)]
    slots = [order[r].pop() for r in seqs]
    token_pos = [int(x) for x in rng.integers(0, 600, n)]
    left_out = sorted(set(int(x) for x in rng.integers(0, n, 60)))
    for j, i in enumerate(left_out):
        if j % 3 == 0:
            slots[i] = -1
        elif j % 3 == 1:
            token_pos[i] = 600 + j
        else:
            slots[i] = 700 + j
    live = torch.ones(n, dtype=torch.bool, device="cuda")
    live[ints(left_out).long()] = False
    rope = tables(be)
    wide = s.randn(n, qh + 2 * kvh, HD)
    q, k, v = wide.split([qh, kvh, kvh], dim=1)
    qn, kn = s.randn(HD), s.randn(HD)
    pos = ints(token_pos).long().clamp(0, 599)
    want_k, want_v, want_w, want_p = s.k.clone(), s.v.clone(), s.w.clone(), s.pos.clone()
    q_out = torch.full((n, qh, HD), 5.0, dtype=torch.bfloat16, device="cuda")
    lens_out = torch.full((n,), 99, dtype=torch.int32, device="cuda")
    with s.cache() as cache:
        be.cache_append(cache, q, k, v, qn, kn, rope, ints(token_pos), ints(slots), q_out, EPS, lens_out=lens_out,
                        row_seq=ints(seqs))
        with pytest.raises(Q3Error):
            cache.sync()
    zq, tq = cu.turn(q, qn, rope.cosine[pos], rope.sine[pos], EPS)
    close(q_out[live], zq[live], tq[live], "query")
    assert (q_out[~live] == 5.0).all() and (lens_out[~live] == 99).all()
    slot, seq = ints(slots).long()[live], ints(seqs).long()[live]
    assert torch.equal(lens_out[live].long(), slot + 1)
    page, at = s.tables[seq, slot // PAGE].long(), slot % PAGE
    zk, tk = cu.turn(k, kn, rope.cosine[pos], rope.sine[pos], EPS)
    close(s.k[page, :, at], zk[live], tk[live], "key")
    want_k[page, :, at] = s.k[page, :, at]
    want_v[page, :, at] = v[live]
    want_w[seq, :, slot] = 0.0
    want_p[seq, :, slot] = ints(token_pos)[live][:, None]
    assert same(s.k, want_k) and same(s.v, want_v) and same(s.w, want_w) and same(s.pos, want_p)


@pytest.mark.parametrize("n,qh,kvh", [(600, 64, 8), (1500, 32, 8), (300, 64, 8)])
def test_append_over_its_inputs(be, n, qh, kvh):
    """Row i into sequence i, the query over the query slice of the QKV rows, the lengths over the slots, rows left out among
    them: by the streaming form (600 and 1500 rows), which reads slots and rows ahead of what it writes, and by the other."""
    import torch

    s = Setup(n, kvh, 150, seed=n + qh)
    rng = np.random.default_rng(n)
    slots = rng.integers(0, 150, n).astype(np.int32)
    slots[rng.integers(0, n, n // 9)] = -1
    token_pos = [int(x) for x in rng.integers(0, 600, n)]
    live = torch.from_numpy(slots >= 0).cuda()
    rope = tables(be)
    wide = s.randn(n, qh + 2 * kvh, HD)
    was = wide.clone()
    q, k, v = wide.split([qh, kvh, kvh], dim=1)
    qn, kn = s.randn(HD), s.randn(HD)
    want_k, want_v, want_w, want_p = s.k.clone(), s.v.clone(), s.w.clone(), s.pos.clone()
    lens = torch.from_numpy(slots).cuda()
    with s.cache() as cache:
        be.cache_append(cache, q, k, v, qn, kn, rope, ints(token_pos), lens, q, EPS, lens_out=lens)
        cache.sync()
    slot = torch.from_numpy(slots).cuda().long()
    assert torch.equal(lens.long(), torch.where(live, slot + 1, slot))
    assert same(wide[:, qh:].contiguous(), was[:, qh:].contiguous())
    assert same(wide[~live].contiguous(), was[~live].contiguous())
    pos, seq, slot = ints(token_pos).long(), torch.arange(n, device="cuda")[live], slot[live]
    zq, tq = cu.turn(was[:, :qh], qn, rope.cosine[pos], rope.sine[pos], EPS)
    close(q[live], zq[live], tq[live], "query")
    page, at = s.tables[seq, slot // PAGE].long(), slot % PAGE
    zk, tk = cu.turn(was[:, qh:qh + kvh], kn, rope.cosine[pos], rope.sine[pos], EPS)
    close(s.k[page, :, at], zk[live], tk[live], "key")
    want_k[page, :, at] = s.k[page, :, at]
    want_v[page, :, at] = was[live, qh + kvh:]
    want_w[seq, :, slot] = 0.0
    want_p[seq, :, slot] = pos[live][:, None].int()
    assert same(s.k, want_k) and same(s.v, want_v) and same(s.w, want_w) and same(s.pos, want_p)


@pytest.mark.parametrize("what,row", [("slot", (200, 5, 0)), ("slot", (-2, 5, 0)), ("position", (3, 600, 0)),
                                      ("position", (3, -1, 0)), ("sequence", (3, 5, 2)), ("sequence", (3, 5, -1)),
                                      ("page", (70, 5, 1))])
def test_append_refuses_bad_device_values(be, what, row):
    """The row is left out, the others are written, the error is reported once."""
    import torch

    from inference_b200 import Q3Error

    s = Setup(2, 2, 200, seed=12)
    s.tables[1, 1] = s.k.shape[0] + 5
    rope = tables(be)
    slots, token_pos, seqs = [1, row[0]], [1, row[1]], [0, row[2]]
    before = [x.clone() for x in (s.k, s.v, s.w, s.pos)]
    q, k, v = s.randn(2, 4, HD), s.randn(2, 2, HD), s.randn(2, 2, HD)
    qn = s.randn(HD)
    q_out = torch.zeros_like(q)
    lens_out = ints([0, 0])
    with s.cache() as cache:
        be.cache_append(cache, q, k, v, qn, qn, rope, ints(token_pos), ints(slots), q_out, EPS, lens_out=lens_out,
                        row_seq=ints(seqs))
        with pytest.raises(Q3Error) as e:
            cache.sync()
        assert e.value.status == 5 and what in str(e.value)
        cache.sync()
    page = int(s.tables[0, 0])
    assert same(s.v[page, :, 1], v[0]) and lens_out.tolist() == [2, 0]
    assert not q_out[1].any() and q_out[0].any()
    for now, was in zip((s.k, s.v), before):
        was[page, :, 1] = now[page, :, 1]
        assert same(now, was)
    assert same(s.w[1], before[2][1]) and same(s.pos[1], before[3][1])


def fill_state(s, lens, seed, ties):
    """Weights (with ties and special values) and distinct positions of each sequence's slots, in any order."""
    rng = np.random.default_rng(seed)
    w = np.exp(2.0 * rng.standard_normal(tuple(s.w.shape))).astype(np.float32)
    if ties:
        w = np.round(w).astype(np.float32)
        w.reshape(-1)[rng.integers(0, w.size, w.size // 10)] = -0.0
    p = np.zeros(w.shape, np.int32)
    for r, n in enumerate(lens):
        for h in range(w.shape[1]):
            p[r, h, :n] = rng.permutation(n) + 10
    s.w.copy_(cu.torch().from_numpy(w))
    s.pos.copy_(cu.torch().from_numpy(p))
    return w, p, [n + 10 for n in lens]


def check_evict(be, s, lens, keep, recent, w, p, next_pos, in_place):
    import torch

    want_lens, moves = cu.evict(lens, next_pos, keep, recent, w, p)
    before = [x.clone() for x in (s.k, s.v, s.w, s.pos)]
    wk, wv, ww, wp = cu.apply_moves(s, moves, *before)
    lens_t = ints(lens)
    lens_out = lens_t if in_place else torch.full_like(lens_t, 77)
    wo = po = None
    if not in_place:
        whole = (s.rows, s.kvh, s.w.stride(1))
        wo = torch.full(whole, 3.0, device="cuda")[:, :, :s.max_len]
        po = torch.full(whole, 3, dtype=torch.int32, device="cuda")[:, :, :s.max_len]
    with s.cache() as cache:
        be.cache_evict(cache, lens_t, ints(next_pos), keep, recent, lens_out, weights_out=wo, positions_out=po)
        cache.sync()
    assert lens_out.tolist() == want_lens
    assert same(s.k, wk) and same(s.v, wv)
    if in_place:
        assert same(s.w, ww) and same(s.pos, wp)
    else:
        assert same(s.w, before[2]) and same(s.pos, before[3])
        for r, n in enumerate(want_lens):
            assert same(wo[r, :, :n], ww[r, :, :n]) and same(po[r, :, :n], wp[r, :, :n])
            assert (wo[r, :, n:] == 3.0).all() and (po[r, :, n:] == 3).all()


EVICT = [([65], 64, 0), ([65], 64, 64), ([1, 0, 5], 1, 0), ([300, 40, 301, 64, 1000], 64, 20),
         ([1000, 999, 0, 500], 500, 499), ([1000, 700], 699, 900), ([5000, 1025, 1024], 1024, 100), ([20000], 333, 64),
         ([33000, 2000], 30000, 1000), ([70], 1 << 19, 3)]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("lens,keep,recent", EVICT, ids=lambda v: str(v).replace(" ", ""))
def test_evict(be, lens, keep, recent, ties, in_place):
    s = Setup(len(lens), 3, max(max(lens), 1), seed=keep, slot_stride=max(lens) + 7)
    w, p, next_pos = fill_state(s, lens, seed=sum(lens), ties=ties)
    check_evict(be, s, lens, keep, recent, w, p, next_pos, in_place)


@pytest.mark.parametrize("rows,kvh,max_len,keep", [(20, 3, 8200, 3000), (10, 3, 8200, 8000), (80, 1, 21000, 5000),
                                                   (1, 1, 200000, 60000), (2, 2, 9000, 8999), (200, 1, 70, 65)])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_shapes(be, rows, kvh, max_len, keep, ties):
    """Clusters of two and four, pieces too long for their keys to be kept, few and many moves, over most sequences short."""
    lens = [max_len if r % 37 == 0 else (r * 977) % min(max_len, 400) for r in range(rows)]
    s = Setup(rows, kvh, max_len, seed=rows)
    w, p, next_pos = fill_state(s, lens, seed=rows + kvh, ties=ties)
    check_evict(be, s, lens, keep, keep // 3, w, p, next_pos, in_place=not ties)


@pytest.mark.parametrize("rows,kvh,max_len,keep", [(80, 1, 3000, 1000), (1, 1, 20000, 6000), (3, 2, 2500, 2400)])
@pytest.mark.parametrize("scale", [1e-24, 1e-13, 1e-7, 1e4, 1e8])
def test_evict_weights_of_any_size(be, rows, kvh, max_len, keep, scale):
    """Weights far below and above the usual ones, all different and in few octaves: as many as a histogram can mix."""
    lens = [max_len - (r * 13) % 40 for r in range(rows)]
    s = Setup(rows, kvh, max_len, seed=rows)
    _, p, next_pos = fill_state(s, lens, seed=7, ties=False)
    w = (scale * (1.0 + np.random.default_rng(rows).random(p.shape))).astype(np.float32)
    s.w.copy_(cu.torch().from_numpy(w))
    check_evict(be, s, lens, keep, keep // 5, w, p, next_pos, True)


def test_evict_equal_and_special_weights(be):
    """All weights equal (ties by slot), NaN last, infinities and negatives in order, denormals, every slot recent."""
    lens = [200] * 5
    s = Setup(5, 1, 200, seed=21)
    w, p, next_pos = fill_state(s, lens, seed=4, ties=False)
    w[0] = 1.25
    w[1, 0, ::3] = np.nan
    w[2, 0, :6] = [np.inf, -np.inf, -1.0, 0.0, -0.0, 1e-42]
    w[2, 0, 6:] = np.float32(1e-41)
    w[3] = np.nan
    s.w.copy_(cu.torch().from_numpy(w))
    next_pos[4] = 0  # every position is recent
    check_evict(be, s, lens, 100, 0, w, p, next_pos, True)


def test_evict_refuses_bad_device_values(be):
    """A bad length or page leaves its sequence as it was and is reported; the others shrink."""
    import torch

    from inference_b200 import Q3Error

    for bad in ("length", "page"):
        lens = [150, 150, 150]
        s = Setup(3, 2, 150, seed=22)
        w, p, next_pos = fill_state(s, lens, seed=5, ties=False)
        if bad == "page":
            s.tables[1, 2] = -7
        given = ints([150, 151 if bad == "length" else 150, 150])
        before = [x.clone() for x in (s.k, s.v, s.w, s.pos)]
        ok = Setup(3, 2, 150, seed=22)
        _, moves = cu.evict([150, 0, 150], next_pos, 64, 10, w, p)
        want = cu.apply_moves(ok, moves, *before)
        with s.cache() as cache:
            be.cache_evict(cache, given, ints(next_pos), 64, 10, given)
            with pytest.raises(Q3Error) as e:
                cache.sync()
            assert e.value.status == 5 and bad in str(e.value)
        assert given.tolist() == [64, 151 if bad == "length" else 150, 64]
        for now, expect in zip((s.k, s.v, s.w, s.pos), want):
            assert same(now, expect)
        torch.cuda.synchronize()


def test_bounded_decode_loop(be):
    """Append, attend, evict as a user runs them: sequences of different lengths decode past their budget.  Every step's
    output is held to the 64-bit form over the slots that the plain form of the earlier evictions left (chosen by the
    weights that the cache reports), and each slot's position says which token it holds."""
    import torch

    qh, kvh, keep, recent, cap, steps = 8, 2, 96, 32, 112, 60
    start = [90, 3, 0]
    s = Setup(3, kvh, cap, seed=31)
    rope = tables(be)
    qn, kn = s.randn(HD), s.randn(HD)
    s.w.zero_()
    keys, values = {}, {}  # (row, position) -> the token's stored key and value rows
    lens = ints(start)
    next_pos = ints(start)
    for r, n in enumerate(start):
        for h in range(kvh):
            s.pos[r, h, :n] = torch.arange(n, dtype=torch.int32, device="cuda")
        for j in range(n):
            page = int(s.tables[r, j // PAGE])
            keys[r, j], values[r, j] = s.k[page, :, j % PAGE].clone(), s.v[page, :, j % PAGE].clone()
    with s.cache() as cache:
        for step in range(steps):
            wide = s.randn(3, qh + 2 * kvh, HD)
            q, k, v = wide.split([qh, kvh, kvh], dim=1)
            q_out = torch.empty(3, qh, HD, dtype=torch.bfloat16, device="cuda")
            slots = lens.clone()
            be.cache_append(cache, q, k, v, qn, kn, rope, next_pos, lens, q_out, EPS, lens_out=lens)
            now = lens.tolist()
            for r in range(3):
                at = int(slots[r])
                page = int(s.tables[r, at // PAGE])
                pos = int(next_pos[r])
                keys[r, pos], values[r, pos] = s.k[page, :, at % PAGE].clone(), s.v[page, :, at % PAGE].clone()
            check_attention(be, s, cache, q_out, now)
            next_pos += 1
            if step % 5 == 4:
                w, p = s.w.cpu().numpy(), s.pos.cpu().numpy()
                want_lens, moves = cu.evict(now, next_pos.tolist(), keep, recent, w, p)
                want = cu.apply_moves(s, moves, s.k, s.v, s.w, s.pos)
                be.cache_evict(cache, lens, next_pos, keep, recent, lens)
                cache.sync()
                assert lens.tolist() == want_lens
                assert all(same(a, b) for a, b in zip((s.k, s.v, s.w, s.pos), want))
        lens_now = lens.tolist()
    assert lens_now == [keep, 63, 60]
    for r, n in enumerate(lens_now):
        for h in range(kvh):
            held = s.pos[r, h, :n].tolist()
            assert len(set(held)) == n and set(range(int(next_pos[r]) - recent, int(next_pos[r]))) <= set(held)
            for j, pos in enumerate(held):
                page = int(s.tables[r, j // PAGE])
                assert same(s.k[page, h, j % PAGE], keys[r, pos][h]) and same(s.v[page, h, j % PAGE], values[r, pos][h])


def test_captured_step_replays(be):
    """One step of the three calls as a CUDA graph: two graphs on the same cache, replayed in turn with lengths and
    positions that advance on the device, against the same calls made one by one."""
    import torch

    qh, kvh, keep, recent, cap = 8, 2, 70, 16, 80
    rope = tables(be)

    def state():
        s = Setup(3, kvh, cap, seed=41)
        s.w.zero_()
        s.pos.copy_(torch.arange(cap, dtype=torch.int32, device="cuda").expand(3, kvh, cap))
        s.lens, s.next = ints([69, 70, 12]), ints([69, 70, 12])
        s.q = [s.randn(3, qh, HD) for _ in range(2)]
        s.kv = [(s.randn(3, kvh, HD), s.randn(3, kvh, HD)) for _ in range(2)]
        s.qn, s.out = s.randn(HD), [torch.zeros(3, qh, HD, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        return s

    def step(s, cache, i):
        q_out = torch.empty_like(s.q[i])
        be.cache_append(cache, s.q[i], *s.kv[i], s.qn, s.qn, rope, s.next, s.lens, q_out, EPS, lens_out=s.lens)
        be.cache_attention(cache, q_out, s.lens, s.out[i])
        s.next.add_(1)
        be.cache_evict(cache, s.lens, s.next, keep, recent, s.lens)

    a, b = state(), state()
    with a.cache() as ca, b.cache() as cb:
        side = torch.cuda.Stream()
        graphs = []
        with torch.cuda.stream(side):
            for i in range(2):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=side):
                    step(b, cb, i)
                graphs.append(g)
        torch.cuda.synchronize()
        for n in range(6):
            step(a, ca, n % 2)
            graphs[n % 2].replay()
            torch.cuda.synchronize()
            for x, y in zip((a.k, a.v, a.w, a.pos, a.lens, a.out[0], a.out[1]),
                            (b.k, b.v, b.w, b.pos, b.lens, b.out[0], b.out[1])):
                assert same(x, y), n
        ca.sync()
        cb.sync()
        del graphs


def test_lengths_written_right_before(be):
    """Lengths that a kernel writes right before each attention, another set every time: the runs of every call are those of
    its own lengths, one call after the other and as a graph."""
    import torch

    rng = np.random.default_rng(17)
    sets = [[int(x) for x in rng.integers(0, 900, 40)] for _ in range(6)]
    s = Setup(40, 2, 900, seed=18)
    q = s.randn(40, 8, HD)
    want = [cu.attention(s, q, lens) for lens in sets]
    given = torch.stack([ints(lens) for lens in sets])
    which, lens = torch.zeros(1, dtype=torch.int64, device="cuda"), ints([0] * 40)
    start, out = s.w.clone(), torch.empty_like(q)

    def step(cache):
        torch.index_select(given, 0, which, out=lens.view(1, -1))
        be.cache_attention(cache, q, lens, out)

    with s.cache() as cache:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                step(cache)
        torch.cuda.synchronize()
        for n in range(60):
            i = n * 5 % 6
            s.w.copy_(start)
            which.fill_(i)
            step(cache) if n % 2 else g.replay()
            o, tol, dw, dw_tol = want[i]
            close(out, o, tol, f"out {n}")
            full = start.double() + dw
            close(s.w, full, dw_tol + full.abs() * 2.0 ** -23, f"weights {n}")
        cache.sync()
        del g


def test_calls_behind_copies_in_a_graph(be):
    """Captured behind a copy and a fill, not a kernel: the calls wait for them."""
    import torch

    lens, other = ints([5, 90, 0]), ints([90, 33, 64])
    s = Setup(3, 2, 90, seed=42)
    q = s.randn(3, 8, HD)
    want, tol, _, _ = cu.attention(s, q, other.tolist())
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    with s.cache() as cache:
        with torch.cuda.stream(side):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                lens.copy_(other)
                be.cache_attention(cache, q, lens, out, accumulate=False)
                lens.zero_()
                be.cache_evict(cache, lens, lens, 10, 0, lens)
        torch.cuda.synchronize()
        for _ in range(3):
            out.zero_()
            lens.fill_(1)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            close(out, want, tol)
            assert lens.tolist() == [0, 0, 0]
        cache.sync()
        del g


def test_python_checks(be):
    """What the Python layer refuses before the C ABI sees it."""
    import torch

    from inference_b200 import PagedCache

    s = Setup(2, 2, 100, seed=1)
    with pytest.raises(ValueError):
        PagedCache(s.k, s.v.float(), s.tables, s.w, s.pos)
    with pytest.raises(ValueError):
        PagedCache(s.k, s.v, s.tables.long(), s.w, s.pos)
    with pytest.raises(ValueError):
        PagedCache(s.k, s.v, s.tables, s.w, None)
    with pytest.raises(ValueError):
        PagedCache(s.k, s.v, s.tables, s.w[:1], s.pos)
    with pytest.raises(ValueError):
        PagedCache(s.k, s.v, s.tables, s.w, s.pos, max_len=101)
    with pytest.raises(ValueError):
        PagedCache(s.k.transpose(0, 1), s.v.transpose(0, 1), s.tables)
    q, lens, out = s.randn(2, 4, HD), ints([5, 5]), torch.empty(2, 4, HD, dtype=torch.bfloat16, device="cuda")
    cache = s.cache()
    for bad in (dict(query=q[:1]), dict(query=q.float()), dict(query=q.transpose(1, 2)), dict(lens=lens.long()),
                dict(lens=lens[:1]), dict(lens=lens.cpu()), dict(output=out[:, :2]), dict(query=s.randn(2, 3, HD))):
        with pytest.raises((ValueError, RuntimeError)):
            be.cache_attention(cache, **{**dict(query=q, lens=lens, output=out), **bad})
    with pytest.raises(ValueError):
        be.cache_evict(cache, lens, lens, 0, 5, lens)
    with pytest.raises(ValueError):
        be.cache_evict(cache, lens, lens, 5, -1, lens)
    with pytest.raises(ValueError):
        be.cache_evict(cache, lens, lens, 5, 1, lens, weights_out=s.w[:, :, :50], positions_out=s.pos[:, :, :50])
    rope = tables(be, 10)
    kv = s.randn(2, 2, HD)
    be.cache_append(cache, q[:0], kv[:0], kv[:0], s.randn(HD), s.randn(HD), rope, lens[:0], lens[:0], out[:0], EPS)
    with pytest.raises(ValueError):
        be.cache_append(cache, q, kv, kv, s.randn(HD)[:64], s.randn(HD), rope, lens, lens, out, EPS)
    with pytest.raises(ValueError):
        be.cache_append(cache, q, kv[:, :1], kv, s.randn(HD), s.randn(HD), rope, lens, lens, out, EPS)
    cache.sync()
    cache.close()
    with pytest.raises(ValueError):
        be.cache_attention(cache, q, lens, out)
    plain = Setup(2, 2, 100, seed=1, weights=False)
    with plain.cache() as c2:
        with pytest.raises(RuntimeError, match="no weights"):
            be.cache_attention(c2, q, lens, out)
        be.cache_attention(c2, q, lens, out, accumulate=False)
        c2.sync()


def test_calls_on_two_streams(be):
    """Two caches, each on its own stream, at the same time: the same results as one after the other."""
    import torch

    lens = [3000, 100, 64]
    sets = [Setup(3, 4, 3000, seed=51 + i) for i in range(2)]
    qs = [s.randn(3, 16, HD) for s in sets]
    alone, start = [], [s.w.clone() for s in sets]
    caches = [s.cache() for s in sets]
    for s, q, c in zip(sets, qs, caches):
        out = torch.empty_like(q)
        be.cache_attention(c, q, ints(lens), out)
        c.sync()
        alone.append((out, s.w.clone()))
    streams = [torch.cuda.Stream() for _ in sets]
    lens_t = ints(lens)
    for _ in range(5):
        for s, w in zip(sets, start):
            s.w.copy_(w)
        outs = [torch.zeros_like(q) for q in qs]
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                be.cache_attention(caches[i], qs[i], lens_t, outs[i])
        torch.cuda.synchronize()
        for i in range(2):
            assert same(outs[i], alone[i][0]) and same(sets[i].w, alone[i][1])
    for c in caches:
        c.close()


def test_cache_dropped_behind_a_call_on_another_stream(be):
    """A cache made on one stream, used on another and dropped while that one is busy: the memory of its state words is not
    given out again before the other stream is done."""
    import torch

    s = Setup(3, 2, 100, seed=61)
    q, lens = s.randn(3, 8, HD), ints([100, 5, 64])
    want, tol, _, _ = cu.attention(s, q, lens.tolist())
    side, out = torch.cuda.Stream(), torch.empty_like(q)
    torch.cuda.synchronize()
    cache = s.cache()
    at = cache.state.data_ptr()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # some 0.2 s
        be.cache_attention(cache, q, lens, out)
    cache.close()
    del cache
    others = [torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(64)]
    assert not side.query() and at not in [t.data_ptr() for t in others]
    torch.cuda.synchronize()
    close(out, want, tol)
    assert not any(bool(t.any()) for t in others)


def test_captured_calls_do_not_mark_streams(be):
    """Calls on a capturing stream leave the allocator's records alone, and the graph replays."""
    import torch

    s = Setup(2, 2, 100, seed=62)
    q, lens, out = s.randn(2, 8, HD), ints([100, 7]), torch.empty(2, 8, HD, dtype=torch.bfloat16, device="cuda")
    want, tol, _, _ = cu.attention(s, q, lens.tolist())
    with s.cache() as cache:
        known = set(cache._streams)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                be.cache_attention(cache, q, lens, out, accumulate=False)
        assert cache._streams == known
        g.replay()
        torch.cuda.synchronize()
        close(out, want, tol)
        with torch.cuda.stream(side):
            be.cache_attention(cache, q, lens, out, accumulate=False)
        assert cache._streams == known | {side.cuda_stream}
        cache.sync()
        del g

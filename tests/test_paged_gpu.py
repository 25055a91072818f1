"""The operators over a pool of cache pages (paged.rope_append, paged.attention) against plain implementations in 64 bits.

Every pool is NaN wherever no position of a sequence lies, and entries of the page table that belong to no position hold nonsense: whatever
is read by mistake shows.

Tolerance of the attention, element by element, with A = the attention of |v| and S = the largest scale * sum_i |q_i k_i|:
  the output's rounding                           h |o|          h = finfo(type).eps / 2
  the probabilities' rounding to the type         h A            (sums of up to 2^-8 p v with weights that sum to one)
  scores: 128 products added in fp32, each add off by up to 2^-23 (tensor cores truncate), to a weight and to the sum of weights
                                                  2 * 130 * 2^-23 S A
  sums over n keys, in output and denominator, exp2 (2^-22) and the rescaling of running sums (n / 16 times at most)
                                                  2 * (n + n / 16 + 8) * 2^-23 A"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def make_pool(g, lens, page, kv_heads, dtype, *, layers=1, order="slots", spare=3, scale=1.0):
    """A poisoned pool, the page table and the true K and V rows [total, kv_heads, 128] of every sequence."""
    from qwen3mk import paged

    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    shape = (layers, pages, page, kv_heads, D)
    if order == "slots":
        k, v = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    else:                                            # heads outside the slots, K and V of a page side by side
        both = torch.full((layers, pages, 2, kv_heads, page, D), float("nan"), dtype=dtype, device="cuda")
        k, v = both[:, :, 0].transpose(2, 3), both[:, :, 1].transpose(2, 3)
    ids = torch.randperm(pages, generator=g).tolist()
    table = torch.randint(-2**31, 2**31 - 1, (len(lens), max(1, max(counts)) + 2), generator=g, dtype=torch.int64).to(torch.int32)
    rows = []
    for b, n in enumerate(lens):
        mine = [ids.pop() for _ in range(counts[b])]
        table[b, :counts[b]] = torch.tensor(mine, dtype=torch.int32)
        kr, vr = ((torch.randn(n, kv_heads, D, generator=g) * scale).to(dtype).cuda() for _ in range(2))
        where = torch.tensor([mine[p // page] for p in range(n)], dtype=torch.long, device="cuda"), torch.arange(n, device="cuda") % page
        k[layers - 1][where], v[layers - 1][where] = kr, vr
        rows.append((kr, vr))
    return paged.PagePool(k, v), table.cuda(), rows


def reference(q, rows, news, lens, scale, there=None):
    """o, A, S of the formula: 64 bits, a sequence and a head at a time, keys that a token does not see left out by index."""
    heads, o, big, most = q.shape[1], torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda"), 0.0
    at = 0
    for b, (new, n) in enumerate(zip(news, lens)):
        kr, vr = rows[b]
        group = heads // kr.shape[1]
        keep = torch.ones(n, dtype=torch.bool, device="cuda") if there is None else there[b]
        pos = torch.arange(n, device="cuda")
        for h in range(heads):
            key, val = kr[:, h // group].double(), vr[:, h // group].double()
            s = q[at:at + new, h].double() @ torch.nan_to_num(key, 0, 0, 0).T * scale
            s = torch.where(torch.isfinite(key).all(dim=1), s, torch.full_like(s, float("nan")))
            seen = keep & (pos <= (n - new + torch.arange(new, device="cuda"))[:, None])
            s = s.masked_fill(~seen, float("-inf"))
            p = torch.softmax(s, dim=-1)
            p = torch.where(seen.any(dim=-1, keepdim=True), p, torch.zeros_like(p)) if n else p.new_zeros(new, 0)
            fin = torch.isfinite(val)
            o[at:at + new, h] = p @ torch.where(fin, val, torch.zeros_like(val))
            spoiled = (seen.double() @ (~fin).double()) > 0
            o[at:at + new, h] = torch.where(spoiled, torch.full_like(o[at:at + new, h], float("nan")), o[at:at + new, h])
            big[at:at + new, h] = p @ torch.where(fin, val, torch.zeros_like(val)).abs()
            if n and new:
                most = max(most, float((q[at:at + new, h].double().abs() @ torch.nan_to_num(key, 0, 0, 0).abs().T).max()) * scale)
        at += new
    return o, big, most


def check(got, q, rows, news, lens, scale=D ** -0.5, there=None):
    o, big, most = reference(q, rows, news, lens, scale, there)
    n, h = max(max(lens), 1), torch.finfo(q.dtype).eps / 2
    tol = h * o.abs() + (h + 2.0 ** -23 * (2 * 130 * most + 2 * (n + n / 16 + 8))) * big + 2.0 ** -24
    nan = torch.isnan(o)
    # (a row spoiled by an infinite value is infinite or NaN)
    assert torch.equal(~torch.isfinite(got), nan), f"{int((~torch.isfinite(got) ^ nan).sum())} values finite on one side only"
    worst = ((got.double() - o).abs() / tol).masked_fill(nan, 0)
    assert float(worst.max()) <= 1.0, f"off by {float(worst.max()):.2f} tolerances at {torch.nonzero(worst == worst.max())[0].tolist()}"


def describe(pool, table, news, lens, **kw):
    from qwen3mk import paged

    start = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda()
    return paged.PagedBatch(pool, table, start, torch.tensor(lens, dtype=torch.int32).cuda(), **kw)


CASES = [
    # (new tokens, all positions) of every sequence, page, q heads, kv heads
    ([(1, 1)], 16, 16, 8),
    ([(1, 1000)], 64, 16, 8),
    ([(1, 63), (1, 64), (1, 65), (1, 1), (1, 128), (1, 129)], 16, 16, 8),
    ([(0, 100), (1, 17), (0, 0), (1, 300), (0, 5)], 32, 16, 8),
    ([(4, 4), (3, 70), (1, 500)], 16, 16, 8),
    ([(5, 5), (8, 333)], 128, 16, 8),
    ([(13, 1313), (16, 16), (2, 900)], 16, 8, 4),
    ([(17, 17), (40, 1000), (1, 77)], 64, 16, 8),
    ([(1, 2000), (2, 130)], 256, 8, 8),
    ([(3, 700), (1, 90)], 64, 8, 2),
    ([(7, 411), (1, 16)], 32, 16, 2),
    ([(33, 33), (31, 200)], 16, 4, 1),
    ([(129, 129), (64, 64), (63, 700), (200, 1100)], 64, 16, 8),
    ([(300, 300)], 128, 16, 8),
    ([(127, 1151), (1, 2100), (1, 3), (66, 66)], 16, 8, 8),
    ([(257, 999), (2, 2)], 256, 8, 1),
    ([(1000, 1000), (0, 300), (1, 4097)], 32, 8, 4),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_matches_the_formula(case, dtype):
    from qwen3mk import paged

    seqs, page, heads, kv_heads = CASES[case]
    news, lens = [s[0] for s in seqs], [s[1] for s in seqs]
    g = torch.Generator().manual_seed(case)
    pool, table, rows = make_pool(g, lens, page, kv_heads, dtype, layers=2, order="heads" if case % 2 else "slots")
    q = torch.randn(sum(news), heads, D, generator=g).to(dtype).cuda()
    batch = describe(pool, table, news, lens)
    out = torch.full_like(q, float("nan"))
    assert paged.attention(batch, q, 1, out=out) is out
    check(out, q, rows, news, lens)
    assert torch.equal(paged.attention(batch, q, 1), out), "another run gives other bits"


def test_many_sequences_of_every_length():
    """A thousand sequences, most of them short, one long, some without a new token."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(3)
    lens = torch.randint(1, 200, (1024,), generator=g).tolist()
    news = [min(n, int(x)) for n, x in zip(lens, torch.randint(0, 3, (1024,), generator=g))]
    lens[500], news[500] = 20000, 2
    pool, table, rows = make_pool(g, lens, 16, 2, torch.bfloat16)
    q = torch.randn(sum(news), 4, D, generator=g).to(torch.bfloat16).cuda()
    check(paged.attention(describe(pool, table, news, lens), q), q, rows, news, lens)


@pytest.mark.parametrize("news,lens", [([1], [70000]), ([12], [33000]), ([90, 1], [9000, 9000])])
def test_long_caches(news, lens):
    from qwen3mk import paged

    g = torch.Generator().manual_seed(4)
    pool, table, rows = make_pool(g, lens, 64, 2, torch.bfloat16)
    q = torch.randn(sum(news), 4, D, generator=g).to(torch.bfloat16).cuda()
    check(paged.attention(describe(pool, table, news, lens), q), q, rows, news, lens)


@pytest.mark.parametrize("new", [1, 3, 16, 100])
def test_offsets_beyond_32_bits(new):
    """Pages whose elements lie more than 2^31 elements (and 2^32 bytes) behind the pool's first."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(5)
    page, kv_heads, n = 64, 8, 400
    k, v = (torch.empty((1, 33000, page, kv_heads, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pool = paged.PagePool(k, v)
    ids = [32999, 5, 32998, 32790, 0, 32999 - 7, 32997]
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    kr, vr = (torch.randn(n, kv_heads, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    for i, p in enumerate(ids):
        m = min(page, n - i * page)
        k[0, p, :m], v[0, p, :m] = kr[i * page:i * page + m], vr[i * page:i * page + m]
    q = torch.randn(new, 16, D, generator=g).to(torch.bfloat16).cuda()
    batch = describe(pool, table, [new], [n])
    check(paged.attention(batch, q), q, [(kr, vr)], [new], [n])
    # the same slots are written where they are read
    rows = torch.randn(new, 32, D, generator=g).cuda()
    paged.rope_append(batch, rows[:, :16], rows[:, 16:24], rows[:, 24:], None)
    for t in range(new):
        p = n - new + t
        assert torch.equal(k[0, ids[p // page], p % page], rows[t, 16:24].to(torch.bfloat16)) and torch.equal(v[0, ids[p // page], p % page], rows[t, 24:].to(torch.bfloat16))


@pytest.mark.parametrize("new", [1, 9, 150])
def test_missing_pages_are_not_attended(new):
    from qwen3mk import paged

    g = torch.Generator().manual_seed(6)
    page, n = 16, 700
    pool, table, rows = make_pool(g, [n, 40], page, 8, torch.bfloat16)
    gone = [0, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 20, 43]
    for i, j in enumerate(gone):
        table[0, j] = (-1, pool.pages, 2**31 - 1, -2**31)[i % 4]
    there = [torch.tensor([p // page not in gone for p in range(n)], device="cuda"), torch.ones(40, dtype=torch.bool, device="cuda")]
    q = torch.randn(new + 2, 16, D, generator=g).to(torch.bfloat16).cuda()
    check(paged.attention(describe(pool, table, [new, 2], [n, 40]), q), q, rows, [new, 2], [n, 40], there=there)
    # a sequence of which nothing is left: zeros
    table[0] = -1
    out = paged.attention(describe(pool, table, [new, 2], [n, 40]), q)
    assert not out[:new].any() and torch.isfinite(out).all() and out[new:].any()


@pytest.mark.parametrize("new,n", [(5, 3), (4, 0), (100, 30), (70, 0), (300, 299)])
def test_tokens_without_a_position_get_zeros(new, n):
    """Fewer positions than new tokens: the first ones see nothing."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(7)
    pool, table, rows = make_pool(g, [n, 200], 16, 8, torch.float16)
    q = torch.randn(new + 1, 16, D, generator=g).to(torch.float16).cuda()
    out = torch.full_like(q, float("nan"))
    paged.attention(describe(pool, table, [new, 1], [n, 200]), q, out=out)
    assert not out[:new - n].any()
    check(out, q, rows, [new, 1], [n, 200])


@pytest.mark.parametrize("new", [2, 7, 16, 60, 200])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_row_that_is_not_seen_does_not_touch_the_result(new, value):
    """A later token's K or V row, and what lies behind the last position, may hold anything; rows that do see such a V row are not finite."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(8)
    n, page = new + 90, 16
    pool, table, rows = make_pool(g, [n, n], page, 8, torch.bfloat16)
    q = torch.randn(2 * new, 16, D, generator=g).to(torch.bfloat16).cuda()
    p = n - 1 - new // 3                             # seen by the last tokens alone
    at, slot = int(table[0, p // page]), p % page
    pool.v[0, at, slot, 3, 17] = value
    rows[0][1][p, 3, 17] = value
    out = paged.attention(describe(pool, table, [new, new], [n, n]), q)
    check(out, q, rows, [new, new], [n, n])
    # a NaN in the last K row: only the last token's heads of that kv head are spoiled
    rows[0][1][p, 3, 17] = pool.v[0, at, slot, 3, 17] = 0.5
    at, slot = int(table[0, (n - 1) // page]), (n - 1) % page
    pool.k[0, at, slot, 5] = float("nan")
    out = paged.attention(describe(pool, table, [new, new], [n, n]), q)
    bad = torch.isnan(out).any(dim=-1)
    assert bad[new - 1, 10:12].all() and int(bad.sum()) == 2


@pytest.mark.parametrize("new", [1, 4, 80])
def test_large_and_equal_scores(new):
    """Scores of several hundred (one key takes all the weight), equal scores (weights of 1 / n), scores of -inf (no weight)."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(9)
    n = 500
    pool, table, rows = make_pool(g, [n], 32, 8, torch.bfloat16, scale=8.0)
    q = (torch.randn(new, 16, D, generator=g) * 8).to(torch.bfloat16).cuda()
    check(paged.attention(describe(pool, table, [new], [n]), q), q, rows, [new], [n])
    zero = torch.zeros_like(q)
    check(paged.attention(describe(pool, table, [new], [n]), zero), zero, rows, [new], [n])
    # the lowest finite K: scores of about -1e38 and below beside ordinary ones
    low = torch.finfo(torch.bfloat16).min
    q = q.abs()
    p = 5
    pool.k[0, int(table[0, p // 32]), p % 32] = low
    out = paged.attention(describe(pool, table, [new], [n]), q)
    keep = [torch.arange(n, device="cuda") != p]
    check(out, q, rows, [new], [n], there=keep)


@pytest.mark.parametrize("new", [1, 2, 48])
def test_strides_padding_rows_and_other_layouts(new):
    """q and out as slices of wider rows; rows behind the last sequence stay as they were."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(10)
    news, lens = [new, 1, new], [new + 31, 90, new]
    pool, table, rows = make_pool(g, lens, 16, 4, torch.bfloat16, order="heads")
    tokens, pad = sum(news), 5
    wide = torch.randn(tokens + pad, 20, 2 * D, generator=g).to(torch.bfloat16).cuda()
    q = wide[:, 3:11, :D]
    wide[tokens:] = float("nan")
    hold = torch.full((8, tokens + pad, 3 * D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = hold[:, :, D:2 * D].transpose(0, 1)
    batch = describe(pool, table, news, lens, tokens=tokens + pad, max_new=new)
    paged.attention(batch, q, out=out)
    check(out[:tokens], q[:tokens], rows, news, lens)
    assert (out[tokens:] == 7).all() and (hold[:, :, :D] == 7).all() and (hold[:, :, 2 * D:] == 7).all()


def test_scale_is_taken():
    from qwen3mk import paged

    g = torch.Generator().manual_seed(11)
    for new in (1, 70):
        pool, table, rows = make_pool(g, [200], 16, 8, torch.bfloat16)
        q = torch.randn(new, 16, D, generator=g).to(torch.bfloat16).cuda()
        check(paged.attention(describe(pool, table, [new], [200]), q, scale=0.25), q, rows, [new], [200], scale=0.25)


@pytest.mark.parametrize("new", [1, 6, 90])
def test_captured_calls_follow_the_descriptors(new):
    """Two graphs, captured one after the other and replayed on two streams at once, with lengths and pages that changed in between."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(12)
    sets = []
    for seed in range(2):
        lens = [new + 700, new + 20 + 300 * seed]
        pool, table, rows = make_pool(g, lens, 16, 8, torch.bfloat16)
        q = torch.randn(2 * new, 16, D, generator=g).to(torch.bfloat16).cuda()
        batch = describe(pool, table, [new, new], lens)
        out = torch.zeros_like(q)
        paged.attention(batch, q, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged.attention(batch, q, out=out)
        sets.append((pool, table, rows, q, batch, out, graph, lens))
    for cut in (0, 123):
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s in sets:
            s[4].kv_len.copy_(torch.tensor([n - cut if n - cut >= new else n for n in s[7]], dtype=torch.int32))
            s[5].fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(10):
            for s, st in zip(sets, streams):
                with torch.cuda.stream(st):
                    s[6].replay()
        torch.cuda.synchronize()
        for pool, table, rows, q, batch, out, graph, lens in sets:
            now = batch.kv_len.tolist()
            check(out, q, [(k[:m], v[:m]) for (k, v), m in zip(rows, now)], [new, new], now)


@pytest.mark.parametrize("new", [1, 70])
def test_two_streams_at_once(new):
    from qwen3mk import paged

    g = torch.Generator().manual_seed(13)
    pool, table, rows = make_pool(g, [2000, 900], 64, 8, torch.bfloat16)
    q = torch.randn(2 * new, 16, D, generator=g).to(torch.bfloat16).cuda()
    batch = describe(pool, table, [new, new], [2000, 900])
    want = paged.attention(batch, q)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(20):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(paged.attention(batch, q))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ------------------------------------------------------------------------------------------------ rope_append

def rope_reference(x, gain, table, pos, interleaved):
    x = x.double()
    if gain is not None:
        x = x / torch.sqrt(x.pow(2).mean(dim=-1, keepdim=True) + 1e-6) * gain.double()
    if table is None:
        return x
    r = table.shape[1]
    c, s = table[pos, None, :r // 2].double(), table[pos, None, r // 2:].double()
    y = x.clone()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    if interleaved:
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    else:
        y[..., :r // 2], y[..., r // 2:r] = a * c - b * s, b * c + a * s
    return y


def near(got, want, big):
    """One rounding of the result, and ten fp32 roundings (norm, gain, two products, a sum) of terms of size `big`."""
    h = torch.finfo(got.dtype).eps / 2
    tol = h * want.abs() + 10 * 2.0 ** -23 * big + torch.finfo(got.dtype).tiny * h
    assert float(((got.double() - want).abs() / tol).max()) <= 1.0


@pytest.mark.parametrize("rotary,interleaved,norm", [(128, False, True), (128, True, False), (64, False, False), (64, True, True), (8, False, True), (24, True, False), (104, False, True), (0, False, True)])
@pytest.mark.parametrize("rows_type,dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float16), (torch.bfloat16, torch.float16)])
def test_rope_append_matches_the_formula(rotary, interleaved, norm, rows_type, dtype):
    from qwen3mk import paged

    g = torch.Generator().manual_seed(rotary + norm)
    heads, kv_heads, page = 16, 8, 16
    news, lens = [3, 0, 37, 1], [40, 9, 37, 4000]
    pool, table, rows = make_pool(g, lens, page, kv_heads, dtype, order="heads" if interleaved else "slots")
    tokens, pad = sum(news), 2
    qkv = torch.randn(tokens + pad, (heads + 2 * kv_heads) * D, generator=g).to(rows_type).cuda()
    q, k, v = (x.view(tokens + pad, -1, D) for x in qkv.split([heads * D, kv_heads * D, kv_heads * D], dim=1))
    gq, gk = ((1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).cuda() if norm else None for _ in range(2))
    rope = paged.rope_table(4000, rotary_dim=rotary) if rotary else None
    batch = describe(pool, table, news, lens, tokens=tokens + pad, max_new=37)
    out = torch.full((tokens + pad, heads, D), 7.0, dtype=dtype, device="cuda")
    old_k, old_v = pool.k.clone(), pool.v.clone()
    paged.rope_append(batch, q, k, v, rope, q_gain=gq, k_gain=gk, interleaved=interleaved, out=out)
    assert (out[tokens:] == 7).all()
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(news, lens)]).cuda()
    owner = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news)).cuda()
    big = lambda x, gain: rope_reference(x.abs(), None if gain is None else gain.abs(), None, pos, False).amax(dim=-1, keepdim=True) * 2 + 0.0  # noqa: E731
    near(out[:tokens], rope_reference(q[:tokens], gq, rope, pos, interleaved), big(q[:tokens], gq))
    at, slot = table[owner, pos // page].long(), pos % page
    near(pool.k[0, at, slot], rope_reference(k[:tokens], gk, rope, pos, interleaved), big(k[:tokens], gk))
    assert torch.equal(pool.v[0, at, slot], v[:tokens].to(dtype))
    # nothing else was written
    pool.k[0, at, slot], pool.v[0, at, slot] = old_k[0, at, slot], old_v[0, at, slot]
    assert torch.equal(torch.nan_to_num(pool.k, 9), torch.nan_to_num(old_k, 9)) and torch.equal(torch.nan_to_num(pool.v, 9), torch.nan_to_num(old_v, 9))


def test_rope_append_positions_missing_slots_and_short_tables():
    from qwen3mk import paged

    g = torch.Generator().manual_seed(21)
    news, lens = [4, 6, 3], [20, 4, 50]              # the second: two tokens without a position
    pool, table, _ = make_pool(g, lens, 16, 2, torch.bfloat16)
    table[2, 3] = -5                                 # positions 48 and 49 of the third have no page
    tokens = sum(news)
    q, k, v = (torch.randn(tokens, h, D, generator=g).cuda() for h in (4, 2, 2))
    rope = paged.rope_table(48)
    old = pool.k.clone()
    batch = describe(pool, table, news, lens)
    out = paged.rope_append(batch, q, k, v, rope)
    pos = torch.tensor([16, 17, 18, 19, -2, -1, 0, 1, 2, 3, 47, 48, 49]).cuda()
    known = (pos >= 0) & (pos < 48)
    assert torch.isnan(out[~known]).all()
    near(out[known], rope_reference(q[known], None, rope, pos[known], False), q[known].double().abs().amax(dim=-1, keepdim=True) * 2)
    p47 = pool.k[0, int(table[2, 2]), 15]
    near(p47, rope_reference(k[10:11], None, rope, pos[10:11], False)[0], k[10].double().abs().amax(dim=-1, keepdim=True) * 2)
    changed = (torch.nan_to_num(pool.k, 9) != torch.nan_to_num(old, 9)).any(dim=-1).any(dim=-1)
    assert int(changed.sum()) == 4 + 4 + 1
    # positions of the caller's: rotated by them, stored where the tokens stand
    given = torch.arange(tokens, dtype=torch.int32, device="cuda") * 3
    out = paged.rope_append(batch, q, k, v, rope, positions=given)
    near(out, rope_reference(q, None, rope, given.long(), False), q.double().abs().amax(dim=-1, keepdim=True) * 2)
    near(pool.k[0, int(table[0, 1]), :4], rope_reference(k[:4], None, rope, given[:4].long(), False), k[:4].double().abs().amax(dim=-1, keepdim=True) * 2)


def test_appended_rows_are_attended():
    """As a server uses them: chunks of uneven conversations, then single tokens, each step rope_append and attention; the whole is one causal attention."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(22)
    page, heads, kv_heads, totals = 16, 16, 8, [150, 37, 81]
    pool = paged.PagePool.empty(layers=3, pages=40, page_size=page)
    pool.k.fill_(float("nan")), pool.v.fill_(float("nan"))
    ids = torch.randperm(40, generator=g)
    table = torch.full((3, 10), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(totals):
        c = -(-n // page)
        table[b, :c] = ids[at:at + c].to(torch.int32)
        at += c
    table = table.cuda()
    rope = paged.rope_table(200)
    full = [torch.randn(n, heads + 2 * kv_heads, D, generator=g).cuda() for n in totals]
    gq, gk = ((1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).cuda() for _ in range(2))
    done, outs, qs = [0, 0, 0], [[], [], []], [[], [], []]
    for news in ([70, 5, 33], [1, 0, 1], [66, 17, 1], [1, 1, 1], [12, 14, 45]):
        rows = torch.cat([f[d:d + m] for f, d, m in zip(full, done, news)])
        done = [d + m for d, m in zip(done, news)]
        batch = describe(pool, table, news, done)
        q = paged.rope_append(batch, rows[:, :heads], rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:], rope, 2, q_gain=gq, k_gain=gk)
        o = paged.attention(batch, q, 2)
        for b, (x, y) in enumerate(zip(q.split(news), o.split(news))):
            qs[b].append(x), outs[b].append(y)
    assert done == totals
    for b, n in enumerate(totals):
        where = table[b, torch.arange(n, device="cuda") // page].long(), torch.arange(n, device="cuda") % page
        check(torch.cat(outs[b]), torch.cat(qs[b]), [(pool.k[2][where], pool.v[2][where])], [n], [n])
        near(pool.k[2][where], rope_reference(full[b][:, heads:heads + kv_heads], gk, rope, torch.arange(n, device="cuda"), False),
             rope_reference(full[b][:, heads:heads + kv_heads].abs(), gk.abs(), None, None, False).amax(dim=-1, keepdim=True) * 2)


def test_refusals():
    from qwen3mk import paged

    g = torch.Generator().manual_seed(23)
    pool, table, _ = make_pool(g, [20], 16, 8, torch.bfloat16)
    batch = describe(pool, table, [2], [20])
    q = torch.randn(2, 16, D, generator=g).to(torch.bfloat16).cuda()
    for bad in (q.float(), q.half(), q[:1], q[:, :, :64], q.cpu(), q.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError, match="attention: q"):
            paged.attention(batch, bad)
    for bad in (q[:, :12], q[:, :3], torch.cat([q] * 8, dim=1)):
        with pytest.raises(ValueError, match="q heads over 8 kv heads"):
            paged.attention(batch, bad)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            paged.attention(batch, q, scale=scale)
    with pytest.raises(ValueError, match="layer 1 outside"):
        paged.attention(batch, q, 1)
    with pytest.raises(ValueError, match="16-byte aligned"):
        paged.attention(batch, torch.empty(2 * 16 * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 16, D))
    with pytest.raises(ValueError, match="page_size"):
        paged.attention(describe(paged.PagePool.empty(layers=1, pages=4, page_size=24), table, [2], [20]), q)
    x = torch.randn(2, 32, D, generator=g).cuda()
    rope = paged.rope_table(32)
    for args in ((x[:, :16], x[:, 16:23], x[:, 24:]), (x[:, :16].half(), x[:, 16:24], x[:, 24:]), (x[:1, :16], x[:, 16:24], x[:, 24:])):
        with pytest.raises(ValueError, match="rope_append"):
            paged.rope_append(batch, *args, rope)
    good = (x[:, :16], x[:, 16:24], x[:, 24:])
    for bad in (rope.double(), rope[:, :100], torch.zeros(4, 12, device="cuda"), torch.zeros(4, 136, device="cuda"), rope.cpu()):
        with pytest.raises(ValueError):
            paged.rope_append(batch, *good, bad)
    with pytest.raises(ValueError, match="k_gain"):
        paged.rope_append(batch, *good, rope, k_gain=torch.ones(D, device="cuda"))
    with pytest.raises(ValueError, match="positions"):
        paged.rope_append(batch, *good, rope, positions=torch.zeros(2, dtype=torch.int64, device="cuda"))
    # no new token at all: nothing to do
    none = describe(pool, table, [0], [20])
    assert paged.attention(none, q[:0]).shape == (0, 16, D)


def test_one_batch_serves_q_of_several_head_counts():
    """The workspace goes by the q heads of the call: 8 new tokens of 16 heads are few rows, of 64 heads many."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(24)
    news, lens = [8, 3], [200, 45]
    pool, table, rows = make_pool(g, lens, 16, 8, torch.bfloat16)
    batch = describe(pool, table, news, lens)
    for heads in (16, 64, 8, 64):
        q = torch.randn(sum(news), heads, D, generator=g).to(torch.bfloat16).cuda()
        check(paged.attention(batch, q), q, rows, news, lens)


def test_q_in_place_and_outputs_that_overlap():
    from qwen3mk import paged

    g = torch.Generator().manual_seed(25)
    pool, table, _ = make_pool(g, [60, 9], 16, 8, torch.bfloat16)
    batch = describe(pool, table, [33, 9], [60, 9])
    x = torch.randn(42, 32, D, generator=g).to(torch.bfloat16).cuda()
    rope, gain = paged.rope_table(64), torch.ones(D, dtype=torch.bfloat16, device="cuda")
    want = paged.rope_append(batch, x[:, :16], x[:, 16:24], x[:, 24:], rope, q_gain=gain)
    q = x[:, :16]
    assert paged.rope_append(batch, q, x[:, 16:24], x[:, 24:], rope, q_gain=gain, out=q) is q and torch.equal(q, want)
    with pytest.raises(ValueError, match="overlap"):
        paged.rope_append(batch, q, x[:, 16:24], x[:, 24:], rope, out=want[:1].expand(42, 16, D))
    with pytest.raises(ValueError, match="out must not be q"):
        paged.attention(batch, want, out=want)


@pytest.mark.parametrize("news,lens,page,heads", [([39] * 8, [5527] * 8, 64, 16), ([28] * 15, [3609] * 15, 32, 8), ([43] + [1] * 28, [2032 - 31 * i for i in range(29)], 64, 16),
                                                   ([130, 131], [700, 2001], 16, 16)])
def test_pages_that_arrive_late(news, lens, page, heads):
    """Cold caches: K and V come late and out of step with one another, over and over with the same bits."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(26)
    pool, table, rows = make_pool(g, lens, page, 8, torch.bfloat16)
    batch = describe(pool, table, news, lens)
    q = torch.randn(sum(news), heads, D, generator=g).to(torch.bfloat16).cuda()
    flush = torch.empty(300_000_000, dtype=torch.uint8, device="cuda")
    first = paged.attention(batch, q)
    check(first, q, rows, news, lens)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(200):
        flush.fill_(i & 1)
        differ += (paged.attention(batch, q).view(torch.int16) != first.view(torch.int16)).any()
    assert int(differ) == 0

"""Attention of chunks over long caches where rows have to be done again (a V row that only later tokens see is not finite, scores leave the range of a
tile's first reference): the result is the formula's however many keys that takes.  Formula and tolerances as in test_paged_gpu.py."""
from __future__ import annotations

import pytest
import torch
from test_paged_gpu import D, check, describe, make_pool

pytestmark = pytest.mark.gpu


def slot(pool, table, b, p):
    return int(table[b, p // pool.page_size]), p % pool.page_size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_the_last_value_row_is_not_finite(dtype, value):
    """Only the chunk's last token sees it: all others are finite, behind 33000 positions."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(200)
    new, n = 64, 33064
    pool, table, rows = make_pool(g, [n], 64, 8, dtype)
    q = torch.randn(new, 16, D, generator=g).to(dtype).cuda()
    at, s = slot(pool, table, 0, n - 1)
    pool.v[0, at, s, :, 17] = value
    rows[0][1][n - 1, :, 17] = value
    batch = describe(pool, table, [new], [n])
    out = paged.attention(batch, q)
    check(out, q, rows, [new], [n])
    assert torch.isfinite(out[:new - 1]).all() and torch.equal(out[:new - 1], paged.attention(batch, q)[:new - 1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scores_that_rise_by_more_than_a_hundred(dtype):
    """Scores grow along the cache by 120: fp32 does not hold their exponentials under the first tile's maximum."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(201)
    news, lens = [64, 1, 70], [33064, 500, 900]
    pool, table, rows = make_pool(g, lens, 64, 8, dtype, scale=0.25)
    c = (120 / D ** 0.5) ** 0.5
    kr = rows[0][0]
    kr += (c * torch.arange(lens[0], device="cuda") / lens[0])[:, None, None]
    p = torch.arange(lens[0], device="cuda")
    pool.k[0][table[0][p // 64].long(), p % 64] = kr
    q = (torch.randn(sum(news), 16, D, generator=g) * 0.25 + c).to(dtype).cuda()
    batch = describe(pool, table, news, lens)
    out = paged.attention(batch, q)
    check(out, q, rows, news, lens)
    assert torch.equal(out, paged.attention(batch, q))


def test_many_chunks_behind_one_long_prefix():
    """Nineteen conversations share 32768 positions, each has 64 new tokens and an infinity in the last one's V row: a block has whole items of 32832 keys, and all their
    rows but two are done again."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(202)
    many, new, page, prefix = 19, 64, 64, 32768
    n = prefix + new
    pages = prefix // page + many
    pool = paged.PagePool(*(torch.full((1, pages, page, 8, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    for x in (pool.k, pool.v):
        x[0] = torch.randn(pages, page, 8, D, generator=g).to(torch.bfloat16).cuda()
    pool.v[0, prefix // page:, new - 1, :, 5] = float("inf")
    table = torch.arange(prefix // page, dtype=torch.int32).repeat(many, 1)
    table = torch.cat([table, torch.arange(prefix // page, pages, dtype=torch.int32)[:, None]], dim=1).contiguous().cuda()
    rows = [tuple(x[0][table[b].long()].reshape(n, 8, D) for x in (pool.k, pool.v)) for b in range(many)]
    q = torch.randn(many * new, 16, D, generator=g).to(torch.bfloat16).cuda()
    check(paged.attention(describe(pool, table, [new] * many, [n] * many), q), q, rows, [new] * many, [n] * many)


@pytest.mark.parametrize("new", [2, 8])
def test_few_rows_behind_a_long_cache(new):
    """The same with the kernel of few rows."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(203)
    n = 20000
    pool, table, rows = make_pool(g, [n, n], 16, 8, torch.bfloat16)
    q = torch.randn(2 * new, 16, D, generator=g).to(torch.bfloat16).cuda()
    at, s = slot(pool, table, 0, n - 1)
    pool.v[0, at, s, :, 3] = float("inf")
    rows[0][1][n - 1, :, 3] = float("inf")
    check(paged.attention(describe(pool, table, [new, new], [n, n]), q), q, rows, [new, new], [n, n])


def median_us(f, runs=9):
    f()
    times = []
    for _ in range(runs):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3)
    return sorted(times)[runs // 2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kept", [0, 1000])
def test_pages_that_are_gone_cost_nothing(dtype, kept):
    """A caller who drops old pages: what is left is attended, and the call takes no longer than with all of them (before, a row that found nothing in a part looked
    for its keys one by one: fifty times as long)."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(204)
    new, n, page = 64, 33064, 64
    pool, table, rows = make_pool(g, [n], page, 8, dtype)
    q = torch.randn(new, 16, D, generator=g).to(dtype).cuda()
    batch = describe(pool, table, [new], [n])
    whole = median_us(lambda: paged.attention(batch, q))
    gone = (n - kept) // page if kept else table.shape[1]
    table[0, :gone] = -1
    out = paged.attention(batch, q)
    there = [torch.arange(n, device="cuda") >= gone * page]
    check(out, q, rows, [new], [n], there=there)
    less = median_us(lambda: paged.attention(batch, q))
    assert less < 2 * whole, f"{less:.0f} us without {gone} pages, {whole:.0f} us with them"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,n", [(64, 33064), (300, 300), (40, 170)])
def test_rows_that_are_no_numbers_cost_nothing(dtype, new, n):
    """Queries that are NaN (positions behind a rotary table's end, say) and a K row that is: their rows are NaN, the others right, and nothing is done again for them
    but where an infinite V row asks for it as well."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(205)
    pool, table, rows = make_pool(g, [n, 50], 64, 8, dtype)
    q = torch.randn(new + 20, 16, D, generator=g).to(dtype).cuda()
    batch = describe(pool, table, [new, 20], [n, 50])
    plain = median_us(lambda: paged.attention(batch, q))
    broken = q.clone()
    broken[:new:2] = float("nan")
    out = paged.attention(batch, broken)
    lost = torch.zeros(new + 20, dtype=torch.bool, device="cuda")
    lost[:new:2] = True
    assert torch.isnan(out[lost]).all()
    kept = ~lost
    want = paged.attention(batch, q)
    check(want, q, rows, [new, 20], [n, 50])
    assert torch.equal(out[kept], want[kept])
    slow = median_us(lambda: paged.attention(batch, broken))
    assert slow < 2 * plain + 20, f"{slow:.0f} us with NaN, {plain:.0f} us without"
    # a K row that every token of the first sequence sees, and an infinite V row that the last one sees
    at, s = slot(pool, table, 0, 0)
    pool.k[0, at, s, 2] = rows[0][0][0, 2] = float("nan")
    at, s = slot(pool, table, 0, n - 1)
    pool.v[0, at, s, 2, 9] = rows[0][1][n - 1, 2, 9] = float("inf")
    pool.v[0, at, s, 4, 9] = rows[0][1][n - 1, 4, 9] = float("inf")
    check(paged.attention(batch, q), q, rows, [new, 20], [n, 50])

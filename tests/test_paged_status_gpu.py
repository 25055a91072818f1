"""Waits of the attention over pages that give up, without a fault: their patience is set to a microsecond, which no page takes to arrive.  They are reported, the rows of
the blocks that gave up are NaN, all others are what they are otherwise, and the next call is whole again."""
from __future__ import annotations

import pytest
import torch
from test_paged_gpu import check, describe, make_pool

pytestmark = pytest.mark.gpu

SHAPES = [
    ([64], [2064], 64, 16, 8),
    ([600], [9000], 64, 16, 8),
    # parts of one tile, of which one group of warps has none, and sequences without a key between them
    ([20, 9, 20, 30, 10] * 12, [0, 100, 0, 60, 128] * 12, 16, 16, 8),
    ([17, 300], [40000, 300], 16, 4, 1),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_wait_that_gives_up_is_reported(shape, dtype):
    from qwen3mk import paged

    news, lens, page, heads, kv_heads = SHAPES[shape]
    g = torch.Generator().manual_seed(400 + shape)
    pool, table, rows = make_pool(g, lens, page, kv_heads, dtype)
    q = torch.randn(sum(news), heads, 128, generator=g).to(dtype).cuda()
    batch = describe(pool, table, news, lens)
    right = paged.attention(batch, q)
    check(right, q, rows, news, lens)
    assert pool.status() == [0, 0, 0, 0]
    short = describe(pool, table, news, lens, wait_limit_us=1)
    for _ in range(5):
        out = paged.attention(short, q)
        with pytest.raises(RuntimeError, match=r"device status: code 2 at site (8|9)\d,"):
            pool.status()
        gone = torch.isnan(out)
        assert gone.any() and torch.equal(gone.any(dim=-1), gone.all(dim=-1)), "a row that was not finished is NaN throughout"
        assert torch.equal(out[~gone], right[~gone])
    assert torch.equal(paged.attention(batch, q), right)
    assert pool.status(torch.cuda.current_stream()) == [0, 0, 0, 0]


def test_extend_reports_to_the_engine():
    """The engine's own limit, and its own status words."""
    from qwen3mk import Megakernel, paged, weights

    inputs = weights.synthetic(0, "cuda", layers=2, vocab=4096)
    pool = paged.PagePool.empty(layers=2, pages=40, page_size=64)
    pool.k.zero_(), pool.v.zero_()
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    ids = torch.randint(0, 4096, (300,), device="cuda")
    results = {}
    for limit in (1, 0):
        mk = Megakernel(layers=2, vocab=4096, max_batch=4, max_tokens=512, wait_limit_us=limit)
        batch = describe(pool, table, [300], [2300])
        results[limit] = mk.extend(inputs, ids, batch)["logits"]
        if limit:
            with pytest.raises(RuntimeError, match=r"device status: code 2 at site (8|9)\d,"):
                mk.status()
        mk.status()
        assert pool.status() == [0, 0, 0, 0]
    assert torch.isfinite(results[0]).all() and not torch.isfinite(results[1]).all()

"""Attention over pages where a row sees nothing of a part of its item: its other parts must count as if that part were not there, whatever their
scores are.  Same pools, formula and tolerances as in test_paged_gpu.py."""
from __future__ import annotations

import pytest
import torch
from test_paged_gpu import D, check, describe, make_pool

pytestmark = pytest.mark.gpu


def low_scores(g, level, news, lens, page, heads, kv_heads, dtype):
    """Queries along a direction, keys against it: every score is about -level."""
    pool, table, rows = make_pool(g, lens, page, kv_heads, dtype, scale=0.25)
    c = (level / D ** 0.5) ** 0.5                    # D c c / sqrt(D) = level
    for b, (n, (kr, _)) in enumerate(zip(lens, rows)):
        kr -= c
        at, slot = table[b].cpu()[torch.arange(n) // page].long(), torch.arange(n) % page
        pool.k[0][at.cuda(), slot.cuda()] = kr
    q = (torch.randn(sum(news), heads, D, generator=g) * 0.25 + c).to(dtype).cuda()
    return pool, table, rows, q


# tiles whose first tokens see nothing of the last unit of 128 keys, few enough units that items are cut at every one of them
SHAPES = [
    ([64], [2064], 64, 16, 8),        # 17 units a head, the last one begins at 2048: tokens 2000..2047 see nothing of it
    ([80], [180], 32, 4, 2),          # tokens 100..127 see keys 0..127 only
    ([40], [300], 16, 8, 1),          # group 8: tiles of 16 tokens, one of them across 256
    ([200, 33], [500, 140], 16, 4, 4),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("level", [-80, 60, 100, 200, 300, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_parts_that_a_row_does_not_see(shape, level, dtype):
    from qwen3mk import paged

    news, lens, page, heads, kv_heads = SHAPES[shape]
    g = torch.Generator().manual_seed(100 + shape)
    pool, table, rows, q = low_scores(g, abs(level), news, lens, page, heads, kv_heads, dtype)
    if level < 0:
        q = -q
    check(paged.attention(describe(pool, table, news, lens), q), q, rows, news, lens)


@pytest.mark.parametrize("level", [60, 100, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,gone", [(64, [2, 3, 30, 31]), (128, [0, 15]), (16, list(range(0, 120))), (16, list(range(5, 129)))])
def test_parts_on_missing_pages(level, dtype, page, gone):
    """Whole parts, and parts of parts, of which no page is there."""
    from qwen3mk import paged

    n, new = 2064, 64
    g = torch.Generator().manual_seed(110)
    pool, table, rows, q = low_scores(g, level, [new], [n], page, 16, 8, dtype)
    table[0, gone] = -1
    there = [torch.tensor([p // page not in gone for p in range(n)], device="cuda")]
    check(paged.attention(describe(pool, table, [new], [n]), q), q, rows, [new], [n], there=there)

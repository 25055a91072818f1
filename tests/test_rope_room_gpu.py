"""rope_append of sequences that have outgrown their row of the page table: what has no slot is not written, and nothing that is cached is written over."""
from __future__ import annotations

import pytest
import torch
from test_paged_gpu import D, describe, make_pool, near, rope_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,past", [(1, 1), (5, 2), (5, 5), (40, 7), (3, 1000), (2, 2**31 - 1 - 64)])
def test_tokens_behind_the_page_table_have_no_slot(dtype, new, past):
    """A table of four pages of 16, the last one shared with another sequence whose rows must stay; `past` tokens too many.  Positions are true all the same: rotated by them."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(30)
    pool, table, _ = make_pool(g, [64, 64], 16, 2, dtype)
    table = table[:, :4].contiguous()
    table[1, 3] = table[0, 3]
    q, k, v = (torch.randn(new + 1, h, D, generator=g).cuda() for h in (4, 2, 2))
    rope = paged.rope_table(2000)
    batch = describe(pool, table, [new, 1], [64 + past, 11])
    old_k, old_v = pool.k.clone(), pool.v.clone()
    out = paged.rope_append(batch, q, k, v, rope)
    pos = torch.cat([64 + past - new + torch.arange(new), torch.tensor([10])]).cuda()
    known = pos < 2000
    big = lambda x: x.double().abs().amax(dim=-1, keepdim=True) * 2  # noqa: E731
    if bool(known.any()):
        near(out[known], rope_reference(q[known], None, rope, pos[known], False), big(q[known]))
    assert torch.isnan(out[~known]).all()
    stored = [(t, int(p)) for t, p in enumerate(pos.tolist()) if p < 64]
    assert len(stored) == max(new - past, 0) + 1
    for t, p in stored:
        page = int(table[0 if t < new else 1, p // 16])
        near(pool.k[0, page, p % 16], rope_reference(k[t:t + 1], None, rope, pos[t:t + 1], False)[0], big(k[t]))
        assert torch.equal(pool.v[0, page, p % 16], v[t].to(dtype))
        pool.k[0, page, p % 16], pool.v[0, page, p % 16] = old_k[0, page, p % 16], old_v[0, page, p % 16]
    assert torch.equal(torch.nan_to_num(pool.k, 9), torch.nan_to_num(old_k, 9)) and torch.equal(torch.nan_to_num(pool.v, 9), torch.nan_to_num(old_v, 9))

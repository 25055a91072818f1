"""Attention of a chunk whose blocks have more pages each than are looked at ahead (2^15): 80 million positions on shared pages."""
from __future__ import annotations

import pytest
import torch
from test_paged_gpu import D, describe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gone", [0, 7])
def test_more_pages_than_are_looked_at_ahead(dtype, gone):
    """A table of 5 million entries names 97 pages over and over (every 7th entry none).  The formula: positions of one page slot weigh alike, so a slot counts as often as it
    is seen.  Tolerance as in test_paged_gpu.py, but for the sums: a block adds its 33800 pages one after the other, a page's 16 products in one step of the matrix unit, and the join
    a part a block; output and sum of weights each, 2^-23 an add."""
    from qwen3mk import paged

    g = torch.Generator().manual_seed(300)
    blocks = torch.cuda.get_device_properties(0).multi_processor_count
    page, distinct, heads, new, entries = 16, 97, 2, 9, 33_800 * blocks
    k, v = ((torch.randn(1, distinct, page, 1, D, generator=g)).to(dtype).cuda() for _ in range(2))
    pool = paged.PagePool(k, v)
    table = (torch.arange(entries, dtype=torch.int64) * 31 % distinct).to(torch.int32)
    if gone:
        table[::gone] = -1
    n = entries * page - 5
    table = table[None].cuda()
    q = torch.randn(new, heads, D, generator=g).to(dtype).cuda()
    out = paged.attention(describe(pool, table, [new], [n]), q)

    live = table[0][table[0] >= 0].long()
    count = torch.bincount(live, minlength=distinct)[:, None].repeat(1, page).double()      # how often a slot is a position
    key, val = k[0, :, :, 0].reshape(-1, D).double(), v[0, :, :, 0].reshape(-1, D).double()
    scale, h, adds = D ** -0.5, torch.finfo(dtype).eps / 2, 33_800 + 2 * blocks + 128
    last = int(table[0, -1])
    for t in range(new):
        seen = count.clone()
        if last >= 0:                                # positions of the last page behind the token's own
            seen[last, page - 5 - (new - 1 - t):] -= 1
        assert new < page - 5
        s = q[t].double() @ key.T * scale
        w = torch.exp(s - s.max(dim=1, keepdim=True).values) * seen.reshape(1, -1)
        p = w / w.sum(dim=1, keepdim=True)
        o, big = p @ val, p @ val.abs()
        most = float((q[t].double().abs() @ key.abs().T).max()) * scale
        tol = h * o.abs() + (h + 2.0 ** -23 * (2 * 130 * most + 2 * adds)) * big + 2.0 ** -24
        assert ((out[t].double() - o).abs() <= tol).all(), f"token {t}: off by {float(((out[t].double() - o).abs() / tol).max()):.2f} tolerances"

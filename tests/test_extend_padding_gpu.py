"""Megakernel.extend with rows that belong to no sequence: a captured step is as wide as its largest batch."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [0, 3])
def test_ids_of_padding_rows_may_be_anything(first):
    from qwen3mk import Megakernel, paged, weights

    inputs = weights.synthetic(0, "cuda", layers=2, vocab=2048)
    mk = Megakernel(layers=2, vocab=2048, max_batch=4, max_tokens=64)
    pool = paged.PagePool.empty(layers=2, pages=8, page_size=64)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    start = torch.tensor([first, first + 30, first + 37], dtype=torch.int32, device="cuda")
    lens = torch.tensor([30, 7], dtype=torch.int32, device="cuda")
    batch = paged.PagedBatch(pool, table, start, lens, tokens=60, max_new=30)
    ids = torch.randint(0, 2048, (60,), generator=torch.Generator().manual_seed(2)).cuda()
    want = mk.extend(inputs, ids, batch)
    mk.status()
    k, v = pool.k.clone(), pool.v.clone()
    padded = ids.clone()
    padded[first + 37:] = torch.tensor([-1, -100, 2048, 2**62, -2**63])[torch.arange(60 - first - 37) % 5].cuda()
    padded[:first] = -1
    got = mk.extend(inputs, padded, batch)
    mk.status()
    assert torch.equal(got["logits"], want["logits"]) and torch.equal(got["next_token"], want["next_token"])
    where = table[0, 0].item(), table[1, 0].item()
    for new, old in ((pool.k, k), (pool.v, v)):
        assert torch.equal(new[:, where[0], :30], old[:, where[0], :30]) and torch.equal(new[:, where[1], :7], old[:, where[1], :7])
    # a sequence's own token is looked at as before
    padded[first + 36] = 2048
    mk.extend(inputs, padded, batch)
    with pytest.raises(RuntimeError, match="code 3 at site 0"):
        mk.status()

"""Megakernel.set_rope beside calls that were captured before it."""
from __future__ import annotations

import gc
import weakref

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_captured_call_keeps_its_table():
    """The engine's own table, then a caller's that nobody else holds, are replaced; memory of their size is written over and over; replays rotate as when they were captured."""
    from qwen3mk import Megakernel, paged, weights

    inputs = weights.synthetic(0, "cuda", layers=2, vocab=2048)
    mk = Megakernel(layers=2, vocab=2048, max_batch=4, max_tokens=64, max_positions=1024)
    pool = paged.PagePool.empty(layers=2, pages=8, page_size=64)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    batch = paged.PagedBatch(pool, table, torch.tensor([0, 40, 60], dtype=torch.int32, device="cuda"), torch.tensor([40, 20], dtype=torch.int32, device="cuda"))
    ids = torch.randint(0, 2048, (60,), generator=torch.Generator().manual_seed(1)).cuda()
    graphs, refs = [], []
    for scale in (None, 8.0, 16.0):
        if scale:
            mk.set_rope(paged.rope_table(1024, scaling={"type": "linear", "factor": scale}))
        want = mk.extend(inputs, ids, batch)["logits"].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mk.extend(inputs, ids, batch)["logits"]
        graphs.append((graph, out, want))
        refs.append(weakref.ref(mk.rope))
    gc.collect()
    torch.cuda.synchronize()
    assert all(r() is not None for r in refs), "a table that captured calls read is gone"
    junk = [torch.full((1024, 128), 7.0, device="cuda") for _ in range(16)]
    for graph, out, want in graphs:
        graph.replay()
        assert torch.equal(out, want)
    mk.status()
    assert not torch.equal(graphs[0][2], graphs[1][2]) and not torch.equal(graphs[1][2], graphs[2][2]) and junk
    mk.set_rope(mk.rope)
    assert len(mk._ropes) == 3

"""The whole model over a pool of pages (Megakernel.extend): against the fp32 oracle, against the engine's own prompt and decode paths, and as a server uses it, with
rope_append and attention inside and sample_rows behind.

The gates are those of a prompt, whose activations are rounded to bf16 in the same places: K/V rows within rel-L2 1e-2, logits within 2e-2 (tests/test_baseline_configs_gpu.py);
here q enters the attention as one bf16 plane instead of two, a score's error of 2^-9 |q||k| / 11 beside the 2^-9 of k itself."""
from __future__ import annotations

import pytest
import torch

LAYERS, VOCAB = 3, 2048


def setup(oracle, seed, **kw):
    from qwen3mk import Megakernel, weights

    inp = oracle.synthetic(seed, oracle.Shape(layers=LAYERS, vocab=kw.get("vocab", VOCAB)), context=1)
    w = {k: inp[k] for k in weights.WEIGHT_NAMES}
    mk = Megakernel(layers=LAYERS, vocab=kw.pop("vocab", VOCAB), max_batch=8, max_tokens=640, **kw)
    return mk, w, {k: v.cuda() for k, v in w.items()}


class Server:
    """Pages of a few conversations: tables and lengths as a server keeps them."""

    def __init__(self, seqs, page, pages, g):
        from qwen3mk import paged

        self.pool = paged.PagePool.empty(layers=LAYERS, pages=pages, page_size=page)
        self.pool.k.fill_(float("nan")), self.pool.v.fill_(float("nan"))
        self.free = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((seqs, 64), -1, dtype=torch.int32)
        self.len = [0] * seqs

    def batch(self, news):
        from qwen3mk import paged

        for b, m in enumerate(news):
            have, need = (-(-n // self.pool.page_size) for n in (self.len[b], self.len[b] + m))
            for i in range(have, need):
                self.table[b, i] = self.free.pop()
            self.len[b] += m
        start = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda()
        return paged.PagedBatch(self.pool, self.table.cuda(), start, torch.tensor(self.len, dtype=torch.int32).cuda())

    def rows(self, b):
        p = torch.arange(self.len[b])
        at, slot = self.table[b, p // self.pool.page_size].long().cuda(), (p % self.pool.page_size).cuda()
        return self.pool.k[:, at, slot].cpu(), self.pool.v[:, at, slot].cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("page,steps", [(16, [[40, 0, 7, 1]]), (64, [[5, 70, 0, 33], [1, 1, 1, 1], [0, 20, 64, 1]]), (128, [[130, 300, 64, 65], [1, 2, 3, 200], [1, 0, 1, 1]]), (16, [[1, 0, 0, 0], [2, 0, 0, 1], [0, 3, 0, 0]])])
def test_chunks_match_the_oracles_prompt(oracle, page, steps):
    g = torch.Generator().manual_seed(page + len(steps))
    mk, w, dev = setup(oracle, 31)
    w32 = oracle.to_fp32(w)
    server = Server(4, page, 120, g)
    ids = [torch.randint(0, VOCAB, (600,), generator=g) for _ in range(4)]
    for news in steps:
        at = list(server.len)
        batch = server.batch(news)
        out = mk.extend(dev, torch.cat([x[n:n + m] for x, n, m in zip(ids, at, news)]).cuda(), batch)
        mk.status()
        for b, m in enumerate(news):
            if m == 0:
                assert not out["logits"][b].any() and int(out["next_token"][b]) == 0
                continue
            kc, vc, logits = oracle.prefill(w32, ids[b][:server.len[b]])
            err = oracle.rel_l2(out["logits"][b].cpu(), logits)
            assert err <= 2e-2, (b, err)
            k, v = server.rows(b)
            assert oracle.rel_l2(k, kc) <= 1e-2 and oracle.rel_l2(v, vc) <= 1e-2
            got = int(out["next_token"][b])
            assert got == int(out["logits"][b].argmax())


@pytest.mark.gpu
def test_full_size_beside_the_engines_own_prompt(oracle):
    """28 layers, 151936 words: a prompt in two chunks beside other conversations, against q3_prefill on the same weights."""
    from qwen3mk import Megakernel, paged, prefill, weights

    w = weights.synthetic(3, "cuda", context=1)
    w = {k: w[k] for k in weights.WEIGHT_NAMES}
    ids = torch.randint(0, 151936, (700,), generator=torch.Generator().manual_seed(3)).cuda()
    mk = Megakernel(max_batch=4, max_tokens=700)
    kc, vc, logits = prefill.prefill(w, ids, engine=mk)
    pool = paged.PagePool.empty(pages=64, page_size=64)
    table = torch.randperm(64, generator=torch.Generator().manual_seed(4)).to(torch.int32).view(4, 16).cuda()
    for news, lens in (([450, 3, 0, 1], [450, 3, 0, 1]), ([250, 30, 17, 1], [700, 33, 17, 2])):
        start = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda()
        batch = paged.PagedBatch(pool, table, start, torch.tensor(lens, dtype=torch.int32).cuda())
        mine = torch.cat([ids[n - m:n] for m, n in zip(news, lens)])
        out = mk.extend(w, mine, batch)
    mk.status()
    # Both sides round to bf16, each may be a gate away from the exact rows: |a - b| <= |a - exact| + |b - exact| <= two gates (|exact| and |b| alike to 1e-2)
    assert oracle.rel_l2(out["logits"][0], logits) <= 4e-2
    p = torch.arange(700, device="cuda")
    at, slot = table[0, p // 64].long(), p % 64
    assert oracle.rel_l2(pool.k[:, at, slot], kc) <= 2e-2 and oracle.rel_l2(pool.v[:, at, slot], vc) <= 2e-2


@pytest.mark.gpu
def test_a_sampled_stream_in_one_graph(oracle):
    """Decode as a server runs it: one captured step (extend, sample_rows into the ids of the next one, lengths advanced on the device) replayed; every step is checked against
    the same calls outside a graph."""
    from qwen3mk import paged, sampling

    g = torch.Generator().manual_seed(5)
    mk, w, dev = setup(oracle, 32)
    streams = []
    for captured in (True, False):
        server = Server(5, 16, 120, torch.Generator().manual_seed(6))
        news = [20, 3, 50, 1, 17]
        batch = server.batch(news)
        ids = torch.randint(0, VOCAB, (sum(news),), generator=torch.Generator().manual_seed(7)).cuda()
        tokens = mk.extend(dev, ids, batch)["next_token"]
        for b in range(5):                                       # room for 30 more positions
            for i in range(-(-server.len[b] // 16), -(-(server.len[b] + 30) // 16)):
                server.table[b, i] = server.free.pop()
        start = torch.arange(6, dtype=torch.int32).cuda()
        length = torch.tensor(server.len, dtype=torch.int32).cuda()
        step = paged.PagedBatch(server.pool, server.table.cuda(), start, length)
        u = torch.zeros(5, device="cuda")
        t, k, p, m = (torch.tensor(x, dtype=d).cuda() for x, d in (([0.0, 0.7, 1.0, 0.9, 1.2], torch.float32), ([0, 20, 0, 50, 0], torch.int32), ([1.0, 0.9, 0.8, 1.0, 1.0], torch.float32), ([0, 0, 0, 0.05, 0.1], torch.float32)))

        def one():
            length.add_(1)
            out = mk.extend(dev, tokens, step)
            sampling.sample_rows(out["logits"], t, k, p, m, u=u, out=tokens)

        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            keep = tokens.clone()
            with torch.cuda.stream(side):
                one()
            torch.cuda.current_stream().wait_stream(side)
            length.sub_(1)
            tokens.copy_(keep)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                one()
        draws = torch.Generator().manual_seed(8)
        got = []
        for _ in range(25):
            u.copy_(torch.rand(5, generator=draws))
            graph.replay() if captured else one()
            got.append(tokens.clone())
        mk.status()
        streams.append(torch.stack(got))
    assert torch.equal(*streams)
    assert streams[0].unique().numel() > 10


@pytest.mark.gpu
def test_a_scaled_rope_table_reaches_the_model(oracle):
    """`set_rope` with a stretched table: extend and the engine's own prompt see the same positions, and other logits than without it."""
    from qwen3mk import paged, prefill

    g = torch.Generator().manual_seed(9)
    mk, w, dev = setup(oracle, 33)
    ids = torch.randint(0, VOCAB, (300,), generator=g).cuda()
    plain = prefill.prefill(dev, ids, engine=mk)[2]
    mk.set_rope(paged.rope_table(4096, scaling={"type": "yarn", "factor": 4.0, "original": 128}))
    want = prefill.prefill(dev, ids, engine=mk)[2]
    server = Server(1, 64, 20, g)
    out = mk.extend(dev, ids, server.batch([300]))
    mk.status()
    assert oracle.rel_l2(out["logits"][0], want) <= 4e-2        # two gates, as above
    assert oracle.rel_l2(plain, want) > 8e-2
    with pytest.raises(ValueError, match="set_rope"):
        mk.set_rope(paged.rope_table(10, rotary_dim=64))


@pytest.mark.gpu
def test_refusals_and_reports(oracle):
    from qwen3mk import Megakernel, paged

    mk, w, dev = setup(oracle, 34, max_positions=256)
    g = torch.Generator().manual_seed(10)
    server = Server(2, 16, 60, g)
    batch = server.batch([4, 6])
    ids = torch.randint(0, VOCAB, (10,), generator=g).cuda()
    for bad in (ids[:9], ids.to(torch.int32), ids.cpu()):
        with pytest.raises(ValueError, match="ids"):
            mk.extend(dev, bad, batch)
    with pytest.raises(ValueError, match="layers"):
        mk.extend(dev, ids, paged.PagedBatch(paged.PagePool.empty(layers=2, pages=4), batch.page_table, batch.q_start, batch.kv_len))
    with pytest.raises(ValueError, match="kv heads"):
        mk.extend(dev, ids, paged.PagedBatch(paged.PagePool.empty(layers=LAYERS, pages=60, page_size=16, kv_heads=4), batch.page_table, batch.q_start, batch.kv_len))
    many = paged.PagedBatch(server.pool, batch.page_table.repeat(5, 1), torch.arange(11, dtype=torch.int32).cuda(), torch.ones(10, dtype=torch.int32).cuda())
    with pytest.raises(ValueError, match="max_batch"):
        mk.extend(dev, ids, many)
    small = Megakernel(layers=LAYERS, vocab=VOCAB, max_batch=2)
    with pytest.raises(RuntimeError, match="at least 4"):
        small.extend(dev, ids, batch)
    out = mk.extend(dev, ids, batch, want_logits=False)
    assert out["logits"] is None
    mk.status()
    # positions beyond the RoPE table, and fewer positions than new tokens
    for lens in ([4, 300], [3, 6]):
        mk.extend(dev, ids, paged.PagedBatch(server.pool, batch.page_table, batch.q_start, torch.tensor(lens, dtype=torch.int32).cuda()))
        with pytest.raises(RuntimeError, match="code 5 at site 1100"):
            mk.status()
    good = mk.extend(dev, ids, batch)
    mk.status()
    assert torch.isfinite(good["logits"]).all()


def test_null_engines_are_refused():
    from qwen3mk import _cabi

    lib = _cabi.load()
    assert lib.q3_extend(None, None, None) == _cabi.ERR_INVALID


@pytest.mark.gpu
def test_a_small_workspace_is_refused_before_anything_is_written(oracle):
    import ctypes

    from qwen3mk import _cabi

    mk, w, dev = setup(oracle, 35)
    g = torch.Generator().manual_seed(11)
    server = Server(2, 16, 20, g)
    batch = server.batch([3, 5])
    mk.extend(dev, torch.randint(0, VOCAB, (8,), generator=g).cuda(), batch)
    k = server.pool.k.clone()
    ids, nxt = torch.randint(0, VOCAB, (8,), generator=g).cuda(), torch.zeros(2, dtype=torch.int64, device="cuda")
    need = batch.workspace_bytes(16)
    space = torch.empty(need, dtype=torch.uint8, device="cuda")
    for at, size in ((space.data_ptr(), need - 1), (None, need), (space.data_ptr() + 4, need)):
        a = _cabi.ExtendArgs(ctypes.pointer(batch.view(0)), server.pool.k.stride(0), ids.data_ptr(), None, nxt.data_ptr(), at, size)
        with pytest.raises(ValueError, match="workspace"):
            _cabi.check(mk.lib, mk.handle, mk.lib.q3_extend(mk.handle, ctypes.byref(a), None), "q3_extend")
    torch.cuda.synchronize()
    assert torch.equal(server.pool.k.view(torch.int16), k.view(torch.int16))

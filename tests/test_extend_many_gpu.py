"""Megakernel.extend with more sequences than a small server has: the LM head's forms for up to 32, 64 and more of them, and a vocabulary that its tiles do not divide."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

LAYERS = 2


def serve(mk, dev, news, ids, table, pool, had):
    from qwen3mk import paged

    start = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda()
    lens = torch.tensor([h + m for h, m in zip(had, news)], dtype=torch.int32).cuda()
    return mk.extend(dev, torch.cat(ids).cuda(), paged.PagedBatch(pool, table, start, lens))


@pytest.mark.parametrize("batch,vocab", [(33, 4096), (40, 2056), (64, 4096), (70, 4096), (70, 2056), (130, 4096)])
def test_many_sequences_beside_small_calls(oracle, batch, vocab):
    """A first chunk, then one or two tokens each, some sequences without any: logits and tokens beside those of the same sequences in calls of three, and three of them beside the
    oracle.  Both sides round activations to bf16: a gate of 2e-2 against the exact rows, so two between them."""
    from qwen3mk import Megakernel, paged, weights

    inp = oracle.synthetic(40, oracle.Shape(layers=LAYERS, vocab=vocab), context=1)
    w = {k: inp[k] for k in weights.WEIGHT_NAMES}
    dev = {k: v.cuda() for k, v in w.items()}
    w32 = {k: v.float() for k, v in w.items()}
    g = torch.Generator().manual_seed(batch)
    first = [int(x) for x in torch.randint(0, 9, (batch,), generator=g)]
    first[0], first[1] = 5, 0
    then = [int(x) for x in torch.randint(0, 3, (batch,), generator=g)]
    then[0], then[1], then[2] = 1, 0, 2
    ids = [torch.randint(0, vocab, (a + b,), generator=g) for a, b in zip(first, then)]
    table = torch.arange(batch, dtype=torch.int32)[:, None].contiguous().cuda()
    mk = Megakernel(layers=LAYERS, vocab=vocab, max_batch=batch, max_tokens=1300)
    few = Megakernel(layers=LAYERS, vocab=vocab, max_batch=4, max_tokens=64)
    pools = [paged.PagePool.empty(layers=LAYERS, pages=batch, page_size=16) for _ in range(2)]
    for step, (news, had) in enumerate(((first, [0] * batch), (then, first))):
        mine = [x[h:h + m] for x, h, m in zip(ids, had, news)]
        out = serve(mk, dev, news, mine, table, pools[0], had)
        mk.status()
        assert torch.equal(out["next_token"], out["logits"].argmax(dim=-1).where(torch.tensor(news).cuda() > 0, torch.zeros((), dtype=torch.int64, device="cuda")))
        for b in range(0, batch, 3):
            part = slice(b, b + 3)
            if sum(news[part]) == 0:
                assert not out["logits"][part].any()
                continue
            small = serve(few, dev, news[part], mine[part], table[part], pools[1], had[part])["logits"]
            few.status()
            for i, m in enumerate(news[part]):
                if m == 0:
                    assert not out["logits"][b + i].any() and not small[i].any()
                else:
                    assert oracle.rel_l2(out["logits"][b + i], small[i]) <= 4e-2, (step, b + i)
        for b in (0, 2, batch - 1):
            if news[b]:
                assert oracle.rel_l2(out["logits"][b].cpu(), oracle.prefill(w32, ids[b][:had[b] + news[b]])[2]) <= 2e-2, (step, b)
        if batch <= 64:                                  # (the same rows are written again)
            again = serve(mk, dev, news, mine, table, pools[0], had)
            assert torch.equal(again["logits"], out["logits"]) and torch.equal(again["next_token"], out["next_token"])
        else:
            again = serve(mk, dev, news, mine, table, pools[0], had)
            assert oracle.rel_l2(again["logits"], out["logits"]) <= 1e-5
    # without logits: the engine's own buffer
    start = torch.tensor([0] + then).cumsum(0).to(torch.int32).cuda()
    lens = torch.tensor([a + b for a, b in zip(first, then)], dtype=torch.int32).cuda()
    quiet = mk.extend(dev, torch.cat([x[h:] for x, h in zip(ids, first)]).cuda(), paged.PagedBatch(pools[0], table, start, lens), want_logits=False)
    assert quiet["logits"] is None and torch.equal(quiet["next_token"], out["next_token"])

"""The operators of a server that keeps many conversations in one pool of cache pages, as cases that can be timed and compared:

  rope    {"op", "seqs", "new", "cached", "ragged", "page", "heads", "kv_heads", "rotary", "interleaved", "norm", "rows", "type"}
          paged.rope_append(): head norm and rotary embedding of the new tokens' q and k rows, k and v rows into the pages
  attend  {"op", "seqs", "new", "chunks", "cached", "ragged", "page", "heads", "kv_heads", "type"}
          paged.attention(): `seqs` sequences of up to `cached` cached positions; `chunks` of them bring up to `new` new tokens, the others one
  sample  {"op", "rows", "temperature", "top_k", "top_p", "min_p", "mixed"}
          sampling.sample_rows(): one token a row; `mixed`: every row has temperature, top-k, top-p and min-p of its own

`own` false: plain torch operations in 32 bits (64 for the sums and borders of sampling); true: the package's operators.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

HEAD_DIM = 128
VOCAB = 151936
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _package():
    root = os.path.join(os.getcwd(), "qwen3-megakernel_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from qwen3mk import paged, sampling

    return paged, sampling


def listed():
    attend = {"op": "attend", "page": 64, "heads": 16, "kv_heads": 8, "type": "bf16"}
    rope = {"op": "rope", "page": 64, "heads": 16, "kv_heads": 8, "rotary": 128, "interleaved": False, "norm": True, "rows": "fp32", "type": "bf16"}
    return [
        # the new tokens' rows: one chat's next token, an odd chunk of a half-rotated interleaved model with bf16 rows, a whole long prompt
        {"name": "rope_1", **rope, "seqs": 1, "new": 1, "cached": 1000, "ragged": False},
        {"name": "rope_777_interleaved", **rope, "seqs": 3, "new": 377, "cached": 2000, "ragged": True, "page": 16, "rotary": 64, "interleaved": True, "norm": False,
         "rows": "bf16"},
        {"name": "rope_2048", **rope, "seqs": 1, "new": 2048, "cached": 0, "ragged": False},
        # one chat's next token; a full serving batch of uneven chats; one very long document
        {"name": "attend_1_1000", **attend, "seqs": 1, "new": 1, "chunks": 0, "cached": 1000, "ragged": False},
        {"name": "attend_64_ragged", **attend, "seqs": 64, "new": 1, "chunks": 0, "cached": 2048, "ragged": True},
        # eight users' short answers (or drafts that are checked at once) over long chats, small pages, fp16
        {"name": "attend_8_answers", **attend, "seqs": 8, "new": 13, "chunks": 8, "cached": 5000, "ragged": True, "page": 16, "type": "fp16"},
        # a chunk of a long document behind what is cached of it; a first chunk beside a batch that decodes
        {"name": "attend_chunk_2048", **attend, "seqs": 1, "new": 2048, "chunks": 1, "cached": 8192, "ragged": False},
        {"name": "attend_mixed", **attend, "seqs": 27, "new": 512, "chunks": 3, "cached": 2048, "ragged": True},
        # choosing the next token: the model's own settings for one chat, a nucleus of the whole vocabulary for a full batch, users with settings of their own
        {"name": "sample_1_top20", "op": "sample", "rows": 1, "temperature": 0.6, "top_k": 20, "top_p": 0.95, "min_p": 0.0, "mixed": False},
        {"name": "sample_64_nucleus", "op": "sample", "rows": 64, "temperature": 0.8, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "mixed": False},
        {"name": "sample_27_mixed", "op": "sample", "rows": 27, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.05, "mixed": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "attend", "attend", "attend", "sample"])
    if op == "sample":
        return {"op": op, "rows": _log_int(rng, 1, 64), "temperature": round(rng.uniform(0.4, 1.2), 3), "top_k": rng.choice([0, 0, 20, 50, 200]),
                "top_p": rng.choice([0.8, 0.9, 0.95, 1.0]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1]), "mixed": rng.random() < 0.4}
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (16, 8), (8, 4), (8, 8), (16, 4), (16, 2)])
    page = rng.choice([16, 32, 64, 128])
    base = {"op": op, "page": page, "heads": heads, "kv_heads": kv_heads, "type": rng.choice(["bf16", "bf16", "fp16"])}
    if op == "rope":
        seqs = _log_int(rng, 1, 64)
        return {**base, "seqs": seqs, "new": _log_int(rng, 1, max(1, 2048 // seqs)), "cached": _log_int(rng, 1, min(8000, 65536 // seqs)), "ragged": rng.random() < 0.6,
                "rotary": rng.choice([128, 128, 64, 32]), "interleaved": rng.random() < 0.4, "norm": rng.random() < 0.6, "rows": rng.choice(["fp32", "bf16"])}
    kind = rng.choice(["decode", "decode", "answers", "chunk", "mixed"])
    if kind == "decode":
        seqs = _log_int(rng, 1, 64)
        return {**base, "seqs": seqs, "new": 1, "chunks": 0, "cached": _log_int(rng, 16, min(32768, 131072 // seqs)), "ragged": rng.random() < 0.6}
    if kind == "answers":
        seqs = _log_int(rng, 1, 16)
        return {**base, "seqs": seqs, "new": _log_int(rng, 2, 40), "chunks": seqs, "cached": _log_int(rng, 64, min(8192, 65536 // seqs)), "ragged": rng.random() < 0.6}
    if kind == "chunk":
        new = _log_int(rng, 64, 2048)
        return {**base, "seqs": 1, "new": new, "chunks": 1, "cached": _log_int(rng, 1, 8192), "ragged": False}
    seqs = _log_int(rng, 4, 32)
    return {**base, "seqs": seqs, "new": _log_int(rng, 32, 512), "chunks": rng.randint(1, 3), "cached": _log_int(rng, 64, 2048), "ragged": True}


def _lengths(case):
    """(new tokens, cached positions) of every sequence: all alike, or spread down to a quarter."""
    n, new, cached = case["seqs"], case["new"], case["cached"]
    chunks = case.get("chunks", n)
    spread = (lambda most, i, of: most - (3 * most * i) // (4 * max(1, of - 1)) if case["ragged"] else most)  # noqa: E731
    news = [max(1, spread(new, i, chunks)) if i < chunks else 1 for i in range(n)]
    olds = [max(0, spread(cached, (i * 7) % n, n)) for i in range(n)]
    return news, olds


def _pool(gen, case, totals):
    """Pages in no particular order, two of them spare; K rows leave a head norm and V rows a projection of normalised activations: elements of size one."""
    page = case["page"]
    counts = np.array([-(-t // page) for t in totals])
    n_pages = int(counts.sum()) + 2
    shape = (1, n_pages, page, case["kv_heads"], HEAD_DIM)
    k, v = (torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=gen).to(TYPES[case["type"]]) for _ in range(2))
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32).cpu().numpy()
    table = np.full((len(totals), max(1, int(counts.max()))), -1, dtype=np.int32)
    table[np.arange(table.shape[1]) < counts[:, None]] = order[:counts.sum()]
    return k, v, torch.from_numpy(table).cuda()


def _rope_rows(positions, rotary):
    """cos | sin of every position, fp32 [positions, rotary], from angles in 64 bits."""
    freq = 1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat([ang.cos(), ang.sin()], dim=1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(2_000_003 + seed)
    s = {"case": case}
    if case["op"] == "sample":
        rows = case["rows"]
        # the logits of a trained model are far from flat: a few words carry most of the weight
        s["logits"] = 5.0 * torch.randn((rows, VOCAB), generator=gen, device="cuda")
        s["u"] = torch.rand(rows, generator=gen, device="cuda")
        one = lambda x, dt: torch.full((rows,), x, dtype=dt, device="cuda")  # noqa: E731
        if case["mixed"]:
            pick = lambda xs, dt: torch.tensor(xs, dtype=dt, device="cuda")[torch.randint(len(xs), (rows,), generator=gen, device="cuda")]  # noqa: E731
            s["temperature"] = pick([case["temperature"], 0.0, 0.6, 1.0, case["temperature"]], torch.float32)
            s["top_k"] = pick([case["top_k"], 0, 20, 1, 100], torch.int32)
            s["top_p"] = pick([case["top_p"], 1.0, 0.95, 0.8], torch.float32)
            s["min_p"] = pick([case["min_p"], 0.0, 0.0, 0.1], torch.float32)
        else:
            s["temperature"], s["top_k"] = one(case["temperature"], torch.float32), one(case["top_k"], torch.int32)
            s["top_p"], s["min_p"] = one(case["top_p"], torch.float32), one(case["min_p"], torch.float32)
        s["out"] = torch.zeros(rows, dtype=torch.int64, device="cuda")
        return s
    news, olds = _lengths(case)
    totals = [n + c for n, c in zip(news, olds)]
    tokens, heads, kv_heads, dt = sum(news), case["heads"], case["kv_heads"], TYPES[case["type"]]
    s["k_pages"], s["v_pages"], s["table"] = _pool(gen, case, totals)
    s["q_start"] = torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(totals, dtype=torch.int32, device="cuda")
    s["max_new"], s["max_total"], s["tokens"] = max(news), max(totals), tokens
    normal = lambda shape, d: torch.randn(shape, generator=gen, device="cuda").to(d)  # noqa: E731
    if case["op"] == "attend":
        s["q"] = normal((tokens, heads, HEAD_DIM), dt)
        s["out"] = torch.zeros((tokens, heads, HEAD_DIM), dtype=dt, device="cuda")
    else:
        # q, k and v rows lie side by side, as one projection writes them
        qkv = normal((tokens, (heads + 2 * kv_heads) * HEAD_DIM), TYPES[case["rows"]])
        s["qkv"] = qkv
        s["q"], s["k"], s["v"] = (x.view(tokens, -1, HEAD_DIM) for x in qkv.split([heads * HEAD_DIM, kv_heads * HEAD_DIM, kv_heads * HEAD_DIM], dim=1))
        s["gq"], s["gk"] = ((1.0 + 0.1 * normal((HEAD_DIM,), torch.float32)).to(torch.bfloat16) if case["norm"] else None for _ in range(2))
        s["rope"] = _rope_rows(s["max_total"], case["rotary"])
        s["out"] = torch.zeros((tokens, heads, HEAD_DIM), dtype=dt, device="cuda")
    return s


def _owners(s):
    """Sequence and position of every new token."""
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["q_start"][1:].long(), t, right=True)
    return b, s["kv_len"][b].long() - s["q_start"][b + 1].long() + t


def _plain_rope(s):
    case, r = s["case"], s["case"]["rotary"]
    b, pos = _owners(s)
    cos, sin = s["rope"][pos, None, :r // 2], s["rope"][pos, None, r // 2:]

    def turn(x, gain):
        x = x.float()
        if gain is not None:
            x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6) * gain.float()
        if case["interleaved"]:
            x0, x1 = x[..., 0:r:2], x[..., 1:r:2]
            y = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], dim=-1).flatten(-2)
        else:
            x0, x1 = x[..., :r // 2], x[..., r // 2:r]
            y = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], dim=-1)
        return torch.cat([y, x[..., r:]], dim=-1)

    page = case["page"]
    at, slot = s["table"][b, pos // page].long(), pos % page
    s["k_pages"][0, at, slot] = turn(s["k"], s["gk"]).to(s["k_pages"].dtype)
    s["v_pages"][0, at, slot] = s["v"].to(s["v_pages"].dtype)
    s["out"].copy_(turn(s["q"], s["gq"]))
    return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attend(s):
    case = s["case"]
    kv_heads, page = case["kv_heads"], case["page"]
    group = case["heads"] // kv_heads
    start, end, total = s["q_start"][:-1].long(), s["q_start"][1:].long(), s["kv_len"].long()
    row = start[:, None] + torch.arange(s["max_new"], device="cuda")
    live = row < end[:, None]
    row = row.clamp(max=s["tokens"] - 1)
    qpos = total[:, None] - end[:, None] + row
    key = torch.arange(s["max_total"], device="cuda")
    at = s["table"][:, key // page].long()
    seen = (at >= 0) & (key < total[:, None])
    at, slot = at.clamp(min=0), (key % page).expand_as(at)
    k = s["k_pages"][0, at, slot].float()                       # [seqs, keys, kv_heads, 128]
    v = s["v_pages"][0, at, slot].float()
    q = s["q"][row].float().unflatten(2, (kv_heads, group))     # [seqs, new, kv_heads, group, 128]
    seqs, new = row.shape
    q = q.permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, group * new, HEAD_DIM)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).view(seqs, kv_heads, group, new, -1)
    scores *= HEAD_DIM ** -0.5
    hidden = ~(seen[:, None, :] & (key <= qpos[..., None]))     # [seqs, new, keys]
    scores.masked_fill_(hidden[:, None, None], float("-inf"))
    scores -= scores.amax(dim=-1, keepdim=True)
    scores.exp_()
    scores /= scores.sum(dim=-1, keepdim=True)
    o = torch.matmul(scores.view(seqs, kv_heads, group * new, -1), v.permute(0, 2, 1, 3))
    o = o.view(seqs, kv_heads, group, new, HEAD_DIM).permute(0, 3, 1, 2, 4).reshape(seqs, new, case["heads"], HEAD_DIM)
    s["out"][row[live]] = o[live].to(s["out"].dtype)
    return s["out"]


def _plain_sample(s):
    rows = s["logits"].double()
    vocab = rows.shape[-1]
    top = rows.amax(dim=-1, keepdim=True)
    greedy = (s["temperature"] <= 0) | (s["top_k"] == 1)
    t = torch.where(s["temperature"] > 0, s["temperature"], torch.ones_like(s["temperature"])).double()
    w = torch.exp((rows - top) / t[:, None])
    most, order = torch.sort(rows, dim=-1, descending=True, stable=True)     # equal words: the lowest index first
    k = torch.where((s["top_k"] > 0) & (s["top_k"] < vocab), s["top_k"].long(), torch.full_like(s["top_k"], vocab).long())
    kth = most.gather(1, k[:, None] - 1)
    ranked = torch.where(most >= kth, w.gather(1, order), torch.zeros_like(w))
    before = ranked.cumsum(dim=-1) - ranked
    p = s["top_p"].double()[:, None]
    kept = (most >= kth) & ((p >= 1) | (before < p * ranked.sum(dim=-1, keepdim=True))) & (w.gather(1, order) >= s["min_p"].double()[:, None])
    kept[:, 0] = True
    w = torch.where(torch.zeros_like(kept).scatter(1, order, kept), w, torch.zeros_like(w))
    cdf = w.cumsum(dim=-1)
    token = (cdf > s["u"].double()[:, None] * cdf[:, -1:]).to(torch.uint8).argmax(dim=-1)
    s["out"].copy_(torch.where(greedy, (rows == top).to(torch.uint8).argmax(dim=-1), token))
    return s["out"]


def run(state):
    s, case = state, state["case"]
    if own:
        paged, sampling = _package()
        if case["op"] != "sample" and "batch" not in s:     # the descriptors that a program keeps for a batch
            s["batch"] = paged.PagedBatch(paged.PagePool(s["k_pages"], s["v_pages"]), s["table"], s["q_start"], s["kv_len"], tokens=s["tokens"], max_new=s["max_new"])
        if case["op"] == "rope":
            q = paged.rope_append(s["batch"], s["q"], s["k"], s["v"], s["rope"], q_gain=s["gq"], k_gain=s["gk"], interleaved=case["interleaved"], out=s["out"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if case["op"] == "attend":
            return paged.attention(s["batch"], s["q"], out=s["out"])
        return sampling.sample_rows(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], u=s["u"], out=s["out"])
    return {"rope": _plain_rope, "attend": _plain_attend, "sample": _plain_sample}[case["op"]](s)


def exact(case, seed):
    if case["op"] == "sample":
        return None                                  # words are whole numbers
    s = prepare(case, seed)
    news, olds = _lengths(case)
    page, table = case["page"], s["table"].tolist()
    kv_heads, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    at = 0
    for b, (new, old) in enumerate(zip(news, olds)):
        total = new + old
        where = torch.tensor([table[b][p // page] * page + p % page for p in range(total)], device="cuda")
        if case["op"] == "attend":
            keys, values = (x[0].flatten(0, 1)[where] for x in (k_pages, v_pages))
            hide = torch.ones((new, total), dtype=torch.bool, device="cuda").triu(old + 1)
            for h in range(case["heads"]):
                score = s["q"][at:at + new, h].double() @ keys[:, h // group].T / math.sqrt(HEAD_DIM)
                out[at:at + new, h] = torch.softmax(score.masked_fill(hide, -math.inf), dim=-1) @ values[:, h // group]
        else:
            r = case["rotary"]
            freq = torch.tensor([1e6 ** (-2 * i / r) for i in range(r // 2)], dtype=torch.float64, device="cuda")
            turn = torch.polar(torch.ones((new, r // 2), dtype=torch.float64, device="cuda"), torch.arange(old, total, device="cuda").double()[:, None] * freq)

            def rotated(x, gain):
                x = x.double()
                if gain is not None:
                    x = x / torch.sqrt(x.pow(2).mean(dim=-1, keepdim=True) + 1e-6) * gain.double()
                head = x[..., :r].unflatten(-1, (r // 2, 2) if case["interleaved"] else (2, r // 2))
                head = head if case["interleaved"] else head.transpose(-1, -2)
                y = torch.view_as_real(torch.view_as_complex(head.contiguous()) * turn[:, None])
                y = y if case["interleaved"] else y.transpose(-1, -2)
                return torch.cat([y.flatten(-2), x[..., r:]], dim=-1)

            out[at:at + new] = rotated(s["q"][at:at + new], s["gq"])
            k_pages[0].view(-1, kv_heads, HEAD_DIM)[where[old:]] = rotated(s["k"][at:at + new], s["gk"])
            v_pages[0].view(-1, kv_heads, HEAD_DIM)[where[old:]] = s["v"][at:at + new].double()
        at += new
    return out if case["op"] == "attend" else {"q": out, "k_pages": k_pages, "v_pages": v_pages}


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (4 * VOCAB + 28), "flops": 6 * case["rows"] * VOCAB}
    news, olds = _lengths(case)
    tokens, heads, kv_heads = sum(news), case["heads"], case["kv_heads"]
    if case["op"] == "rope":
        row = (heads + 2 * kv_heads) * HEAD_DIM
        size = 4 if case["rows"] == "fp32" else 2
        return {"bytes": tokens * (row * (size + 2) + 4 * case["rotary"]), "flops": tokens * row * 6}
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(news, olds))
    cache = sum(n + c for n, c in zip(news, olds)) * kv_heads * HEAD_DIM * 4
    return {"bytes": cache + tokens * heads * HEAD_DIM * 4, "flops": 4 * HEAD_DIM * heads * pairs}

"""Row-wise sampling (q3_sample_rows) against the rule in 64 bits.

The kernel's weights are fp32: exp's argument x is off by up to |x| 2^-23 (two roundings) and exp itself by 2^-21, so a sum of weights w = e^-x is off by at most the mean of
(x 2^-23 + 2^-21) over its weight, with x below 30 on average in every case here 32 * 2^-22 = 7.7e-6; rounding to units of 2^-40 adds vocab * 2^-41, 1e-7.  So the cumulative
distribution may be off by TOL = 1e-5, and a word whose place at a top-p border is nearer to it than that may be kept or not."""
from __future__ import annotations

import pytest
import torch

TOL = 1e-5


def rule(row, t, k, p, m):
    """(kept words by the rule with p shifted down and up by TOL, weights): 64 bits, one row, on the CPU."""
    row = row.double()
    w = torch.where(row > float("-inf"), torch.exp((row - row.max()) / t), torch.zeros_like(row))
    order = torch.sort(row, descending=True, stable=True).indices
    ranked = w[order]
    if 0 < k < row.numel():
        ranked = torch.where(row[order] >= row[order][k - 1], ranked, torch.zeros_like(ranked))
    before = ranked.cumsum(0) - ranked
    kept = []
    for shift in (-TOL, TOL):
        keep = (ranked > 0) & ((before < (p + shift) * ranked.sum()) if p < 1 else True) & (ranked >= m * (1 - shift))
        keep[0] = True
        kept.append(torch.zeros_like(keep).scatter(0, order, keep))
    return kept[0], kept[1], w


def verify(logits, got, u, t, k, p, m):
    logits, got, u = logits.cpu(), got.cpu(), u.cpu()
    exact = 0
    for b in range(logits.shape[0]):
        j, (tb, kb, pb, mb) = int(got[b]), (float(x[b]) if isinstance(x, torch.Tensor) else x for x in (t, k, p, m))
        if not tb > 0 or kb == 1 or pb <= 0:
            assert j == int((logits[b] == logits[b].max()).nonzero()[0]), f"row {b}: not the arg-max"
            continue
        inner, outer, w = rule(logits[b], tb, int(kb), pb, mb)
        assert 0 <= j < logits.shape[1] and bool(outer[j]), f"row {b}: word {j} is not kept"
        if bool((inner != outer).any()):
            continue
        exact += 1
        cdf = torch.where(inner, w, torch.zeros_like(w)).cumsum(0)
        cdf /= cdf[-1].clone()
        lo = float(cdf[j - 1]) if j else 0.0
        assert lo - TOL <= float(u[b]) <= float(cdf[j]) + TOL, f"row {b}: u {float(u[b]):.7f} outside [{lo:.7f}, {float(cdf[j]):.7f}]"
    return exact


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.6, 20, 0.95, 0.0), (0.8, 0, 0.9, 0.0), (1.3, 0, 0.99, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 300, 0.5, 0.02), (0.9, 0, 1.0, 0.1), (1.0, 0, 0.97, 0.003),
            (1.0, 2, 0.3, 0.0), (0.05, 0, 0.9, 0.0), (30.0, 0, 0.9, 0.0), (2.0, 900, 1.0, 0.0), (2.0, 3000, 0.8, 0.0), (0.0, 5, 0.5, 0.0), (1.0, 0, 0.0, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab,batch", [(151936, 3), (151936, 70), (50000, 13), (4099, 33), (1000, 80), (17, 5), (2, 4), (1, 2)])
@pytest.mark.parametrize("setting", range(len(SETTINGS)))
def test_tokens_follow_the_rule(vocab, batch, setting):
    from qwen3mk import sampling

    t, k, p, m = SETTINGS[setting]
    g = torch.Generator().manual_seed(vocab + batch + setting)
    logits = (torch.randn(batch, vocab, generator=g) * 4).cuda()
    u = torch.rand(batch, generator=g).cuda()
    got = sampling.sample_rows(logits, t, k, p, m, u=u)
    verify(logits, got, u, t, k, p, m)
    assert torch.equal(got, sampling.sample_rows(logits, t, k, p, m, u=u)), "another run draws other words"


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [0.0, 0.01, 0.5, 1.5])
@pytest.mark.parametrize("setting", [(1.0, 0, 0.95, 0.0), (1.0, 20000, 0.9, 0.0), (1.0, 3000, 1.0, 0.0), (0.5, 0, 0.6, 0.01), (1.0, 0, 1.0, 0.2)])
def test_wide_sets(spread, setting):
    """Flat rows: tens of thousands of words are kept."""
    from qwen3mk import sampling

    t, k, p, m = setting
    g = torch.Generator().manual_seed(int(100 * spread) + k)
    logits = (torch.randn(6, 151936, generator=g) * spread).cuda()
    u = torch.tensor([0.0, 0.2, 0.5, 0.777, 0.99, 1 - 2.0 ** -24]).cuda()
    verify(logits, sampling.sample_rows(logits, t, k, p, m, u=u), u, t, k, p, m)


@pytest.mark.gpu
def test_equal_words_are_kept_in_the_order_of_their_indices():
    """All logits equal: a nucleus of p is the first ceil(p vocab) words, and the draw is floor(u count); top-k keeps every tie."""
    from qwen3mk import sampling

    for vocab in (30000, 151936, 40):
        logits = torch.full((5, vocab), -3.25, device="cuda")
        u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.875]).cuda()
        for p, count in ((0.5, vocab // 2), (0.25, vocab // 4)):
            got = sampling.sample_rows(logits, 0.7, 0, p, 0.0, u=u).tolist()
            assert got == [int(x * count) for x in u.tolist()]
        got = sampling.sample_rows(logits, 0.7, 7, 1.0, 0.0, u=u).tolist()
        assert got == [int(x * vocab) for x in u.tolist()]
    # 3000 words share the first place, the others are far below
    logits = torch.full((4, 151936), -50.0, device="cuda")
    at = torch.randperm(151936, generator=torch.Generator().manual_seed(1))[:3000].sort().values
    logits[:, at.cuda()] = 2.0
    u = torch.tensor([0.0, 0.3, 0.6, 0.999]).cuda()
    got = sampling.sample_rows(logits, 1.0, 0, 0.5, 0.0, u=u).tolist()
    assert got == [int(at[int(x * 1500 + 1e-4)]) for x in u.tolist()]


@pytest.mark.gpu
@pytest.mark.parametrize("mask", [float("-inf"), -1e9, torch.finfo(torch.float32).min])
def test_masked_words_are_never_drawn(mask):
    from qwen3mk import sampling

    g = torch.Generator().manual_seed(3)
    logits = (torch.randn(24, 50000, generator=g) * 3).cuda()
    allowed = torch.rand(24, 50000, generator=g) < 0.01
    allowed[5] = False
    allowed[5, 31234] = True
    allowed[6] = False
    allowed[6, [7, 49999]] = True
    logits[~allowed.cuda()] = mask
    u = torch.rand(24, generator=g).cuda()
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 3000, 1.0, 0.0), (0.9, 0, 1.0, 0.05), (5.0, 0, 0.999, 0.0), (float("inf"), 0, 1.0, 0.0) if mask == float("-inf") else (2.0, 0, 1.0, 0.0)):
        got = sampling.sample_rows(logits, t, k, p, m, u=u)
        assert allowed[torch.arange(24), got.cpu()].all(), (t, k, p, m)
        if t < 100:
            verify(logits, got, u, t, k, p, m)


@pytest.mark.gpu
def test_rows_with_settings_of_their_own_and_strides():
    from qwen3mk import sampling

    g = torch.Generator().manual_seed(4)
    n, vocab = 45, 70001
    wide = (torch.randn(n, vocab + 11, generator=g) * 4).cuda()
    logits = wide[:, 3:3 + vocab]                    # rows that begin at any word
    pick = lambda xs, dt: torch.tensor(xs, dtype=dt)[torch.randint(len(xs), (n,), generator=g)].cuda()  # noqa: E731
    t, k = pick([0.0, 0.3, 0.8, 1.0, 2.5], torch.float32), pick([0, 1, 5, 50, 2000, 100000, -3], torch.int32)
    p, m = pick([0.0, 0.5, 0.9, 1.0, 2.0], torch.float32), pick([0.0, 0.01, 0.2, -1.0], torch.float32)
    u = torch.rand(n, generator=g).cuda()
    got = sampling.sample_rows(logits, t, k, p, m, u=u)
    assert verify(logits, got, u, t, k.clamp(min=0), p, m.clamp(min=0)) > 10
    # a row alone draws what it draws among others
    for b in (0, 7, 44):
        assert int(sampling.sample_rows(logits[b:b + 1], t[b:b + 1], k[b:b + 1], p[b:b + 1], m[b:b + 1], u=u[b:b + 1])[0]) == int(got[b])


@pytest.mark.gpu
def test_rows_without_a_draw_give_the_arg_max():
    from qwen3mk import sampling

    logits = torch.randn(8, 20000, generator=torch.Generator().manual_seed(5)).cuda()
    logits[:, 1234] = 9.0
    logits[:, 4321] = 9.0                            # a tie: the lowest index
    logits[0, 17] = float("nan")
    logits[1, 15000] = float("inf")
    logits[1, 16000] = float("inf")
    logits[2] = float("-inf")
    logits[3] = float("nan")
    u = torch.tensor([0.5, 0.5, 0.5, 0.5, -0.1, 1.0, float("nan"), 0.5]).cuda()
    t = torch.tensor([1, 1, 1, 1, 1, 1, 1, float("nan")], dtype=torch.float32).cuda()
    for k, p, m in ((0, 1.0, 0.0), (50, 0.9, 0.0), (0, 0.9, 0.1)):
        assert sampling.sample_rows(logits, t, k, p, m, u=u).tolist() == [1234, 15000, 0, 0, 1234, 1234, 1234, 1234]
    assert sampling.sample_rows(logits[4:], 1.0, 0, 1.0, 1.5, u=u[:4] * 0).tolist() == [1234] * 4


@pytest.mark.gpu
def test_draws_follow_the_probabilities():
    from qwen3mk import sampling

    g = torch.Generator().manual_seed(6)
    base = torch.randn(60, generator=g) * 2
    n = 40000
    got = sampling.sample_rows(base.cuda().expand(n, 60), 0.9, 30, 0.9, 0.01, generator=torch.Generator(device="cuda").manual_seed(2)).cpu()
    inner, outer, w = rule(base, 0.9, 30, 0.9, 0.01)
    assert torch.equal(inner, outer)
    prob = torch.where(inner, w, torch.zeros_like(w))
    prob /= prob.sum()
    freq = torch.bincount(got, minlength=60).double() / n
    # five standard deviations of a frequency
    assert bool(((freq - prob).abs() <= 5 * (prob * (1 - prob) / n).sqrt() + 1e-9).all())


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    from qwen3mk import sampling

    g = torch.Generator().manual_seed(7)
    logits = (torch.randn(20, 151936, generator=g) * 4).cuda()
    u = torch.rand(20, generator=g).cuda()
    p = torch.full((20,), 0.9, device="cuda")
    out = torch.zeros(20, dtype=torch.int64, device="cuda")
    sampling.sample_rows(logits, 0.8, 0, p, 0.0, u=u, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampling.sample_rows(logits, 0.8, 0, p, 0.0, u=u, out=out)
    for q in (0.9, 0.3):
        p.fill_(q)
        logits.mul_(0.9)
        out.zero_()
        graph.replay()
        want = sampling.sample_rows(logits, 0.8, 0, q, 0.0, u=u)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        with torch.cuda.stream(torch.cuda.Stream()):
            other = sampling.sample_rows(logits, 0.8, 0, q, 0.0, u=u)
        torch.cuda.synchronize()
        assert torch.equal(other, want)


@pytest.mark.gpu
def test_refusals():
    from qwen3mk import sampling

    x = torch.zeros(3, 100, device="cuda")
    for bad in (x.half(), x.cpu(), x[0], x.t(), x[:0]):
        with pytest.raises(ValueError, match="logits"):
            sampling.sample_rows(bad)
    for kw in (dict(temperature=x[:, 0].double()), dict(top_k=torch.zeros(3, device="cuda")), dict(top_p=torch.zeros(2, device="cuda")), dict(min_p=torch.zeros(3)),
               dict(top_k=-1), dict(top_p=-0.5), dict(min_p=float("nan")), dict(temperature=float("nan")), dict(u=torch.zeros(2, device="cuda")), dict(out=torch.zeros(3, device="cuda"))):
        with pytest.raises(ValueError):
            sampling.sample_rows(x, **kw)


def test_bad_arguments_are_refused_before_the_device_is_touched():
    import ctypes

    from qwen3mk import _cabi

    lib = _cabi.load()
    good = dict(logits=4096, row_stride=100, uniform=4096, out_tokens=4096, batch=2, vocab=100, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    for bad in (dict(logits=None), dict(uniform=None), dict(out_tokens=None), dict(batch=0), dict(batch=(1 << 20) + 1), dict(vocab=0), dict(vocab=(1 << 22) + 1, row_stride=1 << 30), dict(row_stride=99),
                dict(top_k=-1), dict(top_p=-1.0), dict(top_p=float("nan")), dict(min_p=-0.1), dict(temperature=float("nan")), dict(logits=4097), dict(out_tokens=4100), dict(top_ks=4098)):
        assert lib.q3_sample_rows(ctypes.byref(_cabi.SampleRowsArgs(**{**good, **bad})), None) == _cabi.ERR_INVALID, bad
        assert lib.q3_last_error(None).startswith(b"q3_sample_rows: ")
    assert lib.q3_sample_rows(None, None) == _cabi.ERR_INVALID
    assert ctypes.sizeof(_cabi.SampleRowsArgs) == 8 * 8 + 6 * 4


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1e-39, 1e-37, 1e-20, 1e30, 1e37, float("inf")])
@pytest.mark.parametrize("setting", [(0, 1.0, 0.0), (0, 0.9, 0.0), (50, 1.0, 0.0), (0, 1.0, 0.1), (100, 0.9, 0.05)])
def test_extreme_temperatures_and_logits(t, setting):
    from qwen3mk import sampling

    g = torch.Generator().manual_seed(6)
    logits = torch.randn(6, 5000, generator=g) * 4
    logits[1] *= 7e37 / logits[1].abs().max()
    logits[2, ::2], logits[2, 1::2] = 3e38, -3e38
    logits[3] = -7.0
    logits[4, 100:] = float("-inf")
    logits = logits.cuda()
    u = torch.rand(6, generator=g).cuda()
    verify(logits, sampling.sample_rows(logits, t, *setting, u=u), u, t, *setting)

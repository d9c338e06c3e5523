"""Beam search's selection against the definition in 64 bits on the CPU.

Which continuations come out is checked without a tolerance within each beam (its chosen tokens are the first of its tokens by logit, then by number, in that order), and sums by a bound: exponentials in 32 bits
are off by two roundings and 2^-24 of their exponent, sums of 64 of them in four parts by 16 roundings, weighted averages of exponents below a maximum are less than log2 of the vocabulary: 2^-19 in all,
and an output is rounded to 32 bits once.
"""
import numpy as np
import pytest

from test_gpu_parity import bam  # noqa: F401  (the module fixture)

pytestmark = pytest.mark.gpu

OFF = 2.0 ** -19


def _type(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _sums(logits, scores):
    """[requests, beams, vocab] in 64 bits"""
    import torch
    x = logits.double().view(*scores.shape, -1)
    x = x - x.amax(-1, keepdim=True)                 # exact; the largest may be so far from zero that a logarithm beside it is lost
    lse = torch.logsumexp(x, -1, keepdim=True)
    s = scores.double()[..., None]
    y = s + (x - lse)
    lse_ok = torch.isfinite(lse)
    y = torch.where(lse_ok & ~torch.isfinite(s), s.expand_as(y), y)
    return torch.where(lse_ok, y, torch.full_like(y, float("nan")))


def _check(got, logits, scores, width):
    import torch
    sums, beams, tokens = (x.cpu() for x in got)
    requests, n_beams = scores.shape
    vocab = logits.shape[1]
    assert sums.shape == beams.shape == tokens.shape == (requests, width) and sums.dtype is torch.float32 and beams.dtype is tokens.dtype is torch.int32
    every = _sums(logits.cpu(), scores.cpu())
    x = logits.cpu().double().view(requests, n_beams, vocab)
    order = torch.arange(vocab)
    for r in range(requests):
        at = (beams[r].long() - r * n_beams) * vocab + tokens[r]
        assert bool(((beams[r] >= r * n_beams) & (beams[r] < (r + 1) * n_beams) & (tokens[r] >= 0) & (tokens[r] < vocab)).all())
        assert at.unique().numel() == width
        mine = every[r].flatten()[at]
        # the sums that they say they are, in order, NaN last
        nan = torch.isnan(mine)
        assert torch.equal(torch.isnan(sums[r]), nan) and (not bool(nan.any()) or bool(nan[int(nan.int().argmax()):].all()))
        inf = torch.isinf(mine)
        assert torch.equal(sums[r][inf].double(), mine[inf])
        fin = ~nan & ~inf
        assert bool(((sums[r][fin].double() - mine[fin]).abs() <= OFF + 1.01 * 2.0 ** -24 * mine[fin].abs()).all()), (sums[r][fin].double() - mine[fin]).abs().max()
        assert bool((sums[r][~nan][1:] <= sums[r][~nan][:-1]).all())
        # none of the others is larger
        best = torch.sort(torch.nan_to_num(every[r].flatten(), nan=-1e308, neginf=-1e307), descending=True, stable=True)
        have = torch.nan_to_num(mine, nan=-1e308, neginf=-1e307)
        assert bool(((have - best.values[:width]).abs() <= 2 * OFF).all() | torch.equal(have, best.values[:width])), (have - best.values[:width]).abs().max()
        # what is not finite: exactly by place
        odd = ~fin
        if bool(odd.any()) and int(odd.int().argmax()) > 0 or not bool(fin.any()):
            k = int(odd.int().argmax()) if bool(fin.any()) else 0
            assert torch.equal(at[k:], best.indices[k:width]), (at[k:], best.indices[k:width])
        for i in range(n_beams):
            chosen = tokens[r][(beams[r] == r * n_beams + i) & fin]
            if chosen.numel():
                first = order[torch.argsort(torch.nan_to_num(x[r, i], nan=-np.inf), descending=True, stable=True)][:chosen.numel()]
                assert torch.equal(chosen.long(), first), (r, i)


def _inputs(dtype, requests, beams, vocab, seed=1, spread=3.0):
    import torch
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(requests * beams, vocab, generator=gen) * spread).to(_type(dtype))
    scores = -20 * torch.rand(requests, 1, generator=gen) - 4 * torch.rand(requests, beams, generator=gen)
    return logits, scores


@pytest.mark.parametrize("dtype,requests,beams,vocab,width", [
    ("bf16", 1, 4, 32000, 8), ("f16", 3, 1, 5000, 1), ("f32", 2, 5, 10007, 10), ("bf16", 2, 3, 50001, 64), ("f16", 1, 2, 70003, 33), ("f32", 1, 2, 40001, 256), ("bf16", 5, 7, 1, 7), ("f16", 2, 3, 7, 20),
    ("f32", 2, 2, 3, 6), ("bf16", 1, 32, 503, 64), ("bf16", 1, 32, 2049, 200), ("f32", 70, 16, 999, 32), ("f16", 40, 4, 8191, 4), ("bf16", 300, 2, 4099, 5), ("bf16", 600, 4, 20011, 31), ("f32", 2100, 1, 9000, 64), ("bf16", 1, 1024, 40, 77),
])
def test_selection(bam, dtype, requests, beams, vocab, width):
    logits, scores = _inputs(dtype, requests, beams, vocab)
    _check(bam.beam_select(logits.cuda(), scores.cuda(), width=width), logits, scores, width)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("width", [5, 32, 50, 256])
@pytest.mark.parametrize("vocab", [300, 17003, 130000])
def test_equal_numbers(bam, dtype, width, vocab):
    """all logits the same, a few values only, beams alike, zeros of both signs: equal sums in the order of beam and token, exactly"""
    import torch
    gen = torch.Generator().manual_seed(2)
    same = torch.full((3, vocab), 0.5)
    few = torch.randint(0, 3, (1, vocab), generator=gen).float().expand(3, -1)
    zeros = torch.where(torch.rand(1, vocab, generator=gen) < 0.5, 0.0, -0.0).expand(3, -1)
    for x in (same, few, zeros):
        logits = x.to(_type(dtype)).contiguous()
        scores = torch.full((1, 3), -2.5)
        _, beams, tokens = bam.beam_select(logits.cuda(), scores.cuda(), width=width)
        want = torch.argsort(logits.double().flatten(), descending=True, stable=True)[:width]
        assert torch.equal((beams * vocab + tokens).cpu()[0].long(), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("width", [8, 40, 256])
@pytest.mark.parametrize("vocab", [16384, 100000])
@pytest.mark.parametrize("requests", [1, 1200])
def test_large_numbers_side_by_side(bam, dtype, width, vocab, requests):
    """orders that put the large numbers into a few threads' loads, or make every part better than the one before: more candidates than there is room for"""
    import torch
    n = 2 if requests == 1 else 1
    gen = torch.Generator().manual_seed(3)
    i = torch.arange(vocab)
    load = 4 if dtype == "f32" else 8
    rows = [torch.where((i // load) % 256 < 124, 5 + torch.rand(vocab, generator=gen), -torch.rand(vocab, generator=gen)), i.float() / vocab * 50, -i.float() / vocab * 50,
            torch.where(i < vocab // 3, 10.0, 0.0) + torch.rand(vocab, generator=gen)]
    if requests > 1:
        rows = rows[:2]
    for x in rows:
        logits = x.to(_type(dtype)).view(1, -1).expand(n, -1).contiguous()
        scores = -torch.rand(1, n, generator=gen)
        if requests == 1:
            _check(bam.beam_select(logits.cuda(), scores.cuda(), width=width), logits, scores, width)
        else:                      # as one of many: few workgroups to a row
            got = bam.beam_select(logits.cuda().expand(requests, -1), scores.cuda().expand(requests, -1), width=width)
            _check([y[-1:] - (requests - 1 if k == 1 else 0) for k, y in enumerate(got)], logits, scores, width)
            assert bool((got[2] == got[2][:1]).all())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_masked_and_ended(bam, dtype):
    """logits of minus infinity, all but a few tokens or all of them; the type's lowest value; beams whose score is minus infinity or NaN; NaN and infinity among logits"""
    import torch
    inf, nan = float("inf"), float("nan")
    for vocab in (50, 9001):
        for width in (3, 17, 40):
            logits, scores = _inputs(dtype, 2, 4, vocab)
            logits[0, 5:] = -inf
            logits[1, :] = -inf
            logits[2, 40] = nan
            scores[0, 3] = -inf
            logits[4, :] = torch.finfo(logits.dtype).min
            logits[5, 7:] = torch.finfo(logits.dtype).min
            logits[6, 45] = inf
            scores[1, 3] = nan
            _check(bam.beam_select(logits.cuda(), scores.cuda(), width=width), logits, scores, width)
            # the first step of a search: one beam of all
            scores[0, 1:] = -inf
            _check(bam.beam_select(logits[:4].cuda(), scores[:1].cuda(), width=width), logits[:4], scores[:1], width)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_strides(bam, dtype, offset):
    import torch
    logits, scores = _inputs(dtype, 2, 3, 6007)
    wide = torch.full((6, 6007 + 11), 50.0, dtype=logits.dtype, device="cuda")
    wide[:, offset:offset + 6007] = logits.cuda()
    wide_scores = torch.zeros(2, 9, device="cuda")
    wide_scores[:, 2:5] = scores.cuda()
    _check(bam.beam_select(wide[:, offset:offset + 6007], wide_scores[:, 2:5], width=9), logits, scores, 9)
    # one row for all beams
    one = wide[:1, offset:offset + 6007].expand(6, -1)
    _check(bam.beam_select(one, scores.cuda(), width=9), logits[:1].expand(6, -1).contiguous(), scores, 9)


def test_streams_and_graphs(bam):
    """on another stream, and replayed several times with other inputs and other work between, as eagerly"""
    import torch
    logits, scores = (x.cuda() for x in _inputs("bf16", 3, 4, 40000))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = bam.beam_select(logits, scores, width=8)
    side.synchronize()
    _check(other, logits, scores, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bam.beam_select(logits, scores, width=8)
    for seed in range(4):
        x, y = (t.cuda() for t in _inputs("bf16", 3, 4, 40000, seed=seed + 10))
        logits.copy_(x)
        scores.copy_(y)
        graph.replay()
        eager = bam.beam_select(x, y, width=8)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), seed
        _check(out, x, y, 8)


def test_refusals(bam):
    import torch
    x, s = torch.zeros(6, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    for logits, scores, kw in ((x.cpu(), s, {}), (x, s.cpu(), {}), (x.double(), s, {}), (x, s.double(), {}), (x, s[:1], {}), (x[0], s, {}), (x, s[0], {}), (x.T.contiguous().T, s, {}), (x, s.T.contiguous().T, {}),
                               (x, s, {"width": 0}), (x, s, {"width": 257}), (x[:, :2], s, {"width": 7}), (x[:, :0], s, {}), (x, s, {"width": 2.0}), (x, s, {"width": -1}),
                               (x.clone().requires_grad_(), s, {}), (x, s.clone().requires_grad_(), {}), (torch.zeros(1100, 5, device="cuda"), torch.zeros(1, 1100, device="cuda"), {"width": 3})):
        with pytest.raises(bam.BamError):
            bam.beam_select(logits, scores, **kw)
    with torch.no_grad():
        assert bam.beam_select(x.clone().requires_grad_(), s)[0].shape == (2, 3)
    assert bam.beam_select(x[:0], s[:0])[1].shape == (0, 3)

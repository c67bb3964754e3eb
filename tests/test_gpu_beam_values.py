"""Beam selection at logits and scores of any size, against float64 on the GPU: what masks by -1e10 and the like leave, sums whose
terms are all rounded the same way, beams far behind the best, values below float32's range."""
import math

import numpy as np
import pytest
import torch

from test_gpu_beam_search import check_step, cuda, generator, inputs  # noqa: F401

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def shifted(logits):
    """The same rows relative to their largest value, in float64: no library's log_softmax then swallows a sum next to 1e30."""
    x = logits.double()
    return x - x.amax(1, keepdim=True)


# ------------------------------------------------------- logits of large size
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('value', [-1e4, -1e7, -3e9, -1e10, -1e12, -1e30, -1e36])
@pytest.mark.parametrize('where', ['front', 'slices', 'most', 'row', 'best row'])
def test_logits_masked_by_large_values(where, value, dtype):
    """Rows masked by a value as programs write it (masked_fill with -1e10, say): whole groups, slices, all but some, all."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(2, 6, 70001, dtype, 31)
    rows = logits.view(2, 6, -1)
    if where == 'front':
        rows[:, ::2, :30000] = value
    elif where == 'slices':
        rows[:, :, 9000:66000] = value
    elif where == 'most':
        rows[:, :, 100:-3] = value
    else:
        rows[:, 1] = value
        if where == 'best row':
            scores[:, 1] = 12.0
    search = BeamSearch(6)
    step = search.select(logits, scores)
    check_step(step, shifted(logits), scores, 12, 6)
    if where == 'best row':
        assert step.all_parents.tolist() == [[1] * 12] * 2 and step.all_tokens.tolist() == [list(range(12))] * 2
    search.check()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('value', [1e4, 1e7, 3e9, 1e10, 1e12, 1e30, 1e36])
def test_logits_far_above_the_others(value, dtype):
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(2, 6, 70001, dtype, 32)
    logits[::4, 12345] = value
    logits[1, 7::30000] = value  # several that are equal
    search = BeamSearch(6)
    check_step(search.select(logits, scores), shifted(logits), scores, 12, 6)
    search.check()


@pytest.mark.parametrize('middle', [(1 << 21) - 9, (1 << 21) + 9, 9 - (1 << 21), -9 - (1 << 21), 3 << 20, 1 << 22, -(1 << 23), 1 << 24])
def test_rows_about_a_large_value(middle):
    """Rows whose logits all lie near a value of 2^21 and more, a quarter or more apart."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    g = generator(5)
    logits = middle + 3.0 * torch.randn(12, 30011, generator=g, device='cuda')
    scores = -4 * torch.rand(2, 6, generator=g, device='cuda')
    search = BeamSearch(6)
    check_step(search.select(logits, scores), shifted(logits), scores, 12, 6)
    search.check()


# --------------------------------------------- sums rounded the same way in all terms
def exponents(top, tail):
    """What float32 makes of the exponents of tail under top, in two forms, less what they are (units of log2)."""
    one = np.float32(1.4426950408889634)
    exact = (tail.astype(np.float64) - top.astype(np.float64)) * 1.4426950408889634
    apart = ((tail - top) * one).astype(np.float64)
    unit = np.ceil(top * one) - np.float32(6)
    fused = (tail.astype(np.float64) * np.float64(one) - unit).astype(np.float32).astype(np.float64)
    return apart - exact, fused - (tail.astype(np.float64) * 1.4426950408889634 - unit)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [20000, 152704, 262144, 1 << 20])
@pytest.mark.parametrize('form', [0, 1])
@pytest.mark.parametrize('each', [0, 1024, 8192, 65536])
def test_rows_whose_terms_are_rounded_alike(each, form, vocab, dtype):
    """Two beams, each with one value (at one place, or every so many) above a tail of one other value, 6 to 14 below: all terms of
    a sum have the same error.  The values are those of 4,000 pairs whose exponent is rounded up and down the most; the best
    candidates of the two are 1e-8 to 6e-7 apart, both ways, and come in float64's order."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    rng = np.random.default_rng(vocab + form)
    top = rng.uniform(0.5, 2.0, 4000).astype(np.float32)
    tail = (top - rng.uniform(6.0, 14.0, 4000)).astype(np.float32)
    if dtype == torch.bfloat16:
        top, tail = (torch.tensor(x).to(dtype).float().numpy() for x in (top, tail))
    count = vocab // each if each else 1
    share = 1 / (1 + count / (vocab - count) * np.exp(top - tail))  # how much of the sum is the tail
    order = np.argsort(exponents(top, tail)[form] * share)
    gaps = [s * x for x in (1e-8, 3e-8, 1e-7, 2e-7, 4e-7, 6e-7) for s in (1, -1)]
    pick = [(order[-1 - i % 3], order[i % 4]) for i in range(len(gaps))]
    pick = [p if i % 4 < 2 else p[::-1] for i, p in enumerate(pick)]
    logits = torch.empty(2 * len(gaps), vocab, dtype=dtype, device='cuda')
    scores = torch.zeros(len(gaps), 2, device='cuda')
    sums = []
    for i, pair in enumerate(pick):
        for j, p in enumerate(pair):
            logits[2 * i + j] = float(tail[p])
            logits[2 * i + j, 5::each or vocab] = float(top[p])
            n = len(range(5, vocab, each or vocab))
            sums.append(math.log(n + (vocab - n) * math.exp(float(tail[p]) - float(top[p]))))
        scores[i, 1] = sums[-1] - sums[-2] - gaps[i]
    value = -torch.tensor(sums, dtype=torch.float64).view(-1, 2) + scores.double().cpu()
    first = (value[:, 1] > value[:, 0]).int()
    away = value[:, 0] - value[:, 1]
    rounded = 2.0 ** -24 * scores[:, 1].double().abs().cpu() + 1e-12  # of the second score
    assert ((away - torch.tensor(gaps, dtype=torch.float64)).abs() <= rounded).all() and away.abs().min() > 1e-10
    for items in (1, 3, len(gaps)):
        for i in range(0, len(gaps), items):
            step = BeamSearch(1).select(logits[2 * i:2 * (i + items)], scores[i:i + items].contiguous())
            assert torch.equal(step.parents.cpu()[:, 0], first[i:i + items])
            assert (step.tokens == 5).all()


# ------------------------------------------------------ scores of any size
def spread_scores(items, n, far, seed):
    """Beams most of which are far behind: the first of an item alone, or two of them, as a search starts."""
    s = far - torch.rand(items, n, generator=generator(seed), device='cuda')
    s[:, 0] = -0.5
    if n > 3:
        s[::2, 3] = -1.25
    return s


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('far', [-6.0, -20.0, -100.0, -1e4, -1e9, -1e30])
@pytest.mark.parametrize('items,n,vocab,k', [(1, 50, 152704, 100), (3, 50, 32003, 100), (2, 128, 4000, 256), (2, 128, 32000, 256), (9, 10, 70001, 20), (4, 12, 900, 256),
                                             (2, 4, 152833, 256)])
def test_beams_far_behind(items, n, vocab, k, far, dtype):
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, _ = inputs(items, n, vocab, dtype, 41)
    scores = spread_scores(items, n, far, 42)
    search = BeamSearch(n, candidates=k)
    check_step(search.select(logits, scores), logits, scores, k, n)
    logits.view(items, n, -1)[:] = logits.view(items, n, -1)[:, :1].clone()  # and the same logits for all of them
    check_step(search.select(logits, scores), logits, scores, k, n)
    search.check()


@pytest.mark.parametrize('dtype', TYPES)
def test_a_far_score_above(dtype):
    """A beam far above the others takes all places that it has candidates for."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    for far in (30.0, 1e4, 1e9):
        logits, scores = inputs(2, 8, 20011, dtype, 43)
        scores[:, 5] += far
        check_step(BeamSearch(8).select(logits, scores), logits, scores, 16, 8)


def took(search, logits, scores):
    """Of ten calls."""
    best = math.inf
    for _ in range(5):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        search.select(logits, scores)
        start.record()
        for _ in range(10):
            search.select(logits, scores)
        end.record()
        end.synchronize()
        best = min(best, start.elapsed_time(end))
    return best


@pytest.mark.parametrize('far', [-20.0, -100.0, -1e9])
def test_beams_far_behind_take_no_longer(far):
    """At most six times what beams of a kind take (summing every row again, and finding the best bit by bit, is more than a hundred)."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, near = inputs(1, 50, 152704, torch.float32, 44)
    scores = spread_scores(1, 50, far, 45)
    search = BeamSearch(50)

    assert took(search, logits, scores) <= 6 * took(search, logits, near)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('value', [-1e4, -1e9, -math.inf, 'lowest'])
@pytest.mark.parametrize('items,n,vocab,live', [(1, 50, 152704, 1000), (3, 50, 32003, 5), (9, 12, 70001, 300), (1, 128, 5003, 700)])
def test_rows_of_which_a_mask_leaves_few_groups(items, n, vocab, live, value, dtype):
    """Fewer groups of logits than candidates, whose best are asked for, and more that the mask has made equal."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(items, n, vocab, dtype, 61)
    logits[:, live:] = torch.finfo(dtype).min if value == 'lowest' else value
    search = BeamSearch(n)
    check_step(search.select(logits, scores), shifted(logits), scores, 2 * n, n)
    search.check()


def test_masks_take_no_longer():
    """At most six times what rows that are not masked take."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(1, 50, 152704, torch.float32, 62)
    search = BeamSearch(50)
    plain = took(search, logits, scores)
    for value in (-1e4, -1e9, -math.inf, torch.finfo(torch.float32).min):
        logits[:, 1000:] = value
        assert took(search, logits, scores) <= 6 * plain


def check_range(logits, scores, beams):
    """The order is that of the values rounded to float32 where these are below its range, by beam and token."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    items, k, vocab = scores.shape[0], 2 * beams, logits.shape[1]
    search = BeamSearch(beams)
    step = search.select(logits, scores)
    value = shifted(logits)
    value = value - value.logsumexp(1, keepdim=True) + scores.double().view(-1, 1)
    value = torch.where(value.float() == -math.inf, -math.inf, value)
    value, place = value.view(items, -1).sort(dim=1, descending=True, stable=True)
    assert torch.equal(step.all_parents.long() * vocab + step.all_tokens.long(), place[:, :k])
    assert torch.equal(step.all_scores == -math.inf, value[:, :k] == -math.inf)
    search.check()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('top', [1e30, 1e32, 1e37])
def test_values_below_the_range_of_float32(top, dtype):
    """A candidate whose value is below float32's range counts as minus infinity: it ranks by beam and token with the others."""
    logits = torch.full((4, 9001), torch.finfo(dtype).min, dtype=dtype, device='cuda')
    logits[0, 5000] = top
    logits[0, 5001:5005] = -top
    logits[1, 4000] = top
    logits[2:, 8000] = 0
    check_range(logits, torch.tensor([[-1.0, -2.0], [-1.0, -math.inf]], device='cuda'), 8)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('few', [3, 40])
def test_scores_and_logits_at_the_lowest_value(few, dtype):
    """Beams set aside by float32's lowest value, logits masked by their type's: both together are below the range."""
    logits, scores = inputs(3, 4, 9001, dtype, 51)
    keep = torch.zeros(9001, dtype=torch.bool, device='cuda')
    keep[torch.randperm(9001, generator=generator(few), device='cuda')[:few]] = True
    logits = torch.where(keep, logits, torch.finfo(dtype).min)
    scores[:, 1:] = torch.finfo(torch.float32).min
    scores[2] = torch.finfo(torch.float32).min
    check_range(logits, scores, 8)
    check_range(logits, scores, 128)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('far', [-20.0, -1e9])
@pytest.mark.parametrize('share', [0.5, 0.002])
def test_beams_far_behind_with_lists_of_allowed_tokens(share, far, dtype):
    """Rows that start at no multiple of 16 bytes, captured and replayed with other inputs."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    items, n, vocab = 3, 30, 33001
    room = torch.empty(items * n, vocab + 6, dtype=dtype, device='cuda')
    logits, allowed = room[:, 3:3 + vocab], torch.empty(items * n, vocab, dtype=torch.bool, device='cuda')
    scores = torch.zeros(items, n, device='cuda')
    search = BeamSearch(n, eos=5)

    def fill(seed):
        made, _ = inputs(items, n, vocab, dtype, seed)
        logits.copy_(made)
        allowed.copy_(torch.rand(items * n, vocab, generator=generator(seed), device='cuda') < share)
        scores.copy_(spread_scores(items, n, far, seed))

    fill(71)
    check_step(search.select(logits, scores, allowed=allowed), logits, scores, 2 * n, n, eos=5, allowed=allowed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = search.select(logits, scores, allowed=allowed)
    for seed in (72, 73):
        fill(seed)
        graph.replay()
        check_step(step, logits, scores, 2 * n, n, eos=5, allowed=allowed)
    search.check()

"""Beam selection and the reordering of states against float64 on the GPU.

Tokens, parents and reordered states are compared for equality: the order is that of 64-bit arithmetic, equal
values by beam and token.  A score's tolerance counts its roundings: an exponential is off by 2^-22 and by its argument's rounding (up to 2^-23 of
the argument in units of log2, whose mean under the softmax is at most log2(vocabulary) <= 20), and an fp32 sum goes through
fewer than 64 additions (2^-24 each): lse by at most 2^-22 + 20 * 0.7 * 2^-23 + 64 * 2^-24 = 5.8e-6; the score itself is
rounded once, by half a step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

LSE = 5.8e-6


@pytest.fixture(scope='module', autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.fail('CUDA device required for -m gpu tests')


def generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def plain_select(logits, scores, k, beams, eos=None, allowed=None):
    """tokens, parents, values [items, k] in float64, and the places of the next beams among them."""
    items, n = scores.shape
    value = torch.log_softmax(logits.double(), 1) + scores.double().view(-1, 1)
    if allowed is not None:
        value = torch.where(allowed, value, -math.inf)
    bad = logits.isnan().any(1) | (logits == math.inf).any(1)
    value = torch.where(bad[:, None] | value.isnan(), -math.inf, value).view(items, -1)
    value, place = value.sort(dim=1, descending=True, stable=True)
    value, place = value[:, :k], place[:, :k]
    tokens, parents = place % logits.shape[1], place // logits.shape[1]
    on = [[j for j in range(k) if row[j] != eos][:beams] for row in tokens.tolist()]
    return tokens, parents, value, torch.tensor(on, device=logits.device)


def check_step(step, logits, scores, k, beams, eos=None, allowed=None):
    tokens, parents, value, on = plain_select(logits, scores, k, beams, eos, allowed)
    assert torch.equal(step.all_tokens.long(), tokens)
    assert torch.equal(step.all_parents.long(), parents)
    none = value == -math.inf
    assert torch.equal(step.all_scores == -math.inf, none)
    off = (step.all_scores.double() - value).abs()
    assert (off <= LSE + 2.0 ** -24 * value.abs())[~none].all(), off[~none].max()
    for got, all_ in ((step.tokens, step.all_tokens), (step.parents, step.all_parents), (step.scores, step.all_scores)):
        assert torch.equal(got, all_.gather(1, on))


def inputs(items, n, vocab, dtype, seed, gain=2.5):
    g = generator(seed)
    logits = (gain * torch.randn(items * n, vocab, generator=g, device='cuda')).to(dtype)
    return logits, -4 * torch.rand(items, n, generator=g, device='cuda')


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('items,n,beams,vocab,k,eos', [
    (1, 1, 1, 1000, 1, None), (1, 4, 4, 8192, 8, 17), (3, 50, 50, 32003, 100, 5), (2, 1, 50, 151, 100, None),
    (1, 128, 128, 4096, 256, 0), (5, 10, 5, 1, 10, None), (2, 3, 3, 7, 6, 6), (1, 2, 64, 152704, 128, 152703), (70, 3, 3, 2047, 9, None),
    (1, 1, 128, 2000, 256, None), (2, 60, 5, 513, 65, 44), (1, 50, 50, 152832, 100, None), (1, 1, 3, 1 << 20, 6, None),
    (1, 128, 128, 152704, 256, 7), (1, 1, 128, 152704, 256, None), (3, 1, 50, 152704, 100, 1), (2, 33, 33, 32000, 66, None)])
def test_sizes_and_types(items, n, beams, vocab, k, eos, dtype):
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(items, n, vocab, dtype, items + vocab)
    search = BeamSearch(beams, eos=eos, candidates=k)
    check_step(search.select(logits, scores), logits, scores, k, beams, eos)
    search.check()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('items,n,vocab,share', [(2, 20, 152704, 0.5), (1, 128, 40001, 0.01), (3, 1, 152832, 0.9), (40, 10, 5008, 0.2)])
def test_lists_of_allowed_tokens(items, n, vocab, share, dtype):
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(items, n, vocab, dtype, vocab)
    allowed = torch.rand(items * n, vocab, generator=generator(n), device='cuda') < share
    search = BeamSearch(n, eos=3)
    check_step(search.select(logits, scores, allowed=allowed), logits, scores, 2 * n, n, eos=3, allowed=allowed)
    search.check()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('offset,room', [(0, 0), (1, 2), (3, 5), (5, 1), (7, 9)])
def test_rows_that_start_anywhere(dtype, offset, room):
    """Rows of a wider tensor, at no multiple of 16 bytes: what lies between them is not part of them."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(2, 5, 3001, dtype, 7)
    whole = torch.full((10, 3001 + offset + room), 1e4, dtype=dtype, device='cuda')
    whole[:, offset:offset + 3001] = logits
    g = generator(offset)
    allowed = torch.ones(10, 3001 + offset + room, dtype=torch.bool, device='cuda')
    allowed[:, offset:offset + 3001] = torch.rand(10, 3001, generator=g, device='cuda') < 0.1
    search = BeamSearch(5)
    part, mask = whole[:, offset:offset + 3001], allowed[:, offset:offset + 3001]
    check_step(search.select(part, scores), logits, scores, 10, 5)
    check_step(search.select(part, scores, allowed=mask), logits, scores, 10, 5, allowed=mask)
    check_step(search.select(part, scores, allowed=mask[3]), logits, scores, 10, 5, allowed=mask[3:4])
    check_step(search.select(part, scores, allowed=mask[3:4].expand(10, -1)), logits, scores, 10, 5, allowed=mask[3:4])
    other = part.t().contiguous().t()  # tokens outermost: copied
    check_step(search.select(other, scores), logits, scores, 10, 5)
    same = logits[:1].expand(10, -1)
    check_step(search.select(same, scores), same, scores, 10, 5)
    search.check()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('step', [0.25, 1.0, 4.0, 100.0])
def test_ties(dtype, step):
    """Coarse logits: most candidates at the border are equal, within a beam and, where rows are equal, between beams."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(3, 12, 9001, dtype, 3)
    logits = (logits / step).round() * step
    logits[3] = logits[2]
    scores[0, 3] = scores[0, 2]
    logits[12:24] = logits[12]
    scores[1] = -1.5
    check_step(BeamSearch(12).select(logits, scores), logits, scores, 24, 12)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('value', [0.0, -5.0, 'lowest'])
def test_rows_of_one_value(dtype, value):
    """Every candidate of a beam is equal; beams with scores of their own, and all of one score."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    value = torch.finfo(dtype).min if value == 'lowest' else value
    logits = torch.full((20, 40007), value, dtype=dtype, device='cuda')
    scores = torch.stack([torch.arange(10, device='cuda') * -0.25, torch.zeros(10, device='cuda')])
    step = BeamSearch(10).select(logits, scores)
    if value == torch.finfo(dtype).min:
        # the sum of a row is that of 40,007 ones; the value itself swallows it, as in float64
        check_step(step, logits, scores, 20, 10)
        assert step.all_tokens.tolist() == [list(range(20))] * 2
    else:
        check_step(step, logits, scores, 20, 10)
        assert step.all_parents[0].tolist() == [0] * 20 and step.all_tokens[1].tolist() == list(range(20))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('lowest', [False, True])
def test_masks_that_leave_little(dtype, lowest):
    """Logits masked by minus infinity or by the type's lowest value, lists of allowed tokens, beams that have ended: fewer
    candidates than are asked for, or none."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    none = torch.finfo(dtype).min if lowest else -math.inf
    logits, scores = inputs(4, 6, 5003, dtype, 21)
    keep = torch.zeros_like(logits, dtype=torch.bool)
    keep[:, [5, 700, 5002]] = True
    keep[6:12] = False   # nothing at all
    keep[14] = True      # one beam has everything
    masked = torch.where(keep, logits, none)
    scores[3, 1:] = -math.inf
    search = BeamSearch(6)
    check_step(search.select(masked, scores), masked, scores, 12, 6)
    check_step(search.select(logits, scores, allowed=keep), logits, scores, 12, 6, allowed=keep)
    check_step(search.select(masked, scores, allowed=keep), masked, scores, 12, 6, allowed=keep)
    scores[2] = -math.inf
    step = search.select(logits, scores, allowed=keep)
    check_step(step, logits, scores, 12, 6, allowed=keep)
    assert step.all_tokens[2].tolist() == list(range(12)) and (step.all_scores[2] == -math.inf).all()
    search.check()


def test_values_that_are_not_finite():
    from rapidtinyrec_b200 import _native
    from rapidtinyrec_b200.beam_search import BeamSearch
    for dtype in (torch.float32, torch.bfloat16):
        for place, what in ((3, math.nan), (5000, math.nan), (4444, math.inf)):
            logits, scores = inputs(2, 4, 5001, dtype, 4)
            search = BeamSearch(4)
            logits[5, place] = what
            check_step(search.select(logits, scores), logits, scores, 8, 4)
            with pytest.raises(_native.NativeError, match='left out'):
                search.check()
            scores[1, 1] = -math.inf  # an ended beam is not read
            check_step(search.select(logits, scores), logits, scores, 8, 4)
            search.check()
        logits[5] = math.nan
        scores[1, 1] = -1.0
        check_step(search.select(logits, scores), logits, scores, 8, 4)
        with pytest.raises(_native.NativeError, match='left out'):
            search.check()
        logits, scores = inputs(2, 4, 5001, dtype, 4)
        for bad in (math.nan, math.inf):
            scores[0, 2] = bad
            want = scores.clone()
            want[0, 2] = -math.inf
            check_step(search.select(logits, scores), logits, want, 8, 4)
            with pytest.raises(_native.NativeError, match='left out'):
                search.check()


@pytest.mark.parametrize('vocab', [1500, 60001, 70001])
def test_candidates_too_close_for_32_bits(vocab):
    """Candidates of different beams 1e-9 to 3e-7 apart, both ways, closer than fp32 sums tell: the order is float64's."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    g = generator(vocab)
    n = 6
    logits = 1.3 * torch.randn(n, vocab, generator=g, device='cuda') - 6.0
    at = torch.randperm(vocab, generator=g, device='cuda')[:12]
    best = 0.3 * torch.rand(12, generator=g, device='cuda').double()  # near 0, where floats are fine enough
    apart = (torch.rand(n, 12, generator=g, device='cuda').double() - 0.5) * 6e-7
    scores = (-0.01 * torch.arange(n, device='cuda').float())[None]
    for _ in range(40):  # row i's value of candidate j = best[j] - 12 + apart[i, j]
        lse = torch.logsumexp(logits.double(), 1, keepdim=True)
        logits[:, at] = (best + apart + lse - lse[:1] - scores.double().t()).float()
    tokens, _, value, _ = plain_select(logits, scores, 24, 12)
    gaps = value[0, :-1] - value[0, 1:]
    assert (gaps < 1e-6).sum() >= 15 and (gaps[gaps > 0] > 1e-12).all()
    check_step(BeamSearch(12).select(logits, scores), logits, scores, 24, 12)
    for items in (3, 8, 40, 100):  # of 70,001: one block an item, clusters of four, of two, one again
        more, same = logits.repeat(items, 1), scores.repeat(items, 1)
        if items > 3:
            more[6:12] = 1.3 * torch.randn(n, vocab, generator=g, device='cuda')  # an item without doubts
        check_step(BeamSearch(12).select(more, same), more, same, 24, 12)


@pytest.mark.parametrize('seed', range(4))
@pytest.mark.parametrize('vocab', [5003, 152833, 1 << 20])
def test_candidates_too_close_in_rows_of_few_values(vocab, seed):
    """The same where a row's other logits have one value, so that the roundings of its sum do not cancel."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    g = generator(vocab + seed)
    n = 6
    logits = (-6 - torch.rand(n, 1, generator=g, device='cuda')).expand(n, vocab).clone()
    at = torch.randperm(vocab, generator=g, device='cuda')[:12]
    best = 0.3 * torch.rand(12, generator=g, device='cuda').double()
    apart = (torch.rand(n, 12, generator=g, device='cuda').double() - 0.5) * 6e-7
    scores = (-0.01 * torch.arange(n, device='cuda').float())[None]
    for _ in range(40):
        lse = torch.logsumexp(logits.double(), 1, keepdim=True)
        logits[:, at] = (best + apart + lse - lse[:1] - scores.double().t()).float()
    value = plain_select(logits, scores, 24, 12)[2]
    gaps = value[0, :-1] - value[0, 1:]
    assert (gaps < 1e-6).sum() >= 15 and (gaps[gaps > 0] > 1e-12).all()
    check_step(BeamSearch(12).select(logits, scores), logits, scores, 24, 12)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('items,vocab', [(1, 1500), (2, 60001), (9, 70001)])
def test_rows_that_differ_less_than_32_bits_tell(items, vocab, dtype):
    """Beams with one score whose logits are the same but for a token that adds 3e-10 to 2e-9 to their sums: the smaller sums come
    first, and only two that are the same in all places rank by beam."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(items, 5, vocab, dtype, vocab)
    rows = logits.view(items, 5, vocab)
    rows[:] = rows[:, :1].clone()
    scores[:] = scores[:, :1].clone()
    rows[:, :, 7] = -math.inf
    lse = rows[:, 0].double().logsumexp(1)
    for j, away in enumerate((20, 21, 22, 21, 20.5)):
        rows[:, j, 7] = (lse - away).to(dtype)
    sums = rows.double().logsumexp(2)
    gaps = (sums[:, :, None] - sums[:, None]).abs()
    assert (gaps[gaps > 1e-14] > 1e-10).all() and (gaps < 3e-9).all()
    sums[:, 3] = sums[:, 1]  # rows that are the same, however the library adds them
    value = rows.double() - sums[:, :, None] + scores.double()[:, :, None]
    value, place = value.view(items, -1).sort(dim=1, descending=True, stable=True)
    step = BeamSearch(16).select(logits, scores)
    assert torch.equal(step.all_parents.long() * vocab + step.all_tokens.long(), place[:, :32])
    assert ((step.all_scores.double() - value[:, :32]).abs() <= LSE + 2.0 ** -24 * value[:, :32].abs()).all()


def test_every_call_the_same_and_captured():
    from rapidtinyrec_b200.beam_search import BeamSearch
    logits, scores = inputs(4, 20, 30011, torch.bfloat16, 8)
    search = BeamSearch(20, eos=3)
    first = search.select(logits, scores)
    again = search.select(logits, scores)
    assert all(torch.equal(x, y) for x, y in zip(first, again))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    states = torch.zeros(80, 5, device='cuda')
    with torch.cuda.graph(graph, stream=stream):
        step = search.select(logits, scores)
        search.reorder(states, step.parents)
    for seed in (9, 10):
        new, s = inputs(4, 20, 30011, torch.bfloat16, seed)
        logits.copy_(new)
        scores.copy_(s)
        held = torch.randn(80, 5, generator=generator(seed), device='cuda')
        states.copy_(held)
        graph.replay()
        check_step(step, logits, scores, 40, 20, eos=3)
        assert torch.equal(states, held[(step.parents.long() + 20 * torch.arange(4, device='cuda')[:, None]).view(-1)])
    with torch.cuda.stream(stream):
        other = search.select(logits, scores)
    stream.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(step, other))
    search.check()


def test_rows_and_states_beyond_32_bits():
    """Rows and states more than 2^31 values apart."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    far = (1 << 30) + 7
    room = torch.empty(2 * far + 60000, dtype=torch.bfloat16, device='cuda')
    logits = room.as_strided((3, 50021), (far, 1))
    made, scores = inputs(1, 3, 50021, torch.bfloat16, 5)
    logits.copy_(made)
    check_step(BeamSearch(3).select(logits, scores), made, scores, 6, 3)
    state = room.as_strided((3, 2, 1009), (far, 2048, 1))
    made = values((3, 2, 1009), torch.bfloat16, 6)
    state.copy_(made)
    parents = torch.tensor([[2, 0, 0]], dtype=torch.int32, device='cuda')
    BeamSearch(3).reorder(state, parents)
    assert torch.equal(state, moved(made, parents, 0))


def test_two_calls_at_once():
    """Two streams, each with calls of its own; the handle is one."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    search = BeamSearch(30)
    sets = [inputs(2, 30, 60000 + 5 * i, torch.float32, i) for i in range(2)]
    states = [values((60, 40000), torch.float32, i) for i in range(2)]
    want = [x.clone() for x in states]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    steps = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                steps[i].append(search.select(*sets[i]))
                search.reorder(states[i], steps[i][-1].parents)
    torch.cuda.synchronize()
    for i in range(2):
        for step in steps[i]:
            check_step(step, *sets[i], 60, 30)
            want[i] = moved(want[i], step.parents, 0)
        assert torch.equal(states[i], want[i])
    search.check()


def test_no_items():
    from rapidtinyrec_b200.beam_search import BeamSearch
    search = BeamSearch(3)
    step = search.select(torch.zeros(0, 50, device='cuda'), torch.zeros(0, 4, device='cuda'))
    assert step.tokens.shape == (0, 3) and step.all_scores.shape == (0, 6)
    search.reorder(torch.zeros(0, 4, device='cuda'), torch.zeros(0, 3, dtype=torch.int32, device='cuda'))
    search.reorder([], torch.zeros(2, 3, dtype=torch.int32, device='cuda'))
    search.check()


# ----------------------------------------------------------------- reordering
def moved(state, parents, dim):
    items, beams = parents.shape
    rows = (parents.long() + beams * torch.arange(items, device=parents.device)[:, None]).view(-1)
    return state.index_select(dim, rows)


def some_parents(items, beams, seed):
    g = generator(seed)
    p = torch.randint(0, beams, (items, beams), generator=g, device='cuda', dtype=torch.int32)
    p[0] = p[0].sort().values
    return p


def values(shape, dtype, seed):
    x = torch.randint(-100, 100, shape, generator=generator(seed), device='cuda')
    return x.to(torch.uint8).to(dtype) if dtype == torch.uint8 else (x > 0) if dtype == torch.bool else x.to(dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.int64, torch.uint8, torch.bool])
@pytest.mark.parametrize('items,beams,shape,dim', [
    (1, 50, (50, 2, 4, 128), 0), (8, 4, (2, 32, 3, 40), 1), (3, 1, (3, 7), 0), (2, 128, (256, 65), 0), (1, 5, (5,), 0), (5, 7, (6, 3, 35), 2),
    (1, 2, (3, 2, 100001), 1), (70, 3, (210, 16), 0), (1, 64, (2, 2, 64, 1, 1), -3)])
def test_reordering(items, beams, shape, dim, dtype):
    from rapidtinyrec_b200.beam_search import BeamSearch
    search = BeamSearch(beams)
    for seed in range(2):
        state, parents = values(shape, dtype, seed), some_parents(items, beams, seed + 5)
        want = moved(state, parents, dim)
        search.reorder(state, parents, dim=dim)
        assert torch.equal(state, want)
    same = torch.arange(beams, dtype=torch.int32, device='cuda').repeat(items, 1)
    search.reorder(state, same, dim=dim)
    assert torch.equal(state, want)
    search.reorder(state, torch.full_like(same, beams - 1), dim=dim)
    assert torch.equal(state, moved(want, torch.full_like(same, beams - 1), dim))
    search.check()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.uint8])
@pytest.mark.parametrize('tokens', [0, 1, 5, 11])
def test_part_of_the_tokens_of_many_states(dtype, tokens):
    """More states than one launch takes, of several sizes and places in memory; entries behind the tokens stay."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    search = BeamSearch(6)
    parents = some_parents(3, 6, 2)
    states = [values((2, 18, 2, 11, 1 + i % 9 * 8), dtype, i) for i in range(37)]
    states += [values((2, 18, 2, 11, 70), dtype, 50)[..., 3:65], values((2, 18, 2, 11, 64), dtype, 51).transpose(2, 4)[:, :, :, :, :1].transpose(2, 4)]
    want = [s.clone() for s in states]
    for w in want:
        w[:, :, :, :tokens] = moved(w, parents, 1)[:, :, :, :tokens]
    search.reorder(tuple(states), parents, dim=1, token_dim=-2, tokens=tokens)
    assert all(torch.equal(s, w) for s, w in zip(states, want))
    search.check()


def test_parents_that_are_none_of_the_beams():
    from rapidtinyrec_b200 import _native
    from rapidtinyrec_b200.beam_search import BeamSearch
    search = BeamSearch(4)
    state = torch.arange(8, device='cuda').view(8, 1).repeat(1, 9)
    search.reorder(state, torch.tensor([[3, -1, 4, 0], [1, 0, 1 << 30, 3]], dtype=torch.int32, device='cuda'))
    assert state[:, 0].tolist() == [3, 1, 2, 0, 5, 4, 6, 7]
    with pytest.raises(_native.NativeError, match='none of the beams'):
        search.check()
    search.check()


def test_refusals():
    from rapidtinyrec_b200.beam_search import BeamSearch
    search = BeamSearch(4, eos=2)
    logits, scores = inputs(2, 4, 50, torch.float32, 1)
    for args, kw, says in [
            ((logits.cpu(), scores), {}, 'logits'), ((logits.half(), scores), {}, 'logits'), ((logits[:7], scores), {}, 'row for each'),
            ((logits.view(2, 4, 50), scores), {}, 'logits'), ((logits, scores.double()), {}, 'scores'), ((logits, scores.view(-1)), {}, 'scores'),
            ((logits, scores.cpu()), {}, 'scores'), ((logits, scores.t().contiguous().t()), {}, 'scores'),
            ((logits, scores.view(1, 8)), {}, 'at least 12 candidates'), ((logits[:2, :3], scores[:, :1].contiguous()), {}, 'candidates of 3'),
            ((logits, scores), {'allowed': (logits > 0).byte()}, 'allowed'),
            ((logits, scores), {'allowed': (logits > 0)[:, :49]}, 'allowed'), ((logits, scores), {'allowed': (logits > 0)[:3]}, 'allowed'),
            ((logits, scores), {'allowed': (logits > 0).cpu()}, 'allowed'), ((3, scores), {}, 'logits must be a tensor')]:
        with pytest.raises(ValueError, match=says):
            search.select(*args, **kw)
    state, parents = torch.zeros(8, 3, 10, device='cuda'), torch.zeros(2, 4, dtype=torch.int32, device='cuda')
    for args, kw, says in [
            ((state, parents.long()), {}, 'parents'), ((state, parents.view(4, 2)), {}, 'parents'), ((state, parents.cpu()), {}, 'parents'),
            ((state[:7], parents), {}, 'rows'), ((state, parents), {'dim': 1}, 'rows'), ((state, parents), {'dim': 3}, 'rows'),
            ((state.cpu(), parents), {}, 'rows'), (([state, state], parents), {}, 'twice'), (([state, 'x'], parents), {}, 'tensor'),
            (('x', parents), {}, 'states'), ((state[:1].expand(8, 3, 10), parents), {}, 'overlap'),
            ((torch.zeros(40, device='cuda').as_strided((8, 3), (2, 1)), parents), {}, 'overlap'),
            ((state, parents), {'token_dim': 1}, 'belong together'), ((state, parents), {'token_dim': 0, 'tokens': 1}, 'another dimension'),
            ((state, parents), {'token_dim': 2, 'tokens': 11}, 'holds 10'), ((state, parents), {'token_dim': 2, 'tokens': -1}, 'holds 10'),
            ((state.clone().requires_grad_(), parents), {}, 'gradient'),
            ((torch.zeros(8, 3, 3, 3, 3, 8, device='cuda')[:, ::2, :2, :2, :2, :5], parents), {}, 'three strided')]:
        with pytest.raises(ValueError, match=says):
            search.reorder(*args, **kw)
    assert not state.any()


# -------------------------------------------------------------- all of them
def test_a_search_over_a_paged_cache():
    """Four steps of a small model's beam search, as a program of its own runs it: pages and positions for the prompts, rotary
    positions, the 8-bit cache for the prompts and rows of the beams' own for their tokens, selection, reordering; against the same
    search in float64 over the values that the cache holds."""
    from rapidtinyrec_b200.beam_search import BeamSearch
    from rapidtinyrec_b200.kv_cache import KvCache8
    from rapidtinyrec_b200.page_pool import PagePool
    from rapidtinyrec_b200.rotary import Rotary
    g = generator(77)
    items, beams, steps, heads, kv, dim, vocab, eos = 2, 5, 4, 4, 2, 64, 700, 9
    lens = [37, 70]
    width = heads * dim
    emb = torch.randn(vocab, width, generator=g, device='cuda')
    wqkv = torch.randn(width, (heads + 2 * kv) * dim, generator=g, device='cuda') / 16
    wo = torch.randn(width, width, generator=g, device='cuda') / 16
    head = torch.randn(width, vocab, generator=g, device='cuda') / 5
    prompt = torch.randint(0, vocab, (sum(lens),), generator=g, device='cuda')
    rotary = Rotary(dim, theta=1e4)
    search = BeamSearch(beams, eos=eos)
    cache, pool = KvCache8.allocate(20, kv, 16, dim), PagePool(20, 16)

    # the prompts: their keys and values into the cache
    table = torch.zeros(items, 8, dtype=torch.int32, device='cuda')
    zeros = torch.zeros(items, dtype=torch.int32, device='cuda')
    got = pool.grow(table, zeros, torch.tensor(lens, dtype=torch.int32, device='cuda'), rows=sum(lens))
    qkv = (emb[prompt] @ wqkv).view(-1, heads + 2 * kv, dim)
    q, k, v = qkv.split([heads, kv, kv], 1)
    q, k = rotary.rotate(q, k, got.positions)
    cache.write(k, v, table, got.lens, starts=got.starts)
    out = cache.attention(q, table, got.lens, starts=got.starts)
    last = got.starts[1:].long() - 1
    hidden = emb[prompt][last] + out[last].reshape(items, width) @ wo
    step = search.select(hidden @ head, torch.zeros(items, 1, device='cuda'))
    own = torch.zeros(2, items * beams, steps, kv, dim, device='cuda')  # K and V of the beams' own tokens
    history = torch.zeros(items * beams, steps, dtype=torch.int32, device='cuda')
    paths = []
    for t in range(steps):
        history[:, t] = step.tokens.view(-1)
        paths.append(step)
        if t == steps - 1:
            break
        x = emb[step.tokens.view(-1).long()]
        q, k, v = (x @ wqkv).view(-1, heads + 2 * kv, dim).split([heads, kv, kv], 1)
        at = (got.lens + t).repeat_interleave(beams)
        q, k = rotary.rotate(q, k, at)
        own[0, :, t], own[1, :, t] = k, v
        out, lse = cache.attention(q, table, got.lens, causal=False, return_lse=True)
        s = torch.einsum('bgjd,btgd->bgjt', q.view(-1, kv, heads // kv, dim), own[0, :, :t + 1]) / 8
        lse2 = torch.logsumexp(s, -1)
        out2 = torch.einsum('bgjt,btgd->bgjd', torch.softmax(s, -1), own[1, :, :t + 1]).reshape(-1, heads, dim)
        share = torch.sigmoid(lse2.reshape(-1, heads) - lse)[..., None]
        out = out * (1 - share) + out2 * share
        hidden = x + out.reshape(-1, width) @ wo
        step = search.select(hidden @ head, step.scores)
        search.reorder(own, step.parents, dim=1, token_dim=2, tokens=t + 1)
        search.reorder(history, step.parents, token_dim=1, tokens=t + 1)
    for x in (cache, pool, search):
        x.check()

    # the same in float64
    d = torch.float64
    emb, wqkv, wo, head = (x.double() for x in (emb, wqkv, wo, head))
    f = torch.tensor(rotary.frequencies, dtype=d, device='cuda')

    def turn(x, positions):
        c, s = torch.cos(positions[:, None, None] * f), torch.sin(positions[:, None, None] * f)
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    kept = [x.double() for x in cache.read(sum(lens), table, got.lens, starts=got.starts)]
    worst = 0.0
    for b in range(items):
        lo, hi = sum(lens[:b]), sum(lens[:b + 1])
        pk, pv = kept[0][lo:hi], kept[1][lo:hi]

        def attend(q, keys, vals):  # [heads, dim] over [tokens, kv, dim]
            s = torch.einsum('gjd,tgd->gjt', q.view(kv, -1, dim), keys) / 8
            return torch.einsum('gjt,tgd->gjd', torch.softmax(s, -1), vals).reshape(width)

        def logits_of(token, position, keys, vals, mine):
            x = emb[token]
            q, k, v = (x @ wqkv).view(heads + 2 * kv, dim).split([heads, kv, kv])
            p = torch.tensor([float(position)], dtype=d, device='cuda')
            q, k = turn(q[None], p)[0], turn(k[None], p)[0]
            if mine:
                keys, vals = torch.cat([keys, k[None]]), torch.cat([vals, v[None]])
            return (x + attend(q, keys, vals) @ wo) @ head, keys, vals

        start, _, _ = logits_of(prompt[hi - 1], lens[b] - 1, pk, pv, False)
        running = [([], 0.0, pk, pv, start)]
        for t in range(steps):
            ways = []
            for i, (path, score, keys, vals, logits) in enumerate(running):
                value = torch.log_softmax(logits, 0) + score
                top = value.topk(2 * beams)
                ways += [(float(x), i, int(tok)) for x, tok in zip(top.values, top.indices)]
            ways.sort(key=lambda w: -w[0])
            ways = ways[:2 * beams + 1]
            # the fp32 model's logits differ from these by some 1e-5: far less than the candidates are apart
            assert min(x[0] - y[0] for x, y in zip(ways, ways[1:])) > 2e-4
            next_ = [w for w in ways[:2 * beams] if w[2] != eos][:beams]
            assert paths[t].tokens[b].tolist() == [w[2] for w in next_]
            assert paths[t].parents[b].tolist() == [w[1] for w in next_]
            worst = max(worst, max(abs(s - w[0]) for s, w in zip(paths[t].scores[b].tolist(), next_)))
            new = []
            for score, i, token in next_:
                path, _, keys, vals, _ = running[i]
                new.append((path + [token], score) + logits_of(token, lens[b] + t, keys, vals, True)[1:] +
                           (logits_of(token, lens[b] + t, keys, vals, True)[0],))
            running = new
        assert history[b * beams:(b + 1) * beams].tolist() == [r[0] for r in running]
    assert worst < 2e-4

"""Page pool, rotary positions and beam search without a GPU: what their C entry points and Python layers refuse before
anything is enqueued, and the arithmetic that the host does for the kernels."""
import ctypes
import math

import pytest
import torch

from rapidtinyrec_b200 import _native
from rapidtinyrec_b200.beam_search import BeamSearch
from rapidtinyrec_b200.page_pool import PagePool
from rapidtinyrec_b200.rotary import Rotary, frequencies

A = 1 << 20  # an address that is never followed: every refusal comes before device work


def message():
    return _native.load().rtr_last_error(None).decode()


# ------------------------------------------------------------------ page pool
def pool(**change):
    args = dict(free=A, count=A, marks=A, status=A, ticket=A, pages=9, page=16)
    args.update(change)
    return _native.PagePoolC(**args)


def grow(p, table=A, stride=8, width=8, held=A, fresh=A, each=0, seqs=2, rows=6, lens=A, starts=A, positions=A, slots=A):
    return _native.load().rtr_pages_grow(ctypes.byref(p), table, stride, width, held, fresh, each, seqs, rows, lens, starts,
                                         positions, slots, 0, None)


def release(p, table=A, stride=8, width=8, held=A, keep=A, seqs=2):
    return _native.load().rtr_pages_release(ctypes.byref(p), table, stride, width, held, keep, seqs, 0, None)


@pytest.mark.parametrize('change,says', [
    (dict(free=None), 'null pool'), (dict(count=None), 'null pool'), (dict(marks=None), 'null pool'), (dict(status=None), 'null pool'),
    (dict(ticket=None), 'null pool'), (dict(pages=0), 'pages'), (dict(page=0), 'power of two'), (dict(page=48), 'power of two'),
    (dict(page=2048), 'power of two')])
def test_pools_that_are_refused(change, says):
    for call in (grow, release):
        assert call(pool(**change)) == _native.RTR_ERR_ARG
        assert says in message()


@pytest.mark.parametrize('change,says', [
    (dict(table=None), 'null table'), (dict(held=None), 'null table'), (dict(seqs=-1), 'sequences'), (dict(seqs=16385), 'sequences'),
    (dict(width=0), 'table rows'), (dict(stride=7), 'table rows'), (dict(width=1 << 27, stride=1 << 27), '2^31')])
def test_page_tables_that_are_refused(change, says):
    for call in (grow, release):
        assert call(pool(), **change) == _native.RTR_ERR_ARG
        assert says in message()


@pytest.mark.parametrize('change,says', [
    (dict(rows=-1), 'negative'), (dict(each=-1), 'negative'), (dict(lens=None), 'null output'), (dict(starts=None), 'null output'),
    (dict(positions=None), 'null output'), (dict(slots=None), 'null output'), (dict(positions=A + 4), '16 bytes'),
    (dict(slots=A + 8), '16 bytes')])
def test_outputs_of_grow_that_are_refused(change, says):
    assert grow(pool(), **change) == _native.RTR_ERR_ARG
    assert says in message()


def test_releasing_no_sequence_is_no_work():
    assert release(pool(), table=None, held=None, seqs=0) == _native.RTR_OK


def test_pools_without_a_gpu_are_refused():
    for args, kw in [((9, 16), {'device': 'cpu'}), ((9, 16), {'free': torch.arange(9)}), ((0, 16), {}), ((9, 48), {})]:
        with pytest.raises(ValueError):
            PagePool(*args, **kw)


# --------------------------------------------------------------------- rotary
def rows(**change):
    args = dict(in_=A, out=A, in_row=512, in_head=128, out_row=512, out_head=128, heads=4)
    args.update(change)
    return _native.RotaryRowsC(**args)


def rotate(q, k=None, n=6, dim=128, part=128, dtype=0, positions=A, turns=A):
    return _native.load().rtr_rotary(None if q is None else ctypes.byref(q), None if k is None else ctypes.byref(k), n, dim, part, 0,
                                     dtype, positions, 0, turns, 1.0, 0, 0, None)


@pytest.mark.parametrize('change,says', [
    (dict(in_=None), 'null rows'), (dict(out=None), 'null rows'), (dict(heads=0), 'heads'), (dict(out=A + (1 << 20), out_head=64), 'overlap'),
    (dict(out=A + (1 << 20), out_row=64), 'overlap'), (dict(out_row=1024), 'one set'), (dict(in_head=256), 'one set')])
def test_rotary_rows_that_are_refused(change, says):
    for args in ((rows(**change),), (rows(), rows(**change))):
        assert rotate(*args) == _native.RTR_ERR_ARG
        assert says in message()


@pytest.mark.parametrize('change,says', [
    (dict(q=None), 'null rows'), (dict(dim=1, part=2), 'head_dim'), (dict(dim=514), 'head_dim'), (dict(part=0), 'rotary_dim'),
    (dict(part=7), 'rotary_dim'), (dict(part=130), 'rotary_dim'), (dict(dtype=2), 'dtype'), (dict(n=-1), 'negative'),
    (dict(positions=None), 'null positions'), (dict(turns=None), 'null positions')])
def test_rotary_calls_that_are_refused(change, says):
    args = dict(q=rows())
    args.update(change)
    assert rotate(**args) == _native.RTR_ERR_ARG
    assert says in message()


def test_no_rows_to_rotate():
    assert rotate(rows(in_=None, out=None), n=0, positions=None) == _native.RTR_OK


def test_frequencies():
    plain = frequencies(8, theta=1e4)
    assert plain == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    assert frequencies(8, theta=1e4, scaling='linear', factor=4.0) == pytest.approx([x / 4 for x in plain], rel=1e-14)
    ntk = frequencies(8, theta=1e4, scaling='ntk', factor=4.0)
    assert ntk[0] == 1.0 and ntk[3] == pytest.approx(plain[3] / 4, rel=1e-14)
    # turns over 1000 positions: 159, 15.9, 1.59, 0.159; from 1 on a share of (turns - 1) / 9 stays
    bands = frequencies(8, theta=1e4, scaling='bands', factor=4.0, length=1000, low=1.0, high=10.0)
    share = (10 / (2 * math.pi) - 1) / 9
    assert bands == pytest.approx([1.0, 0.1, 0.01 * (share + (1 - share) / 4), 0.001 / 4], rel=1e-14)


@pytest.mark.parametrize('kw', [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling='other'), dict(rotary_dim=8, theta=0.0),
                                dict(rotary_dim=8, factor=-1.0), dict(rotary_dim=2, scaling='ntk'), dict(rotary_dim=8, scaling='bands'),
                                dict(rotary_dim=8, scaling='bands', length=100, low=4.0, high=4.0)])
def test_frequencies_that_are_refused(kw):
    with pytest.raises(ValueError):
        frequencies(**kw)


@pytest.mark.parametrize('kw', [dict(head_dim=1), dict(head_dim=1024), dict(head_dim=64, rotary_dim=65), dict(head_dim=64, rotary_dim=33),
                                dict(head_dim=64, device='cpu'), dict(head_dim=4, given=[1.0]), dict(head_dim=4, given=[1.0, math.inf]),
                                dict(head_dim=64, amplitude=math.nan)])
def test_rotary_handles_that_are_refused(kw):
    with pytest.raises(ValueError):
        Rotary(**kw)


# ---------------------------------------------------------------- beam search
def step(**change):
    args = dict(logits=A, scores=A, allowed=None, logits_stride=1000, allowed_stride=0, dtype=0, items=2, n=4, vocab=1000, k=8, beams=4,
                eos=-1, all_tokens=A, all_parents=A, next_tokens=A, next_parents=A, all_scores=A, next_scores=A, status=A)
    args.update(change)
    return _native.BeamStepC(**args)


@pytest.mark.parametrize('change,says', [
    (dict(dtype=2), 'dtype'), (dict(items=-1), '1 to 128'), (dict(n=0), '1 to 128'), (dict(n=129), '1 to 128'), (dict(vocab=0), 'vocabulary'),
    (dict(vocab=(1 << 20) + 1), 'vocabulary'), (dict(k=0), '1 to 256'), (dict(k=257), '1 to 256'), (dict(n=1, vocab=7, k=8), 'there are'),
    (dict(beams=0), 'next beams'), (dict(beams=9), 'next beams'), (dict(eos=3, k=7), 'eos'), (dict(eos=3, beams=5), 'eos'),
    (dict(logits_stride=999), 'logits overlap'), (dict(allowed=A, allowed_stride=999), 'allowed overlap'), (dict(logits=A + 2), 'multiples'),
    (dict(dtype=1, logits=A + 1), 'multiples')] + [(dict([(name, None)]), 'null buffer') for name in (
        'logits', 'scores', 'all_tokens', 'all_parents', 'all_scores', 'next_tokens', 'next_parents', 'next_scores', 'status')])
def test_steps_that_are_refused(change, says):
    lib, room = _native.load(), ctypes.c_int64()
    s = step(**change)
    assert lib.rtr_beam_select_workspace(ctypes.byref(s), 0, ctypes.byref(room)) == _native.RTR_ERR_ARG
    assert says in message()
    assert lib.rtr_beam_select(ctypes.byref(s), A, 1 << 30, 0, None) == _native.RTR_ERR_ARG
    assert says in message()


def test_steps_without_items_are_no_work():
    s = step(items=0, logits=None, scores=None)
    assert _native.load().rtr_beam_select(ctypes.byref(s), None, 0, 0, None) == _native.RTR_OK


def state(**change):
    args = dict(data=A, row_bytes=4096, inner=256, strides=(ctypes.c_int64 * 3)(0, 0, 256), sizes=(ctypes.c_int32 * 3)(1, 1, 2))
    args.update(change)
    return _native.BeamStateC(**args)


def reorder(states, parents=A, items=2, beams=4, status=A):
    many = (_native.BeamStateC * max(1, len(states)))(*states)
    return _native.load().rtr_beam_reorder(many, len(states), parents, items, beams, status, 0, None)


@pytest.mark.parametrize('change,says', [
    (dict(data=None), 'null state'), (dict(inner=0), 'positive'), (dict(sizes=(ctypes.c_int32 * 3)(1, 0, 2)), 'positive'),
    (dict(row_bytes=0), 'rows of a state'), (dict(strides=(ctypes.c_int64 * 3)(0, 0, 0)), 'dimensions overlap'),
    (dict(inner=(1 << 31) + 1), 'too long'), (dict(inner=17, sizes=(ctypes.c_int32 * 3)(1 << 30, 1 << 30, 2), strides=(ctypes.c_int64 * 3)(1, 1, 1)), 'too long')])
def test_states_that_are_refused(change, says):
    assert reorder([state(), state(**change)]) == _native.RTR_ERR_ARG
    assert says in message()


@pytest.mark.parametrize('kw,says', [(dict(beams=0), '128 beams'), (dict(beams=129), '128 beams'), (dict(items=-1), 'items'),
                                     (dict(items=65536), '65535'), (dict(parents=None), 'null'), (dict(status=None), 'null')])
def test_reorderings_that_are_refused(kw, says):
    assert reorder([state()], **kw) == _native.RTR_ERR_ARG
    assert says in message()


def test_nothing_to_reorder():
    assert reorder([]) == _native.RTR_OK and reorder([state()], items=0) == _native.RTR_OK


@pytest.mark.parametrize('kw', [dict(beams=0), dict(beams=129), dict(beams=4, candidates=3), dict(beams=4, candidates=257), dict(beams=4, eos=-1),
                                dict(beams=4, device='cpu')])
def test_searches_that_are_refused(kw):
    with pytest.raises(ValueError):
        BeamSearch(**kw)

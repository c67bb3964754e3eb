"""Beam selection at logits of any size against float64 on the GPU: what masks by -1e10 and the like leave."""
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

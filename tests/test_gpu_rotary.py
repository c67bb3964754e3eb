"""Rotary positions against the formula in float64.

Tolerance, per pair (a, b) of amplitude m: the angle as a float of half turns is off by at most 2^-25 of a half
turn (1e-7 radians), sine and cosine by a last place of values up to 1 (2^-24) and their product with
the amplitude by 2^-24 more: 2.2e-7 together.  The two products of an output round twice
(2 * 2^-24 of their sizes).  So (|a| + |b|) m * 3.5e-7, plus half a step of the output's type, plus, far out, what the float64 angle of
the formula itself is off by: position * frequency * 2^-52.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module', autouse=True)
def cuda():
    if not torch.cuda.is_available():
        pytest.fail('CUDA device required for -m gpu tests')


def plain(x, positions, frequencies, part, interleaved, amplitude=1.0, back=False):
    """The rotated rows in float64, and the tolerance of each value."""
    dt, x = x.dtype, x.double()
    angle = positions.double()[:, None, None] * torch.tensor(frequencies, dtype=torch.float64, device=x.device)
    far = angle.abs() * 2.0 ** -52
    cos, sin = torch.cos(angle) * amplitude, torch.sin(angle) * (-amplitude if back else amplitude)
    i = torch.arange(part // 2, device=x.device)
    at = (2 * i, 2 * i + 1) if interleaved else (i, i + part // 2)
    a, b = x[..., at[0]], x[..., at[1]]
    out, tol = x.clone(), torch.zeros_like(x)
    out[..., at[0]], out[..., at[1]] = a * cos - b * sin, b * cos + a * sin
    size = (a.abs() + b.abs()) * abs(amplitude)
    tol[..., at[0]] = tol[..., at[1]] = size * (3.5e-7 + far)
    tol[..., :part] += torch.finfo(dt).eps / 2 * out[..., :part].abs()
    return out, tol


def check_rows(got, want):
    out, tol = want
    off = (got.double() - out).abs()
    assert (off <= tol).all(), (off - tol).max()


def rows_of(rows, heads, dim, dtype, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return torch.randn(rows, heads, dim, generator=g, device='cuda').to(dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('rows,heads,kv,dim,part', [(1, 12, 2, 128, 128), (7, 1, 1, 64, 32), (50, 28, 4, 128, 96), (3, 5, 0, 64, 64),
                                                    (33, 3, 1, 36, 20), (2, 2, 1, 65, 2), (5, 40, 8, 512, 512), (1025, 8, 8, 64, 16),
                                                    (9, 300, 1, 2, 2)])
def test_layouts_types_and_sizes(rows, heads, kv, dim, part, dtype, interleaved):
    from rapidtinyrec_b200.rotary import Rotary
    q = rows_of(rows, heads, dim, dtype, 1)
    k = rows_of(rows, kv, dim, dtype, 2) if kv else None
    positions = torch.randint(0, 5000, (rows,), device='cuda', dtype=torch.int32)
    rotary = Rotary(dim, rotary_dim=part, theta=1e4, interleaved=interleaved)
    kept = q.clone()
    for back in (False, True):
        got = rotary.rotate(q, k, positions, back=back)
        for x, y in zip((q, k), got if kv else (got,)):
            check_rows(y, plain(x, positions, rotary.frequencies, part, interleaved, back=back))
            assert torch.equal(y[..., part:], x[..., part:])
    assert torch.equal(q, kept)
    if kv:  # in place
        out = q.clone(), k.clone()
        again = rotary.rotate(*out, positions, out=out, back=True)
        assert again[0].data_ptr() == out[0].data_ptr() and again[1].data_ptr() == out[1].data_ptr()
        assert torch.equal(out[0], got[0]) and torch.equal(out[1], got[1])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('offset', [0, 1, 3])
def test_strides(dtype, interleaved, offset):
    """Rows of a fused projection, heads outermost, and rows that start at no multiple of 16 bytes: what lies
    between them stays."""
    from rapidtinyrec_b200.rotary import Rotary
    rotary = Rotary(64, rotary_dim=48, interleaved=interleaved)
    positions = torch.arange(40, 51, device='cuda')  # int64
    fused = rows_of(11, 9, 64, dtype, 4).reshape(-1)
    fused = torch.cat([fused, fused[:8]])[offset:offset + 11 * 9 * 64].view(11, 9, 64)
    q, k = fused[:, 1:6], fused[:, 6:8]
    want = [plain(x, positions, rotary.frequencies, 48, interleaved) for x in (q, k)]
    got = rotary.rotate(q, k, positions)
    kept = fused.clone()
    rotary.rotate(q, k, positions, out=(q, k))
    for x, y, w in zip((q, k), got, want):
        assert y.is_contiguous()
        check_rows(y, w)
        assert torch.equal(x, y)
    assert torch.equal(fused[:, :1], kept[:, :1]) and torch.equal(fused[:, 8:], kept[:, 8:])
    outer = kept[:, 1:6].transpose(0, 1).contiguous().transpose(0, 1)  # [heads][rows][dim] in memory
    room = torch.full((2, 11, 70), 7.0, dtype=dtype, device='cuda')
    out = torch.empty_like(outer), room[:, :, 3:67].transpose(0, 1)
    rotary.rotate(outer, kept[:, 6:8], positions, out=out)
    for y, w in zip(out, want):
        check_rows(y, w)
    assert (room[:, :, :3] == 7).all() and (room[:, :, 67:] == 7).all()
    apart = kept[:, 1:6].transpose(1, 2).contiguous().transpose(1, 2)  # dimensions that are not contiguous: copied
    check_rows(rotary.rotate(apart, None, positions), want[0])
    wide = kept[:, :8].clone()  # q into the place of k's neighbours: between the rows of the input
    rotary.rotate(wide[:, :2], None, positions, out=wide[:, 4:6])
    check_rows(wide[:, 4:6], plain(kept[:, :2], positions, rotary.frequencies, 48, interleaved))
    assert torch.equal(wide[:, :4], kept[:, :4]) and torch.equal(wide[:, 6:], kept[:, 6:8])


@pytest.mark.parametrize('scaling,kw', [('linear', {'factor': 4.0}), ('ntk', {'factor': 8.0}),
                                        ('bands', {'factor': 8.0, 'length': 8192, 'low': 1.0, 'high': 4.0}),
                                        ('bands', {'factor': 4.0, 'length': 4096, 'low': 1.0, 'high': 32.0, 'amplitude': 1.1386}),
                                        (None, {'given': [0.5 ** i for i in range(32)], 'amplitude': -2.0})])
def test_scalings_at_far_positions(scaling, kw):
    from rapidtinyrec_b200.rotary import Rotary
    rotary = Rotary(64, scaling=scaling, **kw)
    q = rows_of(12, 2, 64, torch.float32, 6)
    positions = torch.tensor([0, 1, 2, 8191, 8192, 130000, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -1, -130001, -(1 << 31)],
                             dtype=torch.int32, device='cuda')
    for p in (positions, positions.long()):
        got = rotary.rotate(q, None, p)
        check_rows(got, plain(q, positions, rotary.frequencies, 64, False, kw.get('amplitude', 1.0)))
    assert torch.equal(got[0], q[0] * torch.tensor(kw.get('amplitude', 1.0), device='cuda'))


def test_positions_beyond_32_bits():
    """Whole turns drop out: a frequency of 2^-20 turns a position at n 2^20 + m stands where it stands at m."""
    from rapidtinyrec_b200.rotary import Rotary
    rotary = Rotary(2, given=[2 * math.pi / (1 << 20)])
    q = rows_of(64, 3, 2, torch.float32, 8)
    m = torch.randint(0, 1 << 20, (64,), device='cuda')
    near = rotary.rotate(q, None, m)
    far = rotary.rotate(q, None, m + (torch.randint(0, 1 << 30, (64,), device='cuda') << 20))
    assert torch.equal(near, far)


def test_gradient_of_rotated_rows():
    """back=True is the transpose: against autograd through the formula, and against differences (the rotation is linear, so
    a difference of any width is the derivative)."""
    from rapidtinyrec_b200.rotary import Rotary
    for interleaved in (False, True):
        rotary = Rotary(64, rotary_dim=32, interleaved=interleaved, amplitude=0.75)
        x, up = rows_of(5, 3, 64, torch.float32, 9), rows_of(5, 3, 64, torch.float32, 10)
        positions = torch.tensor([0, 3, 70, 999, 131071], dtype=torch.int32, device='cuda')
        leaf = x.double().requires_grad_()
        i = torch.arange(16, device='cuda')
        at = (2 * i, 2 * i + 1) if interleaved else (i, i + 16)
        angle = positions.double()[:, None, None] * torch.tensor(rotary.frequencies, dtype=torch.float64, device='cuda')
        cos, sin = 0.75 * torch.cos(angle), 0.75 * torch.sin(angle)
        a, b = leaf[..., at[0]], leaf[..., at[1]]
        value = ((a * cos - b * sin) * up[..., at[0]] + (b * cos + a * sin) * up[..., at[1]]).sum() + (leaf * up)[..., 32:].sum()
        value.backward()
        got = rotary.rotate(up, None, positions, back=True)
        _, tol = plain(up, positions, rotary.frequencies, 32, interleaved, 0.75, back=True)
        assert ((got.double() - leaf.grad).abs() <= tol).all()
        step = rows_of(5, 3, 64, torch.float32, 11)
        moved = rotary.rotate(x + step, None, positions).double() - rotary.rotate(x, None, positions).double()
        slope = (got.double() * ((x + step).double() - x.double())).sum((1, 2))
        # each value of `moved` is off by the tolerance of its two rows, `got` by its own: summed over a row
        _, t1 = plain(x + step, positions, rotary.frequencies, 32, interleaved, 0.75)
        _, t0 = plain(x, positions, rotary.frequencies, 32, interleaved, 0.75)
        room = ((t1 + t0) * up.double().abs() + tol * ((x + step).double() - x.double()).abs()).sum((1, 2))
        assert (((moved * up.double()).sum((1, 2)) - slope).abs() <= room).all()


def test_turning_back_and_forth():
    from rapidtinyrec_b200.rotary import Rotary
    rotary = Rotary(128, theta=1e6)
    q = rows_of(20, 4, 128, torch.float32, 12)
    positions = torch.arange(1000, 1020, dtype=torch.int32, device='cuda')
    back = rotary.rotate(rotary.rotate(q, None, positions), None, positions, back=True)
    pair = q.abs() + q.abs().roll(64, -1)
    assert ((back - q).abs() <= 8e-7 * pair).all()  # twice the tolerance above: the first one's goes through the second rotation


def test_nothing_to_do_and_values_that_are_not_finite():
    from rapidtinyrec_b200.rotary import Rotary
    rotary = Rotary(64)
    q = rows_of(3, 2, 64, torch.bfloat16, 13)
    empty = rotary.rotate(q[:0], q[:0], torch.zeros(0, dtype=torch.int32, device='cuda'))
    assert empty[0].shape == (0, 2, 64)
    q[1, 1, 5], q[2, 0, 40] = float('nan'), float('inf')
    got = rotary.rotate(q, None, torch.tensor([5, 6, 7], dtype=torch.int32, device='cuda'))
    bad = ~got.isfinite()
    want = torch.zeros_like(bad)
    want[1, 1, 5] = want[1, 1, 37] = want[2, 0, 40] = want[2, 0, 8] = True  # the pair alone
    assert torch.equal(bad, want)


def test_rows_beyond_32_bits():
    from rapidtinyrec_b200.rotary import Rotary
    rotary = Rotary(64)
    far = (1 << 30) + 64
    room = torch.empty(2 * far + 256, dtype=torch.bfloat16, device='cuda')
    q = room.as_strided((3, 2, 64), (far, 64, 1))
    made = rows_of(3, 2, 64, torch.bfloat16, 20)
    q.copy_(made)
    positions = torch.tensor([3, 50, 700], device='cuda')
    rotary.rotate(q, None, positions, out=q)
    check_rows(q, plain(made, positions, rotary.frequencies, 64, False))


def test_captured_and_on_another_stream():
    from rapidtinyrec_b200.rotary import Rotary
    rotary = Rotary(64)
    q, k = rows_of(6, 4, 64, torch.float32, 14), rows_of(6, 1, 64, torch.float32, 15)
    positions = torch.arange(6, dtype=torch.int32, device='cuda')
    rotary.rotate(q, k, positions)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = rotary.rotate(q, k, positions)
    for first in (0, 70000):
        positions.copy_(torch.arange(first, first + 6))
        q.copy_(rows_of(6, 4, 64, torch.float32, first + 16))
        graph.replay()
        check_rows(got[0], plain(q, positions, rotary.frequencies, 64, False))
        check_rows(got[1], plain(k, positions, rotary.frequencies, 64, False))


def test_refusals():
    from rapidtinyrec_b200.rotary import Rotary
    rotary = Rotary(64)
    q, k = rows_of(6, 4, 64, torch.float32, 1), rows_of(6, 1, 64, torch.float32, 2)
    at = torch.arange(6, dtype=torch.int32, device='cuda')
    flat = torch.zeros(6 * 4 * 64 + 64, device='cuda')
    over = flat[64:].view(6, 4, 64)
    for args, kw, says in [
            ((q.cpu(), k, at), {}, 'handle'), ((q[0], k, at), {}, r'\[rows'), ((q, k[:5], at), {}, r'\[rows'),
            ((q, k.bfloat16(), at), {}, 'one type'), ((q.half(), None, at), {}, 'float32 or bfloat16'),
            ((q[..., :32], None, at), {}, r'\[rows'), ((q, k, at.float()), {}, 'positions'), ((q, k, at[:5]), {}, 'positions'),
            ((q, k, at.cpu()), {}, 'positions'), ((q, k, torch.arange(12, dtype=torch.int32, device='cuda')[::2]), {}, 'positions'),
            ((q, k, at), {'out': q}, 'pair'), ((q, k, at), {'out': (k, q)}, 'like q'), ((q, k, at), {'out': (q, k.bfloat16())}, 'like k'),
            ((over, None, at), {'out': flat[:-64].view(6, 4, 64)}, 'itself'),
            ((q, None, at), {'out': q[:1].expand(6, 4, 64)}, 'overlap'),
            ((q[:, :1], k, at), {'out': (torch.empty_like(k),) * 2}, 'share'),
            ((q, 3, at), {}, 'k must be a tensor'), (('q', k, at), {}, 'q must be a tensor')]:
        with pytest.raises(ValueError, match=says):
            rotary.rotate(*args, **kw)


def test_a_pair_is_a_tuple_or_a_list():
    from rapidtinyrec_b200.rotary import Rotary
    rotary = Rotary(64)
    q, k = rows_of(6, 4, 64, torch.float32, 1), rows_of(6, 2, 64, torch.float32, 2)
    at = torch.arange(6, dtype=torch.int32, device='cuda')
    want = rotary.rotate(q, k, at)
    room = [torch.empty_like(q), torch.empty_like(k)]
    got = rotary.rotate(q, k, at, out=room)
    assert got[0].data_ptr() == room[0].data_ptr() and got[1].data_ptr() == room[1].data_ptr()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    rotary.rotate(q, k, at, out=[q, k])
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    for out in ([q], [q, k, k], (q,), [q, 'k']):
        with pytest.raises(ValueError, match='pair|tensor'):
            rotary.rotate(q, k, at, out=out)

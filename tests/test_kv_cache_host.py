"""The 8-bit KV cache without a GPU: what its C entry points and its Python layer
refuse (before anything is enqueued), and the arithmetic that hands pages and row
tiles to blocks."""
import ctypes

import pytest
import torch

from rapidtinyrec_b200 import _native
from rapidtinyrec_b200.kv_cache import KvCache8

A = 1 << 20  # an address that is never followed: every refusal comes before device work


def cache(**change):
    args = dict(k=A, v=A, k_scale=A, v_scale=A, page_stride=4 * 16 * 128, head_stride=16 * 128, scale_stride=4, pages=9,
                kv_heads=4, page=16, head_dim=128, status=A)
    args.update(change)
    return _native.KvCacheC(**args)


def batch(**change):
    args = dict(table=A, lens=A, starts=None, table_stride=8, table_width=8, seqs=2, rows=6)
    args.update(change)
    return _native.KvBatchC(**args)


def write(c, b, k=A, v=A, dtype=0, kt=512, kh=128, vt=512, vh=128):
    return _native.load().rtr_kv_write(ctypes.byref(c), ctypes.byref(b), k, v, dtype, kt, kh, vt, vh, 0, None)


def attention(c, b, q=A, dtype=0, heads=8, stride=1024, out=A, work=None, room=0):
    return _native.load().rtr_kv_attention(ctypes.byref(c), ctypes.byref(b), q, dtype, heads, stride, 1, 0.1, out, None,
                                           work, room, 0, None)


def message():
    return _native.load().rtr_last_error(None).decode()


@pytest.mark.parametrize('change,says', [
    (dict(k=None), 'null cache'), (dict(status=None), 'null cache'), (dict(head_dim=96), 'head_dim'),
    (dict(page=48), 'page must'), (dict(page=256), 'page must'), (dict(pages=0), 'pages'), (dict(kv_heads=0), 'KV heads'),
    (dict(kv_heads=20000), 'KV heads'), (dict(head_stride=1024), 'overlap'), (dict(page_stride=128), 'overlap'),
    (dict(scale_stride=0), 'overlap'), (dict(k=A + 8), '16 bytes'), (dict(page_stride=4 * 16 * 128 + 8), '16 bytes')])
def test_caches_that_are_refused(change, says):
    for call in (write, attention):
        assert call(cache(**change), batch()) == _native.RTR_ERR_ARG
        assert says in message()


@pytest.mark.parametrize('change', [dict(page_stride=4 * 16 * 128 - 16), dict(scale_stride=3),
                                    dict(head_stride=1 << 62, page_stride=(1 << 63) - 16)])
def test_pages_that_share_memory_are_refused(change):
    for call in (write, attention):
        assert call(cache(**change), batch()) == _native.RTR_ERR_ARG
        assert 'overlap' in message()
    for fits in (dict(page_stride=7 * 16 * 128, head_stride=2 * 16 * 128), dict(kv_heads=1, page_stride=16 * 128)):
        assert write(cache(**fits), batch(rows=0)) == _native.RTR_OK


def test_heads_may_lie_outermost():
    """[heads][pages][page][dim], as one buffer a head: nothing overlaps."""
    one = 16 * 128
    for fits in (dict(page_stride=one, head_stride=9 * one), dict(page_stride=2 * one, head_stride=40 * one),
                 dict(page_stride=16 * one, head_stride=one, pages=1), dict(page_stride=one, head_stride=one, pages=1)):
        assert write(cache(**fits), batch(rows=0)) == _native.RTR_OK, message()
        assert attention(cache(**fits), batch(rows=0)) == _native.RTR_OK, message()
    for bad in (dict(page_stride=one, head_stride=9 * one - 16), dict(page_stride=one + 16, head_stride=9 * one),
                dict(page_stride=one, head_stride=2 * one), dict(page_stride=one - 16, head_stride=9 * one)):
        for call in (write, attention):
            assert call(cache(**bad), batch()) == _native.RTR_ERR_ARG and 'overlap' in message()


@pytest.mark.parametrize('change,says', [
    (dict(table=None), 'null table'), (dict(lens=None), 'null table'), (dict(seqs=-1), 'negative'),
    (dict(rows=-1), 'negative'), (dict(table_width=0), 'table rows'), (dict(table_stride=7), 'table rows'),
    (dict(table_width=1 << 27, table_stride=1 << 27), '2^31'), (dict(seqs=0), 'without sequences'),
    (dict(rows=7), 'multiple of the sequences')])
def test_batches_that_are_refused(change, says):
    for call in (write, attention):
        assert call(cache(), batch(**change)) == _native.RTR_ERR_ARG
        assert says in message()


def test_rows_that_are_refused():
    for bad, says in ((dict(dtype=2), 'dtype'), (dict(k=None), 'null'), (dict(v=A + 4), '16 bytes'),
                      (dict(kt=510), '16 bytes'), (dict(dtype=1, vh=68), '16 bytes')):
        assert write(cache(), batch(), **bad) == _native.RTR_ERR_ARG
        assert says in message()
    for bad, says in ((dict(dtype=2), 'dtype'), (dict(q=None), 'null'), (dict(out=None), 'null'), (dict(heads=6), 'multiple'),
                      (dict(heads=0), 'multiple'), (dict(q=A + 8), '16 bytes'), (dict(stride=1022), '16 bytes')):
        assert attention(cache(), batch(), **bad) == _native.RTR_ERR_ARG
        assert says in message()
    assert attention(cache(), batch(rows=1 << 30, seqs=1)) == _native.RTR_ERR_ARG and '2^31' in message()
    lib = _native.load()
    assert lib.rtr_kv_attention_workspace(ctypes.byref(cache()), ctypes.byref(batch()), 0, 8, 0, None) == _native.RTR_ERR_ARG
    assert lib.rtr_kv_write(None, None, A, A, 0, 512, 128, 512, 128, 0, None) == _native.RTR_ERR_ARG


def test_the_call_module_loads_and_refuses():
    from rapidtinyrec_b200 import kv_cache
    call = kv_cache._load()
    c = cache()
    t = torch.zeros(2, 2, 128)
    for bad in ((t, t, t, t, None), (None, t, t, t, None), (t, t.double(), t, t, None), (t, t[:1], t, t, None)):
        with pytest.raises(ValueError):
            call.write(ctypes.addressof(c), 0, *bad)  # tensors on the CPU, of wrong types or shapes
    with pytest.raises(ValueError, match='arguments'):
        call.attention(ctypes.addressof(c), 0, t)
    with pytest.raises(ValueError, match='pair'):
        call.read(ctypes.addressof(c), 0, 2, t, t, None, 0, t)
    with pytest.raises(TypeError):
        call.write('cache', 0, t, t, t, t, None)


def test_nothing_to_do_is_done_without_a_device():
    for b in (batch(rows=0), batch(rows=0, seqs=0, table=None, lens=None)):
        assert write(cache(), b) == _native.RTR_OK
        assert attention(cache(), b) == _native.RTR_OK


def test_python_refuses_wrong_caches():
    code = torch.zeros(3, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = torch.ones(3, 2)
    for bad in ((code.float(), code.float(), scale, scale), (code, code[:2], scale, scale), (code[0], code[0], scale, scale),
                (code[:, :, :8], code[:, :, :8], scale, scale), (code, code, scale.double(), scale.double()),
                (code, code, scale[:2], scale[:2]), (code, code, scale.t().contiguous().t(), scale.t().contiguous().t()),
                (code.transpose(0, 1).contiguous().transpose(0, 1), code, scale, scale),
                (code, code, scale, scale)):  # the last one: not on a CUDA device
        with pytest.raises(ValueError):
            KvCache8(*bad)


def test_python_refuses_wrong_status_words():
    code = torch.zeros(3, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = torch.ones(3, 2)
    for bad in (torch.zeros(1), torch.zeros(1, dtype=torch.int64), torch.zeros(2, dtype=torch.int32),
                torch.zeros(0, dtype=torch.int32), torch.zeros(1, dtype=torch.int32, device='meta')):
        with pytest.raises(ValueError, match='status'):
            KvCache8(code, code, scale, scale, bad)


@pytest.mark.parametrize('page', [16, 32, 64, 128])
def test_page_items_cover_every_page_once(page):
    """A sequence's items start at starts[b] // page + 2 b, without starts there are
    (n + page - 2) // page + 1 of them: enough for n rows from any position on."""
    for n in list(range(0, 3 * page + 3)) + [1000, 4097]:
        fixed = (n + page - 2) // page + 1
        for begin in range(0, 2 * page):
            touched = (begin + n - 1) // page - begin // page + 1 if n else 0
            assert touched <= fixed
            for row0 in (0, 1, page - 1, page, 12345):
                assert touched <= (row0 + n) // page + 2 - row0 // page


@pytest.mark.parametrize('group', [1, 2, 6, 7, 8, 12])
@pytest.mark.parametrize('tile', [8, 128])
def test_row_tiles_cover_every_row_once(group, tile):
    """A sequence's row tiles start at starts[b] * group // tile + b."""
    for n in list(range(0, 40)) + [127, 128, 129, 1000]:
        for row0 in (0, 1, 2, 7, 8, 99, 12345):
            assert -(-n * group // tile) <= (row0 + n) * group // tile + 1 - row0 * group // tile

"""An 8-bit KV cache in pages, and the operators on it.

``KvCache8`` holds K and V of many sequences as e4m3 codes, ``[pages, kv_heads, page,
head_dim]``, with one float32 scale for each page and head.  A sequence finds its
pages through its row of a page table.  Three operators work on the cache, each one
call into the native library on the current stream: ``write`` quantises new rows into
the pages, ``read`` gives rows back as the values they stand for, and ``attention``
attends over the pages as they are.

What the three share: ``table`` int32 ``[seqs, width]`` page numbers, ``lens`` int32
``[seqs]`` tokens that each sequence holds (the rows of this call included), and
``starts`` int32 ``[seqs + 1]``: rows ``starts[b] .. starts[b + 1] - 1`` are sequence
``b``'s; without it every sequence has the same number.  All are device tensors and
are not read on the host, so nothing here synchronises and every call can be captured
into a CUDA graph.  What does not fit (a page number outside the cache, a length that
the table cannot hold) leaves its work undone and sets a bit that ``check`` raises for:
attention's rows of that sequence become NaN.  ``starts`` that decrease, or leave the call's
rows, leave out the whole call: no row and no page is written.
The operators serve inference: their results carry no gradient.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _native

PAGES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_DTYPES = {torch.float32: _native.RTR_DTYPE_F32, torch.bfloat16: _native.RTR_DTYPE_BF16}
_STATUS = {1 << 5: 'a length or row range that does not fit the call or the table',
           1 << 8: 'a bounded wait of a kernel that ran out',
           1 << 9: 'a page number outside the cache',
           1 << 10: 'a scale that is not positive and finite'}


_call = None


def _load():
    """The calls' C++ module (kv_call.cpp), bound to the library's entry points."""
    global _call
    if _call is None:
        lib = _native.load()
        try:
            from . import _kv_call
        except ImportError as e:
            raise ImportError('_kv_call.so is not built; run `python -m rapidtinyrec_b200.build`') from e
        entries = (lib.rtr_kv_write, lib.rtr_kv_read, lib.rtr_kv_attention, lib.rtr_kv_attention_workspace,
                   lib.rtr_last_error)
        _kv_call.setup(*(ctypes.cast(f, ctypes.c_void_p).value for f in entries), _native.NativeError)
        _call = _kv_call
    return _call


class KvCache8:
    """The cache: ``k``, ``v`` (float8_e4m3fn ``[pages, kv_heads, page, head_dim]``, the last
    two dimensions contiguous) and ``k_scale``, ``v_scale`` (float32 ``[pages, kv_heads]``).

    Slices of larger tensors serve (one layer's heads of a cache of all layers); k and v
    must then be sliced alike.
    """

    def __init__(self, k, v, k_scale, v_scale, status=None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != torch.float8_e4m3fn or v.dtype != k.dtype:
            raise ValueError('k and v must be float8_e4m3fn [pages, kv_heads, page, head_dim] of one shape')
        pages, heads, page, dim = k.shape
        if page not in PAGES or dim not in HEAD_DIMS:
            raise ValueError(f'page must be one of {PAGES} tokens and head_dim one of {HEAD_DIMS}')
        if k.stride() != v.stride() or k.stride(3) != 1 or k.stride(2) != dim:
            raise ValueError('k and v must have the same strides, tokens and dimensions contiguous')
        for s in (k_scale, v_scale):
            if s.shape != (pages, heads) or s.dtype != torch.float32 or s.stride() != k_scale.stride():
                raise ValueError('scales must be float32 [pages, kv_heads], strided alike')
        if heads > 1 and k_scale.stride(1) != 1:
            raise ValueError('the scales of a page must be contiguous')
        if status is not None and (status.dtype != torch.int32 or status.numel() != 1 or status.device != k.device):
            raise ValueError('status must be one int32 on the cache\'s device')
        if not (k.is_cuda and len({t.device for t in (k, v, k_scale, v_scale)}) == 1):
            raise ValueError('the cache must lie on one CUDA device')
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._call = _load()
        self.k, self.v, self.k_scale, self.v_scale, self.status = k, v, k_scale, v_scale, status
        self.pages, self.kv_heads, self.page, self.head_dim = pages, heads, page, dim
        self.device = k.device
        self._index = k.device.index
        # the stride of a dimension with one entry means nothing
        head_stride = k.stride(1) if heads > 1 else page * dim
        self._c = _native.KvCacheC(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                   k.stride(0) if pages > 1 else heads * head_stride, head_stride,
                                   k_scale.stride(0) if pages > 1 else heads, pages, heads, page, dim,
                                   status.data_ptr())
        self._at = ctypes.addressof(self._c)
        self.kept = {}  # page number -> what the last prefix kept there is known by (BeamEngine.keep_prefix)
        self._scale = 1.0 / math.sqrt(dim)

    @classmethod
    def allocate(cls, pages, kv_heads, page, head_dim, device='cuda'):
        """An empty cache: codes 0 and scales 1."""
        dev = torch.device(device)
        shape = (pages, kv_heads, page, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
        ks, vs = (torch.ones(shape[:2], dtype=torch.float32, device=dev) for _ in range(2))
        return cls(k, v, ks, vs)

    def heads(self, first, count):
        """The cache of ``count`` of its heads from ``first`` on (one layer's, say), same memory."""
        if not (0 <= first and 0 < count and first + count <= self.kv_heads):
            raise ValueError('heads outside the cache')
        cut = slice(first, first + count)
        return KvCache8(self.k[:, cut], self.v[:, cut], self.k_scale[:, cut], self.v_scale[:, cut], self.status)

    def check(self):
        """Raise for what earlier calls, on any stream, left undone (waits for them), and forget it."""
        torch.cuda.synchronize(self.device)
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            torch.cuda.synchronize(self.device)  # before a later call on another stream can set a bit
            raise _native.NativeError(_native.RTR_ERR_DEVICE, '; '.join(t for b, t in _STATUS.items() if bits & b))

    # ------------------------------------------------------------ operators
    def write(self, k, v, table, lens, starts=None):
        """Quantise rows ``k``, ``v`` ``[rows, kv_heads, head_dim]`` (float32 or bfloat16, any row and
        head strides) into the pages: the last positions of their sequences.

        A page's scale is the least power of two, from 2^-48 to 2^48, at which its largest
        magnitude is at most 448.  A page that holds older tokens keeps its scale unless that is
        too small; then their codes are rounded again.  NaN, infinities and magnitudes above
        448 * 2^48 are stored as NaN.  Codes behind a sequence's last token stay as they are.
        No two sequences of a call may write into the same page.
        """
        self._call.write(self._at, self._index, k, v, table, lens, starts)

    def read(self, rows, table, lens, starts=None, dtype=torch.float32, out=None):
        """The last tokens of each sequence as ``(k, v)``, ``[rows, kv_heads, head_dim]`` each: the
        values that the codes stand for, rounded once to ``dtype``.  ``out``: a pair of tensors to
        fill, of one type, which then stands for ``dtype``; rows that belong to no sequence keep what
        they held (new tensors: undefined there).
        """
        if dtype not in _DTYPES:
            raise ValueError('dtype must be float32 or bfloat16')
        return self._call.read(self._at, self._index, rows, table, lens, starts, _DTYPES[dtype],
                               out if out is None else tuple(out))

    def attention(self, q, table, lens, starts=None, causal=True, scale=None, return_lse=False, out=None):
        """``softmax(scale q K^T) V`` of the rows ``q`` ``[rows, heads, head_dim]`` (float32 or bfloat16)
        over their sequences; query head h reads KV head ``h // (heads // kv_heads)``.

        ``causal``: a sequence's rows are its last positions, each sees what is not behind it;
        otherwise every row sees the whole sequence.  A row that sees nothing is 0.  ``scale``:
        ``head_dim ** -0.5`` unless given.  Returns ``out`` (a new tensor, or the contiguous one given,
        which may be ``q`` itself), with ``return_lse`` also the float32 ``[rows, heads]`` log of the softmax's sum, by which
        results over several stretches of keys are merged.  Rows that belong to no sequence are not
        written: a given ``out`` keeps them, new tensors are undefined there.  The work is laid out
        for sequences as long as a row of ``table``: where they are much shorter, pass a slice of it
        (``table[:, :n]``).
        """
        return self._call.attention(self._at, self._index, q, table, lens, starts, causal,
                                    self._scale if scale is None else scale, return_lse, out)

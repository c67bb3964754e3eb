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
the table cannot hold) leaves its work undone and sets a bit that ``check`` raises for.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import _native

PAGES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
_BATCH = struct.Struct('PPPqiii4x')  # rtr_kv_batch; packed bytes cost a third of a ctypes structure
_DTYPES = {torch.float32: _native.RTR_DTYPE_F32, torch.bfloat16: _native.RTR_DTYPE_BF16}
_STATUS = {1 << 5: 'a length or row range that does not fit the call or the table',
           1 << 8: 'a bounded wait of a kernel that ran out',
           1 << 9: 'a page number outside the cache',
           1 << 10: 'a scale that is not positive and finite'}


def _stream(index):
    """The device's current stream (torch.cuda.current_stream without making a Stream object)."""
    return torch._C._cuda_getCurrentRawStream(index)


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
        if not (k.is_cuda and len({t.device for t in (k, v, k_scale, v_scale)}) == 1):
            raise ValueError('the cache must lie on one CUDA device')
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self.lib = _native.load()
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
        self._ref = ctypes.byref(self._c)
        self._scale = 1.0 / math.sqrt(dim)
        self._attend = self.lib.rtr_kv_attention
        self._room = {}  # workspace bytes of the call shapes seen

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
        """Raise for what earlier calls left undone (synchronises), and forget it."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise _native.NativeError(_native.RTR_ERR_DEVICE, '; '.join(t for b, t in _STATUS.items() if bits & b))

    # ------------------------------------------------------------- plumbing
    def _batch(self, rows, table, lens, starts):
        """The call's ``rtr_kv_batch`` (packed)."""
        shape = table.shape
        if table.dtype is not torch.int32 or lens.dtype is not torch.int32 or len(shape) != 2 or lens.shape != shape[:1]:
            raise ValueError('table must be int32 [seqs, width] and lens int32 [seqs]')
        seqs, width = shape
        step = table.stride()
        if (width > 1 and step[1] != 1) or (seqs > 1 and lens.stride(0) != 1):
            raise ValueError('the rows of table and lens must be contiguous')
        index = self._index
        if table.get_device() != index or lens.get_device() != index:
            raise ValueError('table and lens must lie on the cache\'s device')
        if starts is None:
            if rows % seqs if seqs else rows:
                raise ValueError('without starts the rows must be a multiple of the sequences')
            begin = 0
        else:
            if starts.dtype is not torch.int32 or starts.shape != (seqs + 1,) or not starts.is_contiguous():
                raise ValueError('starts must be int32 [seqs + 1], contiguous')
            if starts.get_device() != index:
                raise ValueError('starts must lie on the cache\'s device')
            begin = starts.data_ptr()
        return _BATCH.pack(table.data_ptr(), lens.data_ptr(), begin, step[0] if seqs > 1 else width, width, seqs, rows)

    def _dense(self, x, heads, name):
        """Rows as the kernels take them: one type, dimensions contiguous, 16-byte steps."""
        shape = x.shape
        if len(shape) != 3 or shape[1] != heads or shape[2] != self.head_dim or x.get_device() != self._index:
            raise ValueError(f'{name} must be [rows, {heads}, {self.head_dim}] on the cache\'s device')
        if x.dtype not in _DTYPES:
            raise ValueError(f'{name} must be float32 or bfloat16')
        a, b, c = x.stride()
        step = 4 if x.dtype is torch.float32 else 8
        if c != 1 or a % step or b % step or x.data_ptr() % 16:
            x = x.clone(memory_format=torch.contiguous_format)
        return x

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
        if k.dtype != v.dtype or k.shape != v.shape:
            raise ValueError('k and v must have one type and shape')
        k, v = self._dense(k, self.kv_heads, 'k'), self._dense(v, self.kv_heads, 'v')
        batch = self._batch(k.shape[0], table, lens, starts)
        code = self.lib.rtr_kv_write(self._ref, batch, k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype],
                                     k.stride(0), k.stride(1), v.stride(0), v.stride(1), self._index, _stream(self._index))
        if code:
            _native.check(code)

    def read(self, rows, table, lens, starts=None, dtype=torch.float32, out=None):
        """The last tokens of each sequence as ``(k, v)``, ``[rows, kv_heads, head_dim]`` each: the
        values that the codes stand for, rounded once to ``dtype``.  ``out``: a pair of tensors to
        fill; rows that belong to no sequence keep what they held (new tensors: undefined there).
        """
        shape = (rows, self.kv_heads, self.head_dim)
        if out is None:
            if dtype not in _DTYPES:
                raise ValueError('dtype must be float32 or bfloat16')
            k = self.k_scale.new_empty(shape, dtype=dtype)
            v = torch.empty_like(k)
        else:
            k, v = out
            if k.shape != shape or v.shape != shape or k.dtype != v.dtype:
                raise ValueError(f'out must be two tensors {list(shape)} of one type')
            for x, name in ((k, 'k'), (v, 'v')):
                if self._dense(x, self.kv_heads, name) is not x or any(n > 1 and not d for n, d in zip(shape, x.stride())):
                    raise ValueError('out must have contiguous dimensions and rows of their own at multiples of 16 bytes')
        batch = self._batch(rows, table, lens, starts)
        code = self.lib.rtr_kv_read(self._ref, batch, k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype],
                                    k.stride(0), k.stride(1), v.stride(0), v.stride(1), self._index, _stream(self._index))
        if code:
            _native.check(code)
        return k, v

    def attention(self, q, table, lens, starts=None, causal=True, scale=None, return_lse=False, out=None):
        """``softmax(scale q K^T) V`` of the rows ``q`` ``[rows, heads, head_dim]`` (float32 or bfloat16)
        over their sequences; query head h reads KV head ``h // (heads // kv_heads)``.

        ``causal``: a sequence's rows are its last positions, each sees what is not behind it;
        otherwise every row sees the whole sequence.  A row that sees nothing is 0.  ``scale``:
        ``head_dim ** -0.5`` unless given.  Returns ``out`` (a new tensor, or the contiguous one given),
        with ``return_lse`` also the float32 ``[rows, heads]`` log of the softmax's sum, by which
        results over several stretches of keys are merged.  Rows that belong to no sequence are not
        written: a given ``out`` keeps them, new tensors are undefined there.
        """
        rows, heads = q.shape[:2]
        if q.dim() != 3 or heads < 1 or heads % self.kv_heads:
            raise ValueError(f'q must be [rows, heads, {self.head_dim}], heads a multiple of {self.kv_heads}')
        q = self._dense(q, heads, 'q')
        if heads > 1 and q.stride(1) != self.head_dim:
            q = q.clone(memory_format=torch.contiguous_format)
        batch = self._batch(rows, table, lens, starts)
        key = (rows, heads, table.shape, starts is None, q.dtype)
        room = self._room.get(key)
        if room is None:
            need = ctypes.c_int64()
            _native.check(self.lib.rtr_kv_attention_workspace(self._ref, batch, _DTYPES[q.dtype], heads, self._index,
                                                                   ctypes.byref(need)))
            if len(self._room) >= 4096:
                self._room.clear()
            room = self._room[key] = need.value
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != self._index \
                or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError('out must be contiguous and like q')
        lse = q.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
        work = q.new_empty((room,), dtype=torch.uint8) if room else None
        code = self._attend(self._ref, batch, q.data_ptr(), _DTYPES[q.dtype], heads, q.stride(0), causal,
                            self._scale if scale is None else scale, out.data_ptr(),
                            lse.data_ptr() if return_lse else None, work.data_ptr() if room else None, room,
                            self._index, _stream(self._index))
        if code:
            _native.check(code)
        return (out, lse) if return_lse else out

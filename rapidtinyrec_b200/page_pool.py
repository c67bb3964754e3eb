"""Pages for the sequences of a paged cache, handed out and taken back on the GPU.

``PagePool`` keeps the page numbers that no sequence holds.  ``grow`` gives sequences the pages for
their new tokens and returns what the cache's calls and a program's own kernels want to know about
them, from the lengths alone: ``KvCache8.write`` and ``attention`` take the table with ``lens`` and ``starts``,
``Rotary.rotate`` the rows' ``positions``, and a cache of the program's own the rows' ``slots`` (a slot is a token's place in
the cache, ``page number * page + place in the page``).  ``release`` takes back the pages that a sequence
does not need any more: all when it ends, some when tokens are taken back.

Nothing is read on the host, nothing synchronises, and every call can be captured into a CUDA graph (with
``rows`` for the most that a step may bring).  A call that does not fit as a whole (a table row that
is too narrow, too few pages, a page given back twice) changes nothing, its rows have slot and position -1, and
``check`` raises for it.  Calls on one pool have to follow one another: on one stream, or on streams that wait for each
other.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _native

_STATUS = {1 << 5: 'a length or row count that does not fit the call or the table',
           1 << 9: 'a page number outside the pool',
           1 << 11: 'fewer free pages than were needed',
           1 << 12: 'a page given back that no sequence held'}


class Grown(NamedTuple):
    """What ``PagePool.grow`` returns: int32 ``lens`` [seqs] (tokens held now), ``starts`` [seqs + 1] (first row of each
    sequence) and ``positions`` [rows] (of a row in its sequence), int64 ``slots`` [rows]."""
    lens: torch.Tensor
    starts: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


class PagePool:
    """The page numbers 0 .. ``pages`` - 1 of a cache whose pages hold ``page`` tokens (a power of two up to 1024).

    ``free``: the numbers that it may hand out, last first (int32 or int64, distinct; the others are held by
    sequences); all unless given, in ascending order.
    """

    def __init__(self, pages, page, device='cuda', free=None):
        dev = torch.device(device)
        if free is not None:
            dev = free.device
        if dev.type != 'cuda':
            raise ValueError('the pool must lie on a CUDA device')
        if not 0 < pages < 1 << 31:
            raise ValueError('pages must be positive and fit 32 bits')
        if page not in (1 << i for i in range(11)):
            raise ValueError('page must be a power of two from 1 to 1024 tokens')
        self._call = _native.op_call()
        if dev.index is None:
            dev = torch.device('cuda', torch.cuda.current_device())
        if free is None:
            free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=dev)
        elif free.dim() != 1 or free.dtype not in (torch.int32, torch.int64):
            raise ValueError('free must be int32 or int64 [n]')
        elif free.numel() and not (free.numel() <= pages and 0 <= int(free.min()) and int(free.max()) < pages
                                   and free.unique().numel() == free.numel()):
            raise ValueError('free must be distinct page numbers of the pool')
        self.pages, self.page, self.device, self._index = pages, page, dev, dev.index
        self.free = torch.full((pages,), -1, dtype=torch.int32, device=dev)
        self.free[:free.numel()] = free
        self._marks = torch.ones(pages, dtype=torch.int32, device=dev)
        self._marks[free.long()] = 0
        self._words = torch.tensor([free.numel(), 0, 0], dtype=torch.int32, device=dev)
        self.count, self.status = self._words[:1], self._words[1:2]
        at = self._words.data_ptr()
        self._c = _native.PagePoolC(self.free.data_ptr(), at, self._marks.data_ptr(), at + 4, at + 8, pages, page)
        self._at = ctypes.addressof(self._c)

    def grow(self, table, held, new=1, rows=None):
        """Pages for ``new`` tokens more of each sequence (a number, or int32 ``[seqs]``) behind the ``held``
        (int32 ``[seqs]``) that it has: writes their numbers into ``table`` (int32 ``[seqs, width]``) and returns
        ``Grown``.  ``rows``: the rows that the call's tensors have, at least the sum of ``new`` (needed where that is a
        tensor); those behind the last sequence's have slot and position -1.  At most 16384 sequences.
        """
        return Grown._make(self._call.grow(self._at, self._index, table, held, new, rows))

    def release(self, table, held, keep=None):
        """Takes back the pages that ``keep`` (int32 ``[seqs]``; without it none) of the ``held`` tokens of each sequence do
        not need.  ``table`` stays as it is; growing again by as much gives the same pages in the same places.  A
        sequence of the table that others share pages with must not be among them.
        """
        self._call.release(self._at, self._index, table, held, keep)

    def check(self):
        """Raise for calls, on any stream, that did not fit (waits for them), and forget them."""
        torch.cuda.synchronize(self.device)
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            torch.cuda.synchronize(self.device)  # before a later call on another stream can set a bit
            raise _native.NativeError(_native.RTR_ERR_DEVICE, '; '.join(t for b, t in _STATUS.items() if bits & b))

"""Beam search over a whole vocabulary, for programs with a model of their own.

``BeamEngine`` searches the semantic IDs of a catalog: five steps, at most 256 allowed tokens a beam, the states
in its own layout.  ``BeamSearch`` has the two steps that any other beam search needs after its model's logits:
``select`` chooses the best continuations of all beams (log-softmax, running scores, an optional list of
allowed tokens, the end token) in one pass over the logits, and ``reorder`` puts the beams' states (the keys and values of
their own tokens, say) in the order of the chosen beams' parents, in place.

Neither reads anything on the host; both can be captured into a CUDA graph.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native

_STATUS = {1 << 1: 'a parent that is none of the beams',
           1 << 7: 'a NaN or infinite logit or score: its beam was left out'}


class BeamStep(NamedTuple):
    """What ``BeamSearch.select`` returns: the next beams (int32 ``tokens`` and ``parents``, float32 ``scores``, ``[items, beams]`` each) and
    all candidates that they were chosen from, the best first (``[items, candidates]``), those that end among them."""
    tokens: torch.Tensor
    parents: torch.Tensor
    scores: torch.Tensor
    all_tokens: torch.Tensor
    all_parents: torch.Tensor
    all_scores: torch.Tensor


class BeamSearch:
    """Searches with ``beams`` (1 to 128) beams an item.  ``eos``: the token that ends a beam.  ``candidates``: how many
    continuations of an item ``select`` ranks (up to 256), twice the beams unless given, which leaves enough to go on
    with when each beam has one that ends."""

    def __init__(self, beams, eos=None, candidates=None, device='cuda'):
        if not 1 <= beams <= 128:
            raise ValueError('1 to 128 beams')
        candidates = 2 * beams if candidates is None else candidates
        if not beams <= candidates <= 256:
            raise ValueError('candidates must be at least the beams and at most 256')
        if eos is not None and eos < 0:
            raise ValueError('eos must be a token or None')
        dev = torch.device(device)
        if dev.type != 'cuda':
            raise ValueError('the search must run on a CUDA device')
        self._call = _native.op_call()
        self.beams, self.eos, self.candidates = beams, eos, candidates
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.device = self.status.device
        self._at, self._index = self.status.data_ptr(), self.device.index

    def select(self, logits, scores, allowed=None):
        """The best continuations: ``logits`` float32 or bfloat16 ``[items * n, vocab]`` (any row stride, up to 2^20 tokens), ``scores`` the n
        beams' running log-probabilities, float32 ``[items, n]``.  n may differ from ``beams`` (1 at the first step).

        Candidate (i, v) is worth ``log_softmax(logits[i])[v] + scores[i]`` where ``allowed`` (bool ``[items * n, vocab]``, or ``[vocab]`` for all
        rows) holds, minus infinity elsewhere: the softmax is over the whole vocabulary, as in the constrained request.
        Equal ones rank by beam, then token.  The order within a call is that of 64-bit arithmetic.  The scores are float32, of sums
        in 32 bits where nothing more was needed to tell candidates apart: off by 1.4e-6 at most besides their own rounding, and in their
        last bits a row's may differ with the other rows of the call.
        A beam whose score is minus infinity has ended and is not read; any other score is searched (-1e9 for beams that are to wait is right,
        and slower where it leaves one beam alone).  Beams with NaN or plus infinity among logits or
        scores have nothing to offer, and ``check`` raises for them.  Where fewer than ``candidates`` are finite, the last have score minus
        infinity.  Returns ``BeamStep``.  The result carries no gradient.
        """
        return BeamStep._make(self._call.select(self._at, self._index, self.beams, self.eos, self.candidates, logits, scores, allowed))

    def reorder(self, states, parents, dim=0, token_dim=None, tokens=None):
        """Puts row ``b * beams + parents[b, i]`` of every state in the place of row ``b * beams + i``, all at once and in place.

        ``states``: a tensor or a list of them, of any type, whose dimension ``dim`` is the ``items * beams`` rows; ``parents``
        int32 ``[items, beams]`` (``BeamStep.parents``).  ``token_dim``, ``tokens``: of that dimension only the first
        ``tokens`` entries are moved, where a cache has room for more.  States must not share memory.  A parent that is none
        of the beams leaves its row as it is, and ``check`` raises for it.
        """
        self._call.reorder(self._at, self._index, self.beams, states, parents, dim, token_dim, tokens)

    def check(self):
        """Raise for what earlier calls, on any stream, left out (waits for them), and forget it."""
        torch.cuda.synchronize(self.device)
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            torch.cuda.synchronize(self.device)  # before a later call on another stream can set a bit
            raise _native.NativeError(_native.RTR_ERR_DEVICE, '; '.join(t for b, t in _STATUS.items() if bits & b))

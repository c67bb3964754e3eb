"""Rotary positions for query and key rows, in the layouts and scalings that models use.

``Rotary`` holds a model's frequencies; ``rotate`` turns the pairs of dimensions of ``q`` and ``k`` by
``position * frequency``, as a program of its own does before ``KvCache8.write`` and ``attention`` (the engine's requests
have the rotation in their projection).  Angles are exact at any position: a frequency is kept as a 64-bit
fraction of a turn, and the product with the position drops whole turns by integer arithmetic.
"""
from __future__ import annotations

import math

import torch

from . import _native

SCALINGS = (None, 'linear', 'ntk', 'bands')


def frequencies(rotary_dim, theta=1e6, scaling=None, factor=1.0, length=None, low=1.0, high=4.0):
    """Radians a position of each of the ``rotary_dim / 2`` pairs, as Python floats.

    ``theta^(-2 i / rotary_dim)``, and for contexts ``factor`` times as long as the model was trained with:
    ``linear``: divided by the factor; ``ntk``: with ``theta * factor^(rotary_dim / (rotary_dim - 2))``, which leaves the fastest
    pair and divides the slowest by the factor; ``bands``: pairs that turn less than ``low`` times over the original ``length`` are
    divided by the factor, those that turn more than ``high`` times stay, and in between the share of either
    goes linearly with the number of turns.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError('rotary_dim must be even and positive')
    if scaling not in SCALINGS:
        raise ValueError(f'scaling must be one of {SCALINGS}')
    if not (math.isfinite(theta) and theta > 0 and math.isfinite(factor) and factor > 0):
        raise ValueError('theta and factor must be positive')
    if scaling == 'ntk':
        if rotary_dim < 4:
            raise ValueError('ntk needs a rotary_dim of at least 4')
        theta *= factor ** (rotary_dim / (rotary_dim - 2))
    f = [theta ** (-2 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling == 'linear':
        f = [x / factor for x in f]
    if scaling == 'bands':
        if length is None or length <= 0 or not 0 <= low < high:
            raise ValueError('bands needs the original length and 0 <= low < high')
        share = [min(1.0, max(0.0, (x * length / (2 * math.pi) - low) / (high - low))) for x in f]
        f = [x * (s + (1 - s) / factor) for x, s in zip(f, share)]
    return f


class Rotary:
    """Rotary positions of heads of ``head_dim`` dimensions, the first ``rotary_dim`` (all unless given) of which turn.

    ``interleaved``: pairs are neighbours (2 i, 2 i + 1) instead of half the turning part apart (i, i + rotary_dim / 2).
    ``theta``, ``scaling``, ``factor``, ``length``, ``low``, ``high``: see ``frequencies``; or ``given``: the frequencies
    themselves in radians a position (a sequence or tensor of rotary_dim / 2).  ``amplitude`` multiplies
    what turns (the attention factor of some long-context scalings).
    """

    def __init__(self, head_dim, rotary_dim=None, theta=1e6, interleaved=False, scaling=None, factor=1.0, length=None, low=1.0,
                 high=4.0, amplitude=1.0, given=None, device='cuda'):
        part = head_dim if rotary_dim is None else rotary_dim
        if not 2 <= head_dim <= 512 or not 2 <= part <= head_dim or part % 2:
            raise ValueError('head_dim must be 2 to 512 and rotary_dim even and at most head_dim')
        if given is None:
            given = frequencies(part, theta, scaling, factor, length, low, high)
        else:
            given = [float(x) for x in (given.tolist() if isinstance(given, torch.Tensor) else given)]
            if len(given) != part // 2 or not all(math.isfinite(x) for x in given):
                raise ValueError('given must be rotary_dim / 2 finite frequencies')
        if not math.isfinite(amplitude):
            raise ValueError('amplitude must be finite')
        dev = torch.device(device)
        if dev.type != 'cuda':
            raise ValueError('the handle must lie on a CUDA device')
        self._call = _native.op_call()
        self.head_dim, self.rotary_dim, self.interleaved, self.amplitude = head_dim, part, bool(interleaved), float(amplitude)
        self.frequencies = given
        # turns a position times 2^64, modulo 2^64 (whole turns do not matter), as the bits of an int64
        turns = [round(math.ldexp(math.fmod(x / (2 * math.pi), 1.0), 64)) & ((1 << 64) - 1) for x in given]
        self._turns = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64, device=dev)
        self.device = self._turns.device

    def rotate(self, q, k, positions, back=False, out=None):
        """``q`` ``[rows, heads, head_dim]`` and ``k`` ``[rows, kv_heads, head_dim]`` (or None) at ``positions`` (int32 or int64
        ``[rows]``): the pair (a, b) of frequency f becomes ``amplitude * (a cos t - b sin t, b cos t + a sin t)``, ``t = position * f``.
        float32 or bfloat16, any strides; fp32 arithmetic, one rounding.

        Returns ``(q, k)`` (without k: q alone), new tensors, or ``out``: a pair to fill, which may be ``(q, k)``
        themselves.  ``back``: by -t, which takes the rotation of the same positions back, and is what the gradient of a rotated row
        needs.  The result carries no gradient of its own.
        """
        return self._call.rotate(self._turns, self.head_dim, self.rotary_dim, self.interleaved, self.amplitude, q, k, positions, back,
                                 out)

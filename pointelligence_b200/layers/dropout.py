"""Dropout for ragged batches: of elements, of channels of a sample, of samples (drop path).

The mask is a function of a seed and an offset (a counter-based generator), so it is never stored: the backward pass makes it
again.  The reference leaves dropout to ``torch.nn``, whose layers keep a mask of the activations' size, know samples of equal
length only and have no drop path.
"""
from __future__ import annotations

import torch.nn as nn

from .. import _cabi

__all__ = ["RaggedDropout", "fused_dropout", "draw_rng"]

UNITS = {"element": 0, "channel": 1, "sample": 2}


def _unit(unit):
    if unit not in UNITS:
        raise ValueError(f"unit is one of {sorted(UNITS)}, got {unit!r}")
    return UNITS[unit]


def draw_rng(x):
    """A new (seed, offset) from PyTorch's generator of ``x``'s device: ``torch.manual_seed`` sets the sequence of them.  While a
    graph is captured it is a tensor, which every replay fills anew."""
    return _cabi.host().draw_rng(x)


def fused_dropout(x, p, rng=None, unit="element", lengths=None, residual=None, relu=False):
    """``relu?((residual +) dropout(x))`` in one pass (CUDA tensors only).

    ``unit`` is what is dropped together, with probability ``p``: an "element", a "channel" of a sample, or a whole "sample" (drop
    path); the last two take rows (points, channels) and the ``lengths`` of the samples.  What is kept is scaled by 1 / (1 - p),
    what is dropped is zero, whatever it was.  ``p`` is taken to the nearest multiple of 2^-16 (the scale goes by that).

    ``rng``: None draws a new mask from PyTorch's generator (see ``draw_rng``); a pair (seed, offset), or an int64 tensor of the
    two on the device, names one: the same pair gives the same mask.  The backward pass reads such a tensor again, so it may not be
    written to before that."""
    return _cabi.host().dropout(x, p, rng, _unit(unit), lengths, residual, relu)


class RaggedDropout(nn.Module):
    """``fused_dropout`` while training; without it the residual and the ReLU alone."""

    def __init__(self, p=0.5, unit="element"):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability has to be between 0 and 1, but got {p}")
        self.p = p
        self.unit = unit
        _unit(unit)

    def forward(self, x, lengths=None, residual=None, relu=False, rng=None):
        if self.training and self.p > 0.0:
            return fused_dropout(x, self.p, rng, self.unit, lengths, residual, relu)
        x = x if residual is None else x + residual.to(x.dtype)
        return x.relu() if relu else x

    def extra_repr(self):
        return f"p={self.p}, unit={self.unit}"

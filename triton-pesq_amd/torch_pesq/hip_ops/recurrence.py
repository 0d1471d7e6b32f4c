"""Gated linear recurrence over time, diagonal over channels.

The layer that carries a speech enhancement network's memory from frame to
frame::

    u_t = rate softplus(decay) sigmoid(recur_gate_t)        a_t = exp(-u_t)
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(input_gate_t) x_t

``gated_recurrence`` runs whole sequences, with every gradient;
``gated_recurrence_step`` runs one frame of streams that are live;
``HipGatedRecurrence`` is the module that keeps ``decay``.  States are float32
whatever the type of ``x``.  No counterpart in the reference.
"""

import torch

from .. import _lib

__all__ = ["gated_recurrence", "gated_recurrence_step", "HipGatedRecurrence"]


def gated_recurrence(x, recur_gate, input_gate, decay, *, initial_state=None, reset=None,
                     reverse=False, rate=8.0):
    """``(y, last_state)`` of ``x`` ``[batch, time, channels]``.

    ``x`` and the gates' arguments share one type (float32, bfloat16 or float16)
    and may be strided views, such as the parts of one linear layer's output;
    ``decay`` is floating ``[channels]`` (converted where it is not float32),
    ``initial_state`` float32 ``[batch, channels]`` (zero if ``None``).  Where ``reset`` (bool ``[batch, time]``) is
    true the state before that step is dropped, whatever it holds: the start of
    another utterance in the same row.  ``reverse`` runs from the last step to
    the first; the last state is then the one after step 0.  Differentiable once
    with respect to ``x``, the gates, ``decay`` and ``initial_state``.
    """

    y, last = _lib.torch_ext().gated_recurrence(x, recur_gate, input_gate, decay, initial_state, reset,
                                                bool(reverse), float(rate))
    return y, last


def gated_recurrence_step(x, recur_gate, input_gate, decay, state, *, rate=8.0):
    """``y`` ``[batch, channels]`` of one frame; ``state`` (float32, as
    ``gated_recurrence`` returns it) is updated in place, and cannot require a
    gradient while these are recorded.  No gradient."""

    return _lib.torch_ext().gated_recurrence_step(x, recur_gate, input_gate, decay, state, float(rate))


class HipGatedRecurrence(torch.nn.Module):
    """:func:`gated_recurrence` with its ``decay``: the memory of an open gate
    starts between ``slowest`` and ``fastest`` (``a_t`` there, over the channels)."""

    def __init__(self, channels, *, rate=8.0, fastest=0.9, slowest=0.999):
        super().__init__()
        if channels < 1:
            raise ValueError(f"HipGatedRecurrence needs at least one channel, got {channels}.")
        if not 0.0 < rate <= 2.0**126:
            raise ValueError(f"`rate` has to be positive and at most 2^126, got {rate}.")
        if not 0.0 < fastest <= slowest < 1.0:
            raise ValueError(f"Expected 0 < fastest <= slowest < 1, got {fastest} and {slowest}.")
        self.channels, self.rate = int(channels), float(rate)
        open_gate = torch.empty(channels, dtype=torch.float64).uniform_(fastest, slowest)
        self.decay = torch.nn.Parameter(torch.log(torch.expm1(-torch.log(open_gate) / rate)).float())

    def extra_repr(self):
        return f"{self.channels}, rate={self.rate}"

    def forward(self, x, recur_gate, input_gate, *, initial_state=None, reset=None, reverse=False):
        return gated_recurrence(x, recur_gate, input_gate, self.decay, initial_state=initial_state,
                                reset=reset, reverse=reverse, rate=self.rate)

    def step(self, x, recur_gate, input_gate, state):
        return gated_recurrence_step(x, recur_gate, input_gate, self.decay, state, rate=self.rate)

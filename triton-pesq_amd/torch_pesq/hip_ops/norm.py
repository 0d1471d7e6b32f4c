"""Norms around a residual block, fused with its gate and residual scale.

``pre_norm`` is the start of a first block, ``residual_norm`` the end of a block
and the start of the next::

    y = branch silu(gate)               z = y / rms(y) weight
    x_out = x + scale z                 n = x_out / rms(x_out) next_weight

with ``rms(v)^2 = mean(v^2) + eps`` over the last axis.  Both read and write each
tensor once.  The residual stream ``x`` may be float32 under a bfloat16 or
float16 branch; weights of another type than float32 are converted.
No counterpart in the reference.
"""

from .. import _lib

__all__ = ["pre_norm", "residual_norm"]


def pre_norm(x, weight, *, eps=1e-6, dtype=None):
    """``x / rms(x) weight`` of ``x`` ``[..., channels]``, in ``dtype`` (that of ``x``
    if ``None``); differentiable once."""

    (n,) = _lib.torch_ext().residual_norm(x, None, None, None, None, weight, float(eps), dtype)
    return n


def residual_norm(x, branch, weight, *, gate=None, scale=None, next_weight=None, eps=1e-6):
    """``(x_out, n)``, or ``x_out`` alone where ``next_weight`` is ``None``.

    ``x``, ``branch`` and ``gate`` are ``[..., channels]``, ``weight``, ``scale`` and
    ``next_weight`` ``[channels]``; without ``gate`` or ``scale`` their factor is 1.
    ``n`` is computed from ``x_out`` before that is rounded, and has the branch's
    type.  Differentiable once.
    """

    if branch is None or weight is None:
        raise RuntimeError("residual_norm needs a branch and its weight.")
    out = _lib.torch_ext().residual_norm(x, branch, weight, gate, scale, next_weight, float(eps), None)
    return out[0] if next_weight is None else (out[0], out[1])

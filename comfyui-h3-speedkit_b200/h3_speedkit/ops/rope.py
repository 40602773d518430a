"""Rotary positions with several axes for Q and K, and the QKV op's table (B200).

Images and video place a token on a grid: ``positions`` [T, A] holds one coordinate
per axis (time, height, width, ...), INT32 or FP32 (fractional coordinates).
``sections`` gives the number of channel pairs that each axis turns; pair i of an axis
with n pairs turns by ``position * theta ** (-i / n)``:

    (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos)

The pairs are numbered axis after axis.  With P pairs in all, pair p is the channels
(p, P + p) of the head, or (2 p, 2 p + 1) with ``interleaved``; channels from 2 P on
pass (the partial split-half form of ``ops.qkv``: 96 of 128 channels).  A head's RMS
norm ``x * weight / sqrt(mean(x^2) + eps)`` may come first.  All in FP32 from the
stored inputs (heads whose squares pass its range taken smaller), rounded once; angles in 64
bits.

``rope_axes`` rotates Q and K (``inverse=True`` turns back: the transpose, which is
also the gradient of the rotation); ``rope_table`` makes the BF16 rotation rows that
``ops.qkv.QKV`` takes.  Both through libh3sk_b200.so; inference only.
"""
from __future__ import annotations

from functools import lru_cache

from .. import _lib


@lru_cache(maxsize=64)
def _axes(sections, theta):
    """Each pair's frequency and axis, made once for a model's sections."""
    if any(type(n) is not int for n in sections):
        raise ValueError('sections requires the pairs of each axis, whole numbers from 0')
    return _lib.binding().Axes(sections, theta if isinstance(theta, tuple) else (theta,) * len(sections))


def rope_axes(q, k, positions, *, sections, theta=10000.0, interleaved=False, inverse=False, q_weight=None,
              k_weight=None, eps=1e-6, q_out=None, k_out=None):
    """Q and K (k may be None) turned to their positions; returns (q_out, k_out).

    q [T, Hq, D], k [T, Hk, D]: BF16 or FP16, unit channel stride, any token and head
    strides (slices of one projection are taken as they are), D even up to 256, T from
    0.  q_weight, k_weight: [D] norm weights of q's type or FP32, both or neither.
    q_out, k_out: where to write, q and k themselves for in place; new contiguous
    tensors by default."""
    axes = _axes(tuple(sections), tuple(theta) if isinstance(theta, (tuple, list)) else theta)
    return _lib.binding().rope_axes(q, k, positions, axes, interleaved, inverse, q_weight, k_weight, eps, q_out, k_out)


def rope_table(positions, *, sections, theta=10000.0, out=None):
    """The rotations of every token as BF16 [1, T, 1, P, 2, 2] rows
    ((cos, -sin), (sin, cos)): the ``rope`` operand of ``ops.qkv.QKV`` (with 48 pairs)."""
    axes = _axes(tuple(sections), tuple(theta) if isinstance(theta, (tuple, list)) else theta)
    return _lib.binding().rope_table(positions, axes, out)

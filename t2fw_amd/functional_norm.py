"""The residual's addition and the root-mean-square norm of the stream, in one pass, with gradients or with 8-bit results
(csrc/rmsnorm.hip).  The reference leaves the layers around its recurrence to the caller (README.md:32)."""
from . import _lib
from .functional_scan import _stream


def residual_rms_norm(x, residual, weight, eps=1e-6):
    """``stored = x + residual`` and ``y = weight * stored / sqrt(mean(stored ** 2) + eps)`` over the last axis; returns
    ``(y, stored)``.

    ``x: [..., D]``; ``residual`` has its shape and its type, or float32 next to 16-bit tensors (a stream that is carried in
    32 bits); ``weight: [D]`` has the type of ``x`` or float32.  ``stored`` is rounded to the stream's type, and the norm is that
    of the rounded stream: the one that the backward, and the next layer, read.  ``residual=None``: the norm of ``x`` alone, and
    ``stored`` is ``x``.  The gradient of ``weight`` is summed in a fixed order (float32)."""
    y, stored = _lib.host().residual_rms_norm(x, residual, weight, eps, _stream(x))
    return y, x if stored is None else stored


def residual_rms_norm_fp8(x, residual, weight, eps=1e-6, group=0):
    """The same without gradients and with ``y`` in 8 bits, for a product with 8-bit operands: ``(q, scales, stored)``, ``q`` of
    torch.float8_e4m3fn, with ``y`` = ``q * scales``.  ``group=0``: one scale for a row (``scales: [..., 1]``); a power of two from 8
    to 512: one for that many columns (``scales: [..., ceil(D / group)]``).  A scale is the largest ``|y|`` over 448, the largest number
    of the format, and 1 where all ``y`` are zero; a NaN or an infinity makes NaN of what shares its scale."""
    q, scales, stored = _lib.host().residual_rms_norm_fp8(x, residual, weight, eps, group, _stream(x))
    return q, scales, x if stored is None else stored

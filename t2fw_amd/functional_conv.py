"""The causal convolution of a few taps per channel, which a selective scan's inputs come from (csrc/short_conv.hip).  The reference leaves the
layers around its recurrence to the caller (README.md:32)."""
from . import _lib
from .functional_scan import _stream


def short_conv(x, weight, bias=None, state=None, lengths=None, silu=False):
    """``y_t = bias + sum_j weight[:, j] x_{t - taps + 1 + j}`` per channel, or ``silu`` of that; returns ``(y [B, T, D], last inputs
    [B, taps - 1, D])``, with gradients.

    ``x: [B, T, D]`` (float32, float16 or bfloat16), with its channels next to each other in memory and any strides between rows and steps.
    ``weight: [D, taps]`` with 2 to 8 taps (``weight[:, 0]`` of a depthwise ``Conv1d``) and ``bias: [D]`` have the type of ``x`` or float32.
    ``state: [B, taps - 1, D]``: the inputs before the first, oldest first (``None``: zeros), of the type of ``x``, as are the last inputs: what the
    next call takes as its state.  Sums are float32; those of the weights' gradient over rows and steps are made in a fixed order.

    ``lengths: [B]`` (int32 or int64, on the device), for rows that are padded at their end: steps from ``lengths[b]`` on do not count, whatever
    they hold, NaN included.  Their outputs and gradients are zero, and the last inputs of the row are those before its end."""
    return _lib.host().short_conv(x, weight, bias, state, lengths, silu, _stream(x))


def short_conv_step(x, weight, state, bias=None, silu=False, out=None, inplace=True):
    """One token of ``short_conv`` without gradients: ``x: [B, D]``, whose rows may be apart (part of a projection); ``state: [B, taps - 1, D]`` is
    moved on by one step in place unless ``inplace=False``.  Returns ``(y [B, D], state)``."""
    return _lib.host().short_conv_step(x, weight, state, bias, silu, out, inplace, _stream(x))

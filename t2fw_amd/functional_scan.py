"""The recurrence with a vector for its state, per channel ``h_t = f_t h_{t-1} + x_t``: the layer that stands next to the rules
with a matrix for their state (functional_lfw.py, functional_dfw.py), backed by the HIP kernels of csrc/gscan.hip.  The reference
has nothing of the kind; its decay rule with one key channel, query and key one (t2fw/torch.py:21-29), is this recurrence."""
import torch

from . import _lib


def _stream(x, name="x"):
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if not x.is_cuda:
        raise RuntimeError("%s must be a CUDA tensor" % name)
    return _lib.current_stream(x.device)


def gated_scan(x, f, state=None, lengths=None, logits=False):
    """``h_t = f_t h_{t-1} + x_t`` over a sequence; returns ``(h [B, T, D], last state [B, D])``, with gradients.

    ``x, f: [B, T, D]`` (float32, float16, bfloat16 or float64; one type), with their channels next to each other in memory and any
    strides between rows and steps: parts of a projection need not be copied.  ``state: [B, D]``, the state before the first step
    (``None``: zeros), and the last state are float32 (float64 for float64 tensors) whatever the type of ``x``: a state
    that takes up thousands of steps is not rounded between calls.  Gates may be any numbers, but their products over the steps of a sequence
    have to stay finite: stretches are put together by them, and an infinite one makes NaN even of a state of zero.  So does, next to an
    infinite state or step, a product too small for the accumulators' type, where the recurrence step by step would stay infinite.
    ``logits=True``: ``f`` holds gate logits, the gate is their sigmoid, and the gradient that comes back is the logits'.

    ``lengths: [B]`` (int32 or int64, on the device), for rows that are padded at their end: steps from ``lengths[b]`` on do not count,
    whatever they hold, NaN included.  Their outputs and gradients are zero, and the last state of the row is that after its last
    step (``state`` for a length of zero)."""
    return _lib.host().gated_scan(x, f, state, lengths, logits, _stream(x))


def gated_scan_step(x, f, state, logits=False, out=None, inplace=True):
    """One token of ``gated_scan`` without gradients: ``x, f: [B, D]``; ``state: [B, D]`` (float32, or float64 for float64
    tensors) is updated in place unless ``inplace=False``.  Returns ``(h [B, D], state)``."""
    return _lib.host().gated_scan_step(x, f, state, out, logits, inplace, _stream(x))

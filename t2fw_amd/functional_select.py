"""The selective state space scan: per channel a vector of states whose decays, inputs and outputs each step chooses (csrc/select_fwd.hip,
csrc/select_bwd.hip).  Its decay ``exp(dt_t a)`` is no product of a gate per channel and one per state, so it is not the reference's rule
(t2fw/torch.py:21-29); it stands next to it, as ``gated_scan`` does."""
from . import _lib
from .functional_scan import _stream


def selective_scan(x, dt, a, b, c, state=None, skip=None, gate=None, dt_bias=None, lengths=None, softplus=False):
    """``h_t = exp(dt_t a) h_{t-1} + dt_t x_t b_t`` per channel and state and ``y_t = <c_t, h_t> + skip x_t``, times ``silu(gate_t)`` where there is a
    gate; returns ``(y [B, T, D], last state [B, D, N])``, with gradients.

    ``x, dt, gate: [B, T, D]`` and ``b, c: [B, T, N]`` (float32, float16 or bfloat16; one type), with their channels next to each other in
    memory and any strides between rows and steps: parts of a projection need not be copied.  ``a: [D, N]`` with 1 to 64 states, ``skip, dt_bias:
    [D]``, ``state: [B, D, N]``, the state before the first step (``None``: zeros), and the last state are float32.  ``dt_bias`` is added to
    ``dt``; ``softplus=True``: the step's length is ``log(1 + exp(dt + dt_bias))``, and the gradient that comes back is that of ``dt``.

    The decays over the steps of a row are put together by ``exp(a * sum of dt)``, which has to stay finite: where ``dt * a <= 0``, as it
    is meant, it always does.  Next to an infinite state or input such a product that is too small for float32 makes NaN, where the recurrence step by step
    would stay infinite.  States and sums are float32; sums over channels and rows are made in a fixed order.  A decay is off by its exponent's three
    roundings, 2^-22 of ``dt a``, and by 2^-22; a step by the softplus by 2^-20 of its length.

    For the gradients the forward keeps a state every 16 steps (N / 4 bytes a channel and step), and the backward takes scratch for those of ``b`` and ``c``: per channel
    and step 2 bytes with 9 to 16 states, 8 with 17 to 32, 32 with more.

    ``lengths: [B]`` (int32 or int64, on the device), for rows that are padded at their end: steps from ``lengths[b]`` on do not count, whatever
    they hold, NaN included.  Their outputs and gradients are zero, and the last state of the row is that after its last step."""
    return _lib.host().selective_scan(x, dt, a, b, c, state, skip, gate, dt_bias, lengths, softplus, _stream(x))


def selective_scan_step(x, dt, a, b, c, state, skip=None, gate=None, dt_bias=None, softplus=False, out=None, inplace=True):
    """One token of ``selective_scan`` without gradients: ``x, dt, gate: [B, D]``, ``b, c: [B, N]``, whose rows may be apart (parts of a projection);
    ``state: [B, D, N]`` float32 is updated in place unless ``inplace=False``.  Returns ``(y [B, D], state)``."""
    return _lib.host().selective_scan_step(x, dt, a, b, c, state, skip, gate, dt_bias, softplus, out, inplace, _stream(x))

"""The 2-norm over all gradients of a model, and their clipping (csrc/clip.hip): two launches for up to 144 tensors, and no
synchronisation: the norm stays on the device."""
from . import _lib
from .functional_scan import _stream


def _first(tensors):
    tensors = [tensors] if hasattr(tensors, "is_cuda") else list(tensors)
    if not tensors:
        raise RuntimeError("t2fw: no gradients")
    return tensors, _stream(tensors[0], "every gradient")


def clip_grad_norm(grads, max_norm, out=None):
    """Multiplies ``grads`` (a list of tensors, ``[p.grad for p in model.parameters() if p.grad is not None]``) by
    ``min(1, max_norm / (norm + 1e-6))``, ``norm`` being the 2-norm of all of them together, and returns the norm as it was before, a
    float32 scalar on the device.  In place, or into ``out``, a list of tensors of the same shapes and any type (float32
    gradients for the optimizer from 16-bit ones).  Types may be mixed.  What is written may share memory with nothing else of the call: a tensor that is
    in the list twice is refused.  Within the limit gradients in place are not touched.  Norm and factor
    are computed in float64: gradients whose norm is above the largest float32 are scaled as others are, while the norm returned is
    infinite.  An infinite gradient (or squares beyond float64) makes zeros of the finite ones and NaN of the infinite ones, a NaN makes NaN of
    all of them."""
    grads, stream = _first(grads)
    return _lib.host().clip_grad_norm(grads, max_norm, out, stream)[0]


def grad_norm(grads):
    """The 2-norm of all tensors of ``grads`` together, a float32 scalar on the device."""
    grads, stream = _first(grads)
    return _lib.host().clip_grad_norm(grads, 0.0, False, stream)[0]

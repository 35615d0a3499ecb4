"""The clipped policy loss with a KL term on the logits of a model's tokens, with its gradient (csrc/policy_loss.hip): what a
pre-trained model with fast-weight layers is fine-tuned on once it answers.  The reference stops at its autograd function
(README.md:32)."""
from . import _lib
from .functional_scan import _stream


def policy_loss(logits, targets, old_logp, ref_logp, advantages, mask=None, clip=(0.2, 0.2), kl_coef=0.0, scale=1.0):
    """Returns ``(loss, logp)``: a float32 scalar, and the float32 log probabilities of the targets (no gradient).

    With ``logp = log_softmax(logits)[target]``, ``r = exp(logp - old_logp)`` and ``d = ref_logp - logp``::

        loss = scale * mean over the mask's tokens of  -min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_coef (exp(d) - 1 - d)

    ``logits: [..., V]`` float32, float16 or bfloat16; ``targets`` int64, ``old_logp, ref_logp, advantages`` float32 and ``mask`` bool,
    each of the shape of the tokens.  With ``kl_coef=0`` the values of ``ref_logp`` are not looked at: any tensor of that shape will do.
    No token in the mask: the loss is zero.  A target outside the vocabulary is for tokens
    outside the mask (``logp`` is 0 there); inside it makes the loss NaN.

    Float32 and bfloat16 logits: the forward writes their gradient in the pass that reads them, for a loss that is
    differentiated with a gradient of one (an array of the logits' size, held until the backward takes it), and the backward recomputes
    it for another.  So pass the factor of an accumulated
    or scaled loss as ``scale`` rather than multiply the loss.  Float16: the backward makes the gradient, whatever the loss is multiplied by."""
    low, high = clip
    return _lib.host().policy_loss(logits, targets, old_logp, ref_logp, advantages, mask, 1.0 - low, 1.0 + high, kl_coef, scale,
                                   _stream(logits, "logits"))

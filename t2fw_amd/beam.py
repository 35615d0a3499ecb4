"""Beam search over models whose memory is a state: the best continuations of all beams, and the states moved to the beams that go on from them
(csrc/beam.hip).  The reference has no generation but a benchmark's loop (tests/benchmark.py:104-105)."""
from . import _lib
from .functional_scan import _stream


def beam_select(logits, scores, count=None, finished=None, pad=0):
    """The ``count`` best continuations of each request over all its beams and the vocabulary; returns ``(scores [B, count] float32,
    beams [B, count] int64, tokens [B, count] int64)``, best first.

    A continuation of beam ``k`` by token ``v`` has the score ``scores[k] + log_softmax(logits[k])[v]``.
    ``logits: [B, K, V]``, contiguous, float32, float16 or bfloat16, with up to 256 beams; ``scores: [B, K]`` float32; ``count`` is at most 128
    (``None``: K).  The first step, when all beams are the same prompt: scores of zero for one of them and minus infinity for the others.

    ``finished: [B, K]`` bool: a beam that has ended goes on with the token ``pad`` alone, at its own score.  Scores are compared in float64, from sums of
    float32 exponentials (off by up to 2^-19: candidates of different beams nearer than twice that may change places).  Of equal scores the lower beam comes first,
    within a beam the larger logit, then the lower token: next to a score of -1e30, say, all tokens' scores are equal, and they still come by their logits.

    What cannot be (logits or scores of minus infinity, other tokens of an ended beam, a beam with NaN or plus infinity among its logits) has a
    score of minus infinity and comes last, by its index ``k V + v``; of a beam with NaN or plus infinity in no order that is promised.
    No gradients."""
    return _lib.host().beam_select(logits, scores, count, finished, pad, _stream(logits, "logits"))


def reorder_beams(arrays, beams, out=None):
    """Moves what belongs to beams to the beams that go on from them: ``new[b, k] = old[b, beams[b, k]]`` for every tensor of ``arrays``, and
    returns them.  ``beams: [B, K]`` int64, up to 64 beams; tensors of any type, contiguous, whose first axis is ``B * K`` or a multiple (heads of a
    beam next to each other): states of layers, tokens so far.  In place (a beam that goes on from itself is not touched), or into ``out``, tensors of the same shapes and
    types.  What is written may share memory with nothing else of the call.  One launch for up to 96 tensors.  An index outside ``[0, K)`` stands for
    the beam itself.  No gradients."""
    arrays = [arrays] if hasattr(arrays, "is_cuda") else list(arrays)
    if out is not None:
        out = [out] if hasattr(out, "is_cuda") else list(out)
    _lib.host().reorder_beams(arrays, beams, out, _stream(beams, "beams"))
    return arrays if out is None else out

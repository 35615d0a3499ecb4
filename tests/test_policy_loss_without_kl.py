"""policy_loss with a KL coefficient of zero, the default: the reference's log probabilities are nothing to it, whatever they are.
The bounds are those of test_policy_loss.py."""
import pytest
import torch

from tests.test_policy_loss import CLIP, DTYPES, check, inputs, reference


def run(ins, factor=1.0):
    import t2fw_amd as t2
    z = ins[0].detach().requires_grad_(True)
    loss, logp = t2.policy_loss(z, *ins[1:5], mask=ins[5], clip=CLIP)
    grad, = torch.autograd.grad(loss * factor, z)
    return loss.detach(), logp, grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(9, 40), (5, 3001), (3, 140000)], ids=str)
def test_tokens_far_less_likely_than_the_placeholder(shape, dtype):
    """zeros for a reference that there is none of, next to tokens of log probabilities below -100: exp(ref - logp) is beyond float32"""
    ins = inputs(*shape, dtype, seed=shape[1])
    z, targets, old, ref, mask = ins[0], ins[1], ins[2], ins[3], ins[5]
    rows = torch.arange(0, shape[0], 2, device="cuda")
    z[rows, targets[rows]] = -150.0
    mask[rows] = True
    logp = torch.log_softmax(z.double(), 1).gather(1, targets[:, None])[:, 0]
    old.copy_(logp + 0.05)
    ref.zero_()
    assert float(logp.min()) < -100
    want = reference(*ins, kl=0.0)
    assert bool(torch.isfinite(want["loss"][0])) and bool(torch.isfinite(want["grad"][0]).all())
    got = run(ins)
    for n, v in zip(("loss", "logp", "grad"), got):
        check(n, v, want[n])
    # the gradient that the backward makes, for another gradient of the loss than one
    check("grad", run(ins, 0.5)[2], reference(*ins, kl=0.0, scale=0.5)["grad"])
    for placeholder in (float("nan"), float("inf"), float("-inf"), 3e38, 12.5):
        ref.fill_(placeholder)
        assert all(torch.equal(a, b) for a, b in zip(run(ins), got)), placeholder


@pytest.mark.gpu
def test_a_target_that_is_ruled_out():
    """a logit of minus infinity: its ratio is zero, and the loss without a KL term finite"""
    ins = inputs(4, 300, torch.float32, seed=2)
    z, targets, old, ref, adv, mask = ins
    mask[:] = True
    z[1, targets[1]] = float("-inf")
    adv[1] = 0.7
    loss, logp, grad = run(ins)
    assert float(logp[1]) == float("-inf") and bool(torch.isfinite(loss)) and bool((grad[1] == 0).all())
    kept = torch.tensor([0, 2, 3], device="cuda")
    want = reference(*[t[kept] for t in ins], kl=0.0, scale=0.75)
    check("loss", loss, want["loss"])
    check("grad", grad[kept], want["grad"])

"""The operators around the recurrences under torch's other ways to differentiate and transform a call: what they do not have is refused,
never left out."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def ones(*s, dtype=torch.float32):
    return torch.ones(s, device="cuda", dtype=dtype)


def calls():
    """name -> (call, floating-point inputs)"""
    import t2fw_amd as t2
    targets = torch.zeros(4, dtype=torch.int64, device="cuda")
    return {
        "gated_scan": (lambda x, f, s: t2.gated_scan(x, f, s), [ones(2, 5, 8), ones(2, 5, 8), ones(2, 8)]),
        "gated_scan_step": (lambda x, f, s: t2.gated_scan_step(x, f, s), [ones(2, 8), ones(2, 8), ones(2, 8)]),
        "residual_rms_norm": (lambda x, r, w: t2.residual_rms_norm(x, r, w), [ones(4, 16), ones(4, 16), ones(16)]),
        "residual_rms_norm_fp8": (lambda x, r, w: t2.residual_rms_norm_fp8(x, r, w), [ones(4, 16), ones(4, 16), ones(16)]),
        "policy_loss": (lambda z, o, r, a: t2.policy_loss(z, targets, o, r, a), [ones(4, 9), ones(4), ones(4), ones(4)]),
        "clip_grad_norm": (lambda g, h: t2.clip_grad_norm([g, h], 1.0), [ones(5), ones(3, 3)]),
        "grad_norm": (lambda g, h: t2.grad_norm([g, h]), [ones(5), ones(3, 3)]),
        "clip_grad_norm into others": (lambda g, o: t2.clip_grad_norm([g], 1.0, out=[o]), [ones(5), ones(5)]),
        "gated_scan_step into another": (lambda x, o: t2.gated_scan_step(x, x, x.clone(), out=o), [ones(2, 8), ones(2, 8)]),
    }


NAMES = ["gated_scan", "gated_scan_step", "residual_rms_norm", "residual_rms_norm_fp8", "policy_loss", "clip_grad_norm", "grad_norm",
         "clip_grad_norm into others", "gated_scan_step into another"]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name, grad):
    call, ins = calls()[name]
    with forward_ad.dual_level():
        for i in range(len(ins)):
            duals = [t.clone() for t in ins]
            if grad and name in ("gated_scan", "residual_rms_norm"):
                duals[i].requires_grad_(True)
            duals[i] = forward_ad.make_dual(duals[i], torch.ones_like(ins[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*duals)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(*duals)
            # as in an autograd function's own forward, which brings its derivative itself
            with torch.no_grad(), forward_ad._set_fwd_grad_enabled(False):
                call(*duals)
        call(*[t.clone() for t in ins])


@pytest.mark.parametrize("name", NAMES)
def test_transformed_and_fake_tensors_are_refused(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    call, ins = calls()[name]
    with pytest.raises(RuntimeError):
        torch.vmap(call)(*[torch.stack((t, t)) for t in ins])
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, tuple(ins), tuple(torch.ones_like(t) for t in ins))
    with FakeTensorMode() as mode, pytest.raises(RuntimeError):
        call(*[mode.from_tensor(t) for t in ins])

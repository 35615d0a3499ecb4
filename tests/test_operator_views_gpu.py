"""The operators around the recurrences on tensors whose memory does not hold their values as they are: views that torch negates when it reads
them (the imaginary part of a conjugate), as inputs and as gradients, and sparse ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def negated(t):
    """-t, as a view of t"""
    v = torch._neg_view(t)
    assert v.is_neg() and v.data_ptr() == t.data_ptr()
    return v


def rand(*s, seed=0):
    return torch.randn(s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def calls():
    import t2fw_amd as t2
    targets = torch.tensor([1, 0, 3], device="cuda")
    return {
        "gated_scan": (lambda x, f, s: t2.gated_scan(x, f, s), [rand(2, 5, 8), rand(2, 5, 8), rand(2, 8)]),
        "gated_scan_step": (lambda x, f, s: t2.gated_scan_step(x, f, s), [rand(2, 8), rand(2, 8), rand(2, 8)]),
        "residual_rms_norm": (lambda x, r, w: t2.residual_rms_norm(x, r, w), [rand(4, 16), rand(4, 16), rand(16)]),
        "residual_rms_norm_fp8": (lambda x, r, w: t2.residual_rms_norm_fp8(x, r, w), [rand(4, 16), rand(4, 16), rand(16)]),
        "policy_loss": (lambda z, o, r, a: t2.policy_loss(z, targets, o, r, a), [rand(3, 9), rand(3), rand(3), rand(3)]),
        "clip_grad_norm": (lambda g, h: t2.clip_grad_norm([g, h], 1.0), [rand(5), rand(3, 3)]),
        "clip_grad_norm into others": (lambda g, o: t2.clip_grad_norm([g], 1.0, out=[o]), [rand(5), rand(5)]),
        "gated_scan_step into another": (lambda x, o: t2.gated_scan_step(x, x, x.clone(), out=o), [rand(2, 8), rand(2, 8)]),
    }


@pytest.mark.parametrize("name", ["gated_scan", "gated_scan_step", "residual_rms_norm", "residual_rms_norm_fp8", "policy_loss", "clip_grad_norm",
                                  "clip_grad_norm into others", "gated_scan_step into another"])
def test_negated_views_and_sparse_tensors_are_refused(name):
    call, ins = calls()[name]
    call(*[t.clone() for t in ins])
    for i in range(len(ins)):
        for other in (negated(ins[i].clone()), ins[i].to_sparse()):
            with pytest.raises(RuntimeError):
                call(*[t.clone() for t in ins[:i]], other, *[t.clone() for t in ins[i + 1:]])


def test_gradients_that_are_negated_views():
    import t2fw_amd as t2
    targets, per = torch.tensor([1, 0, 3], device="cuda"), rand(3, seed=1)
    cases = [(lambda *a: t2.gated_scan(*a), [rand(2, 300, 8), rand(2, 300, 8).sigmoid(), rand(2, 8)]),
             (lambda *a: t2.gated_scan(*a), [rand(2, 300, 1), rand(2, 300, 1).sigmoid(), rand(2, 1)]),
             (lambda *a: t2.residual_rms_norm(*a), [rand(4, 16), rand(4, 16), rand(16)]),
             (lambda z: t2.policy_loss(z, targets, per, per, per, kl_coef=0.1)[:1], [rand(3, 9)]),
             (lambda z: t2.policy_loss(z.half(), targets, per, per, per)[:1], [rand(3, 9)])]
    for call, ins in cases:
        ins = [t.requires_grad_(True) for t in ins]
        outs = call(*ins)
        grads = [torch.randn_like(o) for o in outs]
        want = torch.autograd.grad(outs, ins, [-g for g in grads], retain_graph=True)
        got = torch.autograd.grad(outs, ins, [negated(g) for g in grads])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # as they come about: a result that is the imaginary part of a conjugate
    x = rand(2, 40, 1).requires_grad_(True)
    h, _ = t2.gated_scan(x, torch.full_like(x, 0.5))
    got, = torch.autograd.grad(torch.complex(torch.zeros_like(h), h).conj().imag.sum(), x, retain_graph=True)
    want, = torch.autograd.grad(-h.sum(), x)
    assert torch.equal(got, want)

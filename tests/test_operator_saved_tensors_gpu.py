"""The operators around the recurrences under hooks on what their nodes save: it may come back in another order of memory, and nothing of
other sizes or types is handed to a kernel."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ones(*s):
    return torch.ones(s, device="cuda")


def spread(t):
    """the same values, every second element of twice the memory"""
    return torch.stack((t, t), -1)[..., 0]


@pytest.mark.parametrize("unpack", [lambda t: t.cuda(), lambda t: spread(t.cuda())], ids=["host", "spread"])
def test_saved_tensors_that_come_back_in_another_order(unpack):
    import t2fw_amd as t2
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    lengths, targets = torch.tensor([700, 300], device="cuda"), torch.randint(0, 50, (6,), device="cuda", generator=g)
    per = [rand(6) for _ in range(3)]
    x, f, s = rand(2, 700, 24), rand(2, 700, 24), rand(2, 24)
    y, r, w = rand(40, 70), rand(40, 70), rand(70)
    z = rand(6, 50)
    cases = [(lambda *a: t2.gated_scan(*a, lengths=lengths, logits=True), (x, f, s)), (lambda *a: t2.residual_rms_norm(*a), (y, r, w)),
             (lambda a, b: t2.residual_rms_norm(a, None, b), (y, w)),
             (lambda a: t2.policy_loss(a, targets, *per, kl_coef=0.1)[:1], (z,)), (lambda a: t2.policy_loss(a.half(), targets, *per)[:1], (z,))]
    for call, ins in cases:
        ins = [t.requires_grad_(True) for t in ins]

        def grads():
            outs = [o for o in call(*ins) if o.requires_grad]
            return torch.autograd.grad([o.float().square().sum() for o in outs], ins)
        want = grads()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), unpack):
            got = grads()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_tensors_of_other_types_and_sizes_are_refused():
    import t2fw_amd as t2
    x, w, z = ones(2, 6, 8), ones(8), ones(4, 9)
    per, targets = ones(4), torch.zeros(4, dtype=torch.int64, device="cuda")
    cases = [(lambda: t2.gated_scan(x, x)[0], x), (lambda: t2.residual_rms_norm(x, x, w)[0], w),
             (lambda: t2.policy_loss(z, targets, per, per, per)[0], z)]
    for leaf in (x, w, z):
        leaf.requires_grad_(True)
    for call, leaf in cases:
        for unpack in (lambda t: t.double() if t.is_floating_point() else t.int(), lambda t: t[..., :1], lambda t: t.cpu(),
                       lambda t: t[:1] if t.dim() else t):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                out = call()
                with pytest.raises(RuntimeError):
                    torch.autograd.grad(out.sum(), leaf)

"""clip_grad_norm on tensors that share memory: many workgroups write at once, so a place that two results claim, or that one gradient is still
read from while another's result is written, would hold whatever came last."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def flat(n=1000, dtype=torch.float32):
    return torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype).cuda()


def test_results_that_share_memory_are_refused():
    import t2fw_amd as t2
    a, b = flat(), flat(500)
    kept = a.clone(), b.clone()
    half = a.view(torch.float16)[:1000]
    cases = [([a, a], None), ([a, b, a], None), ([a, a[10:20]], None), ([b, a[:600], a[599:]], None), ([a, a.view(10, 100).t()], None),
             ([b, b.clone()], [a[:500], a[499:999]]), ([a, b], [b.new_empty(1000), a[:500]]), ([a[:500], b], [a[1:501], b]),
             ([half], [a]), ([a], [half]), ([a[:999]], [a[1:]])]
    for grads, out in cases:
        with pytest.raises(RuntimeError, match="share"):
            t2.clip_grad_norm(grads, 1.0, out=out)
    assert torch.equal(a, kept[0]) and torch.equal(b, kept[1])


def test_neighbours_read_only_repeats_and_empty_tensors_are_not():
    import t2fw_amd as t2
    a, b = flat(), flat(500)
    norm = float(torch.cat((a, a, b)).double().norm())
    assert abs(float(t2.grad_norm([a, a, b])) / norm - 1) < 1e-6                # nothing is written
    out = [torch.empty_like(t) for t in (a, a, b)]
    t2.clip_grad_norm([a, a, b], norm / 2, out=out)
    for o, t in zip(out, (a, a, b)):
        assert torch.allclose(o, t / 2, rtol=1e-6)
    parts, want = [a[600:], a[:300], a[300:600], a[300:300], a[:0]], a / 2
    t2.clip_grad_norm(parts, float(a.double().norm()) / 2)                       # neighbours in any order
    assert torch.allclose(a, want, rtol=1e-6)
    t2.clip_grad_norm([a[:500], b], 1e9, out=[a[:500], a[500:]])                 # in place for one, next to it for the other
    assert torch.equal(a[500:], b)

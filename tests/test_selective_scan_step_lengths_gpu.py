"""The softplus of the selective scan's steps, and its slope, to their last bits over all of its range.

Bounds, u = 2^-24.  The exponential e = e^-|v| = 2^n e^(-|v| - n log 2): the hardware's last place, 2 u, the remainder's factor, u, and log 2 as a float32 number, 2^-28.4 |n log 2|,
4 u at most.  e / (2 + e) = r: a sum, a reciprocal to its last place, a product, 4 u.  The series: cut at u / 4, one rounding where its terms count, the last multiply-add:
14 u in all, less than 2^-20 of the step.  Its slope, e / (1 + e) or 1 / (1 + e): the same without the series.  Below -86 e is next to the smallest normal number."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def steps(dtype):
    v = torch.cat((torch.linspace(-86, 20, 4001), torch.linspace(-1, 1, 513), torch.linspace(20, 300, 100), -torch.logspace(-30, 1.9, 300))).to(dtype).cuda()
    return v[None, None], torch.nn.functional.softplus(v.double(), threshold=1e9)[None, None]


def call(v, dtype, f):
    """x, b, c and the decays of one: the state is the step"""
    D = v.shape[-1]
    one = torch.ones_like(v)
    return f(one, v, torch.zeros(D, 1, device="cuda"), torch.ones_like(one[..., :1]), torch.ones_like(one[..., :1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_steps_of_any_length(dtype):
    import t2fw_amd as t2
    v, want = steps(dtype)
    assert bool((want > 0).all())
    with torch.no_grad():
        y, last = call(v, dtype, lambda *a: t2.selective_scan(*a, softplus=True))
    off = (last[:, :, 0].double() / want[0] - 1).abs()
    assert float(off.max()) <= 2.0 ** -20, float(off.max()) * 2 ** 20
    state = torch.zeros(1, v.shape[-1], 1, device="cuda")
    with torch.no_grad():
        call(v[:, 0], dtype, lambda x, dt, a, b, c: t2.selective_scan_step(x, dt, a, b, c, state, softplus=True))
    assert float((state[:, :, 0].double() / want[0] - 1).abs().max()) <= 2.0 ** -20
    if dtype == torch.float32:
        assert torch.equal(y[:, 0], last[..., 0])


def test_slopes_of_any_step():
    import t2fw_amd as t2
    v, _ = steps(torch.float32)
    v = v.requires_grad_(True)
    y, _ = call(v, torch.float32, lambda *a: t2.selective_scan(*a, softplus=True))
    slope, = torch.autograd.grad(y.sum(), v)
    want = torch.sigmoid(v.detach().double())
    assert float((slope.double() / want - 1).abs().max()) <= 2.0 ** -20


def test_a_bias_and_steps_that_are_none():
    """dt + bias is one float32 sum; what is below the smallest number is no step, and a very long one is itself"""
    import t2fw_amd as t2
    v = torch.tensor([-104.0, -1000.0, -3e38, -float("inf"), 3e38], device="cuda")[None, None]
    with torch.no_grad():
        _, last = call(v, torch.float32, lambda *a: t2.selective_scan(*a, softplus=True))
        assert last[0, :, 0].tolist() == [0.0, 0.0, 0.0, 0.0, float(v[0, 0, 4])]
        y, last = call(torch.full((1, 1, 3), float("nan"), device="cuda"), torch.float32, lambda *a: t2.selective_scan(*a, softplus=True))
        assert bool(torch.isnan(last).all()) and bool(torch.isnan(y).all())
        v, want = steps(torch.float32)
        bias = torch.full_like(v[0, 0], 0.5)
        _, last = call(v - 0.5, torch.float32, lambda *a: t2.selective_scan(*a, dt_bias=bias, softplus=True))
    raw = ((v - 0.5) + 0.5)[0]
    want = torch.nn.functional.softplus(raw.double(), threshold=1e9)
    assert float((last[..., 0].double() / want - 1).abs().max()) <= 2.0 ** -20

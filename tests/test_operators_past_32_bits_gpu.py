"""Arrays whose element offsets, or byte offsets, pass 32 bits: their ends against the same call on a part of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    yield
    torch.cuda.empty_cache()


def randn(*shape, dtype=torch.bfloat16, seed=0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=dtype)


def test_gated_scan():
    import t2fw_amd as t2
    T, D, near = 66000, 33000, 1300                     # 2.18e9 elements; gates of 0.8 forget within a few hundred steps
    x = randn(1, T, D).requires_grad_(True)
    gate = torch.full((1, 1, D), 0.8, device="cuda", dtype=torch.bfloat16)
    go = torch.ones(1, 1, D, device="cuda", dtype=torch.bfloat16)
    h, last = t2.gated_scan(x, gate.expand(1, T, D))
    dx, = torch.autograd.grad(h, x, go.expand(1, T, D))
    with torch.no_grad():
        end, end_last = t2.gated_scan(x[:, -near:].contiguous(), gate.expand(1, near, D))
    # (chunks lie otherwise, so the last bit may differ)
    assert torch.allclose(h[:, -300:].float(), end[:, -300:].float(), rtol=2.0 ** -7, atol=1e-4) and torch.allclose(last, end_last, rtol=1e-5, atol=1e-5)
    sums = 1 / (1 - 0.80078125)                          # 0.8 in bfloat16; the geometric series of an adjoint of ones
    assert torch.allclose(dx[:, :300].float(), torch.full_like(dx[:, :300], sums).float(), rtol=2.0 ** -7)
    assert torch.equal(dx[:, -1], go[:, 0]) and torch.allclose(dx[:, -2].float(), go[:, 0].float() * 1.80078125, rtol=2.0 ** -7)


def test_residual_rms_norm():
    import t2fw_amd as t2
    N, D, some = 525000, 4100, 8                        # 2.15e9 elements
    x, res, w = randn(N, D), randn(N, D, seed=1), torch.ones(D, device="cuda")
    small = [x[-some:].clone().requires_grad_(True), res[-some:].clone().requires_grad_(True), w]
    q, scales, stored8 = t2.residual_rms_norm_fp8(x, res, w)
    qs, ss, _ = t2.residual_rms_norm_fp8(x[-some:], res[-some:], w)
    assert torch.equal(q[-some:].view(torch.uint8), qs.view(torch.uint8)) and torch.equal(scales[-some:], ss)
    del q, scales, stored8
    y, stored = t2.residual_rms_norm(x.requires_grad_(True), res, w)
    ys, sts = t2.residual_rms_norm(*small)
    assert torch.equal(y[-some:], ys) and torch.equal(stored[-some:], sts)
    g = randn(1, D, seed=2)
    dx, = torch.autograd.grad(y, x, g.expand(N, D))
    dxs, = torch.autograd.grad(ys, small[0], g.expand(some, D))
    assert torch.equal(dx[-some:], dxs)


def test_policy_loss():
    import t2fw_amd as t2
    N, V, some = 43000, 50257, 16                       # 2.16e9 logits
    z = randn(N, V).requires_grad_(True)
    t = torch.randint(0, V, (N,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    per = torch.full((N,), -11.0, device="cuda")
    loss, logp = t2.policy_loss(z, t, per, per, torch.ones_like(per), clip=(1.0, 100.0))
    d, = torch.autograd.grad(loss, z)
    zs = z.detach()[-some:].clone().requires_grad_(True)
    s_loss, s_logp = t2.policy_loss(zs, t[-some:], per[-some:], per[-some:], torch.ones_like(per[-some:]), clip=(1.0, 100.0), scale=some / N)
    ds, = torch.autograd.grad(s_loss, zs)
    # (rows start at other places, so sums are put together otherwise)
    assert torch.allclose(logp[-some:], s_logp, atol=1e-5)
    assert torch.allclose(d[-some:].float(), ds.float(), rtol=2.0 ** -6, atol=0)


def test_clip_grad_norm():
    import t2fw_amd as t2
    n = (1 << 32) + 12345
    g = torch.ones(n, device="cuda", dtype=torch.float16)
    g[-5:] = 4096.0
    want = ((n - 5) + 5 * 4096.0 ** 2) ** 0.5
    assert abs(float(t2.grad_norm([g])) / want - 1) < 1e-6
    norm = t2.clip_grad_norm([g], want / 4)
    assert abs(float(norm) / want - 1) < 1e-6
    assert torch.equal(g[-8:], torch.tensor([0.25] * 3 + [1024.0] * 5, device="cuda", dtype=torch.float16)) and float(g[:1 << 20].amax()) == 0.25

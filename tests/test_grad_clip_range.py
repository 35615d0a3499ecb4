"""clip_grad_norm where 24 bits and float32's range do not do: float64 gradients, and norms above the largest float32.

Bounds: the sum of n squares in double is made of chains of at most a few hundred additions, so the norm is within 2^-45 of itself; the
factor and a product add three roundings of 2^-53."""
import math

import pytest
import torch

from tests.test_gated_scan import STORE, TINY


def make(n, dtype, seed, scale=1.0):
    return (torch.randn(n, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale).to(dtype).cuda()


def exact_norm(ts):
    return math.sqrt(math.fsum(v * v for t in ts for v in t.double().flatten().tolist()))


@pytest.mark.gpu
@pytest.mark.parametrize("most", [0.1, 3.7, 1e9])
def test_float64_gradients_keep_their_bits(most):
    import t2fw_amd as t2
    grads = [make(n, torch.float64, n) for n in (1, 4001, 30000)]
    before = [g.cpu() for g in grads]
    by = min(1.0, most / (exact_norm(before) + 1e-6))
    out = [torch.empty_like(g) for g in grads]
    t2.clip_grad_norm(grads, most, out=out)
    t2.clip_grad_norm(grads, most)
    for g, o, b in zip(grads, out, before):
        assert torch.equal(g, o)
        assert bool(((g.cpu() - b * by).abs() <= 2.0 ** -44 * (b * by).abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("to", [torch.float64, torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dtype,value", [(torch.float32, 3e38), (torch.bfloat16, 2.5e38), (torch.float64, 1e100)], ids=str)
def test_a_finite_norm_beyond_float32(dtype, value, to):
    """the norm that comes back is a float32, and infinite; what the gradients are multiplied by is not"""
    import t2fw_amd as t2
    g = make(3001, dtype, 5).clamp(-1.0, 1.0)
    g = (g.double() * value).to(dtype)
    before = g.double().cpu()
    norm = exact_norm([g.cpu()])
    assert 3.5e38 < norm < math.inf
    for most in (1.0, 60000.0):
        out = torch.empty(g.shape, dtype=to, device="cuda")
        got = t2.clip_grad_norm([g], most, out=[out])
        assert got.dtype == torch.float32 and math.isinf(float(got))
        want = before * (most / (norm + 1e-6))
        # the product is made in double, and then stored, 16-bit numbers by way of 32 bits
        bound = (2.0 ** -44 + STORE[to] + (2.0 ** -24 if STORE[to] > 2.0 ** -24 else 0)) * want.abs() + TINY[to]
        assert bool(((out.double().cpu() - want).abs() <= bound).all())
    # up to float32's largest the norm is what it was
    small = torch.full((4,), 1e38, device="cuda")
    assert abs(float(t2.clip_grad_norm([small], 1.0)) / 2e38 - 1) < 1e-6 and abs(float(small[0]) - 0.5) < 1e-6

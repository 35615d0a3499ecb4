"""The norm over more rows than one launch takes workgroups for: a grid has less than 2^32 threads along an axis."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    free, _ = torch.cuda.mem_get_info()
    if free < 30 << 30:
        pytest.skip("needs 30 GB of free device memory")
    yield
    torch.cuda.empty_cache()


def randn(*shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=dtype)


# a row to a workgroup of 256 threads, and 16 rows
@pytest.mark.parametrize("N,D", [((1 << 24) + 77, 3), ((1 << 28) + 77, 8)], ids=str)
def test_rows_of_every_part(N, D):
    """A row's result does not depend on the rows around it: parts of the rows, those at multiples of 2^22 among them, against calls of their own"""
    import t2fw_amd as t2
    x, w = randn(N, D, dtype=torch.bfloat16, seed=1), randn(D, dtype=torch.bfloat16, seed=2)
    res = randn(N, D, dtype=torch.bfloat16, seed=3)
    with torch.no_grad():
        y, stored = t2.residual_rms_norm(x, res, w)
        q, scales, stored8 = t2.residual_rms_norm_fp8(x, res, w)
        assert torch.equal(stored, x + res) and torch.equal(stored8.view(torch.int16), stored.view(torch.int16))
        starts = list(range(0, N, max(1 << 22, N // 64))) + [N - 3000]
        for at in starts:
            part = slice(max(at - 1000, 0), min(at + 3000, N))
            ys, _ = t2.residual_rms_norm(x[part], res[part], w)
            qs, ss, _ = t2.residual_rms_norm_fp8(x[part], res[part], w)
            assert torch.equal(y[part], ys) and torch.equal(scales[part], ss) and torch.equal(q[part].view(torch.uint8), qs.view(torch.uint8)), at
    grads = torch.autograd.grad(t2.residual_rms_norm(x.requires_grad_(True), res, w)[0], x, y)[0]
    part = slice(N - 1000, N)
    xs = x.detach()[part].clone().requires_grad_(True)
    assert torch.equal(grads[part], torch.autograd.grad(t2.residual_rms_norm(xs, res[part], w)[0], xs, y[part])[0])

"""Steps beyond a row's length have no gradient, whatever state the row ends in."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("N", [1, 6, 16, 30, 64])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_padding_of_rows_that_are_not_finite(bad, N, dtype):
    """a state, its gradient, or a step of its own"""
    import t2fw_amd as t2
    B, T, D = 5, 40, 9
    g = torch.Generator().manual_seed(N)
    make = lambda *s: torch.randn(*s, generator=g)
    x, dt, gate, gy = (make(B, T, D).to(dtype).cuda() for _ in range(4))
    b, c = (make(B, T, N).to(dtype).cuda() for _ in range(2))
    a, state, gs = -make(D, N).exp().cuda(), make(B, D, N).cuda(), make(B, D, N).cuda()
    lengths = torch.tensor([T, 5, 5, 21, 0], device="cuda")
    state[1] = bad
    state[4] = bad
    gs[2, :, N - 1] = bad
    x[3, 20, 2] = bad

    def run(rows):
        ins = [t[rows].detach().requires_grad_(True) for t in (x, dt, b, c, gate, state)]
        rest = a.detach().requires_grad_(True)
        out = t2.selective_scan(ins[0], ins[1], rest, ins[2], ins[3], state=ins[5], gate=ins[4], lengths=lengths[rows], softplus=True)
        return out + torch.autograd.grad(out, ins, (gy[rows], gs[rows]))
    got = run(torch.arange(B, device="cuda"))
    for row, n in enumerate(lengths.tolist()):
        for t in (got[0], *got[2:7]):
            assert not t[row, n:].any(), (row, t.shape)          # (NaN is true)
    # the row that is finite stays so
    assert all(bool(torch.isfinite(t[0]).all()) for t in got)

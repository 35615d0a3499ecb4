"""gated_scan with so many workgroups that they run in another order, and their maps in several groups of chunks: every element of every
result.  Logits of any size.  The bounds are those of test_gated_scan.py."""
import pytest
import torch

from tests.test_gated_scan import STORE, TINY, check, inputs, reference, run, unit

pytestmark = pytest.mark.gpu


# 65 x 33, 32 x 71 and 260 x 9 workgroups: more than 2048, and no whole number of rounds of 128; five, five and two groups of chunks
@pytest.mark.parametrize("shape,dtype,logits", [((8, 4100, 520), torch.bfloat16, True), ((2, 9000, 1021), torch.float32, False),
                                                ((16, 1100, 1035), torch.float16, True)], ids=str)
def test_every_element_and_without_one_another(shape, dtype, logits):
    from t2fw_amd import _lib
    B, T, D = shape
    ins, go, gs = inputs(*shape, dtype, logits, seed=T)
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(D))
    lengths[0] = T
    got = run(ins, lengths.cuda(), logits, go, gs)
    ref = reference(*ins, lengths, logits, unit(dtype, logits), go, gs)
    for n in ref:
        check(n, got[n], ref[n])
    del ref
    # the same bits where no chunk waits for another's map
    lib, (x, f, s), p = _lib.load(), ins, _lib.ptr
    lengths = lengths.cuda()
    code, st = _lib.DTYPE_CODE[dtype], _lib.current_stream_handle(x.device)
    nc, nw = lib.t2fw_gated_scan_checkpoint_bytes(B, T, D, code), lib.t2fw_gated_scan_workspace_bytes(B, T, D, code)
    out, last, dx, df, ds = torch.empty_like(x), torch.empty_like(s), torch.empty_like(x), torch.empty_like(x), torch.empty_like(s)
    ckpt, ws = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in (nc, nw))
    flags = 2 | 4 | (1 if logits else 0)
    _lib.check(lib.t2fw_gated_scan_forward(p(x), p(f), p(s), p(lengths), p(out), p(last), p(ckpt), B, T, D, None, code, flags, p(ws), nw, st))
    _lib.check(lib.t2fw_gated_scan_backward(p(go), p(gs), p(x), p(f), p(lengths), p(ckpt), p(dx), p(df), p(ds), B, T, D, None, code, flags, p(ws), nw, st))
    for n, v in zip(("h", "last", "d_x", "d_f", "d_state"), (out, last, dx, df, ds)):
        assert torch.equal(v, got[n]), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("shape", [(3, 1, 1024), (2, 1, 5)], ids=str)
def test_gates_and_slopes_of_logits_of_any_size(shape, dtype):
    """One step from a state of one, and its gradient: the gate and its slope by themselves, for logits from -40 to 40.  The hardware's exponential is that
    of two to the power of a product that 32 bits round: within |z| (2^-24 + 2^-26, of the factor) and 2^-22 of itself, and the reciprocal and the sum add
    2^-22; a slope has them twice.  The library's, for 32-bit logits, 2^-21 in all."""
    import t2fw_amd as t2
    g = torch.Generator().manual_seed(shape[2])
    z = (torch.rand(shape, generator=g) * 80 - 40).to(dtype)
    one = torch.ones(shape[0], shape[2])
    x, f, s = torch.zeros(shape, dtype=dtype).cuda(), z.cuda().requires_grad_(True), one.cuda()
    h, last = t2.gated_scan(x, f, s, logits=True)
    slope, = torch.autograd.grad(last, f, one.cuda())
    _, stepped = t2.gated_scan_step(x[:, 0], f.detach()[:, 0], s.clone(), logits=True)
    z64 = z.double()
    gate = torch.sigmoid(z64)
    u = 2.0 ** -21 + (z64.abs() * 1.25 * 2.0 ** -24 if dtype != torch.float32 else 0)
    for got, bound in ((last, 0), (stepped, 0), (h, STORE[dtype])):
        got = got.detach().double().cpu().view(shape)
        assert bool(((got - gate).abs() <= (u + bound) * gate + (TINY[dtype] if bound else 0)).all())
    want = gate * torch.sigmoid(-z64)
    assert bool(((slope.double().cpu() - want).abs() <= (2 * u + STORE[dtype]) * want + TINY[dtype]).all())

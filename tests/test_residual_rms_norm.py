"""residual_rms_norm and its 8-bit form against the formula in float64.

Bounds, u = 2^-24 (2^-53 for float64): a row's sum of squares is added up by at most 64 numbers after one another (16 to a lane,
then the lanes), its mean, root and reciprocal add 4: r is within 40 u of itself, y within 44 u before it is stored.  The
backward's sum is within 72 u of the sum of its absolute terms, d_x within 128 u of that of its own.  A weight's gradient adds up at most 160 numbers in
a row on top of the 44 u of each.  Storing rounds to half a unit in the last place."""
import pytest
import torch

from tests.test_gated_scan import STORE, TINY

U = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -24}
EPS = 1e-5
# (tokens' type, stream's, weight's)
TYPES = [(torch.float32,) * 3, (torch.float64,) * 3, (torch.float16,) * 3, (torch.bfloat16,) * 3, (torch.bfloat16, torch.float32, torch.float32),
         (torch.float16, torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16, torch.float32)]
# rows of less than a chunk, of one wave, of a workgroup, past what stays in registers; odd ones
SHAPES = [(1, 1), (3, 7), (5, 8), (2, 9), (7, 511), (130, 768), (33, 1021), (1, 1024), (3, 1025), (9, 2047), (2, 4096), (3, 5003), (2, 8192), (2, 8200), (3, 16384), (2, 16390), (9, 100), (65, 256)]


def inputs(N, D, types, seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g)
    x, res, w = make(N, D).to(types[0]).cuda(), (2 * make(N, D)).to(types[1]).cuda(), (1 + 0.2 * make(D)).to(types[2]).cuda()
    return [x, res, w], make(N, D).to(types[0]).cuda(), make(N, D).to(types[1]).cuda()


def reference(x, res, w, gy=None, gres=None):
    u = U[x.dtype]
    stored = x.detach().cpu()
    if res is not None:
        stored = (x.detach().double() + res.detach().double()).to(res.dtype).cpu()
    h, w = stored.double(), w.detach().double().cpu()
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    y = h * r * w
    out = {"stored": (h, torch.zeros_like(h)), "y": (y, 44 * u * y.abs())}
    if gy is None:
        return out
    gy = gy.double().cpu()
    gres = torch.zeros_like(h) if gres is None else gres.double().cpu()
    t = gy * w
    dh = r * (t - h * r * r * (t * h).mean(-1, keepdim=True)) + gres
    size = r * (t.abs() + h.abs() * r * r * (t * h).abs().mean(-1, keepdim=True)) + gres.abs()
    dw = gy * h * r
    out["d_x"] = out["d_res"] = (dh, 128 * u * size)
    out["d_w"] = (dw.sum(0), 204 * u * dw.abs().sum(0))
    return out


def check(name, got, ref):
    value, bound = ref
    got64 = got.detach().double().cpu()
    assert got64.shape == value.shape, name
    bound = bound + STORE[got.dtype] * (value.abs() + bound) + TINY[got.dtype]
    off = (got64 - value).abs() - bound
    assert bool((off <= 0).all()), "%s: %d of %d outside, worst by %.3e" % (name, int((off > 0).sum()), off.numel(), float(off.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, types):
    import t2fw_amd as t2
    ins, gy, gres = inputs(*shape, types, seed=sum(shape))
    ins = [t.requires_grad_(True) for t in ins]
    y, stored = t2.residual_rms_norm(*ins, eps=EPS)
    grads = torch.autograd.grad((y, stored), ins, (gy, gres))
    ref = reference(*ins, gy, gres)
    for n, v in zip(("y", "stored", "d_x", "d_res", "d_w"), (y, stored) + grads):
        assert v.dtype == {"y": types[0], "d_x": types[0], "d_w": types[2]}.get(n, types[1])
        check(n, v, ref[n])


@pytest.mark.gpu
@pytest.mark.parametrize("types", [TYPES[0], TYPES[3], TYPES[4]], ids=str)
@pytest.mark.parametrize("shape", [(5000, 64), (6001, 1500), (2000, 3000)], ids=str)
def test_many_rows(shape, types):
    """more rows than workgroups: a weight's gradient from several rows of each"""
    test_values_and_gradients(shape, types)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_without_a_residual_and_with_one_result_used(dtype):
    import t2fw_amd as t2
    (x, res, w), gy, gres = inputs(10, 300, (dtype,) * 3, seed=0)
    for t in (x, res, w):
        t.requires_grad_(True)
    y, stored = t2.residual_rms_norm(x, None, w, eps=EPS)
    assert stored is x
    ref = reference(x, None, w, gy)
    d_x, d_w = torch.autograd.grad(y, (x, w), gy)
    for n, v in (("y", y), ("d_x", d_x), ("d_w", d_w)):
        check(n, v, ref[n])
    y, stored = t2.residual_rms_norm(x, res, w, eps=EPS)
    for grads, pair in ((torch.autograd.grad(y, (x, res, w), gy, retain_graph=True), (gy, None)),
                        (torch.autograd.grad(stored, (x, res, w), gres), (torch.zeros_like(gy), gres))):
        ref = reference(x, res, w, *pair)
        for n, v in zip(("d_x", "d_res", "d_w"), grads):
            check(n, v, ref[n])
    # one array for both sides of the addition must not become one gradient that is added to twice
    a, b = x.detach().clone().requires_grad_(True), res.detach().clone().requires_grad_(True)
    for _ in range(2):
        torch.autograd.backward(t2.residual_rms_norm(a, b, w, eps=EPS), (gy, gres))
    single = torch.autograd.grad(t2.residual_rms_norm(a, b, w, eps=EPS), a, (gy, gres))[0]
    assert torch.equal(a.grad, 2 * single) and torch.equal(b.grad, 2 * single)
    lead = t2.residual_rms_norm(x.view(2, 5, 300), res.view(2, 5, 300), w, eps=EPS)
    assert lead[0].shape == (2, 5, 300) and torch.equal(lead[0].view(10, 300), y)
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.gpu
def test_gradients_against_differences():
    import t2fw_amd as t2
    (x, res, w), _, _ = inputs(3, 20, (torch.float64,) * 3, seed=2)
    ins = [t.requires_grad_(True) for t in (x, res, w)]
    assert torch.autograd.gradcheck(lambda *a: t2.residual_rms_norm(*a, eps=EPS), ins)


@pytest.mark.gpu
@pytest.mark.parametrize("types", [TYPES[0], TYPES[3], TYPES[5]], ids=str)
@pytest.mark.parametrize("group", [0, 8, 64, 128, 512])
@pytest.mark.parametrize("shape", [(1, 8), (3, 5), (4, 100), (5, 768), (3, 1021), (2, 1536), (2, 4100), (2, 9000), (2, 16500), (17, 128)], ids=str)
def test_eight_bits(shape, group, types):
    import t2fw_amd as t2
    (x, res, w), _, _ = inputs(*shape, types, seed=group + shape[1])
    x[0] = 0
    res[0] = 0
    q, scales, stored = t2.residual_rms_norm_fp8(x, res, w, eps=EPS, group=group)
    ref = reference(x, res, w)
    check("stored", stored, ref["stored"])
    assert q.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32
    D = shape[1]
    width = group or D
    y = ref["y"][0]
    pads = torch.nn.functional.pad(y, (0, -D % width)).view(shape[0], -1, width)
    want = pads.abs().amax(-1) / 448
    want = torch.where(want > 0, want, torch.ones_like(want))
    got = scales.double().cpu()
    assert got.shape == want.shape and bool(((got - want).abs() <= 48 * 2.0 ** -24 * want).all())
    each = got.repeat_interleave(width, 1)[:, :D]
    # half a unit in the last place of the 8-bit number (three bits after the leading one, down to 2^-9), and the 50 u that the
    # number which is rounded is off by
    v = (y / each).abs()
    ulp = torch.exp2(torch.floor(torch.log2(v.clamp(min=2.0 ** -6))) - 3)
    off = (q.double().cpu() - y / each).abs() - (ulp / 2 + 50 * 2.0 ** -24 * v)
    assert bool((off <= 0).all()), float(off.max())
    assert bool((q[0].double() == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("types", [TYPES[0]] + TYPES[2:6], ids=str)
@pytest.mark.parametrize("shape,group", [((500, 768), 0), ((300, 1021), 0), ((40, 4096), 128), ((300, 1021), 64), ((6, 9000), 0),
                                         ((5, 20000), 512), ((300, 5), 0)], ids=str)
def test_eight_bits_are_those_of_the_exact_quotient(shape, group, types):
    """the quotient of the products h w, which 64 bits hold, rounded to 32 bits and then to 8.  16-bit products are exact in 32 bits too, and
    no quotient of two of them is nearer to the middle between two 8-bit numbers than 32 bits tell apart; of others what their
    rounding left out is carried, and one in 2^20 or so may be off by one unit of 32 bits, of which one in 2^18 meets such a middle"""
    import t2fw_amd as t2
    (x, res, w), _, _ = inputs(*shape, types, seed=shape[1])
    q, _, stored = t2.residual_rms_norm_fp8(x, res, w, eps=EPS, group=group)
    D, width = shape[1], group or shape[1]
    p = stored.double().cpu() * w.double().cpu()
    top = torch.nn.functional.pad(p, (0, -D % width)).view(shape[0], -1, width).abs().amax(-1).repeat_interleave(width, 1)[:, :D]
    want = (448 * p / top).float().to(torch.float8_e4m3fn)
    assert torch.equal(q.cpu().double(), want.double())


@pytest.mark.gpu
def test_small_large_and_not_finite_rows():
    import t2fw_amd as t2
    w = torch.ones(256, device="cuda")
    x = torch.zeros(5, 256, device="cuda")
    x[1, 3] = float("nan")
    x[2, 200] = float("inf")
    x[3] = 1e-25
    x[4] = 3e4
    y, _ = t2.residual_rms_norm(x, None, w, eps=1e-12)
    assert bool((y[0] == 0).all()) and bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[2, 200])) and bool((y[2, :200] == 0).all())
    assert torch.allclose(y[4], torch.ones(256, device="cuda"))
    q, s, _ = t2.residual_rms_norm_fp8(x, None, w, eps=1e-12, group=64)
    q, s = q.float(), s.cpu()
    assert bool((q[0] == 0).all()) and bool((s[0] == 1).all())
    assert bool(torch.isnan(q[1]).all())
    assert bool(torch.isnan(q[2, 192:]).any()) and bool((q[2, :192] == 0).all())
    assert bool((q[3] == 448).all())                    # 1e-19 everywhere, and its own largest
    tiny = torch.full((1, 64), 1e-30, device="cuda")
    q, s, _ = t2.residual_rms_norm_fp8(tiny, None, torch.full((64,), 1e-12, device="cuda"), eps=1.0)    # y = 1e-42, a scale of nearly nothing
    assert bool(torch.isfinite(q.float()).all())


@pytest.mark.gpu
def test_the_same_bits_again_on_another_stream_and_in_a_graph():
    import t2fw_amd as t2
    types = TYPES[4]
    ins, gy, gres = inputs(4099, 200, types, seed=1)

    def run(ins):
        ins = [t.detach().requires_grad_(True) for t in ins]
        y, stored = t2.residual_rms_norm(*ins)
        return (y, stored) + torch.autograd.grad((y, stored), ins, (gy, gres))
    want = run(ins)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(ins)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    buffers = [t.clone() for t in ins]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(buffers)
    for seed in (5, 6, 7):
        fresh, _, _ = inputs(4099, 200, types, seed=seed)
        for b, t in zip(buffers, fresh):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(run(fresh), captured))


@pytest.mark.gpu
def test_refusals():
    import t2fw_amd as t2
    (x, res, w), _, _ = inputs(4, 16, TYPES[3], seed=0)
    for bad in (dict(x=x.cpu()), dict(residual=res[:2]), dict(residual=res.half()), dict(weight=w[:8]), dict(weight=w.double()),
                dict(x=x.t()), dict(residual=torch.zeros(16, 4, device="cuda", dtype=x.dtype).t()), dict(x=x.long())):
        for fn in (t2.residual_rms_norm, t2.residual_rms_norm_fp8):
            with pytest.raises(RuntimeError):
                fn(**{**dict(x=x, residual=res, weight=w), **bad})
    with pytest.raises(RuntimeError):
        t2.residual_rms_norm(x.float(), res, w)         # a stream of fewer bits than the tokens
    for group in (4, 24, 1024, -8):
        with pytest.raises(RuntimeError):
            t2.residual_rms_norm_fp8(x, res, w, group=group)
    with pytest.raises(RuntimeError, match="gradients"):
        t2.residual_rms_norm_fp8(x.clone().requires_grad_(True), res, w)
    with pytest.raises(RuntimeError):
        t2.residual_rms_norm_fp8(x.double(), res.double(), w.double())
    assert t2.residual_rms_norm(x[:0], res[:0], w)[0].shape == (0, 16)
    empty = [t.requires_grad_(True) for t in (x[:0].clone(), res[:0].clone(), w.clone())]
    y, stored = t2.residual_rms_norm(*empty)
    assert bool((torch.autograd.grad(y.sum() + stored.sum(), empty[2])[0] == 0).all())


def test_host_memory_and_bad_c_calls_are_refused():
    import ctypes
    import t2fw_amd as t2
    from t2fw_amd import _lib
    with pytest.raises(RuntimeError, match="CUDA"):
        t2.residual_rms_norm(torch.zeros(1, 8), None, torch.ones(8))
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p(ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 64)
    forward = lambda ptrs=(p,) * 5, N=1, D=8, dtype=0, flags=0: lib.t2fw_rms_norm_forward(*ptrs, N, D, 1e-6, dtype, flags, None)
    assert forward(dtype=7) == 2 and forward(N=-1) == 3 and forward(D=0) == 3 and forward(flags=8) == 5 and forward(dtype=3, flags=1) == 5
    assert forward(ptrs=(None, p, p, p, p)) == 1 and forward(ptrs=(p, p, p, p, None)) == 1
    assert forward(ptrs=(ctypes.c_void_p(p.value + 1),) + (p,) * 4) == 4 and forward(N=0) == 0
    assert lib.t2fw_rms_norm_forward_fp8(*(p,) * 6, 1, 8, 12, 1e-6, 0, 0, None) == 3
    assert lib.t2fw_rms_norm_forward_fp8(*(p,) * 6, 1, 8, 0, 1e-6, 3, 0, None) == 2
    assert lib.t2fw_rms_norm_backward(*(p,) * 7, 4, 8, 1e-6, 0, 0, p, 0, None) == 6
    assert lib.t2fw_rms_norm_backward(*(p,) * 5, None, p, 4, 8, 1e-6, 1, 1, p, 4096, None) == 1      # two types, one gradient

"""short_conv and short_conv_step against the sum written out in float64.

Bounds, u = 2^-24.  z is a sum of W + 1 terms by fused multiply-adds: off by (W + 1) u of the sum of their absolute values S.  silu'(z) is at most 1.1 in
size, so y is off by 1.1 of that, and by the sigmoid's own error relative to y: 2^-20 for 16-bit tensors (hardware exponential and reciprocal, 2^-22 each,
and |z| 2^-24 for the exponential's argument, |z| < 40 here), 2^-22 for float32.  The slope s (1 + z (1 - s)) is off by 2^-20 (1 + |z|) or 2^-22 (1 + |z|) and, as
silu'' is at most 0.5 in size, half of the error of z.  dz multiplies that by gy.  A gradient is a sum of products of such numbers: the products' errors and n u of the sum
of their absolute values for n terms in any order.  What is stored is rounded to half a unit in the last place of its type."""
import pytest
import torch

STORE = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def windows(xs, W):
    """[B, W - 1 + T, D] -> [B, T, D, W]"""
    return xs.unfold(1, W, 1)


def reference(x, w, bias, state, lengths, silu, gy=None, gs=None):
    """name -> (value, bound before storing), in float64 on the CPU"""
    act = 2.0 ** -22 if x.dtype == torch.float32 else 2.0 ** -20
    B, T, D = x.shape
    W = w.shape[1]
    x, w = x.detach().double().cpu(), w.detach().double().cpu()
    bias = torch.zeros(D).double() if bias is None else bias.detach().double().cpu()
    state = torch.zeros(B, W - 1, D).double() if state is None else state.detach().double().cpu()
    ends = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    live = (torch.arange(T)[None] < ends[:, None])[:, :, None]
    xs = torch.cat((state, torch.where(live, x, torch.zeros(()).double())), 1)
    zero = torch.zeros(B, 0, D).double()
    z = bias + (windows(xs, W) * w).sum(-1) if T else zero
    ze = (W + 1) * U * (bias.abs() + (windows(xs, W) * w).abs().sum(-1)) if T else zero
    s = torch.sigmoid(z)
    y, ye = (z * s, 1.1 * ze + act * (z * s).abs()) if silu else (z, ze)
    at = ends[:, None] + torch.arange(W - 1)[None]
    gather = at[:, :, None].expand(-1, -1, D)
    out = {"y": (y * live, ye * live), "last": (xs.gather(1, gather), torch.zeros(B, W - 1, D).double())}
    if gy is None:
        return out
    gy, gs = torch.where(live, gy.double().cpu(), torch.zeros(()).double()), gs.double().cpu()
    dz, de = gy, torch.zeros_like(gy)
    if silu:
        dz, de = gy * s * (1 + z * (1 - s)), gy.abs() * (act * (1 + z.abs()) + 0.5 * ze) + 2 * U * gy.abs()
    n = B * T
    dw = torch.stack([(dz * xs[:, j:j + T]).sum((0, 1)) for j in range(W)], 1)
    dwe = torch.stack([((de + n * U * dz.abs()) * xs[:, j:j + T].abs()).sum((0, 1)) for j in range(W)], 1)
    dxs, dxe = torch.zeros_like(xs), torch.zeros_like(xs)
    for j in range(W):
        dxs[:, j:j + T] += dz * w[:, j]
        dxe[:, j:j + T] += (de + (W + 2) * U * dz.abs()) * w[:, j].abs()
    dxs.scatter_add_(1, gather, gs)
    dxe.scatter_add_(1, gather, (W + 2) * U * gs.abs())
    out.update(d_x=(dxs[:, W - 1:] * live, dxe[:, W - 1:] * live), d_state=(dxs[:, :W - 1], dxe[:, :W - 1]), d_w=(dw, dwe),
               d_bias=(dz.sum((0, 1)), (de + n * U * dz.abs()).sum((0, 1))))
    return out


def check(name, got, ref):
    value, bound = ref
    got64 = got.detach().double().cpu()
    assert got64.shape == value.shape, name
    bound = bound + STORE[got.dtype] * (value.abs() + bound) + TINY[got.dtype]
    off = (got64 - value).abs() - bound
    assert bool((off <= 0).all()), "%s: %d of %d outside, worst by %.3e" % (name, int((off > 0).sum()), off.numel(), float(off.max()))


def inputs(B, T, D, W, dtype, seed, weight=None):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g)
    ins = [make(B, T, D).to(dtype), (make(D, W) * W ** -0.5).to(weight or dtype), make(D).to(weight or dtype), make(B, W - 1, D).to(dtype)]
    return [t.cuda() for t in ins], make(B, T, D).to(dtype).cuda(), make(B, W - 1, D).to(dtype).cuda()


NAMES = ("y", "last", "d_x", "d_w", "d_bias", "d_state")


def run(ins, lengths, silu, gy, gs):
    import t2fw_amd as t2
    ins = [t.detach().requires_grad_(True) for t in ins]
    x, w, bias, state = ins
    out = t2.short_conv(x, w, bias=bias, state=state, lengths=lengths, silu=silu)
    return dict(zip(NAMES, out + torch.autograd.grad(out, ins, (gy, gs))))


# one token, fewer steps than taps, one less and one more than a lane's steps and than a workgroup's; widths of less than a vector, odd ones, several workgroups
SHAPES = [(1, 1, 1), (2, 2, 5), (3, 8, 64), (1, 9, 7), (2, 127, 65), (5, 64, 8), (1, 1500, 24), (4, 257, 200), (2, 300, 333), (37, 31, 9), (200, 3, 140)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("taps,silu", [(4, True), (2, False), (3, True), (8, True)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, taps, silu, dtype):
    ins, gy, gs = inputs(*shape, taps, dtype, seed=sum(shape))
    got, ref = run(ins, None, silu, gy, gs), reference(*ins, None, silu, gy, gs)
    for n in NAMES:
        check(n, got[n], ref[n])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,weight", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.float32, None), (torch.bfloat16, None)], ids=str)
@pytest.mark.parametrize("taps", [2, 3, 4, 5, 6, 7, 8])
def test_every_number_of_taps_over_rows_that_end_early(taps, dtype, weight):
    T = 70
    lengths = torch.tensor([0, 1, T, T - 1, 2, taps - 1, T + 7, -3, 33])
    ins, gy, gs = inputs(len(lengths), T, 37, taps, dtype, seed=taps, weight=weight)
    for b, n in enumerate(lengths.tolist()):
        n = max(0, min(T, n))
        for t in (ins[0], gy):
            t[b, n:] = float("nan")
            t[b, n + 1:n + 2] = float("inf")
    for kind in (torch.int64, torch.int32):
        got = run(ins, lengths.to(kind).cuda(), True, gy, gs)
        ref = reference(ins[0].nan_to_num(0, 0, 0), *ins[1:], lengths, True, gy.nan_to_num(0, 0, 0), gs)
        for n in NAMES:
            check(n, got[n], ref[n])
    # nothing of a row without steps: its inputs pass as they are
    assert torch.equal(got["last"][0], ins[3][0]) and torch.equal(got["d_state"][0], gs[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_many_rows_and_steps(dtype):
    """several tiles of a stretch, many stretches and workgroups"""
    for shape in ((3, 4000, 260), (900, 40, 50)):
        ins, gy, gs = inputs(*shape, 4, dtype, seed=1)
        lengths = torch.randint(0, shape[1] + 1, (shape[0],), generator=torch.Generator().manual_seed(1))
        got, ref = run(ins, lengths.cuda(), True, gy, gs), reference(*ins, lengths, True, gy, gs)
        for n in NAMES:
            check(n, got[n], ref[n])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_parts_of_a_projection_and_other_orders(dtype):
    import t2fw_amd as t2
    ins, gy, gs = inputs(3, 50, 40, 4, dtype, seed=3)
    x, w, bias, state = ins
    both = torch.randn(3, 50, 2 * 40 + 1, device="cuda").to(dtype)
    both[..., 1:41] = x
    both.requires_grad_(True)
    y, last = t2.short_conv(both[..., 1:41], w, bias, state, silu=True)
    d_both, = torch.autograd.grad((y, last), both, (gy.transpose(0, 1).contiguous().transpose(0, 1), gs))
    ref = reference(*ins, None, True, gy, gs)
    check("y", y, ref["y"])
    check("last", last, ref["last"])
    check("d_x", d_both[..., 1:41], ref["d_x"])
    assert not d_both[..., 41:].any() and not d_both[..., 0].any()
    # time before batch in memory; a gradient that is one value everywhere; results that nothing depends on; no bias, no state
    xt = x.transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True)
    y, last = t2.short_conv(xt, w)
    ones = reference(x, w, None, None, None, False, torch.ones_like(x), torch.zeros_like(gs))
    check("d_x", torch.autograd.grad(y.sum(), xt, retain_graph=True)[0], ones["d_x"])
    only = reference(x, w, None, None, None, False, torch.zeros_like(x), gs)
    check("d_x", torch.autograd.grad(last, xt, gs)[0], only["d_x"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_token_by_token_and_in_pieces(dtype):
    import t2fw_amd as t2
    for B, D, W in ((5, 37, 4), (3, 5, 2), (64, 64, 8), (1, 8, 3)):
        (x, w, bias, state), _, _ = inputs(B, 11, D, W, dtype, seed=D)
        whole, last = t2.short_conv(x, w, bias, state, silu=True)
        a, mid = t2.short_conv(x[:, :4], w, bias, state, silu=True)
        b, end = t2.short_conv(x[:, 4:], w, bias, mid, silu=True)
        assert torch.equal(torch.cat((a, b), 1), whole) and torch.equal(end, last)
        st, wide = state.clone(), torch.randn(B, 2 * D + 1, device="cuda").to(dtype)
        for t in range(11):
            wide[:, 1:D + 1] = x[:, t]
            before = st.clone()
            y, new = t2.short_conv_step(wide[:, 1:D + 1], w, st, bias, silu=True)
            assert new is st and torch.equal(y, whole[:, t])
            out = torch.empty_like(y)
            y2, st2 = t2.short_conv_step(wide[:, 1:D + 1], w, before, bias, silu=True, out=out, inplace=False)
            assert y2.data_ptr() == out.data_ptr() and torch.equal(out, y) and torch.equal(st2, st)
            assert torch.equal(before[:, 1:], st[:, :-1])
        assert torch.equal(st, last)


@pytest.mark.gpu
def test_no_steps_and_no_rows():
    import t2fw_amd as t2
    (x, w, bias, state), _, gs = inputs(2, 1, 6, 4, torch.float32, seed=0)
    state.requires_grad_(True)
    w.requires_grad_(True)
    y, last = t2.short_conv(x[:, :0], w, bias, state)
    assert y.shape == (2, 0, 6) and torch.equal(last, state)
    ds, dw = torch.autograd.grad(last, (state, w), gs)
    assert torch.equal(ds, gs) and not dw.any()
    x0 = x[:0].requires_grad_(True)
    y, last = t2.short_conv(x0, w)
    assert y.shape == (0, 1, 6) and last.shape == (0, 3, 6)
    assert not torch.autograd.grad(y.sum(), w)[0].any()
    y, st = t2.short_conv_step(x0.detach()[:, 0], w.detach(), state.detach()[:0])
    assert y.shape == (0, 6)


@pytest.mark.gpu
def test_gradient_against_differences():
    """Directional differences of the sum in float64 at distance 1e-5: off by h^2 / 6 of the third derivative and by rounding, 1e-8 here; the gradients'
    own float32 errors are within 2^-18 of their terms (the bounds above: slopes to 2^-22 (1 + |z|), z to 5 u, sums of 63 terms)"""
    ins, gy, gs = inputs(2, 40, 6, 4, torch.float32, seed=9)
    lengths = torch.tensor([40, 23])
    got = run(ins, lengths.cuda(), True, gy, gs)
    g = torch.Generator().manual_seed(2)
    for i, name in enumerate(("d_x", "d_w", "d_bias", "d_state")):
        way = torch.randn(ins[i].shape, generator=g).double()

        def at(h):
            moved = [t.double().cpu() + (h * way if i == j else 0) for j, t in enumerate(ins)]
            r = reference(*moved, lengths, True)
            return float((r["y"][0] * gy.double().cpu()).sum() + (r["last"][0] * gs.double().cpu()).sum())
        want = (at(1e-5) - at(-1e-5)) / 2e-5
        terms = (got[name].double().cpu() * way)
        assert abs(float(terms.sum()) - want) <= 2.0 ** -18 * float(terms.abs().sum()) + 1e-6, name


@pytest.mark.gpu
def test_captured_forward_and_backward_replay():
    import t2fw_amd as t2
    ins, gy, gs = inputs(2, 200, 40, 4, torch.bfloat16, seed=5)
    leaves = [t.clone().requires_grad_(True) for t in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        out = t2.short_conv(leaves[0], leaves[1], leaves[2], leaves[3], silu=True)
        return out + torch.autograd.grad(out, leaves, (gy, gs))
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for k in range(3):
        new, _, _ = inputs(2, 200, 40, 4, torch.bfloat16, seed=6 + k)
        with torch.no_grad():
            for l, t in zip(leaves, new):
                l.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = run(new, None, True, gy, gs)
        for n, v in zip(NAMES, res):
            assert torch.equal(v, want[n]), n


def bad_calls():
    import t2fw_amd as t2
    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)
    x, w, s, both = z(2, 5, 8), z(8, 4), z(2, 3, 8), z(2, 16)
    h = torch.float16
    return {
        "x is flat": lambda: t2.short_conv(z(2, 8), w),
        "x has no channels": lambda: t2.short_conv(z(2, 5, 0), z(0, 4)),
        "x by steps": lambda: t2.short_conv(z(2, 8, 5).transpose(1, 2), w),
        "x in 64 bits": lambda: t2.short_conv(x.double(), w.double()),
        "x is a number": lambda: t2.short_conv(z(), w),
        "weight is a number": lambda: t2.short_conv(x, z()),
        "bias is a number": lambda: t2.short_conv(x, w, z()),
        "state is a number": lambda: t2.short_conv(x, w, state=z()),
        "one tap": lambda: t2.short_conv(x, z(8, 1)),
        "nine taps": lambda: t2.short_conv(x, z(8, 9)),
        "weight of other channels": lambda: t2.short_conv(x, z(7, 4)),
        "weight of another type": lambda: t2.short_conv(x, w.half()),
        "weight in bfloat16 next to float16": lambda: t2.short_conv(x.half(), w.bfloat16()),
        "bias of another type than the weight": lambda: t2.short_conv(x.half(), w, z(8, dtype=h)),
        "bias of other channels": lambda: t2.short_conv(x, w, z(7)),
        "state of other taps": lambda: t2.short_conv(x, w, state=z(2, 4, 8)),
        "state of another type": lambda: t2.short_conv(x.half(), w, state=s),
        "lengths of other rows": lambda: t2.short_conv(x, w, lengths=z(3, dtype=torch.int64)),
        "lengths that are numbers": lambda: t2.short_conv(x, w, lengths=z(2)),
        "x in host memory": lambda: t2.short_conv(x.cpu(), w),
        "weight in host memory": lambda: t2.short_conv(x, w.cpu()),
        "step with gradients": lambda: t2.short_conv_step(x[:, 0].contiguous(), w.clone().requires_grad_(True), s),
        "step of a sequence": lambda: t2.short_conv_step(x, w, s),
        "step's state of other rows": lambda: t2.short_conv_step(x[:, 0], w, z(3, 3, 8)),
        "step's state apart": lambda: t2.short_conv_step(x[:, 0], w, z(2, 8, 3).transpose(1, 2)),
        "step's result is its state": lambda: t2.short_conv_step(x[:, 0], w, s, out=s[:, 0]),
        "step's input is its state": lambda: t2.short_conv_step(s[:, 0], w, s),
        "step's result is another part of its input": lambda: t2.short_conv_step(both[:, :8], w, s, out=both.view(4, 8)[1:3]),
        "twice differentiated": lambda: torch.autograd.grad(t2.short_conv(x.clone().requires_grad_(True), w.requires_grad_(True))[0].sum(), w, create_graph=True),
    }


@pytest.mark.gpu
def test_refusals():
    for name, call in bad_calls().items():
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(name)


def test_c_abi_refusals():
    import ctypes
    from t2fw_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p(ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 64)
    fwd = lambda B=1, T=1, D=1, W=4, dtype=0, flags=0, ptrs=None, strides=None: lib.t2fw_short_conv_forward(*(ptrs or [p] * 7), B, T, D, W, strides, dtype, flags, None)
    assert fwd(dtype=3) == 2 and fwd(dtype=9) == 2
    assert fwd(W=1) == 3 and fwd(W=9) == 3 and fwd(D=0) == 3 and fwd(B=-1) == 3 and fwd(B=1 << 40, T=1 << 20, D=1 << 10) == 3
    assert fwd(flags=8) == 5
    assert fwd(strides=(ctypes.c_int64 * 2)(-1, 1)) == 3
    for i in (0, 1, 5, 6):
        ptrs = [p] * 7
        ptrs[i] = None
        assert fwd(ptrs=ptrs) == 1
    assert fwd(ptrs=[ctypes.c_void_p(p.value + 1)] + [p] * 6) == 4
    assert fwd(B=0) == 0
    assert lib.t2fw_short_conv_backward_workspace_bytes(8, 1024, 1536, 4, 2) > 0 and lib.t2fw_short_conv_backward_workspace_bytes(8, 1024, 1536, 1, 2) == 0
    assert lib.t2fw_short_conv_backward(*[p] * 11, 1, 1, 1, 4, None, 0, 0, p, 0, None) == 6
    assert b"workspace" in lib.t2fw_last_error()
    assert lib.t2fw_short_conv_step(*[p] * 6, 1, 1, 4, -1, 0, 0, None) == 3

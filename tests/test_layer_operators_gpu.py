"""short_conv, selective_scan, beam_select and reorder_beams as calls: other ways to differentiate and transform them, hooks on what their nodes save, memory
that does not hold its values as they are, arrays whose offsets pass 32 bits, streams side by side.  What they do not have is refused."""
import gc

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def rand(*s, seed=0):
    return torch.randn(s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def calls():
    """name -> (call, floating-point inputs)"""
    import t2fw_amd as t2
    beams = torch.tensor([[1, 0, 0], [2, 2, 1]], device="cuda")
    x, w, b, st = rand(2, 5, 8), rand(8, 4), rand(8), rand(2, 3, 8)
    a, n, h, one = -rand(8, 4).abs(), rand(2, 5, 4), rand(2, 8, 4), rand(2, 4)
    scan = lambda x, dt, a, b, c, h, s, z, e: t2.selective_scan(x, dt, a, b, c, state=h, skip=s, gate=z, dt_bias=e, softplus=True)
    step = lambda x, dt, a, b, c, h, s, z, e: t2.selective_scan_step(x, dt, a, b, c, h, skip=s, gate=z, dt_bias=e, softplus=True)
    return {
        "short_conv": (lambda x, w, b, s: t2.short_conv(x, w, b, s, silu=True), [x, w, b, st]),
        "short_conv_step": (lambda x, w, s, b: t2.short_conv_step(x, w, s, b), [x[:, 0].clone(), w, st, b]),
        "short_conv_step into another": (lambda x, s, o: t2.short_conv_step(x, w, s, out=o), [x[:, 0].clone(), st, rand(2, 8)]),
        "selective_scan": (scan, [x, rand(2, 5, 8, seed=1), a, n, rand(2, 5, 4, seed=1), h, rand(8), rand(2, 5, 8, seed=2), rand(8, seed=1)]),
        "selective_scan_step": (step, [rand(2, 8), rand(2, 8, seed=1), a, rand(2, 4), rand(2, 4, seed=1), h, rand(8), rand(2, 8, seed=2), rand(8, seed=1)]),
        "selective_scan_step into another": (lambda x, h, o: t2.selective_scan_step(x, x, a, one, one, h, out=o), [rand(2, 8), h, rand(2, 8)]),
        "beam_select": (lambda z, s: t2.beam_select(z, s), [rand(2, 3, 9), rand(2, 3)]),
        "reorder_beams": (lambda t, u: t2.reorder_beams([t, u], beams), [rand(6, 4), rand(12, 2)]),
        "reorder_beams into another": (lambda t, o: t2.reorder_beams([t], beams, out=[o]), [rand(6, 4), rand(6, 4)]),
    }


NAMES = ["short_conv", "short_conv_step", "short_conv_step into another", "selective_scan", "selective_scan_step", "selective_scan_step into another", "beam_select",
         "reorder_beams", "reorder_beams into another"]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name, grad):
    call, ins = calls()[name]
    with forward_ad.dual_level():
        for i in range(len(ins)):
            duals = [t.clone() for t in ins]
            if grad and name in ("short_conv", "selective_scan"):
                duals[i].requires_grad_(True)
            duals[i] = forward_ad.make_dual(duals[i], torch.ones_like(ins[i]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*duals)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(*duals)
            with torch.no_grad(), forward_ad._set_fwd_grad_enabled(False):
                call(*duals)
        call(*[t.clone() for t in ins])


@pytest.mark.parametrize("name", NAMES)
def test_transformed_and_fake_tensors_are_refused(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    call, ins = calls()[name]
    with pytest.raises(RuntimeError):
        torch.vmap(call)(*[torch.stack((t, t)) for t in ins])
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, tuple(ins), tuple(torch.ones_like(t) for t in ins))
    with FakeTensorMode() as mode, pytest.raises(RuntimeError):
        call(*[mode.from_tensor(t) for t in ins])


@pytest.mark.parametrize("name", NAMES)
def test_negated_views_and_sparse_tensors_are_refused(name):
    call, ins = calls()[name]
    call(*[t.clone() for t in ins])
    for i in range(len(ins)):
        for other in (torch._neg_view(ins[i].clone()), ins[i].to_sparse()):
            with pytest.raises(RuntimeError):
                call(*[t.clone() for t in ins[:i]], other, *[t.clone() for t in ins[i + 1:]])


@pytest.mark.parametrize("name", ["short_conv", "selective_scan"])
def test_gradients_that_are_negated_views(name):
    call, ins = calls()[name]
    ins = [t.clone().requires_grad_(True) for t in ins]
    outs = call(*ins)
    grads = [torch.randn_like(o) for o in outs]
    want = torch.autograd.grad(outs, ins, [-g for g in grads], retain_graph=True)
    got = torch.autograd.grad(outs, ins, [torch._neg_view(g) for g in grads])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def spread(t):
    """the same values, every second element of twice the memory"""
    return torch.stack((t, t), -1)[..., 0]


@pytest.mark.parametrize("unpack", [lambda t: t.cuda(), lambda t: spread(t.cuda())], ids=["host", "spread"])
@pytest.mark.parametrize("name", ["short_conv", "selective_scan"])
def test_saved_tensors_that_come_back_in_another_order(name, unpack):
    call, ins = calls()[name]
    ins = [t.clone().requires_grad_(True) for t in ins]

    def grads():
        return torch.autograd.grad([o.square().sum() for o in call(*ins)], ins)
    want = grads()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), unpack):
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", ["short_conv", "selective_scan"])
def test_saved_tensors_of_other_types_and_sizes_are_refused(name):
    call, ins = calls()[name]
    ins = [t.clone().requires_grad_(True) for t in ins]
    for unpack in (lambda t: t.double() if t.is_floating_point() else t.int(), lambda t: t[..., :1], lambda t: t.cpu(), lambda t: t[:1] if t.dim() else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            out = call(*ins)[0]
            with pytest.raises(RuntimeError):
                torch.autograd.grad(out.sum(), ins[0])


def test_inputs_that_want_no_gradient():
    for name in ("short_conv", "selective_scan"):
        call, ins = calls()[name]
        every = [t.clone().requires_grad_(True) for t in ins]
        want = torch.autograd.grad([o.square().sum() for o in call(*every)], every)
        for i in range(len(ins)):
            some = [t.clone().requires_grad_(i == j) for j, t in enumerate(ins)]
            got, = torch.autograd.grad([o.square().sum() for o in call(*some)], some[i])
            assert torch.equal(got, want[i]), (name, i)


@pytest.fixture
def large():
    gc.collect()                                         # (tensors in cycles that earlier tests have left)
    torch.cuda.empty_cache()
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    yield
    gc.collect()
    torch.cuda.empty_cache()                             # (what the tests after this hold would be parts of these blocks)


def test_offsets_past_32_bits(large):
    """rows of 2^31 elements and more apart, in one array of 8.6 GB: the same results as from the rows brought together"""
    import t2fw_amd as t2
    B, T, D, N = 2, 60, 40, 6
    big = torch.empty(B, (1 << 31) + 5000, dtype=torch.bfloat16, device="cuda")
    wide = 3 * D + 2 * N + 1
    at = torch.as_strided(big, (B, T, wide), (big.stride(0), wide, 1), (1 << 31) - 4000)
    at.copy_(rand(B, T, wide))
    near = at.contiguous()
    w, a, state = rand(D, 4), -rand(D, N).abs() - 0.1, rand(B, D, N)

    def both(u):
        x, dt, z, b, c, _ = u.split([D, D, D, N, N, 1], dim=-1)
        conv = t2.short_conv(x, w, silu=True)
        scan = t2.selective_scan(x, dt, a, b, c, state=state, gate=z, softplus=True)
        step = t2.selective_scan_step(x[:, 0], dt[:, 0], a, b[:, 0], c[:, 0], state, gate=z[:, 0], inplace=False)
        return conv + scan + step + t2.short_conv_step(x[:, 3], w, torch.zeros(B, 3, D, dtype=x.dtype, device="cuda"))
    assert all(torch.equal(p, q) for p, q in zip(both(at), both(near)))
    leaf_far, leaf_near = at.detach().requires_grad_(True), near.detach().requires_grad_(True)
    for u in (leaf_far, leaf_near):
        out = both_train(t2, u, w, a, state, D, N)
        u.given = torch.autograd.grad([o.float().square().sum() for o in out], u)[0]
    assert torch.equal(leaf_far.given, leaf_near.given)
    del leaf_far, at
    # steps further apart than a tile's offsets reach: time before batch in memory, few rows of it used
    tall = torch.empty(20, (1 << 27) + 64, dtype=torch.bfloat16, device="cuda")
    u = torch.as_strided(tall, (1, 20, D), (D, tall.stride(0), 1))
    u.copy_(rand(1, 20, D))
    b, c = rand(1, 20, N).bfloat16(), rand(1, 20, N, seed=1).bfloat16()
    far, close = t2.selective_scan(u, u, a, b, c, softplus=True), t2.selective_scan(u.contiguous(), u.contiguous(), a, b, c, softplus=True)
    assert all(torch.equal(p, q) for p, q in zip(far, close))
    far, close = t2.short_conv(u, w), t2.short_conv(u.contiguous(), w)
    assert all(torch.equal(p, q) for p, q in zip(far, close))


def both_train(t2, u, w, a, state, D, N):
    x, dt, z, b, c, _ = u.split([D, D, D, N, N, 1], dim=-1)
    return t2.short_conv(x, w, silu=True) + t2.selective_scan(x, dt, a, b, c, state=state, gate=z, softplus=True)


def test_large_arrays_of_beams(large):
    import t2fw_amd as t2
    V = 131072
    logits = torch.empty(1100, 16, V, dtype=torch.bfloat16, device="cuda").normal_()
    scores = rand(1100, 16) * 0.01
    assert logits.numel() > 1 << 31
    s, k, v = t2.beam_select(logits, scores)
    for b in (0, 1023, 1024, 1099):
        one = t2.beam_select(logits[b:b + 1].contiguous(), scores[b:b + 1].contiguous())
        assert torch.equal(k[b:b + 1], one[1]) and torch.equal(v[b:b + 1], one[2]) and bool(((s[b:b + 1] - one[0]).abs() <= 2.0 ** -18).all())
    beams = torch.randint(0, 4, (3, 4), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    flat = logits.view(-1)[:12 * 180_000_001].view(12, -1)
    want = [flat[4 * b + int(beams[b, j]), -1000:].clone() for b in range(3) for j in range(4)]
    t2.reorder_beams([flat], beams)
    assert all(torch.equal(flat[i, -1000:], w) for i, w in enumerate(want))


def test_two_streams_at_once():
    """calls that overlap in time share nothing"""
    import t2fw_amd as t2
    cases = []
    for seed in range(2):
        x, dt, z = (rand(2, 300, 70, seed=10 * seed + i).bfloat16() for i in range(3))
        b, c = (rand(2, 300, 16, seed=10 * seed + 3 + i).bfloat16() for i in range(2))
        cases.append(dict(x=x, dt=dt, a=-rand(70, 16, seed=seed).abs(), b=b, c=c, gate=z, softplus=True, w=rand(70, 4, seed=seed), logits=rand(3, 4, 9000, seed=seed), scores=rand(3, 4, seed=seed)))

    def work(k):
        k = dict(k)
        w, logits, scores = k.pop("w"), k.pop("logits"), k.pop("scores")
        ins = [k[n].detach().requires_grad_(True) for n in ("x", "dt", "a")]
        y, last = t2.selective_scan(*ins, k["b"], k["c"], gate=k["gate"], softplus=True)
        u, end = t2.short_conv(ins[0], w, silu=True)
        return (y, last, u, end) + torch.autograd.grad((y.float().sum() + u.float().square().sum()), ins) + t2.beam_select(logits, scores)
    want = [[t.detach().clone() for t in work(k)] for k in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for _ in range(5):
        for i, (s, k) in enumerate(zip(streams, cases)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = [t.detach() for t in work(k)]
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(w, g))


class Frame:
    """arrays with a margin on either side, of NaN (inputs) or of a number that has to stay (results)"""
    MARGIN = 4096

    def __init__(self):
        self.kept = []

    def given(self, t):
        whole = torch.full((t.numel() + 2 * self.MARGIN,), float("nan"), dtype=t.dtype, device="cuda")
        part = whole[self.MARGIN:self.MARGIN + t.numel()].view(t.shape)
        part.copy_(t)
        return part

    def result(self, *shape, dtype=torch.float32):
        n = torch.Size(shape).numel()
        whole = torch.full((n + 2 * self.MARGIN,), 77.0, dtype=dtype, device="cuda")
        self.kept.append((whole, n))
        return whole[self.MARGIN:self.MARGIN + n].view(shape)

    def check(self):
        for whole, n in self.kept:
            assert bool((whole[:self.MARGIN] == 77).all()) and bool((whole[self.MARGIN + n:] == 77).all()), (n, whole.dtype)


def pointer(t):
    return None if t is None else t.data_ptr()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 5, 16), (2, 5, 70, 16), (3, 17, 7, 6), (1, 33, 300, 1), (2, 7, 9, 64), (1, 200, 5, 16), (2, 31, 33, 30)], ids=str)
def test_nothing_around_the_arrays_of_the_scan(shape, dtype):
    """neither read into a result nor written"""
    import t2fw_amd as t2
    from t2fw_amd import _lib
    lib, (B, T, D, N), code = _lib.load(), shape, 0 if dtype == torch.float32 else 2
    NP = max(4, 1 << (N - 1).bit_length())
    tiles = (T + 15) // 16
    x, dt, z, gy = (rand(B, T, D, seed=i).to(dtype) for i in range(4))
    b, c = (rand(B, T, N, seed=4 + i).to(dtype) for i in range(2))
    a, s0, gs, skip, bias = -rand(D, N).abs(), rand(B, D, N), rand(B, D, N, seed=1), rand(D), rand(D, seed=1)
    f = Frame()
    ins = [f.given(t) for t in (x, dt, a, b, c, skip, z, bias)]
    s0_, gs_, gy_ = f.given(s0), f.given(gs), f.given(gy)
    y, last, ckpt = f.result(B, T, D, dtype=dtype), f.result(B, D, N), f.result(B, tiles, D, NP)
    assert lib.t2fw_selective_scan_checkpoint_bytes(B, T, D, N) == ckpt.numel() * 4
    room = lib.t2fw_selective_scan_workspace_bytes(B, T, D, N)
    space = f.result((room + 3) // 4)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.t2fw_selective_scan_forward(*map(pointer, ins), s0_.data_ptr(), None, *map(pointer, (y, last, ckpt)), B, T, D, N, None, code, 1, space.data_ptr(), room, stream) == 0
    room = lib.t2fw_selective_scan_backward_workspace_bytes(B, T, D, N)
    space = f.result((room + 3) // 4)
    like = [f.result(B, T, D, dtype=dtype), f.result(B, T, D, dtype=dtype), f.result(D, N), f.result(B, T, N, dtype=dtype), f.result(B, T, N, dtype=dtype), f.result(D),
            f.result(B, T, D, dtype=dtype), f.result(D), f.result(B, D, N)]
    assert lib.t2fw_selective_scan_backward(gy_.data_ptr(), gs_.data_ptr(), *map(pointer, ins), None, ckpt.data_ptr(), *map(pointer, like), B, T, D, N, None, code, 1,
                                            space.data_ptr(), room, stream) == 0
    torch.cuda.synchronize()
    f.check()
    leaves = [t.clone().requires_grad_(True) for t in (x, dt, a, b, c, skip, z, bias, s0)]
    out = t2.selective_scan(*leaves[:5], skip=leaves[5], gate=leaves[6], dt_bias=leaves[7], state=leaves[8], softplus=True)
    grads = torch.autograd.grad(out, leaves, (gy, gs))
    assert torch.equal(out[0], y) and torch.equal(out[1], last)
    assert all(torch.equal(p, q) for p, q in zip(grads, like))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 5, 4), (2, 5, 70, 2), (3, 17, 7, 8), (1, 33, 300, 3), (2, 9, 3, 5), (1, 200, 1, 4), (2, 31, 33, 7)], ids=str)
def test_nothing_around_the_arrays_of_the_convolution(shape, dtype):
    import t2fw_amd as t2
    from t2fw_amd import _lib
    lib, (B, T, D, taps), code = _lib.load(), shape, 0 if dtype == torch.float32 else 2
    x, gy = rand(B, T, D).to(dtype), rand(B, T, D, seed=1).to(dtype)
    w, bias, s0, gs = rand(D, taps).to(dtype), rand(D).to(dtype), rand(B, taps - 1, D).to(dtype), rand(B, taps - 1, D, seed=1).to(dtype)
    f = Frame()
    x_, w_, bias_, s0_, gy_, gs_ = map(f.given, (x, w, bias, s0, gy, gs))
    y, last = f.result(B, T, D, dtype=dtype), f.result(B, taps - 1, D, dtype=dtype)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.t2fw_short_conv_forward(*map(pointer, (x_, w_, bias_, s0_)), None, y.data_ptr(), last.data_ptr(), B, T, D, taps, None, code, 1, stream) == 0
    room = lib.t2fw_short_conv_backward_workspace_bytes(B, T, D, taps, code)
    space = f.result((room + 3) // 4)
    like = [f.result(*t.shape, dtype=dtype) for t in (x, w, bias, s0)]
    assert lib.t2fw_short_conv_backward(*map(pointer, (gy_, gs_, x_, w_, bias_, s0_)), None, *map(pointer, like), B, T, D, taps, None, code, 1, space.data_ptr(), room, stream) == 0
    torch.cuda.synchronize()
    f.check()
    leaves = [t.clone().requires_grad_(True) for t in (x, w, bias, s0)]
    out = t2.short_conv(*leaves, silu=True)
    grads = torch.autograd.grad(out, leaves, (gy, gs))
    assert torch.equal(out[0], y) and torch.equal(out[1], last)
    assert all(torch.equal(p, q) for p, q in zip(grads, like))

"""policy_loss against its formula in float64, and against differences of itself.

Bounds.  A log-sum-exp of V terms: the exponentials are within e of themselves (2^-19 for 16-bit logits, of which the hardware's
exponential takes arguments down to -40; 2^-22 for float32), the sum adds at most V / 4096 + 32 roundings, its logarithm and the
subtraction from the logit one of |z| each: logp is within d = e + (V / 4096 + 32) 2^-24 + 4 max|z| 2^-24.  The ratio and exp(ref - logp)
are within d (and 2^-22) of themselves; a row's coefficient within share (|A| r + kl e^(ref - logp)) 2 (d + 2^-21), and the gradient within
p of that plus |c| p (e + d).  Storing rounds to half a unit in the last place."""
import pytest
import torch

from tests.test_gated_scan import STORE, TINY

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
CLIP, KL = (0.2, 0.3), 0.1


def inputs(N, V, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(N, V, generator=g) * spread).to(dtype)
    targets = torch.randint(0, V, (N,), generator=g)
    logp = torch.log_softmax(logits.double(), 1).gather(1, targets[:, None])[:, 0]
    # ratios well away from the edges of the clip, on both sides of them
    step = torch.tensor([-0.6, -0.15, 0.05, 0.18, 0.5])[torch.randint(0, 5, (N,), generator=g)]
    old, ref = (logp - step).float(), (logp + 0.3 * torch.randn(N, generator=g)).float()
    adv, mask = torch.randn(N, generator=g), torch.rand(N, generator=g) < 0.7
    if N:
        mask[0] = True
    return [t.cuda() for t in (logits, targets, old, ref, adv, mask)]


def reference(logits, targets, old, ref, adv, mask, scale=1.0, kl=KL):
    z, old, ref, adv = (t.detach().double().cpu() for t in (logits, old, ref, adv))
    targets = targets.cpu()
    N, V = z.shape
    m = torch.ones(N, dtype=torch.bool) if mask is None else mask.cpu()
    z.requires_grad_(True)
    lp_all = torch.log_softmax(z, 1)
    logp = lp_all[torch.arange(N), targets]
    r, d = torch.exp(logp - old), ref - logp
    each = -torch.minimum(r * adv, r.clamp(1 - CLIP[0], 1 + CLIP[1]) * adv) + kl * (torch.exp(d) - 1 - d)
    M = max(int(m.sum()), 1)
    loss = scale * (each * m).sum() / M
    grad, = torch.autograd.grad(loss, z)
    with torch.no_grad():
        big = z.abs().amax(1) if V else torch.zeros(N)
        e = 2.0 ** -22 if logits.dtype == torch.float32 else 2.0 ** -19
        dl = e + (V / 4096 + 32) * 2.0 ** -24 + 4 * big * 2.0 ** -24
        rough = (adv.abs() * r + kl * torch.exp(d)) * 2 * (dl + 2.0 ** -21)
        p = lp_all.exp()
        onehot = torch.zeros_like(p).scatter_(1, targets[:, None], 1.0)
        c = scale / M * (adv.abs() * r + kl * (torch.exp(d) + 1))
        b_grad = (m * (scale / M))[:, None].abs() * rough[:, None] * (p + onehot) + (c * m).abs()[:, None] * p * (e + dl[:, None]) + grad.abs() * 2.0 ** -22
        b_loss = abs(scale) / M * float((m * (rough + kl * d.abs() * 2.0 ** -22 + each.abs() * 2.0 ** -22)).sum()) + float(loss.abs()) * 2.0 ** -22
    return {"loss": (loss.detach(), torch.tensor(b_loss)), "logp": (logp.detach(), dl + logp.detach().abs() * 2.0 ** -23), "grad": (grad, b_grad)}


def check(name, got, ref):
    value, bound = ref
    got64 = got.detach().double().cpu()
    assert got64.shape == value.shape, name
    bound = bound + STORE[got.dtype] * (value.abs() + bound) + TINY[got.dtype]
    off = (got64 - value).abs() - bound
    assert bool((off <= 0).all()), "%s: %d of %d outside, worst by %.3e" % (name, int((off > 0).sum()), off.numel(), float(off.max()))


def call(ins, **more):
    import t2fw_amd as t2
    return t2.policy_loss(*ins[:5], mask=ins[5], clip=CLIP, kl_coef=KL, **more)


# vocabularies of one word, of less than a vector, odd, one more than the threads' vectors, more than what fits their registers
SHAPES = [(1, 1), (3, 2), (5, 7), (2, 1000), (70, 513), (3, 8193), (9, 20011), (4, 50257), (2, 70001), (2, 140000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, dtype):
    ins = inputs(*shape, dtype, seed=sum(shape))
    ins[0].requires_grad_(True)
    loss, logp = call(ins)
    assert loss.dtype == logp.dtype == torch.float32 and loss.shape == () and not logp.requires_grad
    grad, = torch.autograd.grad(loss, ins[0])
    ref = reference(*ins)
    for n, v in (("loss", loss), ("logp", logp), ("grad", grad)):
        check(n, v, ref[n])
    with torch.no_grad():
        again, logp_again = call(ins)
    assert torch.equal(again, loss) and torch.equal(logp_again, logp)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(7, 300), (40, 8000), (3, 140000)], ids=str)
def test_a_common_offset_of_the_logits_changes_no_bit(shape):
    """32-bit logits in steps of 1/64, 4096 more of each: nothing is rounded in the addition, nor in a difference of two"""
    ins = inputs(*shape, torch.float32, seed=11)
    results = []
    for offset in (0.0, 4096.0):
        z = ((ins[0] * 64).round() / 64 + offset).requires_grad_(True)
        loss, logp = call([z] + ins[1:])
        results.append((loss, logp, torch.autograd.grad(loss, z, retain_graph=True)[0], torch.autograd.grad(3 * loss, z)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_any_factor_of_the_loss(dtype):
    """a factor as `scale`, one that the loss is multiplied by, and a second backward of one forward"""
    ins = inputs(50, 3001, dtype, seed=5)
    z = ins[0].requires_grad_(True)
    factor = 1024.0 if dtype == torch.float16 else 0.37
    ref = reference(*ins, scale=factor)
    loss, _ = call(ins, scale=factor)
    check("loss", loss, ref["loss"])
    first, = torch.autograd.grad(loss, z, retain_graph=True)
    kept = first.clone()
    second, = torch.autograd.grad(loss, z)
    assert torch.equal(first, kept) and torch.equal(second, kept) and second.data_ptr() != first.data_ptr()
    check("grad", first, ref["grad"])
    loss, _ = call(ins)
    outer, = torch.autograd.grad(loss * factor, z, retain_graph=True)
    check("grad", outer, ref["grad"])
    one, = torch.autograd.grad(loss, z)
    check("grad", one, reference(*ins)["grad"])
    # accumulated by torch: the second backward must not find its own buffer in the first's place
    z.grad = None
    loss, _ = call(ins)
    loss.backward(retain_graph=True)
    loss.backward()
    assert torch.equal(z.grad, 2 * one)
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(call(ins)[0], z, create_graph=True)


@pytest.mark.gpu
def test_masks_that_leave_nothing_and_tokens_outside():
    ins = inputs(12, 700, torch.bfloat16, seed=1)
    z, targets, mask = ins[0], ins[1], ins[5]
    mask[:] = False
    z.requires_grad_(True)
    loss, _ = call(ins)
    assert float(loss) == 0.0 and bool((torch.autograd.grad(loss, z)[0] == 0).all())
    # padding: any target, any logits
    mask[:6] = True
    targets[6:9] = torch.tensor([-100, 700, 1 << 40], device="cuda")
    with torch.no_grad():
        z[9] = float("nan")
        z[10] = float("-inf")
        z[11, :300] = float("inf")
    loss, logp = call(ins)
    grad, = torch.autograd.grad(loss, z)
    ref = reference(*[t[:6] for t in ins])
    check("loss", loss, ref["loss"])
    check("logp", logp[:6], ref["logp"])
    check("grad", grad[:6], ref["grad"])
    assert bool((grad[6:] == 0).all()) and bool((logp[6:9] == 0).all())
    mask[6] = True                                      # a token that counts has to be one
    assert bool(torch.isnan(call(ins)[0]))
    assert bool(torch.isfinite(call(ins[:5] + [None])[0])) is False


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_words_that_are_ruled_out(dtype):
    """logits of minus infinity, and of the type's lowest value"""
    ins = inputs(8, 5000, dtype, seed=2)
    z, targets = ins[0], ins[1]
    out = torch.zeros_like(z, dtype=torch.bool)
    out[:, 1000:] = True
    out[torch.arange(8), targets] = False
    low = z.masked_fill(out, torch.finfo(dtype).min)
    none = z.masked_fill(out, float("-inf"))
    results = []
    for logits in (low, none):
        logits.requires_grad_(True)
        loss, logp = call([logits] + ins[1:])
        results.append((loss, logp, torch.autograd.grad(loss, logits)[0]))
        assert all(bool(torch.isfinite(t).all()) for t in results[-1]) and bool((results[-1][2][out] == 0).all())
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_gradient_against_differences():
    """Along random directions, steps of 2^-6: the difference quotient is off by a third derivative times 2^-12 / 6 (below 1e-3 for these
    sizes) and the losses' rounding, 2^-23 of about one, over the step"""
    ins = inputs(6, 40, torch.float32, seed=3, spread=1.0)
    z = ins[0].requires_grad_(True)
    loss, _ = call(ins)
    grad, = torch.autograd.grad(loss, z)
    g = torch.Generator(device="cuda").manual_seed(0)
    for _ in range(5):
        v = torch.randn(z.shape, generator=g, device="cuda")
        v /= v.norm()
        step = 2.0 ** -6
        with torch.no_grad():
            diff = (call([z + step * v] + ins[1:])[0] - call([z - step * v] + ins[1:])[0]) / (2 * step)
        assert abs(float(diff) - float((grad * v).sum())) < 1e-3 * max(1.0, float(grad.norm()))


@pytest.mark.gpu
def test_leading_axes_another_stream_and_a_graph():
    import t2fw_amd as t2
    ins = inputs(60, 2001, torch.bfloat16, seed=9)

    def run(ins):
        z = ins[0].detach().requires_grad_(True)
        loss, logp = call([z] + ins[1:])
        return loss.detach(), logp, torch.autograd.grad(loss, z)[0]
    want = run(ins)
    shaped = run([ins[0].view(4, 15, 2001)] + [t.view(4, 15) for t in ins[1:]])
    assert shaped[1].shape == (4, 15) and all(torch.equal(a.view(b.shape), b) for a, b in zip(shaped, want))
    assert all(torch.equal(a, b) for a, b in zip(run(ins), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(ins)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    buffers = [t.clone() for t in ins]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(buffers)
    for seed in (21, 22, 23):
        fresh = inputs(60, 2001, torch.bfloat16, seed=seed)
        for b, t in zip(buffers, fresh):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(run(fresh), captured))


@pytest.mark.gpu
def test_refusals():
    import t2fw_amd as t2
    z, t, old, ref, adv, mask = inputs(6, 30, torch.float32, seed=0)
    good = dict(logits=z, targets=t, old_logp=old, ref_logp=ref, advantages=adv, mask=mask)
    for bad in (dict(logits=z.double()), dict(logits=z.cpu()), dict(logits=z.t()), dict(targets=t[:3]), dict(targets=t.int()), dict(old_logp=old.half()),
                dict(ref_logp=ref.cpu()), dict(advantages=adv[:, None]), dict(mask=mask.int()), dict(mask=mask[:2]), dict(clip=(-1.0, -3.0)),
                dict(advantages=adv.clone().requires_grad_(True)), dict(logits=z[:, :0])):
        with pytest.raises(RuntimeError):
            t2.policy_loss(**{**good, **bad})
    loss, logp = t2.policy_loss(z[:0], t[:0], old[:0], ref[:0], adv[:0])
    assert float(loss) == 0 and logp.shape == (0,)


def test_host_memory_and_bad_c_calls_are_refused():
    import ctypes
    import t2fw_amd as t2
    from t2fw_amd import _lib
    with pytest.raises(RuntimeError, match="CUDA"):
        t2.policy_loss(*(torch.zeros(1, 2),) * 5)
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.c_void_p(ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 64)

    def forward(ptrs=(p,) * 11, N=1, V=8, low=0.8, high=1.2, dtype=0, ws=p, n=4096):
        return lib.t2fw_policy_loss_forward(*ptrs, N, V, low, high, 0.0, 1.0, dtype, ws, n, None)
    assert forward(dtype=3) == 2 and forward(N=-1) == 3 and forward(V=0) == 3 and forward(N=1 << 31) == 3 and forward(low=2.0) == 3
    assert forward(low=float("nan")) == 3 and forward(n=0) == 6 and forward(ws=None) == 1
    assert forward(ptrs=(None,) + (p,) * 10) == 1 and forward(ptrs=(ctypes.c_void_p(p.value + 1),) + (p,) * 10) == 4
    assert lib.t2fw_policy_loss_backward(*(p,) * 6, 1, 8, 0, 4, None) == 5 and lib.t2fw_policy_loss_backward(*(None,) * 6, 1, 8, 0, 0, None) == 1

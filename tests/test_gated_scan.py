"""gated_scan and gated_scan_step against the recurrence written out in float64.

Bounds.  A step rounds the gate, a product and a sum, and the composition of stretches rounds no more often than that per step: with
A_t the recurrence of the absolute values, the error of h_t is at most E_t = |f_t| E_{t-1} + 4 u A_t, u the larger of 2^-24
(2^-53 for float64) and the gate's own error where it comes from a logit (2^-20 by the hardware's exponential and
reciprocal, 2^-22 by the library's, 2^-50 in float64).  The adjoint obeys the same; a product of two such numbers adds their
relative errors.  What is stored is rounded to half a unit in the last place of its type."""
import pytest
import torch

STORE = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float64: 0.0, torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
DTYPES = [torch.float32, torch.float16, torch.bfloat16, torch.float64]


def unit(dtype, logits):
    if dtype == torch.float64:
        return 2.0 ** -50 if logits else 2.0 ** -53
    if not logits:
        return 2.0 ** -24
    return 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -20


def wide(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def reference(x, f, s, lengths, logits, u, go=None, gs=None):
    """name -> (value, bound before storing), all in float64 on the CPU"""
    x, f, s = (t.detach().double().cpu() for t in (x, f, s))
    gate = torch.sigmoid(f) if logits else f
    B, T, D = x.shape
    live = torch.ones(B, T, 1, dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(T)[None, :, None] < lengths.cpu().long().clamp(0, T)[:, None, None]
    x, gate_in = torch.where(live, x, torch.zeros(())), torch.where(live, gate, torch.ones(()).double())
    h, a, e = s, s.abs(), torch.zeros_like(s)
    hs, befores, es = [], [], []
    for t in range(T):
        befores.append((h, e))
        h = gate_in[:, t] * h + x[:, t]
        a = gate_in[:, t].abs() * a + x[:, t].abs()
        e = gate_in[:, t].abs() * e + 4 * u * a
        hs.append(h)
        es.append(e)
    zero = x.new_zeros(B, T, D)
    out = {"h": (torch.stack(hs, 1) * live if T else zero, torch.stack(es, 1) * live if T else zero), "last": (h, e)}
    if go is None:
        return out
    go = torch.where(live, go.double().cpu(), torch.zeros(()).double())
    adj, aa, ae = gs.double().cpu(), gs.double().cpu().abs(), torch.zeros_like(s)
    dx, df = [None] * T, [None] * T
    for t in reversed(range(T)):
        g, ga, ge = adj + go[:, t], aa + go[:, t].abs(), ae
        before, before_e = befores[t]
        d, de = g * before, ge * before.abs() + g.abs() * before_e + 4 * u * (ga * before.abs())
        if logits:
            slope = torch.sigmoid(f[:, t]) * torch.sigmoid(-f[:, t])
            d, de = d * slope, de * slope + 8 * u * (d * slope).abs()
        k = live[:, t]
        dx[t], df[t] = (g * k, (ge + 4 * u * ga) * k), (torch.where(k, d, torch.zeros(()).double()), torch.where(k, de, torch.zeros(()).double()))
        adj, aa, ae = gate_in[:, t] * g, gate_in[:, t].abs() * ga, gate_in[:, t].abs() * ge + 4 * u * (gate_in[:, t].abs() * ga)
    out["d_state"] = (adj, ae)
    out["d_x"] = (torch.stack([v for v, _ in dx], 1), torch.stack([b for _, b in dx], 1)) if T else (zero, zero)
    out["d_f"] = (torch.stack([v for v, _ in df], 1), torch.stack([b for _, b in df], 1)) if T else (zero, zero)
    return out


def check(name, got, ref):
    value, bound = ref
    got64 = got.detach().double().cpu()
    assert got64.shape == value.shape, name
    bound = bound + STORE[got.dtype] * (value.abs() + bound) + TINY[got.dtype]
    off = (got64 - value).abs() - bound
    assert bool((off <= 0).all()), "%s: %d of %d outside, worst by %.3e" % (name, int((off > 0).sum()), off.numel(), float(off.max()))


def inputs(B, T, D, dtype, logits, seed, mean=2.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, T, D, generator=g) + mean
    make = lambda *s: torch.randn(*s, generator=g)
    x, f, s = make(B, T, D).to(dtype), (z if logits else torch.sigmoid(z)).to(dtype), make(B, D).to(wide(dtype))
    return [t.cuda() for t in (x, f, s)], make(B, T, D).to(dtype).cuda(), make(B, D).to(wide(dtype)).cuda()


def run(ins, lengths, logits, go, gs):
    import t2fw_amd as t2
    ins = [t.detach().requires_grad_(True) for t in ins]
    h, last = t2.gated_scan(*ins, lengths=lengths, logits=logits)
    grads = torch.autograd.grad((h, last), ins, (go, gs))
    return dict(zip(("h", "last", "d_x", "d_f", "d_state"), (h, last) + grads))


# one token, one less and one more than a chunk, many chunks; widths of less than a vector, odd ones, several workgroups
SHAPES = [(1, 1, 1), (2, 3, 5), (3, 128, 64), (1, 129, 7), (2, 127, 65), (5, 64, 8), (1, 1500, 24), (4, 257, 200), (2, 700, 333), (37, 31, 9)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("logits", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, logits, dtype):
    ins, go, gs = inputs(*shape, dtype, logits, seed=sum(shape))
    got = run(ins, None, logits, go, gs)
    ref = reference(*ins, None, logits, unit(dtype, logits), go, gs)
    for n in ref:
        check(n, got[n], ref[n])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(3000, 7, 90), (2901, 1, 97), (700, 20, 100), (667, 32, 103), (66000, 3, 5), (1400, 13, 96), (341, 60, 97), (5000, 16, 3)], ids=str)
def test_few_steps_of_many_rows(shape, dtype):
    """more channels to a workgroup, which has the whole sequence; ragged"""
    ins, go, gs = inputs(*shape, dtype, True, seed=sum(shape))
    lengths = torch.randint(0, shape[1] + 1, (shape[0],), generator=torch.Generator().manual_seed(1))
    got = run(ins, lengths.cuda(), True, go, gs)
    ref = reference(*ins, lengths, True, unit(dtype, True), go, gs)
    for n in ref:
        check(n, got[n], ref[n])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("D", [24, 70, 130])
def test_many_chunks(D, dtype):
    """several groups of chunks, one to three workgroups side by side"""
    ins, go, gs = inputs(1, 17001, D, dtype, True, seed=D, mean=5.0)
    lengths = torch.tensor([16890])
    got = run(ins, lengths.cuda(), True, go, gs)
    ref = reference(*ins, lengths, True, unit(dtype, True), go, gs)
    for n in ref:
        check(n, got[n], ref[n])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.int64, torch.int32], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("T,D", [(5, 16), (300, 24), (513, 65)])
def test_rows_end_at_their_lengths_whatever_follows(T, D, dtype, kind):
    lengths = torch.tensor([0, 1, T, T - 1, T // 2, T + 7, -3], dtype=kind)
    ins, go, gs = inputs(len(lengths), T, D, dtype, True, seed=T)
    for b, n in enumerate(lengths.tolist()):
        n = max(0, min(T, n))
        for t in (ins[0], ins[1], go):
            t[b, n:] = float("nan")
            t[b, n + 1:n + 2] = float("inf")
    got = run(ins, lengths.cuda(), True, go, gs)
    ref = reference(*[t.nan_to_num(0, 0, 0) for t in ins], lengths, True, unit(dtype, True), go.nan_to_num(0, 0, 0), gs)
    for n in ref:
        check(n, got[n], ref[n])
    # nothing of a row without steps: its state passes as it is
    assert torch.equal(got["last"][0], ins[2][0]) and torch.equal(got["d_state"][0], gs[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=str)
def test_parts_of_a_projection_and_broadcast_gates(dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    both = torch.randn(3, 200, 2 * 40 + 1, generator=g, device="cuda").to(dtype).requires_grad_(True)
    import t2fw_amd as t2
    x, f = both[..., 1:41], both[..., 41:]
    h, last = t2.gated_scan(x, f, None, logits=True)
    go, gs = torch.randn(h.shape, generator=g, device="cuda").to(dtype), torch.randn(last.shape, generator=g, device="cuda")
    d_both, = torch.autograd.grad((h, last), both, (go, gs))
    ref = reference(x, f, torch.zeros(3, 40), None, True, unit(dtype, True), go, gs)
    for n, v in (("h", h), ("last", last), ("d_x", d_both[..., 1:41]), ("d_f", d_both[..., 41:])):
        check(n, v, ref[n])
    # time before batch in memory, one gate for every step and row
    xt = torch.randn(200, 3, 40, generator=g, device="cuda").to(dtype).transpose(0, 1)
    gate = torch.sigmoid(torch.randn(40, generator=g, device="cuda")).to(dtype).requires_grad_(True)
    h, last = t2.gated_scan(xt, gate.expand(3, 200, 40))
    ref = reference(xt, gate.expand(3, 200, 40), torch.zeros(3, 40), None, False, unit(dtype, False), go, torch.zeros_like(gs))
    check("h", h, ref["h"])
    # a gradient that is one value everywhere, as that of a sum
    d_gate, = torch.autograd.grad(h.sum(), gate)
    one = reference(xt, gate.expand(3, 200, 40), torch.zeros(3, 40), None, False, unit(dtype, False), torch.ones(3, 200, 40), torch.zeros(3, 40))
    value, bound = one["d_f"]
    assert bool(((d_gate.double().cpu() - value.sum((0, 1))).abs() <= (bound + 2 * STORE[dtype] * value.abs()).sum((0, 1)) +
                 STORE[dtype] * value.sum((0, 1)).abs()).all())


@pytest.mark.gpu
def test_results_that_nothing_depends_on_and_inputs_without_gradients():
    import t2fw_amd as t2
    ins, go, gs = inputs(2, 150, 20, torch.float32, False, seed=4)
    x, f, s = (t.requires_grad_(True) for t in ins)
    h, last = t2.gated_scan(x, f, s)
    by_last = torch.autograd.grad(last, (x, f, s), gs, retain_graph=True)
    by_h = torch.autograd.grad(h, (x, f, s), go)
    ref_last = reference(x, f, s, None, False, 2.0 ** -24, torch.zeros_like(go), gs)
    ref_h = reference(x, f, s, None, False, 2.0 ** -24, go, torch.zeros_like(gs))
    for got, ref in ((by_last, ref_last), (by_h, ref_h)):
        for n, v in zip(("d_x", "d_f", "d_state"), got):
            check(n, v, ref[n])
    only_x, = torch.autograd.grad(t2.gated_scan(x, f.detach(), s.detach())[0], x, go)
    assert torch.equal(only_x, by_h[0])
    with torch.no_grad():
        assert not t2.gated_scan(x, f, s)[0].requires_grad
    with pytest.raises(RuntimeError, match="once only"):
        torch.autograd.grad(t2.gated_scan(x, f, s)[0].sum(), x, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("logits", [False, True])
def test_gradients_against_differences(logits):
    import t2fw_amd as t2
    ins, _, _ = inputs(2, 70, 3, torch.float64, logits, seed=1)
    lengths = torch.tensor([70, 41], device="cuda")
    ins = [t.requires_grad_(True) for t in ins]
    assert torch.autograd.gradcheck(lambda x, f, s: t2.gated_scan(x, f, s, lengths=lengths, logits=logits), ins, fast_mode=True)


@pytest.mark.gpu
def test_gates_of_zero_one_and_above_and_values_that_are_not_finite():
    import t2fw_amd as t2
    x = torch.ones(1, 400, 16, device="cuda")
    f = torch.ones_like(x)
    f[:, 100] = 0.0                                     # forgets everything
    h, last = t2.gated_scan(x, f)
    count = torch.cat((torch.arange(1, 101), torch.arange(1, 301))).float().cuda()
    assert torch.equal(h[0, :, 3], count) and torch.equal(last, h[:, -1])
    f = torch.full_like(x, 1.0)
    f[:, 7] = -1.5                                      # gates are any numbers
    assert torch.equal(t2.gated_scan(x, f)[0][0, 7], torch.full((16,), -9.5, device="cuda"))
    x[0, 200, 2] = float("nan")
    x[0, 200, 4] = float("inf")
    h, _ = t2.gated_scan(x, torch.ones_like(x))
    assert torch.isfinite(h[0, :200]).all() and torch.isnan(h[0, 200:, 2]).all() and torch.isinf(h[0, 200:, 4]).all()
    assert torch.isfinite(h[0, :, [0, 1, 3, 5]]).all()
    z = torch.full_like(x, 200.0)
    z[:, ::2] = -200.0                                  # logits whose gates are zero and one
    assert torch.isfinite(t2.gated_scan(torch.ones_like(x), z, logits=True)[0]).all()


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits_and_parts_join():
    import t2fw_amd as t2
    ins, go, gs = inputs(3, 1999, 100, torch.bfloat16, True, seed=7)
    first = run(ins, None, True, go, gs)
    for _ in range(3):
        again = run(ins, None, True, go, gs)
        assert all(torch.equal(first[n], again[n]) for n in first)
    # a sequence cut in two, the state handed on: float32 states, so the cut adds no rounding to 16 bits
    x, f, s = ins
    a, mid = t2.gated_scan(x[:, :777], f[:, :777], s, logits=True)
    b, last = t2.gated_scan(x[:, 777:], f[:, 777:], mid, logits=True)
    ref = reference(x, f, s, None, True, unit(torch.bfloat16, True))
    check("h", torch.cat((a, b), 1), ref["h"])
    check("last", last, ref["last"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("B,D", [(1, 1), (3, 7), (64, 768), (5, 1001)])
def test_steps_follow_the_sequence(B, D, dtype):
    import t2fw_amd as t2
    (x, f, s), _, _ = inputs(B, 4, D, dtype, True, seed=B + D)
    state, outs = s.clone(), []
    for t in range(4):
        out, same = t2.gated_scan_step(x[:, t].contiguous(), f[:, t].contiguous(), state, logits=True)
        assert same is state
        outs.append(out)
    ref = reference(x, f, s, None, True, unit(dtype, True))
    check("h", torch.stack(outs, 1), ref["h"])
    check("last", state, ref["last"])
    kept, mine = state.clone(), torch.empty_like(out)
    got, nxt = t2.gated_scan_step(x[:, 0].contiguous(), f[:, 0].contiguous(), state, out=mine, inplace=False)
    assert got is mine and nxt is not state and torch.equal(state, kept)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    import t2fw_amd as t2
    ins, go, gs = inputs(4, 700, 96, torch.bfloat16, True, seed=3)
    want = run(ins, None, True, go, gs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(ins, None, True, go, gs)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want[n], got[n]) for n in want)
    buffers = [t.clone() for t in ins]
    with torch.cuda.stream(side):
        run(buffers, None, True, go, gs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(buffers, None, True, go, gs)
    for seed in (11, 12, 13):
        fresh, _, _ = inputs(4, 700, 96, torch.bfloat16, True, seed=seed)
        for b, t in zip(buffers, fresh):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(fresh, None, True, go, gs)
        assert all(torch.equal(eager[n], captured[n]) for n in eager)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape,ragged", [((2, 900, 40), False), ((1, 2600, 7), True), ((3, 1300, 5), False), ((2, 5000, 65), True), ((1, 17001, 24), False)], ids=str)
def test_chunks_that_do_without_one_another(shape, ragged, dtype):
    """the same bits where no chunk waits for another's map and makes those before it itself"""
    from t2fw_amd import _lib
    lib = _lib.load()
    B, T, D = shape
    (x, f, s), go, gs = inputs(B, T, D, dtype, True, seed=T)
    lengths = torch.tensor([T - 130, T, T // 3][:B], device="cuda") if ragged else None
    code, st = _lib.DTYPE_CODE[dtype], _lib.current_stream_handle(x.device)
    nc, nw = lib.t2fw_gated_scan_checkpoint_bytes(B, T, D, code), lib.t2fw_gated_scan_workspace_bytes(B, T, D, code)
    assert nw > 0
    results = []
    for flags in (3, 3 | 4):
        out, last, dx, df, ds = torch.empty_like(x), torch.empty_like(s), torch.empty_like(x), torch.empty_like(x), torch.empty_like(s)
        ckpt, ws = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in (nc, nw))
        p = _lib.ptr
        _lib.check(lib.t2fw_gated_scan_forward(p(x), p(f), p(s), p(lengths), p(out), p(last), p(ckpt), B, T, D, None, code, flags, p(ws), nw, st))
        _lib.check(lib.t2fw_gated_scan_backward(p(go), p(gs), p(x), p(f), p(lengths), p(ckpt), p(dx), p(df), p(ds), B, T, D, None, code, flags,
                                                p(ws), nw, st))
        torch.cuda.synchronize()
        results.append((out, last, dx, df, ds))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_refusals():
    import t2fw_amd as t2
    x = torch.zeros(2, 3, 8, device="cuda")
    s = torch.zeros(2, 8, device="cuda")
    for bad in (dict(x=x[0], f=x[0]), dict(f=x[:, :2]), dict(f=x.half()), dict(state=s[:1]), dict(state=s.half()), dict(state=s.cpu()),
                dict(f=x.cpu()), dict(lengths=torch.zeros(3, dtype=torch.int64, device="cuda")), dict(lengths=torch.zeros(2, device="cuda")),
                dict(lengths=torch.zeros(2, dtype=torch.int64)), dict(x=x.transpose(1, 2), f=x.transpose(1, 2)),
                dict(x=x.long(), f=x.long()), dict(x=torch.zeros(2, 3, 0, device="cuda"), f=torch.zeros(2, 3, 0, device="cuda"))):
        with pytest.raises(RuntimeError):
            t2.gated_scan(**{**dict(x=x, f=x), **bad})
    for bad in (dict(x=x), dict(f=x[0]), dict(state=s.half()), dict(state=s[:, :4]), dict(out=torch.zeros(2, 8, device="cuda").half()),
                dict(x=x[:, 0].requires_grad_(True))):
        with pytest.raises(RuntimeError):
            t2.gated_scan_step(**{**dict(x=s, f=s, state=s.clone()), **bad})
    empty, last = t2.gated_scan(x[:, :0], x[:, :0], s)
    assert empty.shape == (2, 0, 8) and torch.equal(last, s)
    assert t2.gated_scan(x[:0], x[:0])[1].shape == (0, 8)


def test_host_memory_is_refused():
    import t2fw_amd as t2
    with pytest.raises(RuntimeError, match="CUDA"):
        t2.gated_scan(torch.zeros(1, 1, 1), torch.zeros(1, 1, 1))
    with pytest.raises(TypeError):
        t2.gated_scan_step(None, None, None)


def test_c_entries_refuse_bad_arguments():
    import ctypes
    from t2fw_amd import _lib
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    at = ctypes.addressof(buf)
    p = ctypes.c_void_p(at + (-at) % 64)

    def forward(ptrs=(p,) * 7, B=1, T=1, D=8, strides=None, dtype=0, flags=0, ws=p, n=4096):
        return lib.t2fw_gated_scan_forward(*ptrs, B, T, D, strides, dtype, flags, ws, n, None)

    assert forward(dtype=9) == 2 and forward(B=-1) == 3 and forward(D=0) == 3 and forward(flags=64) == 5
    assert forward(B=1 << 40, T=1 << 20, D=1 << 20) == 3
    assert forward(ptrs=(None,) + (p,) * 6) == 1 and b"x" in lib.t2fw_last_error()
    assert forward(ptrs=(p,) * 5 + (None, p)) == 1
    assert forward(ptrs=(ctypes.c_void_p(p.value + 2),) + (p,) * 6) == 4
    assert forward(T=5000, n=0) == 6 and forward(T=5000, ws=None) == 1
    assert forward(strides=(ctypes.c_int64 * 4)(-1, 1, 1, 1)) == 3
    assert forward(B=0) == 0
    assert lib.t2fw_gated_scan_backward(*(None,) * 9, 1, 1, 8, None, 0, 0, None, 0, None) == 1
    assert lib.t2fw_gated_scan_step(*(None,) * 5, 1, 8, 0, 0, None) == 1
    assert lib.t2fw_gated_scan_workspace_bytes(4, 1, 8, 0) == 0 and lib.t2fw_gated_scan_workspace_bytes(4, 5000, 8, 0) > 0
    assert lib.t2fw_gated_scan_checkpoint_bytes(0, 1, 8, 0) == 0 and lib.t2fw_gated_scan_checkpoint_bytes(4, 1, 8, 9) == 0

"""selective_scan and selective_scan_step against the recurrence written out in float64.

Bounds, u = 2^-24; M and GM are the recurrence and its adjoint of absolute values.
* A step's length by the softplus is off by 2^-20 of itself (hardware exponential and reciprocal, 2^-22 each, a series cut at 2^-26, six roundings) and
  by twice the rounding of dt + bias; without the softplus by that alone.
* A decay exp(dt a): the length's error times |a|, three roundings of the exponent, 2^-22 |dt a|, and the exponential's own 2^-22 and a product's rounding, 2^-21.
  Over chunks the exponent is a times a sum of lengths, in four shares of at most T / 4 terms each: T 2^-25 |dt a| more for every step.
  (Of more than 48 chunks, T / 16 at most, the sums are put together by chunks / 64 + 7 additions, which with a chunk's own T / 4 / 48 are fewer still.)
* A state: E_t = decay E_{t-1} + (its error) decay M_{t-1} + (the input's error) + 2 u M_t.  The adjoint obeys the same.
* A sum of n products of such numbers: the products' errors, and (n + 4) u of the sum of absolute values, in any order.
* The gate's sigmoid: 2^-20 (16-bit tensors, |z| < 40) or 2^-21; its slope that times 1 + |z|.
What is stored is rounded to half a unit in the last place of its type."""
import pytest
import torch

STORE = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24
NAMES = ("x", "dt", "a", "b", "c", "state", "skip", "gate", "dt_bias")


def reference(p, lengths, softplus, gy=None, gs=None):
    """name -> (value, bound before storing), in float64 on the CPU; the gradients by the names of what they belong to"""
    act = 2.0 ** -21 if p["x"].dtype == torch.float32 else 2.0 ** -20
    p = {n: None if t is None else t.detach().double().cpu() for n, t in p.items()}
    (B, T, D), (_, N) = p["x"].shape, p["a"].shape
    zero = torch.zeros(()).double()
    ends = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    live = (torch.arange(T)[None] < ends[:, None])[:, :, None]
    clean = lambda t: torch.where(live, t, zero)
    x, b, c = clean(p["x"]), clean(p["b"]), clean(p["c"])
    a, skip = p["a"], zero.expand(D) if p["skip"] is None else p["skip"]
    bias = zero.expand(D) if p["dt_bias"] is None else p["dt_bias"]
    raw = clean(p["dt"]) + bias
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    dt = clean(torch.logaddexp(raw, zero) if softplus else raw)
    dte = clean((2.0 ** -20 * dt.abs() if softplus else 0) + 2 * U * raw.abs() * slope)
    z = None if p["gate"] is None else clean(p["gate"])
    sig = None if z is None else torch.sigmoid(z)
    state = torch.zeros(B, D, N).double() if p["state"] is None else p["state"]
    h, M, E = state, state.abs(), torch.zeros_like(state)
    saved, y, ye, y0s = [], [], [], []
    for t in range(T):
        A = torch.exp(dt[:, t, :, None] * a)
        Ae = a.abs() * dte[:, t, :, None] + (dt[:, t, :, None] * a).abs() * (2.0 ** -22 + T * 2.0 ** -25) + 2.0 ** -21
        push = (dt[:, t] * x[:, t])[..., None] * b[:, t, None]
        pushe = (dte[:, t] * x[:, t].abs())[..., None] * b[:, t, None].abs() + 3 * U * push.abs()
        saved.append((h, M, E, A, Ae))
        E = A * E + Ae * A * M + pushe
        h, M = A * h + push, A * M + push.abs()
        E = E + 2 * U * M
        E = torch.where(live[:, t, :, None], E, saved[-1][2])
        y0 = (h * c[:, t, None]).sum(-1) + skip * x[:, t]
        y0e = (E * c[:, t, None].abs()).sum(-1) + (N + 4) * U * (M * c[:, t, None].abs()).sum(-1) + 3 * U * (skip * x[:, t]).abs()
        y0s.append((y0, y0e, h, M, E))
        g = torch.ones_like(y0) if z is None else z[:, t] * sig[:, t]
        y.append(y0 * g * live[:, t])
        ye.append((y0e * g.abs() + (0 if z is None else act * (y0 * g).abs()) + 2 * U * (y0 * g).abs()) * live[:, t])
    none = torch.zeros(B, 0, D).double()
    out = {"y": (torch.stack(y, 1) if T else none, torch.stack(ye, 1) if T else none), "last": (h, E)}
    if gy is None:
        return out
    gy = clean(gy.double().cpu())
    adj, AM, AE = gs.double().cpu(), gs.double().cpu().abs(), torch.zeros_like(h)
    grads = {n: [None] * T for n in ("x", "dt", "b", "c", "gate")}
    sums = {n: [torch.zeros(s).double() for _ in range(2)] for n, s in (("a", (D, N)), ("skip", (D,)), ("dt_bias", (D,)))}
    n_all = B * T

    def add(name, value, bound, size):
        sums[name][0] += value.sum(0)
        sums[name][1] += (bound + (n_all + 4) * U * size).sum(0)
    for t in reversed(range(T)):
        hp, Mp, Ep, A, Ae = saved[t]
        y0, y0e, h, M, E = y0s[t]
        k = live[:, t]
        k3 = k[..., None]
        dy, dye = gy[:, t], torch.zeros_like(gy[:, t])
        if z is not None:
            zt, st = z[:, t], sig[:, t]
            dy = dy * zt * st
            dye = (act + 2 * U) * dy.abs()
            sl = st * (1 + zt * (1 - st))
            sle = act * (1 + zt.abs())
            grads["gate"][t] = (gy[:, t] * y0 * sl * k, (gy[:, t].abs() * (y0e * sl.abs() + (y0.abs() + y0e) * sle + 4 * U * (y0 * sl).abs())) * k)
        ct, bt, xt, dtt, dtet, slt = c[:, t, None], b[:, t, None], x[:, t], dt[:, t], dte[:, t], slope[:, t]
        G = adj + dy[..., None] * ct
        GM = AM + dy[..., None].abs() * ct.abs()
        GE = AE + dye[..., None] * ct.abs() + 2 * U * GM
        gb, gbM = (G * bt).sum(-1), (GM * bt.abs()).sum(-1)
        gbe = (GE * bt.abs()).sum(-1) + (N + 4) * U * gbM
        nadj, nAM = A * G, A * GM
        nAE = A * GE + Ae * A * GM + 2 * U * nAM
        q, qM = nadj * hp, nAM * Mp
        qe = nAE * Mp + nAM * Ep + 3 * U * qM
        pa, paM = (q * a).sum(-1), (qM * a.abs()).sum(-1)
        pae = (qe * a.abs()).sum(-1) + (N + 8) * U * paM
        ddt = (pa + xt * gb) * slt * k
        size = (paM + xt.abs() * gbM) * slt
        slope_error = 2.0 ** -20 + U * raw[:, t].abs() if softplus else 0.0
        ddte = ((pae + xt.abs() * gbe) * slt + size * (4 * U + slope_error)) * k
        grads["dt"][t] = (ddt, ddte)
        add("dt_bias", ddt, ddte, size * k)
        grads["x"][t] = ((dtt * gb + skip * dy) * k, (dtt.abs() * gbe + dtet * gbM + skip.abs() * dye + 3 * U * (dtt.abs() * gbM + (skip * dy).abs())) * k)
        add("a", q * dtt[..., None] * k3, (qe * dtt.abs()[..., None] + qM * dtet[..., None]) * k3, qM * dtt.abs()[..., None] * k3)
        add("skip", dy * xt * k, dye * xt.abs() * k, (dy * xt).abs() * k)
        ux = (dtt * xt).abs()[..., None]
        grads["b"][t] = ((G * (dtt * xt)[..., None]).sum(1) * k, ((GE * ux + GM * (dtet * xt.abs())[..., None]).sum(1) + (D + 6) * U * (GM * ux).sum(1)) * k)
        grads["c"][t] = ((dy[..., None] * h).sum(1) * k,
                         ((dye[..., None] * M + dy.abs()[..., None] * E).sum(1) + (D + 6) * U * (dy.abs()[..., None] * M).sum(1)) * k)
        adj, AM, AE = torch.where(k3, nadj, adj), torch.where(k3, nAM, AM), torch.where(k3, nAE, AE)
    for n, v in grads.items():
        if n == "gate" and z is None:
            continue
        shape = (B, T, N) if n in "bc" else (B, T, D)
        out["d_" + n] = tuple(torch.stack([e[i] for e in v], 1) if T else torch.zeros(shape).double() for i in range(2))
    for n, v in sums.items():
        out["d_" + n] = tuple(v)
    out["d_state"] = (adj, AE)
    return out


def check(name, got, ref):
    value, bound = ref
    got64 = got.detach().double().cpu()
    assert got64.shape == value.shape, name
    bound = bound + STORE[got.dtype] * (value.abs() + bound) + TINY[got.dtype]
    off = (got64 - value).abs() - bound
    assert bool((off <= 0).all()), "%s: %d of %d outside, worst by %.3e" % (name, int((~(off <= 0)).sum()), off.numel(), float(off.max()))


def inputs(B, T, D, N, dtype, seed, gated=True, long=False):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g)
    p = {"x": make(B, T, D).to(dtype), "dt": (make(B, T, D) * 0.7).to(dtype),
         "a": -torch.arange(1, N + 1) * torch.exp(0.3 * make(D, N)), "b": make(B, T, N).to(dtype), "c": make(B, T, N).to(dtype), "state": make(B, D, N),
         "skip": make(D), "gate": make(B, T, D).to(dtype) if gated else None, "dt_bias": (make(D) - (5.0 if long else 3.0))}
    return {n: None if t is None else t.cuda() for n, t in p.items()}, make(B, T, D).to(dtype).cuda(), make(B, D, N).cuda()


def run(p, lengths, softplus, gy, gs):
    import t2fw_amd as t2
    p = {n: None if t is None else t.detach().requires_grad_(True) for n, t in p.items()}
    out = t2.selective_scan(*[p[n] for n in NAMES[:5]], lengths=lengths, softplus=softplus, **{n: p[n] for n in NAMES[5:]})
    there = [n for n in NAMES if p[n] is not None]
    grads = torch.autograd.grad(out, [p[n] for n in there], (gy, gs))
    return dict(zip(["y", "last"] + ["d_" + n for n in there], out + grads))


def compare(p, lengths, softplus, gy, gs, ref=None):
    got = run(p, lengths, softplus, gy, gs)
    ref = reference(ref or p, lengths, softplus, gy.nan_to_num(0, 0, 0), gs)
    for n in got:
        check(n, got[n], ref[n])
    return got


# one step, one less and one more than a tile, several chunks; channels of less than a workgroup, one, odd ones; every number of lanes of a channel
SHAPES = [(1, 1, 1, 1), (2, 3, 5, 2), (3, 16, 64, 16), (1, 17, 7, 4), (2, 15, 65, 5), (2, 33, 130, 8), (1, 100, 24, 16), (4, 130, 70, 10), (2, 70, 33, 64),
          (1, 50, 9, 17), (1, 40, 20, 33), (5, 20, 300, 3), (1, 700, 20, 16), (2, 300, 40, 7), (1, 260, 17, 40), (1, 500, 70, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, gated, dtype):
    p, gy, gs = inputs(*shape, dtype, seed=sum(shape), gated=gated)
    compare(p, None, True, gy, gs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("N", [1, 6, 16, 30, 64])
def test_rows_end_at_their_lengths_whatever_follows(N, dtype):
    T = 150
    lengths = torch.tensor([0, 1, T, T - 1, 16, 64, T + 7, -3, 100])
    p, gy, gs = inputs(len(lengths), T, 21, N, dtype, seed=N)
    clean = dict(p)
    for n in ("x", "dt", "b", "c", "gate"):
        p[n] = p[n].clone()
        for b, k in enumerate(lengths.tolist()):
            k = max(0, min(T, k))
            p[n][b, k:] = float("nan")
            p[n][b, k + 1:k + 2] = float("inf")
    for b, k in enumerate(lengths.tolist()):
        gy[b, max(0, min(T, k)):] = float("nan")
    for kind in (torch.int64, torch.int32):
        got = compare(p, lengths.to(kind).cuda(), True, gy, gs, ref=clean)
        # nothing of a row without steps: its state passes as it is
        assert torch.equal(got["last"][0], p["state"][0]) and torch.equal(got["d_state"][0], gs[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_lengths_as_given_and_nothing_that_may_be_missing(dtype):
    """dt as it is, of either sign; no state, skip, gate or bias"""
    import t2fw_amd as t2
    p, gy, gs = inputs(2, 90, 37, 12, dtype, seed=2, gated=False)
    p["dt"] = (p["dt"] * 0.1).contiguous()
    for n in ("state", "skip", "dt_bias"):
        p[n] = None
    got = compare(p, None, False, gy, gs)
    assert set(got) == {"y", "last", "d_x", "d_dt", "d_a", "d_b", "d_c"}
    with torch.no_grad():
        y, last = t2.selective_scan(*[p[n] for n in NAMES[:5]])
    assert torch.equal(y, got["y"]) and torch.equal(last, got["last"]) and not y.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(1, 3000, 12, 16), (3, 1100, 40, 16), (40, 40, 300, 16), (1, 1000, 1030, 14)], ids=str)
def test_many_chunks_and_many_rows(shape, dtype):
    p, gy, gs = inputs(*shape, dtype, seed=7, long=True)
    lengths = torch.randint(0, shape[1] + 1, (shape[0],), generator=torch.Generator().manual_seed(1))
    lengths[0] = shape[1] - 3
    compare(p, lengths.cuda(), True, gy, gs)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 6, 16, 30, 64])
def test_chunks_by_the_hundred(N):
    """their maps put together by a launch of its own: for every number of lanes, with rows that end in the first chunk, before it, and in the last one"""
    B, T, D = 4, 1100, 9
    p, gy, gs = inputs(B, T, D, N, torch.float32, seed=N, long=True)
    compare(p, torch.tensor([T - 1, 0, 7, 530]).cuda(), True, gy, gs)
    got = run(p, None, True, gy, gs)
    alone = [run({n: None if t is None else t[b:b + 1].contiguous() if n in ("x", "dt", "b", "c", "state", "gate") else t for n, t in p.items()}, None, True,
                 gy[b:b + 1].contiguous(), gs[b:b + 1].contiguous()) for b in range(B)]
    # (rows alone are cut in other chunks)
    ref = reference(p, None, True, gy, gs)
    for n in ("y", "last", "d_x", "d_state"):
        check(n, got[n], ref[n])
        check(n, torch.cat([o[n] for o in alone]), ref[n])
    p["state"] = None
    got, ref = run(p, None, True, gy, torch.zeros_like(gs)), reference(p, None, True, gy, torch.zeros_like(gs))
    for n in ("y", "last", "d_x", "d_a"):
        check(n, got[n], ref[n])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_parts_of_a_projection_and_other_orders(dtype):
    import t2fw_amd as t2
    B, T, D, N = 2, 60, 24, 6
    p, gy, gs = inputs(B, T, D, N, dtype, seed=3)
    wide = torch.cat([p["x"], p["dt"], p["gate"], p["b"], p["c"], p["x"][..., :1]], -1).requires_grad_(True)
    x, dt, gate, b, c, _ = wide.split([D, D, D, N, N, 1], dim=-1)
    rest = {n: p[n] for n in ("state", "skip", "dt_bias")}
    y, last = t2.selective_scan(x, dt, p["a"], b, c, gate=gate, softplus=True, **rest)
    ref = reference(p, None, True, gy, gs)
    check("y", y, ref["y"])
    d_wide, = torch.autograd.grad((y, last), wide, (gy.transpose(0, 1).contiguous().transpose(0, 1), gs))
    for n, v in zip(("x", "dt", "gate", "b", "c"), d_wide.split([D, D, D, N, N, 1], dim=-1)):
        check(n, v, ref["d_" + n])
    # time before batch in memory; a gradient that is one value everywhere; a result that nothing depends on
    xt = p["x"].transpose(0, 1).contiguous().transpose(0, 1).requires_grad_(True)
    args = (p["dt"], p["a"], p["b"], p["c"])
    y, last = t2.selective_scan(xt, *args, gate=p["gate"], softplus=True, **rest)
    for out, g, ref in ((y, torch.ones_like(y), reference(p, None, True, torch.ones_like(gy), torch.zeros_like(gs))),
                        (last, gs, reference(p, None, True, torch.zeros_like(gy), gs))):
        check("d_x", torch.autograd.grad((out * g).sum(), xt, retain_graph=True)[0], ref["d_x"])
    check("d_x", torch.autograd.grad(y.sum(), xt)[0], reference(p, None, True, torch.ones_like(gy), torch.zeros_like(gs))["d_x"])
    # one row of b and c for the whole batch
    b1 = p["b"][:1].detach().requires_grad_(True)
    y, last = t2.selective_scan(p["x"], p["dt"], p["a"], b1.expand(B, T, N), p["c"], gate=p["gate"], softplus=True, **rest)
    same = dict(p, b=p["b"][:1].expand(B, T, N))
    value, bound = reference(same, None, True, gy, gs)["d_b"]
    d_b, = torch.autograd.grad((y, last), b1, (gy, gs))
    each = bound + STORE[dtype] * (value.abs() + bound)
    assert bool(((d_b.double().cpu() - value.sum(0, keepdim=True)).abs() <= each.sum(0, keepdim=True) + 2 * STORE[dtype] * (value.abs() + each).sum(0, keepdim=True) + TINY[dtype]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_token_by_token(dtype):
    import t2fw_amd as t2
    for B, D, N, gated in ((5, 37, 16, True), (3, 5, 1, False), (2, 130, 10, True), (1, 9, 64, True)):
        T = 9
        p, _, _ = inputs(B, T, D, N, dtype, seed=D, gated=gated)
        ref = reference(p, None, True)
        state = p["state"].clone()
        wide = torch.randn(B, 3 * D + 2 * N + 1, device="cuda").to(dtype)
        for t in range(T):
            parts = wide.split([D, D, D, N, N, 1], dim=-1)
            for part, n in zip(parts, ("x", "dt", "gate", "b", "c")):
                if p[n] is not None:
                    part.copy_(p[n][:, t])
            args = (parts[0], parts[1], p["a"], parts[3], parts[4])
            options = {"skip": p["skip"], "gate": parts[2] if gated else None, "dt_bias": p["dt_bias"], "softplus": True}
            before = state.clone()
            y, new = t2.selective_scan_step(*args, state, **options)
            assert new is state
            check("y", y, (ref["y"][0][:, t], ref["y"][1][:, t]))
            out = torch.empty_like(y)
            y2, other = t2.selective_scan_step(*args, before, out=out, inplace=False, **options)
            assert y2.data_ptr() == out.data_ptr() and torch.equal(out, y) and torch.equal(other, state) and not torch.equal(before, state)
        check("last", state, ref["last"])


@pytest.mark.gpu
def test_no_steps_and_no_rows():
    import t2fw_amd as t2
    p, gy, gs = inputs(2, 1, 6, 4, torch.float32, seed=0)
    none = {n: p[n][:, :0] if n in ("x", "dt", "b", "c", "gate") else p[n] for n in NAMES}
    got = run(none, None, True, gy[:, :0], gs)
    assert got["y"].shape == (2, 0, 6) and torch.equal(got["last"], p["state"]) and torch.equal(got["d_state"], gs)
    assert not got["d_a"].any() and not got["d_skip"].any() and not got["d_dt_bias"].any() and got["d_b"].shape == (2, 0, 4)
    empty = {n: p[n][:0] if n in ("x", "dt", "b", "c", "gate", "state") else p[n] for n in NAMES}
    got = run(empty, None, True, gy[:0], gs[:0])
    assert got["y"].shape == (0, 1, 6) and not got["d_a"].any()
    with torch.no_grad():
        y, st = t2.selective_scan_step(*[empty[n][:, 0] if n != "a" else empty[n] for n in NAMES[:5]], empty["state"])
    assert y.shape == (0, 6) and st.shape == (0, 6, 4)


@pytest.mark.gpu
def test_long_steps_and_large_numbers():
    """lengths and decays at the ends of their range: nothing forgotten, all forgotten, softplus far out on both sides"""
    p, gy, gs = inputs(1, 64, 16, 4, torch.float32, seed=5)
    p["dt_bias"].zero_()
    p["dt"][0, :16] = -100.0
    p["dt"][0, 16:32] = -12.0
    p["dt"][0, 32:48] = 30.0
    p["dt"][0, 48:] = torch.linspace(-8, 8, 16, device="cuda")[:, None]
    compare(p, None, True, gy, gs)
    p["a"][:, 0] = 0.0                                   # a sum that forgets nothing
    compare(p, None, True, gy, gs)


@pytest.mark.gpu
def test_states_that_forget_at_once_and_steps_that_do_not_count():
    """a decay rate of minus infinity: what is before a step is gone; steps beyond a row's length leave the state all the same"""
    import t2fw_amd as t2
    p, gy, gs = inputs(2, 40, 16, 4, torch.float32, seed=6)
    p["a"][:, 1] = -float("inf")
    lengths = torch.tensor([40, 13], device="cuda")
    out = run(p, lengths, True, gy, gs)
    assert all(bool(torch.isfinite(v).all()) for v in out.values())
    dt = torch.nn.functional.softplus(p["dt"][:, :, :] + p["dt_bias"])
    at = torch.tensor([39, 12], device="cuda")
    row = torch.arange(2, device="cuda")
    want = dt[row, at] * p["x"][row, at] * p["b"][row, at, 1:2]
    assert bool(((out["last"][..., 1] - want).abs() <= 2.0 ** -19 * want.abs()).all())


@pytest.mark.gpu
def test_gradient_against_differences():
    """Directional differences of the float64 sum at distance 1e-5: off by h^2 / 6 of the third derivative and by rounding, 1e-7 of the terms here;
    the gradients' own errors are the bounds above, summed along the direction"""
    p, gy, gs = inputs(2, 40, 6, 5, torch.float32, seed=9)
    lengths = torch.tensor([40, 23])
    got, ref = run(p, lengths.cuda(), True, gy, gs), reference(p, lengths, True, gy, gs)
    g = torch.Generator().manual_seed(2)
    for name in NAMES:
        way = torch.randn(p[name].shape, generator=g).double()

        def at(h):
            moved = {n: t.double().cpu() + (h * way if n == name else 0) for n, t in p.items()}
            r = reference(moved, lengths, True)
            return float((r["y"][0] * gy.double().cpu()).sum() + (r["last"][0] * gs.double().cpu()).sum())
        want = (at(1e-5) - at(-1e-5)) / 2e-5
        v = got["d_" + name].double().cpu()
        most = float(((ref["d_" + name][1] + U * v.abs()) * way.abs()).sum()) + 1e-6 * float((v * way).abs().sum())
        assert abs(float((v * way).sum()) - want) <= most, name


@pytest.mark.gpu
def test_same_bits_every_time_and_whatever_stands_beside():
    """no sum depends on the order in which workgroups are done"""
    p, gy, gs = inputs(3, 400, 100, 16, torch.bfloat16, seed=4)
    first = run(p, None, True, gy, gs)
    for _ in range(3):
        again = run(p, None, True, gy, gs)
        assert all(torch.equal(first[n], again[n]) for n in first)


@pytest.mark.gpu
def test_on_another_stream_and_captured():
    p, gy, gs = inputs(2, 300, 40, 16, torch.bfloat16, seed=5)
    import t2fw_amd as t2
    leaves = {n: t.clone().requires_grad_(True) for n, t in p.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        out = t2.selective_scan(*[leaves[n] for n in NAMES[:5]], softplus=True, **{n: leaves[n] for n in NAMES[5:]})
        return out + torch.autograd.grad(out, [leaves[n] for n in NAMES], (gy, gs))
    with torch.cuda.stream(side):
        eager = [t.detach() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want = run(p, None, True, gy, gs)
    names = ["y", "last"] + ["d_" + n for n in NAMES]
    assert all(torch.equal(want[n], v) for n, v in zip(names, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for k in range(3):
        new, _, _ = inputs(2, 300, 40, 16, torch.bfloat16, seed=6 + k)
        with torch.no_grad():
            for n in NAMES:
                leaves[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        want = run(new, None, True, gy, gs)
        assert all(torch.equal(want[n], v) for n, v in zip(names, res))


def bad_calls():
    import t2fw_amd as t2
    z = lambda *s, **k: torch.zeros(s, device="cuda", **k)
    x, a, b, st = z(2, 5, 8), z(8, 4), z(2, 5, 4), z(2, 8, 4)
    scan = lambda x=x, dt=x, a=a, b=b, c=b, **k: t2.selective_scan(x, dt, a, b, c, **k)
    x1, b1 = z(2, 8), z(2, 4)
    step = lambda x=x1, dt=x1, a=a, b=b1, c=b1, state=st, **k: t2.selective_scan_step(x, dt, a, b, c, state, **k)
    return {
        "x is flat": lambda: scan(x=x1),
        "x has no channels": lambda: scan(x=z(2, 5, 0), dt=z(2, 5, 0), a=z(0, 4)),
        "x by steps": lambda: scan(x=z(2, 8, 5).transpose(1, 2)),
        "x in 64 bits": lambda: t2.selective_scan(x.double(), x.double(), a, b.double(), b.double()),
        "dt of another shape": lambda: scan(dt=z(2, 5, 7)),
        "dt is a number": lambda: scan(dt=z()),
        "gate is a number": lambda: scan(gate=z()),
        "b is a number": lambda: scan(b=z()),
        "a is a number": lambda: scan(a=z()),
        "state is a number": lambda: scan(state=z()),
        "x is a number": lambda: scan(x=z()),
        "dt of another type": lambda: scan(dt=x.half()),
        "b of another type": lambda: scan(b=b.half()),
        "b of other states": lambda: scan(b=z(2, 5, 3)),
        "c of other steps": lambda: scan(c=z(2, 4, 4)),
        "b by states": lambda: scan(b=z(2, 4, 5).transpose(1, 2)),
        "a of other channels": lambda: scan(a=z(7, 4)),
        "a in 16 bits": lambda: scan(a=a.half()),
        "a by states": lambda: scan(a=z(4, 8).t()),
        "no states": lambda: scan(a=z(8, 0), b=z(2, 5, 0), c=z(2, 5, 0)),
        "too many states": lambda: scan(a=z(8, 65), b=z(2, 5, 65), c=z(2, 5, 65)),
        "gate of another shape": lambda: scan(gate=z(2, 5, 4)),
        "gate of another type": lambda: scan(gate=x.half()),
        "state of another shape": lambda: scan(state=z(2, 4, 8)),
        "state in 16 bits": lambda: scan(state=st.half()),
        "skip of other channels": lambda: scan(skip=z(7)),
        "skip in 16 bits": lambda: scan(skip=z(8).half()),
        "bias of other channels": lambda: scan(dt_bias=z(9)),
        "lengths of other rows": lambda: scan(lengths=z(3, dtype=torch.int64)),
        "lengths that are numbers": lambda: scan(lengths=z(2)),
        "a in host memory": lambda: scan(a=a.cpu()),
        "x in host memory": lambda: scan(x=x.cpu()),
        "step with gradients": lambda: step(a=a.clone().requires_grad_(True)),
        "step of a sequence": lambda: step(x=x),
        "step's state of other rows": lambda: step(state=z(3, 8, 4)),
        "step's state in 16 bits": lambda: step(state=st.half()),
        "step's result is its input": lambda: step(out=x1),
        "step's result of another type": lambda: step(out=x1.half()),
        "step's bias is its state": lambda: step(dt_bias=st[0, :2].reshape(8)[:8]),
        "twice differentiated": lambda: torch.autograd.grad(scan(x=x.clone().requires_grad_(True), a=a.requires_grad_(True))[0].sum(), a, create_graph=True),
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
    def fwd(B=1, T=1, D=1, N=4, dtype=0, flags=0, ptrs=None, strides=None, room=1 << 30):
        return lib.t2fw_selective_scan_forward(*(ptrs or [p] * 13), B, T, D, N, strides, dtype, flags, p, room, None)
    assert fwd(dtype=3) == 2 and fwd(N=0) == 3 and fwd(N=65) == 3 and fwd(D=0) == 3 and fwd(T=-1) == 3 and fwd(B=1 << 40, T=1 << 20, D=1 << 10) == 3
    assert fwd(flags=4) == 5 and fwd(strides=(ctypes.c_int64 * 10)(*[1] * 9, -1)) == 3 and fwd(B=0) == 0
    assert fwd(T=4096, room=0) == 6
    for i in (0, 1, 2, 3, 4, 10, 11):
        ptrs = [p] * 13
        ptrs[i] = None
        assert fwd(ptrs=ptrs) == 1
    assert lib.t2fw_selective_scan_checkpoint_bytes(2, 33, 10, 16) == 2 * 3 * 10 * 16 * 4
    assert lib.t2fw_selective_scan_backward(*[p] * 21, 1, 4, 1, 4, None, 0, 0, p, 0, None) == 6
    assert lib.t2fw_selective_scan_step(*[p] * 11, 1, 1, 0, None, 0, 0, None) == 3

"""A selective state space layer and beam search over recurrent states, as they are measured.

Four operators, which a model with such layers runs in training and in generation:

* ``short_conv`` / ``short_conv_step``: the causal convolution of a few taps per channel before the scan;
* ``selective_scan`` / ``selective_scan_step``: ``h_t = exp(dt_t A) h_{t-1} + dt_t B_t x_t`` per channel and state, ``y_t = C_t h_t + D x_t``;
* ``beam_select``: the best continuations over all beams and the vocabulary;
* ``reorder_beams``: the states of all layers moved to the beams that go on from them.

``run`` computes them in their plain form, in 32 bits (the beams' scores in 64), or through the framework's entry points where ``own`` is true.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
HEAD = 64                                # channels of a head of the decay rule, on both sides of its state


def listed():
    return [
        # one token of 64 running requests through a layer of twice 768 channels: launch and host latency
        {"name": "conv_step", "kind": "conv_step", "dtype": "bfloat16", "rows": 64, "steps": 1, "width": 1536, "taps": 4, "silu": True,
         "weight": "bfloat16"},
        # training on a batch of padded sequences, float32 weights
        {"name": "conv_train", "kind": "conv_train", "dtype": "bfloat16", "rows": 8, "steps": 1024, "width": 1536, "taps": 4, "silu": True,
         "weight": "float32", "ragged": True},
        # the prompt of one long request, three taps, a length and a width that are no multiples of anything
        {"name": "conv_prompt_odd", "kind": "conv_forward", "dtype": "float32", "rows": 1, "steps": 32749, "width": 1021, "taps": 3, "silu": False,
         "weight": "float32", "ragged": False},
        # one token of 64 requests, sixteen states a channel
        {"name": "select_step", "kind": "select_step", "dtype": "bfloat16", "rows": 64, "steps": 1, "width": 1536, "states": 16, "gated": True},
        # the prompt of a single long request
        {"name": "select_prompt", "kind": "select_forward", "dtype": "bfloat16", "rows": 1, "steps": 8191, "width": 1536, "states": 16,
         "gated": True, "ragged": False},
        # training on a batch of padded sequences
        {"name": "select_train", "kind": "select_train", "dtype": "bfloat16", "rows": 8, "steps": 1024, "width": 1536, "states": 16,
         "gated": True, "ragged": True},
        # training in full precision, without a gate, odd sizes
        {"name": "select_train_odd", "kind": "select_train", "dtype": "float32", "rows": 3, "steps": 4099, "width": 509, "states": 10,
         "gated": False, "ragged": False},
        # the first step of one request with four beams, logits in 32 bits
        {"name": "beams_small", "kind": "beams", "dtype": "float32", "rows": 1, "beams": 4, "vocab": 8000, "count": 8, "first": True},
        # 32 requests with eight beams, some of which have ended; twice as many candidates as beams
        {"name": "beams_batch", "kind": "beams", "dtype": "bfloat16", "rows": 32, "beams": 8, "vocab": 50257, "count": 16, "first": False},
        # the states of a small model's two layers under four beams: latency
        {"name": "reorder_small", "kind": "reorder", "dtype": "bfloat16", "rows": 1, "beams": 4, "layers": 2, "heads": 2, "states": 16, "tokens": 33},
        # twelve layers under 32 requests of eight beams
        {"name": "reorder_batch", "kind": "reorder", "dtype": "bfloat16", "rows": 32, "beams": 8, "layers": 12, "heads": 12, "states": 16,
         "tokens": 1024},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _within(rng, lo, hi, most):
    """The same, at most ``most``."""
    return _between(rng, lo, max(lo, min(hi, int(most))))


def draw(rng):
    kind = rng.choice(["conv_step", "conv_forward", "conv_train", "select_step", "select_forward", "select_train", "beams", "reorder"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind.startswith("conv"):
        case = {"kind": kind, "dtype": dtype, "width": _between(rng, 16, 4096), "taps": rng.choice([2, 3, 4, 4, 5, 7]), "silu": rng.random() < 0.7,
                "weight": rng.choice([dtype, "float32"])}
        if kind == "conv_step":
            return {**case, "rows": _between(rng, 1, 2048), "steps": 1}
        rows = _between(rng, 1, 32)
        return {**case, "rows": rows, "steps": _within(rng, 1, 32768, 2 ** 25 // (rows * case["width"])), "ragged": rng.random() < 0.5}
    if kind.startswith("select"):
        width, states = _between(rng, 16, 4096), rng.choice([16, 16, _between(rng, 1, 64)])
        case = {"kind": kind, "dtype": dtype, "width": width, "states": states, "gated": rng.random() < 0.7}
        if kind == "select_step":
            return {**case, "rows": _within(rng, 1, 1024, 2 ** 25 // (width * states)), "steps": 1}
        rows = _between(rng, 1, 32)
        return {**case, "rows": rows, "steps": _within(rng, 1, 16384, 2 ** 27 // (rows * width * states)), "ragged": rng.random() < 0.5}
    if kind == "beams":
        vocab, beams = _between(rng, 100, 131072), rng.randint(1, 16)
        return {"kind": kind, "dtype": dtype, "rows": _within(rng, 1, 64, 12e6 / (vocab * beams)), "beams": beams, "vocab": vocab,
                "count": beams * rng.choice([1, 2]), "first": rng.random() < 0.3}
    return {"kind": kind, "dtype": dtype, "rows": _between(rng, 1, 32), "beams": rng.randint(2, 8), "layers": rng.randint(1, 12),
            "heads": rng.randint(1, 12), "states": rng.choice([8, 16]), "tokens": _between(rng, 1, 1024)}


# ---- what a program has in hand before the call -------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return torch.randn(shape, generator=gen, device="cuda").mul_(std).add_(mean).to(to)

    st = {"case": case, "lengths": None}
    step, train = kind.endswith("_step"), kind.endswith("_train")
    if kind.startswith(("conv", "select")):
        B, T, D = case["rows"], case["steps"], case["width"]
        lead = (B, D) if step else (B, T, D)
        if case.get("ragged"):
            st["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device="cuda")
    if kind.startswith("conv"):
        W = case["taps"]
        st["x"] = normal(*lead)
        st["w"] = normal(D, W, std=W ** -0.5, to=DTYPES[case["weight"]])
        st["bias"] = normal(D, std=0.1, to=DTYPES[case["weight"]])
        st["state"] = normal(B, W - 1, D)
        if train:
            st["gy"], st["gs"] = normal(*lead), normal(B, W - 1, D)
            for n in ("x", "w", "bias", "state"):
                st[n].requires_grad_(True)
    elif kind.startswith("select"):
        N, f32 = case["states"], torch.float32
        # as such layers begin: decays of 1 to N, steps of 0.001 to 0.1 around which the input moves them
        st["a"] = normal(D, N, std=0.2, to=f32).exp_().mul_(-torch.arange(1, N + 1, device="cuda"))
        about = torch.rand(D, generator=gen, device="cuda").mul_(math.log(100.0)).add_(math.log(0.001)).exp_()
        st["dt_bias"] = about + torch.log(-torch.expm1(-about))
        st["skip"] = normal(D, std=0.2, mean=1.0, to=f32)
        st["x"], st["dt"] = normal(*lead, std=0.5), normal(*lead, std=0.5)
        st["b"], st["c"] = (normal(*lead[:-1], N) for _ in range(2))
        st["gate"] = normal(*lead) if case["gated"] else None
        st["state"] = normal(B, D, N, std=0.3, to=f32)
        if train:
            st["gy"], st["gs"] = normal(*lead), normal(B, D, N, std=0.3, to=f32)
            for n in _SELECT_INPUTS:
                if st[n] is not None:
                    st[n].requires_grad_(True)
    elif kind == "beams":
        B, K, V = case["rows"], case["beams"], case["vocab"]
        st["logits"] = normal(B, K, V, std=3.0)
        # tokens that the answer's grammar forbids
        st["logits"][:, :, torch.randint(0, V, (V // 16,), generator=gen, device="cuda")] = float("-inf")
        st["scores"] = normal(B, K, std=1.0, mean=-12.0, to=torch.float32)
        st["finished"] = torch.rand(B, K, generator=gen, device="cuda") < 0.15
        if case["first"]:                # all beams are the same prompt: one of them counts
            st["scores"] = torch.zeros_like(st["scores"])
            st["scores"][:, 1:] = float("-inf")
            st["finished"] = None
    else:
        rows, width = case["rows"] * case["beams"], case["heads"] * HEAD
        st["arrays"] = [torch.randint(0, 50000, (rows, case["tokens"]), generator=gen, device="cuda")]
        for i in range(case["layers"]):
            if i % 2 == 0:               # the decay rule's state
                st["arrays"].append(normal(rows * case["heads"], HEAD, HEAD))
            else:                        # a selective layer's: of its scan and of its convolution
                st["arrays"].append(normal(rows, 2 * width, case["states"], to=torch.float32))
                st["arrays"].append(normal(rows, 3, 2 * width))
        st["beams"] = torch.randint(0, case["beams"], (case["rows"], case["beams"]), generator=gen, device="cuda")
    return st


_SELECT_INPUTS = ("x", "dt", "a", "b", "c", "state", "skip", "gate", "dt_bias")
PAD = 0                                  # the token that an ended beam goes on with


# ---- the plain forms ----------------------------------------------------------------------------------------------

def _live(st):
    """[B, T, 1], whether a step is within its row's length"""
    T = st["x"].shape[1]
    return None if st["lengths"] is None else (torch.arange(T, device="cuda")[None] < st["lengths"][:, None])[:, :, None]


def _kept(t, live):
    return t if live is None else t.where(live, torch.zeros_like(t))


def _silu(z):
    return z * torch.sigmoid(z)


def _silu_slope(z):
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def _last_rows(st, W):
    """[B, W - 1], where the last inputs of each row are in its state and inputs together"""
    B, T = st["x"].shape[:2]
    ends = torch.full((B,), T, device="cuda") if st["lengths"] is None else st["lengths"]
    return ends[:, None] + torch.arange(W - 1, device="cuda")[None]


def _plain_conv(st):
    live, w = _live(st), st["w"].detach().float()
    W, T = w.shape[1], st["x"].shape[1]
    xs = torch.cat((st["state"].detach().float(), _kept(st["x"].detach().float(), live)), dim=1)
    z = st["bias"].detach().float() + sum(xs[:, j:j + T] * w[:, j] for j in range(W))
    y = _kept(_silu(z) if st["case"]["silu"] else z, live)
    last = xs.gather(1, _last_rows(st, W)[:, :, None].expand(-1, -1, xs.shape[2]))
    return live, w, xs, z, y.to(st["x"].dtype), last.to(st["x"].dtype)


def _plain_conv_forward(st):
    return _plain_conv(st)[4:]


def _plain_conv_train(st):
    live, w, xs, z, y, last = _plain_conv(st)
    W, T, dtype = w.shape[1], z.shape[1], st["x"].dtype
    dz = _kept(st["gy"].float() * _silu_slope(z) if st["case"]["silu"] else st["gy"].float(), live)
    dxs = torch.zeros_like(xs)
    for j in range(W):
        dxs[:, j:j + T] += dz * w[:, j]
    dw = torch.stack([(dz * xs[:, j:j + T]).sum((0, 1), dtype=torch.float64) for j in range(W)], dim=1)
    dxs.scatter_add_(1, _last_rows(st, W)[:, :, None].expand(-1, -1, xs.shape[2]), st["gs"].float())
    dx = _kept(dxs[:, W - 1:], live)
    return (y, last, dx.to(dtype), dw.to(st["w"].dtype), dz.sum((0, 1), dtype=torch.float64).to(st["bias"].dtype), dxs[:, :W - 1].to(dtype))


def _plain_conv_step(st):
    xs = torch.cat((st["state"], st["x"][:, None]), dim=1)
    z = st["bias"].float() + (xs.float() * st["w"].float().t()).sum(1)
    st["state"].copy_(xs[:, 1:])
    return (_silu(z) if st["case"]["silu"] else z).to(st["x"].dtype), st["state"]


def _softplus(v):
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))


def _shifted(t, by, fill):
    """[B, T, D, N] moved ``by`` steps to later times"""
    return torch.cat((t.new_full((t.shape[0], by) + t.shape[2:], fill), t[:, :t.shape[1] - by]), dim=1)


def _recurrence(u, a, state):
    """All h_t = a_t h_{t-1} + u_t by doubling: after the round of ``by``, every step holds the sum over its last 2 by inputs"""
    h = torch.cat((u[:, :1] + a[:, :1] * state[:, None], u[:, 1:]), dim=1)
    by = 1
    while by < u.shape[1]:
        h = h + a * _shifted(h, by, 0.0)
        a = a * _shifted(a, by, 0.0)
        by *= 2
    return h


def _plain_select(st):
    live = _live(st)
    p = {n: st[n].detach().float() if st[n] is not None else None for n in _SELECT_INPUTS}
    for n in ("x", "dt", "b", "c", "gate"):
        if p[n] is not None:
            p[n] = _kept(p[n], live)
    p["raw"] = p["dt"] + p["dt_bias"]
    p["dt"] = _kept(_softplus(p["raw"]), live)
    p["decay"] = torch.exp(p["dt"][..., None] * p["a"])
    h = _recurrence((p["dt"] * p["x"])[..., None] * p["b"][:, :, None], p["decay"], p["state"])
    y = (h * p["c"][:, :, None]).sum(-1) + p["skip"] * p["x"]
    out = y if p["gate"] is None else y * _silu(p["gate"])
    return p, live, h, y, _kept(out, live).to(st["x"].dtype), h[:, -1].clone()


def _plain_select_forward(st):
    return _plain_select(st)[4:]


def _plain_select_train(st):
    p, live, h, y, out, last = _plain_select(st)
    dtype, gy = st["x"].dtype, _kept(st["gy"].float(), live)
    dgate = None if p["gate"] is None else gy * y * _silu_slope(p["gate"])
    dy = gy if p["gate"] is None else gy * _silu(p["gate"])
    # the adjoint is the same recurrence from the end, its decay at step t that of step t + 1; step T holds the last state's gradient
    later = torch.cat((p["decay"], torch.ones_like(p["decay"][:, :1])), dim=1)[:, 1:]
    G = _recurrence((dy[..., None] * p["c"][:, :, None]).flip(1), later.flip(1), st["gs"]).flip(1)
    db = (G * (p["dt"] * p["x"])[..., None]).sum(2)
    dc = (h * dy[..., None]).sum(2)
    by_decay = G * p["decay"] * torch.cat((p["state"][:, None], h[:, :-1]), dim=1)
    da = (by_decay * p["dt"][..., None]).sum((0, 1), dtype=torch.float64).float()
    by_input = (G * p["b"][:, :, None]).sum(-1)
    ddt = _kept(((by_decay * p["a"]).sum(-1) + by_input * p["x"]) * torch.sigmoid(p["raw"]), live)
    dx = p["dt"] * by_input + p["skip"] * dy
    grads = {"x": dx.to(dtype), "dt": ddt.to(dtype), "a": da, "b": db.to(dtype), "c": dc.to(dtype), "state": p["decay"][:, 0] * G[:, 0],
             "skip": (dy * p["x"]).sum((0, 1), dtype=torch.float64).float(), "dt_bias": ddt.sum((0, 1), dtype=torch.float64).float()}
    if dgate is not None:
        grads["gate"] = dgate.to(dtype)
    return (out, last) + tuple(grads[n] for n in _SELECT_INPUTS if n in grads)


def _plain_select_step(st):
    x, dt = st["x"].float(), _softplus(st["dt"].float() + st["dt_bias"])
    st["state"].mul_(torch.exp(dt[..., None] * st["a"])).add_((dt * x)[..., None] * st["b"].float()[:, None])
    y = (st["state"] * st["c"].float()[:, None]).sum(-1) + st["skip"] * x
    return (y if st["gate"] is None else y * _silu(st["gate"].float())).to(st["x"].dtype), st["state"]


def _plain_beams(st):
    # scores of different beams may be next to one another: 64 bits
    z = st["logits"].double()
    top = z.amax(-1, keepdim=True)
    total = st["scores"].double()[..., None] + (z - top - torch.log(torch.exp(z - top).sum(-1, keepdim=True)))
    if st["finished"] is not None:
        only = torch.full_like(total[:1, :1], float("-inf")).expand_as(total).clone()
        only[..., PAD] = st["scores"].double()
        total = torch.where(st["finished"][..., None], only, total)
    B, K, V = z.shape
    best, at = torch.sort(total.view(B, -1), dim=1, descending=True, stable=True)
    best, at = best[:, :st["case"]["count"]], at[:, :st["case"]["count"]]
    return best.float(), at // V, at % V


def _plain_reorder(st):
    rows, K = st["beams"].shape
    at = (torch.arange(rows, device="cuda")[:, None] * K + st["beams"]).flatten()
    st["arrays"] = [t.view(rows * K, -1).index_select(0, at).view(t.shape) for t in st["arrays"]]
    return st["arrays"]


_PLAIN = {"conv_step": _plain_conv_step, "conv_forward": _plain_conv_forward, "conv_train": _plain_conv_train, "select_step": _plain_select_step,
          "select_forward": _plain_select_forward, "select_train": _plain_select_train, "beams": _plain_beams, "reorder": _plain_reorder}


# ---- the framework's calls ----------------------------------------------------------------------------------------

def _own(st):
    import t2fw_amd as t2
    case = st["case"]
    kind = case["kind"]
    if kind == "conv_step":
        return t2.short_conv_step(st["x"], st["w"], st["state"], bias=st["bias"], silu=case["silu"])
    if kind.startswith("conv"):
        def conv():
            return t2.short_conv(st["x"], st["w"], bias=st["bias"], state=st["state"], lengths=st["lengths"], silu=case["silu"])
        if kind == "conv_forward":
            with torch.no_grad():
                return conv()
        out = conv()
        return out + torch.autograd.grad(out, (st["x"], st["w"], st["bias"], st["state"]), (st["gy"], st["gs"]))
    if kind.startswith("select"):
        options = {"skip": st["skip"], "gate": st["gate"], "dt_bias": st["dt_bias"], "softplus": True}
        main = (st["x"], st["dt"], st["a"], st["b"], st["c"])
        if kind == "select_step":
            return t2.selective_scan_step(*main, st["state"], **options)
        if kind == "select_forward":
            with torch.no_grad():
                return t2.selective_scan(*main, state=st["state"], lengths=st["lengths"], **options)
        out = t2.selective_scan(*main, state=st["state"], lengths=st["lengths"], **options)
        return out + torch.autograd.grad(out, [st[n] for n in _SELECT_INPUTS if st[n] is not None], (st["gy"], st["gs"]))
    if kind == "beams":
        return t2.beam_select(st["logits"], st["scores"], count=case["count"], finished=st["finished"], pad=PAD)
    return t2.reorder_beams(st["arrays"], st["beams"])


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _exact_conv(case, st):
    """Windows of the inputs with the state before them, differentiated by torch"""
    ins = [st[n].detach().double().requires_grad_(True) for n in ("x", "w", "bias", "state")]
    x, w, bias, state = ins
    if case["kind"] == "conv_step":
        x = x[:, None]
    B, T, D = x.shape
    W = w.shape[1]
    ends = [T] * B if st["lengths"] is None else st["lengths"].tolist()
    ys, lasts = [], []
    for b, n in enumerate(ends):
        xs = torch.cat((state[b], x[b, :n]))
        z = bias + (xs.unfold(0, W, 1) * w).sum(-1) if n else xs[:0]
        ys.append(torch.cat((z / (1 + torch.exp(-z)) if case["silu"] else z, z.new_zeros(T - n, D))))
        lasts.append(xs[n:])
    y, last = torch.stack(ys), torch.stack(lasts)
    if case["kind"] == "conv_step":
        return y[:, 0].detach(), last.detach()
    if case["kind"] == "conv_forward":
        return y.detach(), last.detach()
    grads = torch.autograd.grad((y, last), ins, (st["gy"].double(), st["gs"].double()))
    return (y.detach(), last.detach()) + grads


def _exact_select(case, st):
    """Step by step, as the recurrence is written"""
    p = {n: st[n].detach().double() if st[n] is not None else None for n in _SELECT_INPUTS}
    step, train = case["kind"] == "select_step", case["kind"] == "select_train"
    if step:
        p.update({n: p[n][:, None] for n in ("x", "dt", "b", "c", "gate") if p[n] is not None})
    T, h, a = p["x"].shape[1], p["state"], p["a"]
    raw = p["dt"] + p["dt_bias"]
    dt = torch.where(raw > 30, raw + torch.exp(-raw), torch.log1p(torch.exp(raw.clamp(max=30))))
    gate = None if p["gate"] is None else 1 / (1 + torch.exp(-p["gate"]))
    ones = torch.ones(T, 1, 1, dtype=torch.bool, device="cuda")
    live = (ones if st["lengths"] is None else torch.arange(T, device="cuda")[:, None, None] < st["lengths"][None, :, None]).unbind(0)
    before, ys, outs = [], [], []
    for t in range(T):
        if train:
            before.append(h)
        new = torch.exp(dt[:, t, :, None] * a) * h + (dt[:, t] * p["x"][:, t])[..., None] * p["b"][:, t, None]
        h = torch.where(live[t][..., None], new, h)
        y = (h @ p["c"][:, t, :, None])[..., 0] + p["skip"] * p["x"][:, t]
        ys.append(y)
        outs.append((y if gate is None else y * p["gate"][:, t] * gate[:, t]) * live[t])
    out = torch.stack(outs, 1)
    if step:
        return out[:, 0], h
    if not train:
        return out, h
    adj, sums = st["gs"].double(), {n: torch.zeros_like(p[n]) for n in ("a", "skip", "dt_bias")}
    per_step = {n: [] for n in ("x", "dt", "b", "c", "gate")}
    for t in reversed(range(T)):
        x, d, b, c = p["x"][:, t], dt[:, t], p["b"][:, t], p["c"][:, t]
        gy = st["gy"][:, t].double() * live[t]
        dy = gy if gate is None else gy * p["gate"][:, t] * gate[:, t]
        decay = torch.exp(d[..., None] * a)
        G = adj + dy[..., None] * c[:, None]
        now = decay * before[t] + (d * x)[..., None] * b[:, None]
        by_decay = G * decay * before[t] * live[t][..., None]
        by_input = (G @ b[..., None])[..., 0] * live[t]
        slope = 1 / (1 + torch.exp(-raw[:, t]))
        ddt = ((by_decay * a).sum(-1) + by_input * x) * slope
        per_step["x"].append(d * by_input + p["skip"] * dy)
        per_step["dt"].append(ddt)
        per_step["b"].append(((d * x)[:, None] @ G)[:, 0] * live[t])
        per_step["c"].append((dy[:, None] @ now)[:, 0] * live[t])
        if gate is not None:
            s, z = gate[:, t], p["gate"][:, t]
            per_step["gate"].append(gy * ys[t] * s * (1 + z * (1 - s)))
        sums["a"] += (by_decay * d[..., None]).sum(0)
        sums["skip"] += (dy * x).sum(0)
        sums["dt_bias"] += ddt.sum(0)
        adj = torch.where(live[t][..., None], decay * G, adj)
    grads = {n: torch.stack(v[::-1], 1) for n, v in per_step.items() if v}
    grads.update(sums, state=adj)
    return (out, h) + tuple(grads[n] for n in _SELECT_INPUTS if n in grads)


def _exact_beams(case, st):
    """Beam by beam: the best of each row's tokens, then the best of all of them"""
    B, K, V = st["logits"].shape
    n = case["count"]
    found = []
    for b in range(B):
        options = []
        for k in range(K):
            score = float(st["scores"][b, k])
            if st["finished"] is not None and bool(st["finished"][b, k]):
                options += [(score, k * V + PAD)] + [(float("-inf"), k * V + v) for v in range(n + 1) if v != PAD]
                continue
            logp = torch.log_softmax(st["logits"][b, k].double(), dim=0)
            order = torch.sort(logp, descending=True, stable=True)[1][:n]
            options += [(score + p, k * V + v) for p, v in zip(logp[order].tolist(), order.tolist())]
        found.append(sorted(options, key=lambda o: (-o[0], o[1]))[:n])
    at = torch.tensor([[o[1] for o in f] for f in found], device="cuda")
    return torch.tensor([[o[0] for o in f] for f in found], dtype=torch.float64, device="cuda"), at // V, at % V


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"].startswith("conv"):
        return _exact_conv(case, st)
    if case["kind"].startswith("select"):
        return _exact_select(case, st)
    if case["kind"] == "beams":
        return _exact_beams(case, st)
    rows, K = st["beams"].shape
    where = st["beams"].tolist()
    moved = []
    for t in st["arrays"]:
        parts = t.view(rows, K, -1)
        new = torch.stack([torch.stack([parts[r, k] for k in where[r]]) for r in range(rows)]).view(t.shape)
        moved.append(new.double() if new.is_floating_point() else new)
    return moved


def _size(dtype):
    return torch.empty(0, dtype=DTYPES[dtype]).element_size()


def work(case):
    """Each input read once, each output written once.  Operations: convolution two a tap and four for its activation, with gradients three times
    that; scan seven per channel and state (the decay's product and exponential, the input's, two to update, two to read), with gradients 21;
    beams four a logit."""
    kind, es = case["kind"], _size(case["dtype"])
    if kind.startswith("conv"):
        n, W = case["rows"] * case["steps"] * case["width"], case["taps"]
        states, weights = case["rows"] * (W - 1) * case["width"] * es, case["width"] * (W + 1) * _size(case["weight"])
        if kind == "conv_train":         # x and the gradient coming in; y and the input's gradient
            return {"bytes": 4 * n * es + 4 * states + 2 * weights, "flops": 3.0 * n * (2 * W + 4)}
        return {"bytes": 2 * n * es + 2 * states + weights, "flops": 1.0 * n * (2 * W + 4)}
    if kind.startswith("select"):
        steps, D, N = case["rows"] * case["steps"], case["width"], case["states"]
        states, weights = case["rows"] * D * N * 4, D * (N + 2) * 4
        per_step = D * (3 + case["gated"]) + 2 * N       # x, dt, the gate, b and c; y
        if kind == "select_train":       # ... and their gradients, the one coming in among them
            return {"bytes": 2 * steps * per_step * es + 4 * states + 2 * weights, "flops": 21.0 * steps * D * N}
        return {"bytes": steps * per_step * es + 2 * states + weights, "flops": 7.0 * steps * D * N}
    if kind == "beams":
        n = case["rows"] * case["beams"] * case["vocab"]
        return {"bytes": n * es + case["rows"] * (case["beams"] * 5 + case["count"] * 20), "flops": 4.0 * n}
    rows, width = case["rows"] * case["beams"], case["heads"] * HEAD
    odd = case["layers"] // 2
    each = case["tokens"] * 8 + (case["layers"] - odd) * width * HEAD * es + odd * 2 * width * (case["states"] * 4 + 3 * es)
    # beams that go on from themselves stay where they are
    return {"bytes": 2 * rows * each * (1 - 1 / case["beams"]), "flops": 0.0}

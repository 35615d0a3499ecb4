"""The operators of a training and a generation step around the recurrences, as they are measured.

Four operators, which a step of a recurrent language model runs one after the other:

* ``gated_scan`` / ``gated_scan_step``: ``h_t = f_t h_{t-1} + x_t`` per channel, the layer with a vector for its state;
* ``residual_rms_norm`` / ``residual_rms_norm_fp8``: the residual's addition and the norm of what is stored, also in 8 bits;
* ``policy_loss``: the clipped policy loss with a KL term on the logits of the tokens, and its gradient;
* ``clip_grad_norm``: the 2-norm of all gradients together, and their clipping.

``run`` computes them in their plain form, in 32 bits, or through the framework's entry points where ``own`` is true.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
FP8_MAX = 448.0
CLIP_LOW, CLIP_HIGH, KL_COEF, EPS = 0.2, 0.28, 0.05, 1e-6


def listed():
    return [
        # one token of 64 running requests through a recurrent layer, gates from logits: launch and host latency
        {"name": "scan_step", "kind": "scan_step", "dtype": "bfloat16", "rows": 64, "steps": 1, "width": 768, "logits": True},
        # the prompt of a single long request, a length that is no multiple of anything
        {"name": "scan_prompt", "kind": "scan_forward", "dtype": "bfloat16", "rows": 1, "steps": 8191, "width": 768, "logits": True,
         "ragged": False},
        # training on a batch of padded sequences, 12 heads of 64 channels side by side
        {"name": "scan_train", "kind": "scan_train", "dtype": "bfloat16", "rows": 8, "steps": 1024, "width": 768, "logits": True,
         "ragged": True},
        # long-context training in full precision, gates given
        {"name": "scan_train_long", "kind": "scan_train", "dtype": "float32", "rows": 2, "steps": 32768, "width": 1024,
         "logits": False, "ragged": False},
        # one token of 64 requests: the norm before a projection with 8-bit operands, a scale for each row
        {"name": "norm_token", "kind": "norm_fp8", "dtype": "bfloat16", "rows": 64, "width": 768, "residual": "bfloat16",
         "weight": "bfloat16", "group": 0},
        # prompts in 8 bits, a scale for every 128 columns
        {"name": "norm_prompt", "kind": "norm_fp8", "dtype": "bfloat16", "rows": 32768, "width": 4096, "residual": "bfloat16",
         "weight": "bfloat16", "group": 128},
        # a training batch of 8 x 1024 tokens
        {"name": "norm_train", "kind": "norm_train", "dtype": "bfloat16", "rows": 8192, "width": 768, "residual": "bfloat16",
         "weight": "float32", "group": 0},
        # packed tokens of an odd number and width, the residual stream held in 32 bits
        {"name": "norm_train_odd", "kind": "norm_train", "dtype": "float16", "rows": 12345, "width": 1021, "residual": "float32",
         "weight": "float32", "group": 0},
        # the answers to a few prompts, a small vocabulary, logits in 32 bits
        {"name": "loss_small", "kind": "loss", "dtype": "float32", "rows": 333, "vocab": 8000},
        # a batch of 8 x 1024 tokens; the rows of an odd vocabulary start at odd places
        {"name": "loss_train", "kind": "loss", "dtype": "bfloat16", "rows": 8192, "vocab": 50257},
        # a small model whose gradients are under the limit, in place: latency
        {"name": "clip_small", "kind": "clip", "dtype": "float32", "layers": 2, "width": 64, "vocab": 500, "out": ""},
        # twelve layers of 768 channels: 16-bit gradients, clipped into the optimizer's 32-bit copies
        {"name": "clip_model", "kind": "clip", "dtype": "bfloat16", "layers": 12, "width": 768, "vocab": 50257, "out": "float32"},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _within(rng, lo, hi, most):
    """The same, at most ``most``."""
    return _between(rng, lo, max(lo, min(hi, int(most))))


def draw(rng):
    kind = rng.choice(["scan_step", "scan_forward", "scan_train", "norm_fp8", "norm_train", "loss", "clip"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind == "scan_step":
        return {"kind": kind, "dtype": dtype, "rows": _between(rng, 1, 4096), "steps": 1, "width": _between(rng, 16, 4096),
                "logits": rng.random() < 0.5}
    if kind.startswith("scan"):
        rows, width = _between(rng, 1, 32), _between(rng, 16, 4096)
        return {"kind": kind, "dtype": dtype, "rows": rows, "steps": _within(rng, 1, 32768, 2 ** 26 // (rows * width)), "width": width,
                "logits": rng.random() < 0.5, "ragged": rng.random() < 0.5}
    if kind.startswith("norm"):
        width = rng.choice([128 * _between(rng, 1, 23), _between(rng, 16, 8191)])
        return {"kind": kind, "dtype": dtype, "rows": _within(rng, 1, 65536, 2 ** 27 // width), "width": width,
                "residual": rng.choice([dtype, "float32"]), "weight": rng.choice([dtype, "float32"]),
                "group": rng.choice([0, 0, 128, 64]) if kind == "norm_fp8" else 0}
    if kind == "loss":
        vocab = _between(rng, 100, 131072)
        return {"kind": kind, "dtype": dtype, "rows": _within(rng, 1, 16384, 2 ** 28 // vocab), "vocab": vocab}
    return {"kind": kind, "dtype": dtype, "layers": rng.randint(1, 16), "width": _between(rng, 16, 768), "vocab": _between(rng, 100, 50257),
            "out": rng.choice(["", dtype, "float32"])}


# ---- what a program has in hand before the call -------------------------------------------------------------------

def _shapes(case):
    """The parameters of a model of ``layers`` decay-rule layers: five projections in one, the output's, two norms, a two-matrix
    block of 8/3 of the width, the embedding and the last norm."""
    w = case["width"]
    wide = 8 * w // 3
    return [(case["vocab"], w), (w,)] + [(w, 5 * w), (w, w), (w,), (w, wide), (wide, w), (w,)] * case["layers"]


def _flat_views(flat, shapes):
    sizes = [math.prod(s) for s in shapes]
    return [v.view(s) for v, s in zip(flat.split(sizes), shapes)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, to=dtype):
        return torch.randn(shape, generator=gen, device="cuda").mul_(std).add_(mean).to(to)

    state = {"case": case}
    if kind.startswith("scan"):
        B, T, D = case["rows"], case["steps"], case["width"]
        lead = (B, D) if kind == "scan_step" else (B, T, D)
        gate = normal(*lead, mean=3.0, to=torch.float32)
        state["x"] = normal(*lead, std=0.3)
        state["f"] = (gate if case["logits"] else torch.sigmoid(gate)).to(dtype)
        state["state"] = normal(B, D, to=torch.float32)
        state["lengths"] = None
        if case.get("ragged"):
            state["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device="cuda")
        if kind == "scan_train":
            state["go"], state["gs"] = normal(*lead), normal(B, D, to=torch.float32)
            for n in ("x", "f", "state"):
                state[n].requires_grad_(True)
    elif kind.startswith("norm"):
        N, D, res = case["rows"], case["width"], DTYPES[case["residual"]]
        state["x"], state["res"] = normal(N, D), normal(N, D, std=2.0, to=res)
        state["w"] = normal(D, std=0.2, mean=1.0, to=DTYPES[case["weight"]])
        if kind == "norm_train":
            state["gy"], state["gres"] = normal(N, D), normal(N, D, to=res)
            for n in ("x", "res", "w"):
                state[n].requires_grad_(True)
    elif kind == "loss":
        N, V = case["rows"], case["vocab"]
        targets = torch.randint(0, V, (N, 1), generator=gen, device="cuda")
        # the tokens were drawn from the policy: their logits are among the largest of their rows
        logits = normal(N, V, std=2.0).scatter_add_(1, targets, normal(N, 1, std=2.0, mean=10.0))
        logp = (logits.gather(1, targets).float() - logits.float().logsumexp(1, keepdim=True)).squeeze(1)
        state["logits"], state["targets"] = logits.requires_grad_(True), targets.squeeze(1)
        state["old"] = logp + normal(N, std=0.2, to=torch.float32)
        state["ref"] = logp + normal(N, std=0.4, to=torch.float32)
        state["adv"] = normal(N, mean=0.5, to=torch.float32)
        state["mask"] = torch.rand(N, generator=gen, device="cuda") < 0.8        # the answers' tokens, not the prompts'
    else:
        shapes = _shapes(case)
        n = sum(math.prod(s) for s in shapes)
        state["flat"] = normal(n, std=1.0 / math.sqrt(n))                        # a norm of about one
        state["grads"] = _flat_views(state["flat"], shapes)
        state["out"] = None
        if case["out"]:
            state["flat_out"] = torch.zeros(n, dtype=DTYPES[case["out"]], device="cuda")
            state["out"] = _flat_views(state["flat_out"], shapes)
    return state


# ---- the plain forms ----------------------------------------------------------------------------------------------

def _shifted(t, by, fill):
    """[B, T, D] moved ``by`` steps to later times"""
    return torch.cat((t.new_full((t.shape[0], by, t.shape[2]), fill), t[:, :t.shape[1] - by]), dim=1)


def _plain_scan(x, f, state):
    """All h_t = f_t h_{t-1} + x_t by doubling: after the round of ``by``, every step holds the sum over its last 2 by inputs"""
    h = torch.cat((x[:, :1] + f[:, :1] * state[:, None], x[:, 1:]), dim=1) if x.shape[1] else x
    by = 1
    while by < x.shape[1]:
        h = h + f * _shifted(h, by, 0.0)
        f = f * _shifted(f, by, 0.0)
        by *= 2
    return h


def _plain_scan_inputs(state):
    x, raw, s = state["x"].detach().float(), state["f"].detach().float(), state["state"].detach()
    f = torch.sigmoid(raw) if state["case"]["logits"] else raw
    if state["lengths"] is None:
        return x, f, s, f, None
    live = (torch.arange(x.shape[1], device=x.device)[None] < state["lengths"][:, None])[:, :, None]
    return x.where(live, torch.zeros_like(x)), f.where(live, torch.ones_like(f)), s, f, live


def _plain_scan_forward(state):
    dtype = state["x"].dtype
    x, f, s, _, live = _plain_scan_inputs(state)
    h = _plain_scan(x, f, s)
    return (h if live is None else h * live).to(dtype), h[:, -1].clone()


def _plain_scan_train(state):
    dtype = state["x"].dtype
    x, f, s, gate, live = _plain_scan_inputs(state)
    h = _plain_scan(x, f, s)
    go = state["go"].float()
    if live is not None:
        go = go.where(live, torch.zeros_like(go))
    # the adjoint is the same recurrence from the end, its gate at step t that of step t + 1; step T holds the last state's gradient
    later = torch.cat((f, torch.ones_like(f[:, :1])), dim=1)[:, 1:]
    g = _plain_scan(go.flip(1), later.flip(1), state["gs"]).flip(1)
    df = g * torch.cat((s[:, None], h[:, :-1]), dim=1)
    if state["case"]["logits"]:
        df = df * gate * torch.sigmoid(-state["f"].detach().float())
    dx, ds = g, f[:, 0] * g[:, 0]
    out = h
    if live is not None:
        out, dx, df = h * live, dx * live, df * live
    return out.to(dtype), h[:, -1].clone(), dx.to(dtype), df.to(dtype), ds


def _plain_scan_step(state):
    x, f = state["x"].float(), state["f"].float()
    if state["case"]["logits"]:
        f = torch.sigmoid(f)
    state["state"].mul_(f).add_(x)
    return state["state"].to(state["x"].dtype), state["state"]


def _plain_norm(state):
    x, res, w = state["x"].detach(), state["res"].detach(), state["w"].detach().float()
    stored = (x.float() + res.float()).to(res.dtype)               # the norm is of the stream as it is stored
    h = stored.float()
    r = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
    return stored, h, r, w


def _plain_norm_train(state):
    stored, h, r, w = _plain_norm(state)
    y = (h * r * w).to(state["x"].dtype)
    gy = state["gy"].float()
    u = gy * w
    dh = r * (u - h * (r * r) * (u * h).mean(dim=1, keepdim=True)) + state["gres"].float()
    dw = (gy * h * r).sum(dim=0)
    return y, stored, dh.to(state["x"].dtype), dh.to(state["res"].dtype), dw.to(state["w"].dtype)


def _plain_norm_fp8(state):
    stored, h, r, w = _plain_norm(state)
    y = h * r * w
    N, D = y.shape
    group = state["case"]["group"] or D
    grouped = torch.nn.functional.pad(y, (0, -D % group)).view(N, -1, group)
    scale = grouped.abs().amax(dim=2, keepdim=True) / FP8_MAX
    scale = scale.where(scale > 0, torch.ones_like(scale))
    q = (grouped / scale).clamp(-FP8_MAX, FP8_MAX).reshape(N, -1)[:, :D].to(torch.float8_e4m3fn)
    return q, scale.squeeze(2), stored


def _plain_loss(state):
    z, t, keep = state["logits"].detach().float(), state["targets"][:, None], state["mask"]
    top = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    logp = (z.gather(1, t) - top - torch.log(total)).squeeze(1)
    ratio, d, a = torch.exp(logp - state["old"]), state["ref"] - logp, state["adv"]
    free, held = ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a
    each = -torch.minimum(free, held) + KL_COEF * (torch.expm1(d) - d)
    share = keep.float() / keep.sum().clamp(min=1)
    loss = (each * share).sum()
    inside = (ratio >= 1 - CLIP_LOW) & (ratio <= 1 + CLIP_HIGH)
    c = share * (-(free * ((free < held) | inside)) - KL_COEF * torch.expm1(d))
    dz = (e * (-c[:, None] / total)).scatter_add_(1, t, c[:, None])
    return loss, logp, dz.to(state["logits"].dtype)


def _max_norm(case):
    """In place: a limit that the gradients keep, so that a further pass finds them as they were"""
    return 0.25 if case["out"] else 100.0


def _plain_clip(state):
    flat = torch.cat([g.reshape(-1).float() for g in state["grads"]])
    norm = torch.sqrt((flat * flat).sum())
    scaled = flat * (_max_norm(state["case"]) / (norm + 1e-6)).clamp(max=1.0)
    to = state["flat_out"] if state["out"] else state["flat"]
    return norm, to.copy_(scaled)


_PLAIN = {"scan_step": _plain_scan_step, "scan_forward": _plain_scan_forward, "scan_train": _plain_scan_train,
          "norm_fp8": _plain_norm_fp8, "norm_train": _plain_norm_train, "loss": _plain_loss, "clip": _plain_clip}


# ---- the framework's calls ----------------------------------------------------------------------------------------

def _own(state):
    import t2fw_amd as t2
    case = state["case"]
    kind = case["kind"]
    if kind == "scan_step":
        return t2.gated_scan_step(state["x"], state["f"], state["state"], logits=case["logits"])
    if kind == "scan_forward":
        with torch.no_grad():
            return t2.gated_scan(state["x"], state["f"], state["state"], lengths=state["lengths"], logits=case["logits"])
    if kind == "scan_train":
        ins = (state["x"], state["f"], state["state"])
        out, last = t2.gated_scan(*ins, lengths=state["lengths"], logits=case["logits"])
        return (out, last) + torch.autograd.grad((out, last), ins, (state["go"], state["gs"]))
    if kind == "norm_fp8":
        return t2.residual_rms_norm_fp8(state["x"], state["res"], state["w"], eps=EPS, group=case["group"])
    if kind == "norm_train":
        ins = (state["x"], state["res"], state["w"])
        y, stored = t2.residual_rms_norm(*ins, eps=EPS)
        return (y, stored) + torch.autograd.grad((y, stored), ins, (state["gy"], state["gres"]))
    if kind == "loss":
        loss, logp = t2.policy_loss(state["logits"], state["targets"], state["old"], state["ref"], state["adv"], mask=state["mask"],
                                    clip=(CLIP_LOW, CLIP_HIGH), kl_coef=KL_COEF)
        return loss, logp, torch.autograd.grad(loss, state["logits"])[0]
    norm = t2.clip_grad_norm(state["grads"], _max_norm(case), out=state["out"])
    return norm, state["flat_out"] if state["out"] else state["flat"]


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def _exact_scan(case, st):
    """Step by step, as the recurrence is written"""
    step = case["kind"] == "scan_step"
    x, raw, h = st["x"].detach().double(), st["f"].detach().double(), st["state"].detach().double()
    if step:
        x, raw = x[:, None], raw[:, None]
    f = 1 / (1 + torch.exp(-raw)) if case["logits"] else raw
    T = x.shape[1]
    lengths = st.get("lengths")
    live = [None] * T if lengths is None else (torch.arange(T, device=x.device)[:, None, None] < lengths[None, :, None]).unbind(0)
    before, outs = [], []
    for t in range(T):
        before.append(h)
        new = f[:, t] * h + x[:, t]
        h = new if live[t] is None else torch.where(live[t], new, h)
        outs.append(h if live[t] is None else h * live[t])
    if step:
        return outs[0], h
    out = torch.stack(outs, dim=1)
    if case["kind"] == "scan_forward":
        return out, h
    adj, dxs, dfs = st["gs"].double(), [], []
    for t in reversed(range(T)):
        g = adj + st["go"][:, t].double()
        gate = f[:, t]
        dl = g * before[t]
        if case["logits"]:
            dl = dl * gate * (1 - gate)
        if live[t] is None:
            adj = gate * g
        else:
            adj, g, dl = torch.where(live[t], gate * g, adj), g * live[t], dl * live[t]
        dxs.append(g)
        dfs.append(dl)
    return out, h, torch.stack(dxs[::-1], dim=1), torch.stack(dfs[::-1], dim=1), adj


def _exact_norm(case, st):
    stored = (st["x"].detach().double() + st["res"].detach().double()).to(st["res"].dtype)
    h, w = stored.double(), st["w"].detach().double()
    rms = torch.sqrt(h.square().mean(dim=-1, keepdim=True) + EPS)
    unit = h / rms
    y = unit * w
    if case["kind"] == "norm_train":
        gy = st["gy"].double()
        u = gy * w
        dh = (u - unit * (u * unit).mean(dim=-1, keepdim=True)) / rms + st["gres"].double()
        return y, stored.double(), dh, dh, (gy * unit).sum(dim=0)
    N, D = y.shape
    group = case["group"] or D
    scales = [y[:, c:c + group].abs().amax(dim=1) / FP8_MAX for c in range(0, D, group)]
    q = torch.cat([y[:, i * group:(i + 1) * group] / s[:, None] for i, s in enumerate(scales)], dim=1)
    return q.float().to(torch.float8_e4m3fn).double(), torch.stack(scales, dim=1), stored.double()


def _exact_loss(st):
    keep, rows = st["mask"].double(), torch.arange(len(st["targets"]), device="cuda")
    per_row, grads = [], []
    M = max(float(keep.sum()), 1.0)
    for at in rows.split(1024):                                    # 64-bit copies of the logits of 1024 rows at a time
        logp_all = torch.log_softmax(st["logits"].detach()[at].double(), dim=1)
        t = st["targets"][at]
        logp = logp_all[torch.arange(len(at), device="cuda"), t].requires_grad_(True)
        ratio, d, a = torch.exp(logp - st["old"][at].double()), st["ref"][at].double() - logp, st["adv"][at].double()
        each = KL_COEF * (torch.exp(d) - d - 1) - torch.minimum(ratio * a, ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * a)
        part = (each * keep[at]).sum() / M
        c, = torch.autograd.grad(part, logp)
        grad = logp_all.exp_().mul_(-c[:, None])
        grad[torch.arange(len(at), device="cuda"), t] += c
        per_row.append((part.detach(), logp.detach()))
        grads.append(grad)
    return torch.stack([p for p, _ in per_row]).sum(), torch.cat([v for _, v in per_row]), torch.cat(grads)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"].startswith("scan"):
        return _exact_scan(case, st)
    if case["kind"].startswith("norm"):
        return _exact_norm(case, st)
    if case["kind"] == "loss":
        return _exact_loss(st)
    flat = st["flat"].double()
    norm = flat.norm()
    return norm, flat * min(1.0, _max_norm(case) / (float(norm) + 1e-6))


def _size(dtype):
    return torch.empty(0, dtype=DTYPES[dtype]).element_size()


def work(case):
    """Each input read once, each output written once.  Operations per element: scan 2, with its gradients 6; norm 5, with its
    gradients 14; loss 8 (the largest, exponential and sum, gradient); norm and clipping 3."""
    kind, es = case["kind"], _size(case["dtype"])
    if kind.startswith("scan"):
        n, states = case["rows"] * case["steps"] * case["width"], case["rows"] * case["width"] * 4
        if kind == "scan_train":
            return {"bytes": 6 * n * es + 4 * states, "flops": 6.0 * n}
        return {"bytes": 3 * n * es + 2 * states, "flops": 2.0 * n}
    if kind.startswith("norm"):
        n, rs, ws = case["rows"] * case["width"], _size(case["residual"]), case["width"] * _size(case["weight"])
        if kind == "norm_train":
            # x, residual, both gradients coming in; y, the stream, the gradient of the sum (in both types where they are two)
            return {"bytes": n * (4 * es + 3 * rs + (0 if case["dtype"] == case["residual"] else rs)) + 2 * ws, "flops": 14.0 * n}
        scales = case["rows"] * -(-case["width"] // (case["group"] or case["width"])) * 4
        return {"bytes": n * (es + 2 * rs + 1) + scales + ws, "flops": 5.0 * n}
    if kind == "loss":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2 * n * es + case["rows"] * 25, "flops": 8.0 * n}
    n = sum(math.prod(s) for s in _shapes(case))
    # in place and under the limit nothing has to be written
    return {"bytes": n * es + (n * _size(case["out"]) if case["out"] else 0), "flops": 3.0 * n}

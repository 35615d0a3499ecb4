"""The selective layer and beam search as a model runs them (t2fw_amd/finetune.py): a training step's gradients against the same model written in plain
torch operations (float64), generation against the whole sequence, beam search against the model's own probabilities and an exhaustive search."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain_logits(model, params, tokens):
    """RecurrentLM.forward with selective layers in elementary operations of the parameters' type"""
    from t2fw_amd.finetune import HEAD, STATES, TAPS
    p = dict(params)
    layers = len(model.ins)
    branch, stream = p["embed"][tokens], 0
    B, T = tokens.shape

    def norm(i):
        h = branch + stream
        return h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * p["norms.%d" % i], h
    for i in range(layers):
        y, stream = norm(i)
        u = y @ p["ins.%d" % i]
        outs = []
        if i % 2 == 0:
            x, f, q, k, fk = (t.unflatten(-1, (model.heads, HEAD)) for t in u.chunk(5, dim=-1))
            s = 0
            for t in range(T):
                gate = torch.sigmoid(f[:, t] + 2)[..., :, None] * torch.sigmoid(fk[:, t] + 2)[..., None, :]
                s = s * gate + (0.25 * x[:, t])[..., :, None] * (0.25 * k[:, t])[..., None, :]
                outs.append((s * (0.25 * q[:, t])[..., None, :]).sum(-1).flatten(1))
        else:
            x, z = u.chunk(2, dim=-1)
            padded = torch.cat((x.new_zeros(B, TAPS - 1, x.shape[2]), x), 1)
            x = torch.nn.functional.silu((padded.unfold(1, TAPS, 1) * p["convs.%d" % (i // 2)]).sum(-1))
            dt, b, c = (x @ p["steps.%d" % (i // 2)]).split([model.width, STATES, STATES], -1)
            dt = torch.nn.functional.softplus(dt + p["biases.%d" % (i // 2)])
            a, s = -torch.exp(p["rates.%d" % (i // 2)]), 0
            for t in range(T):
                s = torch.exp(dt[:, t, :, None] * a) * s + (dt[:, t] * x[:, t])[..., None] * b[:, t, None]
                outs.append(((s * c[:, t, None]).sum(-1) + p["skips.%d" % (i // 2)] * x[:, t]) * torch.nn.functional.silu(z[:, t]))
        branch = torch.stack(outs, 1) @ p["outs.%d" % i]
    y, _ = norm(layers)
    return y @ p["head"]


def test_a_step_against_plain_operations():
    """The bound of the same test without selective layers, 5 % of a gradient's norm, for every parameter (about twenty bfloat16 roundings of 2^-9 in a
    row add in quadrature to 2 %, half again for the matrix-core operands); a selective layer puts five more on the way (convolution, projection,
    step, results, gate) for one of the vector's recurrence."""
    from t2fw_amd.finetune import PolicyTrainer, RecurrentLM
    model = RecurrentLM(vocab=97, width=128, layers=4, seed=3, selective=True).cuda()
    exact = {n: p.detach().double().requires_grad_(True) for n, p in model.named_parameters()}
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, 97, (3, 40), generator=g, device="cuda")
    trainer = PolicyTrainer(model, lr=0.0, max_norm=1e9, clip=(0.2, 0.2), kl_coef=0.1)
    old = trainer.log_probabilities(tokens)
    adv = torch.randn(3, 1, generator=g, device="cuda").expand(3, 39).contiguous()
    mask = (torch.arange(39, device="cuda") >= 9).expand(3, 39).contiguous()
    ref = old + 0.3 * torch.randn(3, 39, generator=g, device="cuda")
    loss, norm = trainer.step(tokens, old, ref, adv, mask)
    logp = torch.log_softmax(plain_logits(model, exact, tokens[:, :-1]), -1).gather(-1, tokens[:, 1:, None])[..., 0]
    r, d = torch.exp(logp - logp.detach()), ref.double() - logp
    want = ((-r * adv + 0.1 * (torch.exp(d) - 1 - d)) * mask).sum() / mask.sum()
    assert bool((logp - old).abs().max() < 0.15)
    grads = torch.autograd.grad(want, list(exact.values()))
    for (n, p), e in zip(model.named_parameters(), grads):
        off = float((p.grad.double() - e).norm() / e.norm())
        assert off < 0.05, (n, off)
    total = float(torch.sqrt(sum((e * e).sum() for e in grads)))
    assert abs(float(norm) / total - 1) < 0.05
    assert all(torch.equal(v, p.grad.float()) for v, p in zip(trainer.grad_views, trainer.params))


def test_generation_follows_the_whole_sequence():
    """token by token and all at once, as for the other layers: within 0.05 of the logits' spread, with 8-bit operands within 0.2"""
    from t2fw_amd.finetune import RecurrentLM
    model = RecurrentLM(vocab=200, width=128, layers=4, seed=5, selective=True).cuda()
    prompt = torch.randint(0, 200, (16, 7), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    for eight_bit, most in ((False, 0.05), (True, 0.2)):
        tokens, seen = model.generate(prompt, 30, generator=torch.Generator(device="cuda").manual_seed(2), eight_bit=eight_bit)
        with torch.no_grad():
            whole = model(tokens[:, :-1]).float()
        assert float((seen.float() - whole).norm() / whole.norm()) < most


def test_padded_rows_do_not_see_their_padding():
    from t2fw_amd.finetune import RecurrentLM
    model = RecurrentLM(vocab=50, width=64, layers=2, seed=1, selective=True).cuda()
    tokens = torch.randint(0, 50, (2, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    other = tokens.clone()
    other[1, 12:] = 0
    lengths = torch.tensor([20, 12], device="cuda")
    with torch.no_grad():
        a, b = model(tokens, lengths), model(other, lengths)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1, :12], b[1, :12])


def test_a_round_of_training_and_search_runs():
    from t2fw_amd.finetune import finetune
    said = []
    history = finetune(rounds=2, batch=8, answer=12, selective=True, beams=3, say=said.append)
    assert len(history) == 3 and len(said) == 3 and "beam search of 3" in said[-1]
    assert all(0.0 <= h <= 1.0 for h in history)


@pytest.mark.parametrize("selective", [False, True])
def test_beam_search_scores_and_order(selective):
    """The scores are the answers' log probabilities: by the same steps on the answers themselves (the same kernels on as many rows), to float32 sums of ten
    terms; one beam is the most probable token each time."""
    from t2fw_amd.finetune import RecurrentLM
    model = RecurrentLM(vocab=40, width=64, layers=4, seed=5, selective=selective).cuda()
    prompt = torch.randint(0, 40, (3, 5), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    tokens, scores = model.beam_search(prompt, 10, beams=6)
    assert tokens.shape == (3, 6, 15) and scores.shape == (3, 6) and bool((tokens[:, :, :5] == prompt[:, None]).all())
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())
    flat = tokens.view(18, 15)
    assert len({tuple(t) for t in flat.tolist()}) == 18
    with torch.no_grad():
        step, _ = model._stepper(18, False)
        total = torch.zeros(18, dtype=torch.float64, device="cuda")
        for t in range(14):
            logp = torch.log_softmax(step(flat[:, t]).double(), -1)
            if t >= 4:
                total += logp.gather(1, flat[:, t + 1:t + 2])[:, 0]
    assert bool((total.view(3, 6) - scores).abs().max() <= 10 * (2.0 ** -19 + 2.0 ** -24 * 40))
    one, _ = model.beam_search(prompt, 10, beams=1)
    with torch.no_grad():
        step, _ = model._stepper(3, False)
        for t in range(14):
            logits = step(one[:, 0, t])
            if t >= 4:
                # (of equal 16-bit logits the lowest)
                best = (logits == logits.amax(-1, keepdim=True)).int().argmax(-1)
                assert torch.equal(best, one[:, 0, t + 1])


def test_wide_beam_search_is_exhaustive():
    """as many beams as there are answers: all of them, in order"""
    from t2fw_amd.finetune import RecurrentLM
    model = RecurrentLM(vocab=8, width=64, layers=2, seed=7, selective=True).cuda()
    prompt = torch.tensor([[3, 1]], device="cuda")
    tokens, scores = model.beam_search(prompt, 2, beams=64)
    assert len({tuple(t) for t in tokens[0].tolist()}) == 64 and bool(torch.isfinite(scores).all())
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())
    # their probabilities are those of all there is
    assert abs(float(scores.double().exp().sum()) - 1) <= 64 * 2.0 ** -17


def test_answers_that_end():
    from t2fw_amd.finetune import RecurrentLM
    model = RecurrentLM(vocab=6, width=64, layers=2, seed=2, selective=True).cuda()
    prompt = torch.randint(0, 6, (4, 3), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    tokens, scores = model.beam_search(prompt, 12, beams=5, end=2)
    answers = tokens[:, :, 3:]
    ended = (answers == 2).int().cumsum(-1) > 0
    assert bool(ended.any()) and bool((answers[ended] == 2).all())
    # an ended answer's score is that of its tokens up to its end
    flat = tokens.view(20, 15)
    with torch.no_grad():
        step, _ = model._stepper(20, False)
        total, over = torch.zeros(20, dtype=torch.float64, device="cuda"), torch.zeros(20, dtype=torch.bool, device="cuda")
        for t in range(14):
            logp = torch.log_softmax(step(flat[:, t]).double(), -1).gather(1, flat[:, t + 1:t + 2])[:, 0]
            if t >= 2:
                total += torch.where(over, torch.zeros_like(logp), logp)
                over |= flat[:, t + 1] == 2
    assert bool((total.view(4, 5) - scores).abs().max() <= 12 * (2.0 ** -19 + 2.0 ** -24 * 40))

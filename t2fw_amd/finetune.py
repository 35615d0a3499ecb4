"""A fine-tuning step and generation of a small recurrent language model, through every operator that stands around the recurrences.

    python -m t2fw_amd.finetune                       # a few rounds: answers, their reward, a clipped policy step on them
    python -m t2fw_amd.finetune --rounds 40 --width 256 --layers 4
    python -m t2fw_amd.finetune --selective --beams 4 # selective state space layers; the last answers by beam search

The layers alternate between the decay rule (``LFWHeadsFunction``, a 64 x 64 state per head) and the recurrence with a vector for its
state (``gated_scan``), or, with ``--selective``, the selective state space scan behind its convolution (``short_conv``, ``selective_scan``).  Each is
a residual branch: ``residual_rms_norm`` adds the branch before to a float32 stream and normalises it, a projection makes the recurrence's inputs,
another its output.

* Training: logits of whole sequences, ``policy_loss`` on the answers' tokens, backward, ``clip_grad_norm`` of the 16-bit gradients into
  float32 ones, a gradient step on float32 parameters.
* Generation: one token per call, states updated in place (``lfw_step``, ``gated_scan_step``, ``short_conv_step``, ``selective_scan_step``); with
  ``--eight-bit`` the norms come from ``residual_rms_norm_fp8`` and the projections are 8-bit products.
* Beam search: the same with the beams of all prompts for rows; ``beam_select`` takes the best continuations, ``reorder_beams`` moves the states of all
  layers and the tokens so far.

There is no task and no data here: a token of an answer is rewarded if it is in the lower half of the vocabulary, and the steps have to
raise their share.
"""
import argparse

import torch

from .beam import beam_select, reorder_beams
from .functional_conv import short_conv, short_conv_step
from .functional_lfw import LFWHeadsFunction, lfw_step
from .functional_loss import policy_loss
from .functional_norm import residual_rms_norm, residual_rms_norm_fp8
from .functional_scan import gated_scan, gated_scan_step
from .functional_select import selective_scan, selective_scan_step
from .grad_clip import clip_grad_norm

HEAD = 64                                # channels of a head, on both sides of the decay rule's state
TAPS, STATES = 4, 16                     # of a selective layer's convolution, and of each of its channels


class Projection:
    """A weight ``[in, out]`` for generation, as it is or in 8 bits with a scale for each of its outputs"""

    def __init__(self, weight, eight_bit):
        self.weight, self.scales, self.outputs = weight, None, weight.shape[1]
        if eight_bit:
            weight = torch.nn.functional.pad(weight, (0, -self.outputs % 16))      # (the product takes multiples of 16)
            self.scales = (weight.float().abs().amax(0, keepdim=True) / 448).clamp(min=1e-12)
            self.weight = (weight.float() / self.scales).to(torch.float8_e4m3fn).t().contiguous().t()     # (the product wants columns)

    def __call__(self, x, scales=None):
        if scales is None:
            return x @ self.weight
        return torch._scaled_mm(x, self.weight, scale_a=scales, scale_b=self.scales, out_dtype=torch.bfloat16)[:, :self.outputs]


class RecurrentLM(torch.nn.Module):
    def __init__(self, vocab=512, width=128, layers=4, dtype=torch.bfloat16, seed=0, selective=False):
        super().__init__()
        assert width % HEAD == 0, "the width is whole heads of %d channels" % HEAD
        g = torch.Generator().manual_seed(seed)
        new = lambda *s, std: torch.nn.Parameter((torch.randn(*s, generator=g) * std).to(dtype))
        self.width, self.heads = width, width // HEAD
        self.embed = new(vocab, width, std=1.0)
        self.norms = torch.nn.ParameterList([torch.nn.Parameter(torch.ones(width)) for _ in range(layers + 1)])
        self.selective = selective
        # even layers: value, gate, query, key, key gate of the decay rule; odd ones: input and gate of the vector's (selective: input and the
        # output's gate)
        self.ins = torch.nn.ParameterList([new(width, (5 if i % 2 == 0 else 2) * width, std=width ** -0.5) for i in range(layers)])
        self.outs = torch.nn.ParameterList([new(width, width, std=width ** -0.5) for _ in range(layers)])
        self.head = new(width, vocab, std=width ** -0.5)
        if selective:
            odd, full = range(layers // 2), lambda *s: torch.nn.Parameter(torch.zeros(*s))
            self.convs = torch.nn.ParameterList([new(width, TAPS, std=TAPS ** -0.5) for _ in odd])
            # from the convolution's results: step, and input and output of the states
            self.steps = torch.nn.ParameterList([new(width, width + 2 * STATES, std=0.5 * width ** -0.5) for _ in odd])
            # decays of 1 to STATES, steps of 0.002 to 0.1, softplus(-2.25) the largest
            self.rates = torch.nn.ParameterList([torch.nn.Parameter(torch.arange(1.0, STATES + 1).log().repeat(width, 1)) for _ in odd])
            self.biases = torch.nn.ParameterList([torch.nn.Parameter(torch.linspace(-6.2, -2.25, width)) for _ in odd])
            self.skips = torch.nn.ParameterList([torch.nn.Parameter(torch.ones(width)) for _ in odd])

    def _decay_inputs(self, u):
        x, f, q, k, fk = (t.unflatten(-1, (self.heads, HEAD)).contiguous() for t in u.chunk(5, dim=-1))
        return x * 0.25, f + 2, q * 0.25, k * 0.25, fk + 2              # (gates of mostly remembering)

    def _selective(self, i, u, conv, scan, conv_state, scan_state, **options):
        """A selective layer on its projection ``u``: whole sequences or a token, by the calls and states given; (results, states after it)"""
        x, gate = u.chunk(2, dim=-1)                                     # parts of the projection, as they lie
        x, conv_state = conv(x, self.convs[i], state=conv_state, silu=True, **options)
        dt, b, c = (x @ self.steps[i]).split([self.width, STATES, STATES], dim=-1)
        h, scan_state = scan(x, dt, -torch.exp(self.rates[i]), b, c, state=scan_state, skip=self.skips[i], gate=gate, dt_bias=self.biases[i], softplus=True,
                             **options)
        return h, conv_state, scan_state

    def forward(self, tokens, lengths=None):
        """logits [B, T, V] of every next token; ``lengths``: rows end there (right-padded)"""
        B = tokens.shape[0]
        branch = self.embed[tokens]
        stream = torch.zeros(*branch.shape, dtype=torch.float32, device=branch.device)
        for i, (norm, w_in, w_out) in enumerate(zip(self.norms, self.ins, self.outs)):
            y, stream = residual_rms_norm(branch, stream, norm)
            u = y @ w_in
            if i % 2 == 0:
                state = u.new_zeros(B, self.heads, HEAD, HEAD)
                h, _ = LFWHeadsFunction.apply(*self._decay_inputs(u), state, True)
                h = h.flatten(2)
            elif self.selective:
                h, _, _ = self._selective(i // 2, u, short_conv, selective_scan, None, None, lengths=lengths)
            else:
                x, f = u.chunk(2, dim=-1)                                # parts of the projection, as they lie
                h, _ = gated_scan(x, f + 2, lengths=lengths, logits=True)
            branch = h @ w_out
        y, _ = residual_rms_norm(branch, stream, self.norms[-1])
        return y @ self.head

    def _stepper(self, rows, eight_bit):
        """(a function of the next tokens [rows] to their logits [rows, V], the states of all layers that it updates in place)"""
        dev = self.embed.device
        norms = residual_rms_norm_fp8 if eight_bit else residual_rms_norm
        ins, outs = [Projection(w, eight_bit) for w in self.ins], [Projection(w, False) for w in self.outs]
        head = Projection(self.head, eight_bit)
        states = [torch.zeros(rows * self.heads, HEAD, HEAD, dtype=w.dtype, device=dev) if i % 2 == 0 else
                  torch.zeros(rows, self.width, STATES, device=dev) if self.selective else torch.zeros(rows, self.width, device=dev)
                  for i, w in enumerate(self.ins)]
        convs = [torch.zeros(rows, TAPS - 1, self.width, dtype=w.dtype, device=dev) for w in self.ins[1::2]] if self.selective else []

        def step(tokens):
            branch = self.embed[tokens]
            stream = torch.zeros(rows, self.width, device=dev)
            for i, norm in enumerate(self.norms):
                *y, stream = norms(branch, stream, norm)
                if i == len(self.ins):
                    break
                u = ins[i](*y)
                if i % 2 == 0:
                    x, f, q, k, fk = (v.reshape(rows * self.heads, HEAD) for v in self._decay_inputs(u))
                    h, _ = lfw_step(x, torch.sigmoid(f), q, k, torch.sigmoid(fk), states[i])
                    h = h.view(rows, self.width)
                elif self.selective:
                    h, _, _ = self._selective(i // 2, u, short_conv_step, selective_scan_step, convs[i // 2], states[i])
                else:
                    x, f = u.chunk(2, dim=-1)
                    h, _ = gated_scan_step(x.contiguous(), f + 2, states[i], logits=True)
                branch = outs[i](h)
            return head(*y)
        return step, states + convs

    @torch.no_grad()
    def generate(self, prompt, steps, generator=None, eight_bit=False):
        """[B, T] tokens -> ([B, T + steps] tokens, logits [B, T + steps - 1, V] that they were drawn from): token by token, a state per layer"""
        B, T = prompt.shape
        step, _ = self._stepper(B, eight_bit)
        tokens, seen = [prompt[:, t] for t in range(T)], []
        for t in range(T + steps - 1):
            logits = step(tokens[t])
            seen.append(logits)
            if t >= T - 1:
                p = torch.softmax(logits.float(), dim=-1)
                tokens.append(torch.multinomial(p, 1, generator=generator)[:, 0])
        return torch.stack(tokens, 1), torch.stack(seen, 1)

    @torch.no_grad()
    def beam_search(self, prompt, steps, beams=4, end=None, eight_bit=False):
        """[B, T] tokens -> ([B, beams, T + steps] tokens, their answers' log probabilities [B, beams] float32), best first.  An answer ends at the
        token ``end`` (``None``: nowhere) and is filled up with it."""
        B, T = prompt.shape
        if T < 1:
            raise ValueError("a search goes on from at least one token")
        step, states = self._stepper(B * beams, eight_bit)
        tokens = torch.zeros(B * beams, T + steps, dtype=torch.int64, device=prompt.device)
        tokens[:, :T] = prompt.repeat_interleave(beams, dim=0)
        for t in range(T - 1):
            step(tokens[:, t])
        # all beams of a prompt are the same so far: one of them counts
        scores = torch.full((B, beams), float("-inf"), device=prompt.device)
        scores[:, 0] = 0.0
        finished = None if end is None else torch.zeros(B, beams, dtype=torch.bool, device=prompt.device)
        for t in range(T, T + steps):
            logits = step(tokens[:, t - 1]).view(B, beams, -1).contiguous()
            scores, came_from, chosen = beam_select(logits, scores, finished=finished, pad=0 if end is None else end)
            moved = states + [tokens] + ([] if end is None else [finished.view(-1)])
            reorder_beams(moved, came_from)
            tokens[:, t] = chosen.view(-1)
            if end is not None:
                finished |= chosen == end
        return tokens.view(B, beams, -1), scores


class PolicyTrainer:
    """Policy steps on a model with 16-bit parameters: float32 copies that the steps are made on, in one buffer, and their gradients in another"""

    def __init__(self, model, lr=0.5, max_norm=1.0, clip=(0.2, 0.28), kl_coef=0.01):
        self.model, self.lr, self.max_norm, self.clip, self.kl_coef = model, lr, max_norm, clip, kl_coef
        self.params = list(model.parameters())
        sizes = [p.numel() for p in self.params]
        self.master = torch.cat([p.detach().float().flatten() for p in self.params])
        self.grads = torch.empty_like(self.master)
        self.grad_views = [v.view_as(p) for v, p in zip(self.grads.split(sizes), self.params)]
        self.master_views = [v.view_as(p) for v, p in zip(self.master.split(sizes), self.params)]

    def log_probabilities(self, tokens):
        """of every token after the first, [B, T - 1]"""
        with torch.no_grad():
            zero = torch.zeros(tokens.shape[0], tokens.shape[1] - 1, device=tokens.device)
            return policy_loss(self.model(tokens[:, :-1]), tokens[:, 1:].contiguous(), zero, zero, zero)[1]

    def step(self, tokens, old_logp, ref_logp, advantages, mask):
        """One clipped step; tokens [B, T], the others [B, T - 1].  Returns (loss, the gradients' norm), on the device."""
        for p in self.params:
            p.grad = None
        loss, _ = policy_loss(self.model(tokens[:, :-1]), tokens[:, 1:].contiguous(), old_logp, ref_logp, advantages, mask=mask, clip=self.clip,
                              kl_coef=self.kl_coef)
        loss.backward()
        norm = clip_grad_norm([p.grad for p in self.params], self.max_norm, out=self.grad_views)
        with torch.no_grad():
            self.master.sub_(self.grads, alpha=self.lr)
            for p, m in zip(self.params, self.master_views):
                p.copy_(m)
        return loss.detach(), norm


def rewards(tokens, vocab):
    return (tokens < vocab // 2).float()


def finetune(rounds=10, batch=64, prompt=16, answer=48, vocab=512, width=128, layers=4, steps=2, eight_bit=False, seed=0, say=print,
             selective=False, beams=0):
    """The mean reward of each round's answers; with ``beams``, of the best ones that a beam search finds at the end too"""
    model = RecurrentLM(vocab, width, layers, seed=seed, selective=selective).cuda()
    trainer = PolicyTrainer(model)
    reference = RecurrentLM(vocab, width, layers, seed=seed, selective=selective).cuda()
    at_start = PolicyTrainer(reference)
    g = torch.Generator(device="cuda").manual_seed(seed)
    history, asked = [], None
    prompts = lambda: torch.randint(0, vocab, (batch, prompt), generator=g, device="cuda")
    for r in range(rounds):
        asked = prompts()
        tokens, _ = model.generate(asked, answer, generator=g, eight_bit=eight_bit)
        reward = rewards(tokens[:, 1:], vocab)
        old, ref = trainer.log_probabilities(tokens), at_start.log_probabilities(tokens)
        mask = (torch.arange(tokens.shape[1] - 1, device="cuda") >= prompt - 1).expand_as(old).contiguous()
        mean = (reward * mask).sum() / mask.sum()
        advantage = (reward - mean) / ((mean * (1 - mean)).sqrt() + 1e-3)
        for _ in range(steps):
            loss, norm = trainer.step(tokens, old, ref, advantage, mask)
        history.append(float(mean))
        say("round %3d  reward %.3f  loss %+.4f  gradient norm %.3f" % (r, history[-1], float(loss), float(norm)))
    if beams:
        asked = prompts() if asked is None else asked                    # (those of the last round)
        tokens, scores = model.beam_search(asked, answer, beams=beams, eight_bit=eight_bit)
        history.append(float(rewards(tokens[:, 0, prompt:], vocab).mean()))
        say("beam search of %d: reward %.3f  log probability %.2f" % (beams, history[-1], float(scores[:, 0].mean())))
    return history


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("rounds", 10), ("batch", 64), ("prompt", 16), ("answer", 48), ("vocab", 512), ("width", 128), ("layers", 4), ("steps", 2),
                        ("seed", 0), ("beams", 0)):
        p.add_argument("--" + name, type=int, default=value)
    p.add_argument("--eight-bit", action="store_true")
    p.add_argument("--selective", action="store_true")
    finetune(**vars(p.parse_args()))


if __name__ == "__main__":
    main()

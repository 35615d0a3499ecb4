"""A fine-tuning step and generation of a small recurrent language model, through every operator that stands around the recurrences.

    python -m t2fw_amd.finetune                       # a few rounds: answers, their reward, a clipped policy step on them
    python -m t2fw_amd.finetune --rounds 40 --width 256 --layers 4

The layers alternate between the decay rule (``LFWHeadsFunction``, a 64 x 64 state per head) and the recurrence with a vector for its
state (``gated_scan``).  Each is a residual branch: ``residual_rms_norm`` adds the branch before to a float32 stream and normalises it,
a projection makes the recurrence's inputs, another its output.

* Training: logits of whole sequences, ``policy_loss`` on the answers' tokens, backward, ``clip_grad_norm`` of the 16-bit gradients into
  float32 ones, a gradient step on float32 parameters.
* Generation: one token per call, states updated in place (``lfw_step``, ``gated_scan_step``); with ``--eight-bit`` the
  norms come from ``residual_rms_norm_fp8`` and the projections are 8-bit products.

There is no task and no data here: a token of an answer is rewarded if it is in the lower half of the vocabulary, and the steps have to
raise their share.
"""
import argparse

import torch

from .functional_lfw import LFWHeadsFunction, lfw_step
from .functional_loss import policy_loss
from .functional_norm import residual_rms_norm, residual_rms_norm_fp8
from .functional_scan import gated_scan, gated_scan_step
from .grad_clip import clip_grad_norm

HEAD = 64                                # channels of a head, on both sides of the decay rule's state


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
    def __init__(self, vocab=512, width=128, layers=4, dtype=torch.bfloat16, seed=0):
        super().__init__()
        assert width % HEAD == 0, "the width is whole heads of %d channels" % HEAD
        g = torch.Generator().manual_seed(seed)
        new = lambda *s, std: torch.nn.Parameter((torch.randn(*s, generator=g) * std).to(dtype))
        self.width, self.heads = width, width // HEAD
        self.embed = new(vocab, width, std=1.0)
        self.norms = torch.nn.ParameterList([torch.nn.Parameter(torch.ones(width)) for _ in range(layers + 1)])
        # even layers: value, gate, query, key, key gate of the decay rule; odd ones: input and gate of the vector's
        self.ins = torch.nn.ParameterList([new(width, (5 if i % 2 == 0 else 2) * width, std=width ** -0.5) for i in range(layers)])
        self.outs = torch.nn.ParameterList([new(width, width, std=width ** -0.5) for _ in range(layers)])
        self.head = new(width, vocab, std=width ** -0.5)

    def _decay_inputs(self, u):
        x, f, q, k, fk = (t.unflatten(-1, (self.heads, HEAD)).contiguous() for t in u.chunk(5, dim=-1))
        return x * 0.25, f + 2, q * 0.25, k * 0.25, fk + 2              # (gates of mostly remembering)

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
            else:
                x, f = u.chunk(2, dim=-1)                                # parts of the projection, as they lie
                h, _ = gated_scan(x, f + 2, lengths=lengths, logits=True)
            branch = h @ w_out
        y, _ = residual_rms_norm(branch, stream, self.norms[-1])
        return y @ self.head

    @torch.no_grad()
    def generate(self, prompt, steps, generator=None, eight_bit=False):
        """[B, T] tokens -> ([B, T + steps] tokens, logits [B, T + steps - 1, V] that they were drawn from): token by token, a state per layer"""
        B, T = prompt.shape
        dev = prompt.device
        norms = residual_rms_norm_fp8 if eight_bit else residual_rms_norm
        ins, outs = [Projection(w, eight_bit) for w in self.ins], [Projection(w, False) for w in self.outs]
        head = Projection(self.head, eight_bit)
        states = [torch.zeros(B * self.heads, HEAD, HEAD, dtype=w.dtype, device=dev) if i % 2 == 0 else
                  torch.zeros(B, self.width, device=dev) for i, w in enumerate(self.ins)]
        tokens, seen = [prompt[:, t] for t in range(T)], []
        for t in range(T + steps - 1):
            branch = self.embed[tokens[t]]
            stream = torch.zeros(B, self.width, device=dev)
            for i, norm in enumerate(self.norms):
                *y, stream = norms(branch, stream, norm)
                if i == len(self.ins):
                    break
                u = ins[i](*y)
                if i % 2 == 0:
                    x, f, q, k, fk = (v.reshape(B * self.heads, HEAD) for v in self._decay_inputs(u))
                    h, _ = lfw_step(x, torch.sigmoid(f), q, k, torch.sigmoid(fk), states[i])
                    h = h.view(B, self.width)
                else:
                    x, f = u.chunk(2, dim=-1)
                    h, _ = gated_scan_step(x.contiguous(), f + 2, states[i], logits=True)
                branch = outs[i](h)
            logits = head(*y)
            seen.append(logits)
            if t >= T - 1:
                p = torch.softmax(logits.float(), dim=-1)
                tokens.append(torch.multinomial(p, 1, generator=generator)[:, 0])
        return torch.stack(tokens, 1), torch.stack(seen, 1)


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


def finetune(rounds=10, batch=64, prompt=16, answer=48, vocab=512, width=128, layers=4, steps=2, eight_bit=False, seed=0, say=print):
    """The mean reward of each round's answers"""
    model = RecurrentLM(vocab, width, layers, seed=seed).cuda()
    trainer = PolicyTrainer(model)
    reference = RecurrentLM(vocab, width, layers, seed=seed).cuda()
    at_start = PolicyTrainer(reference)
    g = torch.Generator(device="cuda").manual_seed(seed)
    history = []
    for r in range(rounds):
        asked = torch.randint(0, vocab, (batch, prompt), generator=g, device="cuda")
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
    return history


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("rounds", 10), ("batch", 64), ("prompt", 16), ("answer", 48), ("vocab", 512), ("width", 128), ("layers", 4), ("steps", 2),
                        ("seed", 0)):
        p.add_argument("--" + name, type=int, default=value)
    p.add_argument("--eight-bit", action="store_true")
    finetune(**vars(p.parse_args()))


if __name__ == "__main__":
    main()

"""Hardware-aware tuning of a small language model on crossbar layers.

    python -m memintelli_flash_b200.lm_tuning preference [--steps 40] [--noisy]
    python -m memintelli_flash_b200.lm_tuning policy [--steps 40] [--noisy]

The model is a token embedding (``EmbeddingScaled``), residual ``LinearMem`` blocks over each token and the running
mean of the tokens before it, and a ``LinearMem`` head: every matrix product runs on the simulated crossbars, with
straight-through gradients.  The task is a rule, "token t is followed by 3 t + 1": ``preference`` learns it from pairs of
continuations that follow it and random ones, ``policy`` from sampled continuations and the share of their tokens that
follow it.  One step is: logits, ``tuning.preference_loss`` or ``tuning.policy_loss`` against the log-probabilities of
the frozen start (``tuning.token_logprobs``), backward, ``tuning.clip_grad_norm_``, an AdamW update, and the crossbars
programmed again (``update_weight``).
"""
from __future__ import annotations

import argparse

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import tuning
from .NN_layers import EmbeddingScaled, LinearMem
from .pimpy import DPETensor

IGNORE = -100


def make_engine(device, noisy=False):
    """The example device of the package's benchmarks; noisy: read variation and voltage noise of 2%."""
    noise = 0.02 if noisy else 0.0
    return DPETensor(HGS=1e-5, LGS=1e-8, write_variation=0.0, rate_stuck_HGS=0.0, rate_stuck_LGS=0.0,
                     read_variation=noise, vnoise=noise, rdac=4, g_level=4, radc=4096, device=device)


class SmallCimLM(nn.Module):
    """(B, T) token ids -> (B, T, vocab) logits of the next token."""

    def __init__(self, engine, vocab=128, hidden=64, blocks=2, seed=0):
        super().__init__()
        torch.manual_seed(seed)
        mem = dict(input_slice=(1, 1, 2, 2, 2), weight_slice=(1, 1, 2, 2, 2), device=engine.device,
                   input_paral_size=(1, 32), weight_paral_size=(32, 32), input_quant_gran=(1, 64),
                   weight_quant_gran=(64, 64))
        self.embed = EmbeddingScaled(vocab, hidden, scale=hidden ** 0.5, device=engine.device)
        self.blocks = nn.ModuleList(LinearMem(engine, 2 * hidden, hidden, **mem) for _ in range(blocks))
        self.head = LinearMem(engine, hidden, vocab, bias=False, **mem)

    def forward(self, ids):
        B, T = ids.shape
        h = self.embed(ids)
        count = torch.arange(1, T + 1, device=ids.device, dtype=h.dtype)[:, None]
        for block in self.blocks:
            seen = torch.cumsum(h, 1) / count
            h = h + F.gelu(block(torch.cat([h, seen], -1).reshape(B * T, -1))).view(B, T, -1)
        return self.head(h.reshape(B * T, -1)).view(B, T, -1)

    def update_weight(self):
        """Programs the crossbars with the current weights."""
        for layer in (*self.blocks, self.head):
            layer.update_weight()


def shifted(ids, prompt):
    """Targets of each position: the next token, ignored inside the prompt and at the last position."""
    targets = torch.full_like(ids, IGNORE)
    targets[:, prompt - 1:-1] = ids[:, prompt:]
    return targets


def follow_rule(first, length, vocab):
    out = [first]
    for _ in range(length - 1):
        out.append((3 * out[-1] + 1) % vocab)
    return torch.stack(out, 1)


class Tuner:
    """A model, its frozen start as the reference policy, and the update after a loss."""

    def __init__(self, engine, vocab=128, hidden=64, lr=5e-3, max_norm=1.0, seed=0):
        self.model = SmallCimLM(engine, vocab, hidden, seed=seed)
        self.start = SmallCimLM(engine, vocab, hidden, seed=seed)
        self.start.load_state_dict(self.model.state_dict())
        self.start.update_weight()
        self.vocab, self.max_norm = vocab, max_norm
        self.optimizer = torch.optim.AdamW(self.model.parameters(), lr=lr)
        self.gen = torch.Generator(device=engine.device).manual_seed(seed)

    def random_tokens(self, *shape):
        return torch.randint(0, self.vocab, shape, generator=self.gen, device=self.model.head.weight.device)

    def reference_logps(self, ids, targets):
        with torch.no_grad():
            return tuning.token_logprobs(self.start(ids), targets, ignore_index=IGNORE)

    def update(self, loss):
        """Backward, clipping, the weights' update and the crossbars'; returns the gradient norm before clipping."""
        self.optimizer.zero_grad(set_to_none=True)
        loss.backward()
        norm = tuning.clip_grad_norm_(self.model.parameters(), self.max_norm)
        self.optimizer.step()
        self.model.update_weight()
        return norm

    def preference_step(self, pairs=16, length=24, prompt=4, beta=0.5):
        first = follow_rule(self.random_tokens(pairs), length, self.vocab)
        second = first.clone()
        second[:, prompt:] = self.random_tokens(pairs, length - prompt)
        ids = torch.cat([first, second])
        targets = shifted(ids, prompt)
        r = tuning.preference_loss(self.model(ids), targets, self.reference_logps(ids, targets), beta=beta)
        norm = self.update(r.loss)
        return {"loss": r.loss.detach(), "margin": (r.chosen_rewards - r.rejected_rewards).mean(), "norm": norm}

    @torch.no_grad()
    def sample(self, ids, length):
        while ids.shape[1] < length:
            p = torch.softmax(self.model(ids)[:, -1], -1)
            ids = torch.cat([ids, torch.multinomial(p, 1, generator=self.gen)], 1)
        return ids

    def policy_step(self, groups=8, samples=8, length=12, prompt=4, kl_coef=0.01, epochs=2):
        """Sampled continuations of the same prompts, advantages relative to their group, ``epochs`` updates on them."""
        start = follow_rule(self.random_tokens(groups), prompt, self.vocab).repeat_interleave(samples, 0)
        ids = self.sample(start, length)
        targets = shifted(ids, prompt)
        reward = (ids[:, prompt:] == (3 * ids[:, prompt - 1:-1] + 1) % self.vocab).float().mean(1)
        g = reward.view(groups, samples)
        adv = ((g - g.mean(1, keepdim=True)) / (g.std(1, keepdim=True) + 1e-4)).reshape(-1)
        with torch.no_grad():
            old = tuning.token_logprobs(self.model(ids), targets, ignore_index=IGNORE)
        ref = self.reference_logps(ids, targets)
        for _ in range(epochs):
            r = tuning.policy_loss(self.model(ids), targets, old, adv, ref, clip_low=0.2, clip_high=0.28,
                                   kl_coef=kl_coef, reduction="sequence", ignore_index=IGNORE)
            norm = self.update(r.loss)
        return {"loss": r.loss.detach(), "reward": reward.mean(), "kl": r.kl.detach(), "norm": norm}


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("kind", choices=("preference", "policy"))
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--noisy", action="store_true")
    ap.add_argument("--device", default="cuda:0")
    a = ap.parse_args()
    t = Tuner(make_engine(torch.device(a.device), a.noisy))
    step = t.preference_step if a.kind == "preference" else t.policy_step
    for i in range(a.steps):
        r = step()
        if i % 5 == 0 or i + 1 == a.steps:
            print(f"step {i}: " + ", ".join(f"{k} {v.item():.4f}" for k, v in r.items()), flush=True)


if __name__ == "__main__":
    main()

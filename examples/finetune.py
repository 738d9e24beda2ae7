"""A fine-tuning loop on one MI355X: preference loss, then policy loss, stepped by AdamW.

    python examples/finetune.py [--steps N]

A small random language model learns to prefer answers that use one half of the
vocabulary (pairs of answers, a frozen copy of the model as the reference, 8-bit
moments), then to emit tokens of one residue class (sampled answers, advantages
within the group, 32-bit moments).  Synthetic data; prints the losses.
"""
import argparse
import copy
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gefen-x_amd"))

import gefen  # noqa: E402

VOCAB, WIDTH, PROMPT, ANSWER = 4096, 256, 8, 24
IGNORE = -100


class Model(nn.Module):
    """Next-token logits from the token and the mean of the ones before it."""

    def __init__(self):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, WIDTH)
        self.mix = nn.Sequential(nn.Linear(2 * WIDTH, WIDTH), nn.SiLU(), nn.LayerNorm(WIDTH))
        self.head = nn.Linear(WIDTH, VOCAB, bias=False)

    def forward(self, tokens):
        x = self.embed(tokens)
        past = x.cumsum(1) / torch.arange(1, x.shape[1] + 1, device=x.device, dtype=x.dtype)[:, None]
        return self.head(self.mix(torch.cat([x, past], -1)))


def shifted(tokens):
    """Labels: logits[:, t] predicts tokens[:, t + 1]; the prompt is not learned from."""
    labels = torch.full_like(tokens, IGNORE)
    labels[:, PROMPT - 1:-1] = tokens[:, PROMPT:]
    return labels


def prefer(model, steps, pairs=16):
    """Answers of low tokens are chosen over answers of high ones."""
    reference = copy.deepcopy(model).requires_grad_(False)
    opt = gefen.AdamW(model.named_parameters(), lr=2e-3, weight_decay=0.0, state_bits=8, max_grad_norm=1.0)
    losses = []
    for _ in range(steps):
        dev = model.head.weight.device
        prompt = torch.randint(0, VOCAB, (pairs, PROMPT), device=dev)
        low = torch.randint(0, VOCAB // 2, (pairs, ANSWER), device=dev)
        tokens = torch.cat([torch.cat([prompt, low], 1), torch.cat([prompt, low + VOCAB // 2], 1)])
        labels = shifted(tokens)
        ref = gefen.token_logps(reference(tokens), labels)
        out = gefen.preference_loss(model(tokens), labels, ref, beta=0.1)
        opt.zero_grad()
        out.loss.backward()
        opt.step()
        losses.append(out.loss.detach())
    return torch.stack(losses).tolist()


@torch.no_grad()
def sample(model, prompt):
    tokens = prompt
    for _ in range(ANSWER):
        p = torch.softmax(model(tokens)[:, -1].float(), -1)
        tokens = torch.cat([tokens, torch.multinomial(p, 1)], 1)
    return tokens


def reinforce(model, steps, group=64):
    """Answers are rewarded for tokens that are multiples of 4; two updates from each batch of samples."""
    opt = gefen.AdamW(model.named_parameters(), lr=3e-3, weight_decay=0.0, max_grad_norm=1.0)
    reference = copy.deepcopy(model).requires_grad_(False)
    rewards = []
    for _ in range(steps):
        prompt = torch.randint(0, VOCAB, (1, PROMPT), device=model.head.weight.device).expand(group, -1)
        tokens = sample(model, prompt)
        labels = shifted(tokens)
        reward = (tokens[:, PROMPT:] % 4 == 0).float().mean(1)
        advantage = (reward - reward.mean()) / (reward.std() + 1e-4)
        with torch.no_grad():
            old, ref = gefen.token_logps(model(tokens), labels), gefen.token_logps(reference(tokens), labels)
        for _ in range(2):
            logits = model(tokens)
            _, grad = gefen.policy_loss_and_grad(logits, labels, old, advantage, ref, kl_coef=1e-3, reduction="sequence")
            opt.zero_grad()
            logits.backward(grad)
            opt.step()
        rewards.append(reward.mean())
    return torch.stack(rewards).tolist()


def main(steps=60, dtype=torch.bfloat16):
    torch.manual_seed(0)
    model = Model().to("cuda", dtype)
    losses = prefer(model, steps)
    print("preference loss: first {:.4f}, last {:.4f}".format(losses[0], losses[-1]))
    rewards = reinforce(model, steps)
    print("mean reward: first {:.4f}, last {:.4f}".format(rewards[0], rewards[-1]))
    return losses, rewards


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    main(ap.parse_args().steps)

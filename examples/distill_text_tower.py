"""A small text tower learns from a large one's top logits, beside the contrastive loss.

The teacher scores the captions once: log probabilities of their tokens, and for
every position its 16 most probable tokens, which is all that is kept of its
logits.  The student (half the features) is then trained on

    CLIP loss of captions and images  +  weight * distillation from the kept logits

and scored in the end the way the teacher was.  Captions and images are synthetic.

    python examples/distill_text_tower.py [--steps 150] [--texts 256] [--vocab 4096]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from memoryefficientclip_amd import (  # noqa: E402
    MemoryEfficientCLIPLoss,
    ScaledTokenEmbedding,
    TopKDistillationLoss,
    token_log_probs,
)

PAD = 0


class TextTower(nn.Module):
    """Tokens to a feature per text and to logits of each next token: the token's
    embedding and the mean of those so far, two layers, and the embedding again
    as the output layer."""

    def __init__(self, vocab, dim, device, dtype):
        super().__init__()
        self.embed = ScaledTokenEmbedding(vocab, dim, padding_idx=PAD, device=device, dtype=dtype)
        self.layers = nn.Sequential(nn.Linear(2 * dim, 2 * dim, device=device, dtype=dtype), nn.GELU(),
                                    nn.Linear(2 * dim, dim, device=device, dtype=dtype))

    def forward(self, tokens):
        e = self.embed(tokens)
        steps = torch.arange(1, tokens.shape[1] + 1, device=tokens.device)[:, None]
        h = self.layers(torch.cat([e, (e.float().cumsum(1) / steps).to(e.dtype)], -1))
        real = (tokens != PAD)[..., None]
        text = (h * real).float().sum(1) / real.sum(1)
        return text, (h.reshape(-1, h.shape[-1]) @ self.embed.weight.t()).view(*tokens.shape, -1)


def captions(texts, length, vocab, device, generator):
    """Token t is often followed by a token near 3 t: something to learn."""
    tok = torch.randint(1, vocab, (texts, 1), generator=generator)
    rows = [tok]
    for _ in range(length - 1):
        near = (3 * rows[-1] + torch.randint(0, 4, (texts, 1), generator=generator)) % (vocab - 1) + 1
        rows.append(near)
    tok = torch.cat(rows, 1)
    ends = torch.randint(length // 2, length + 1, (texts, 1), generator=generator)
    return tok.masked_fill(torch.arange(length) >= ends, PAD).to(device)


def next_tokens(tokens):
    """The token that follows each position; -100 where there is none."""
    return torch.where(tokens[:, 1:] == PAD, -100, tokens[:, 1:])


def scores(tower, tokens, top_k=0):
    """The tower's scores of the captions, positions without a next token left out."""
    with torch.no_grad():
        _, logits = tower(tokens)
        return token_log_probs(logits[:, :-1], next_tokens(tokens), top_k=top_k)


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=150)
    p.add_argument("--texts", type=int, default=256)
    p.add_argument("--length", type=int, default=24)
    p.add_argument("--vocab", type=int, default=4096)
    p.add_argument("--dim", type=int, default=128)
    p.add_argument("--top-k", type=int, default=16)
    args = p.parse_args(argv)
    device, dtype = "cuda", torch.float32
    torch.manual_seed(0)
    g = torch.Generator().manual_seed(1)
    tokens = captions(args.texts, args.length, args.vocab, device, g)
    images = torch.randn(args.texts, args.dim, generator=g).to(device)
    real = (next_tokens(tokens) != -100).sum()

    # the teacher learns the captions: minus the log probability of their tokens
    teacher = TextTower(args.vocab, 2 * args.dim, device, dtype)
    opt = torch.optim.Adam(teacher.parameters(), lr=3e-3)
    for _ in range(args.steps):
        opt.zero_grad(set_to_none=True)
        _, logits = teacher(tokens)
        loss = -token_log_probs(logits[:, :-1], next_tokens(tokens)).log_probs.sum() / real
        loss.backward()
        opt.step()
    kept = scores(teacher, tokens, args.top_k)
    print(f"teacher: {-(kept.log_probs.sum() / real).item():.3f} nats a token, "
          f"entropy {(kept.entropy.sum() / real).item():.3f}", flush=True)

    student = TextTower(args.vocab, args.dim, device, dtype)
    contrast = MemoryEfficientCLIPLoss(temperature=0.07)
    distill = TopKDistillationLoss(temperature=1.0, weight=0.5)
    opt = torch.optim.Adam(student.parameters(), lr=3e-3)
    first = None
    for step in range(args.steps):
        opt.zero_grad(set_to_none=True)
        text, logits = student(tokens)
        from_teacher = distill(logits[:, :-1], kept.top_tokens, kept.top_log_probs)
        total = contrast(images, text) + from_teacher
        total.backward()
        opt.step()
        if first is None:
            first = (from_teacher.detach(), total.detach())
        if step % 50 == 0 or step == args.steps - 1:
            print(f"step {step}: distillation {from_teacher.item():.3f}, total {total.item():.3f}", flush=True)
    end = scores(student, tokens, args.top_k)
    # how often the student's first choice is the teacher's
    same = ((end.top_tokens[..., 0] == kept.top_tokens[..., 0]) & (end.top_tokens[..., 0] >= 0)).sum() / real
    print(f"student: {-(end.log_probs.sum() / real).item():.3f} nats a token, first choice as the teacher's "
          f"{100 * same.item():.0f}%", flush=True)
    return {"first": [v.item() for v in first], "last": [from_teacher.item(), total.item()], "agreement": same.item()}


if __name__ == "__main__":
    main()

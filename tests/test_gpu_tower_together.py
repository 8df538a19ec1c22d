"""The operators as a tower runs them together: token embedding, a fused projection, the
norm and rotation of queries and keys, attention over padded texts, and the contrastive
loss; forward and backward against the same tower in 64 bits."""
import pytest
import torch

import memoryefficientclip_amd as mec
import oracle
import tower_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TEXTS, TOKENS, VOCAB, HEADS, KEY_HEADS, DIM = 12, 29, 50, 4, 2, 16


def tower(embed, qkv, norms, tokens, lengths, rotate, attend, lookup):
    width = HEADS * DIM
    x = lookup(tokens, embed)
    q, k, v = (x @ qkv).view(*tokens.shape, HEADS + 2 * KEY_HEADS, DIM).split([HEADS, KEY_HEADS, KEY_HEADS], 2)
    q, k = rotate(q, k, norms)
    y = x + attend(q, k, v, lengths).flatten(2)
    real = torch.arange(tokens.shape[1], device=tokens.device) < lengths[:, None]
    return (y * real[..., None]).sum(1) / lengths.clamp(min=1)[:, None], width


@pytest.mark.parametrize("causal", [False, True])
def test_a_tower(causal):
    g = torch.Generator().manual_seed(0)
    width = HEADS * DIM
    embed = torch.randn(VOCAB, width, generator=g) / width ** 0.5
    qkv = torch.randn(width, (HEADS + 2 * KEY_HEADS) * DIM, generator=g) / width ** 0.5
    norms = [1 + 0.1 * torch.randn(DIM, generator=g) for _ in "qk"]
    tokens = torch.randint(0, VOCAB, (TEXTS, TOKENS), generator=g)
    lengths = torch.randint(1, TOKENS + 1, (TEXTS,), generator=g)
    images = torch.randn(TEXTS, width, generator=g)
    positions, sections = torch.arange(TOKENS)[:, None], (DIM // 2,)

    # this package, fp32
    leaves = [t.to(DEV).requires_grad_(True) for t in (embed, qkv, *norms)]
    pos = positions.to(DEV)
    text, _ = tower(leaves[0], leaves[1], leaves[2:], tokens.to(DEV), lengths.to(DEV),
                    lambda q, k, w: mec.norm_rotary(q, k, pos, sections, *w, eps=1e-6),
                    lambda q, k, v, n: mec.attention(q, k, v, causal=causal, query_lengths=n, key_lengths=n),
                    lambda t, e: mec.scaled_embedding(t, e, width ** 0.5))
    loss = mec.MemoryEfficientCLIPLoss(temperature=0.5)(images.to(DEV), text)
    loss.backward()

    # 64 bits
    wide = [t.double().requires_grad_(True) for t in (embed, qkv, *norms)]

    def rotate(q, k, w):
        angle = (positions.double() * ref.frequencies(sections, 10000.0))[:, None]

        def one(x, w):
            x = x * w / torch.sqrt(x.square().mean(3, keepdim=True) + 1e-6)
            a, b = x.chunk(2, 3)
            return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], 3)

        return one(q, w[0]), one(k, w[1])

    def attend(q, k, v, n):
        see = ref.sees(TEXTS, TOKENS, TOKENS, causal, n, n)[:, None]
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        k, v = (t.repeat_interleave(HEADS // KEY_HEADS, 1) for t in (k, v))
        s = (q @ k.transpose(2, 3) / DIM ** 0.5).masked_fill(~see, -1e9)
        return (torch.softmax(s, 3) * see.any(3, keepdim=True) @ v).transpose(1, 2)

    text64, _ = tower(wide[0], wide[1], wide[2:], tokens, lengths, rotate, attend, lambda t, e: e[t] * width ** 0.5)
    loss64, _, dtext = oracle.clip_loss_and_grads(images.double(), text64.detach(), 0.5)
    text64.backward(dtext)
    # Six stages in fp32, each off by at most n E of the sizes of its n <= 128 terms, whose sum is at most 16 times
    # the largest result here: 6 * 128 * 16 E = 2^-10.4 of the largest value.
    assert abs(loss.item() - loss64.item()) <= 2.0 ** -10 * abs(loss64.item())
    for name, got, want in zip(("embedding", "projection", "query norm", "key norm"), leaves, wide):
        ref.close(name, got.grad, want.grad, 2.0 ** -10 * want.grad.abs().max())


def test_offloaded_and_recomputed():
    """Saved tensors that go through the host, or are made again, give the same gradients."""
    from torch.utils.checkpoint import checkpoint

    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(3, 40, 8, 32, generator=g).to(DEV, torch.bfloat16)
    w = torch.ones(32, device=DEV, dtype=torch.bfloat16)
    pos, n = torch.arange(40, device=DEV)[:, None], torch.tensor([40, 0, 17], device=DEV)

    def f(x, w):
        q, k, v = x.split([4, 2, 2], 2)
        q, k = mec.norm_rotary(q, k, pos, (16,), w, w, eps=1e-6)
        return mec.attention(q, k, v, causal=True, query_lengths=n, key_lengths=n)

    grads = []
    for way in ("plain", "host", "again"):
        leaves = [qkv.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        if way == "host":
            with torch.autograd.graph.save_on_cpu():
                out = f(*leaves)
        elif way == "again":
            out = checkpoint(f, *leaves, use_reentrant=False)
        else:
            out = f(*leaves)
        out.float().square().sum().backward()
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(a, b) for way in grads[1:] for a, b in zip(grads[0], way))

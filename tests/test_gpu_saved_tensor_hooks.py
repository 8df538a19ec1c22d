"""Gradients under saved-tensor hooks are the gradients without them, bit for bit:
the kernels read what came back, wherever and in whatever strides it lies."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu

import memoryefficientclip_amd as mec

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# slices of positions and columns, other orders of the positions, rows that are one in memory
CUTS = [lambda x: x[:, :-1], lambda x: x[:, 1:], lambda x: x[..., 3:900], lambda x: x.transpose(0, 1),
        lambda x: x[:, :1].expand(-1, 5, -1), lambda x: x[..., ::2], lambda x: x]


def logits(dtype=torch.float32):
    g = torch.Generator().manual_seed(1)
    return torch.randn(4, 6, 1003, generator=g).to(dtype).to(DEV).requires_grad_(True)


@pytest.mark.parametrize("pin", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("cut", CUTS)
def test_token_scores(cut, dtype, pin):
    x = logits(dtype)
    tokens = torch.arange(cut(x)[..., 0].numel(), device=DEV).reshape(cut(x).shape[:-1])

    def grad():
        r = mec.token_log_probs(cut(x), tokens, temperature=0.7)
        return torch.autograd.grad(r.log_probs.sum() + 0.5 * r.entropy.sum(), x)[0]

    want = grad()
    with save_on_cpu(pin_memory=pin):
        got = grad()
    assert torch.equal(got, want)


@pytest.mark.parametrize("pin", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("cut", CUTS)
def test_distillation(cut, dtype, pin):
    """Where the backward makes the gradient: no common grad_output, one other than 1, a second backward."""
    x = logits(dtype)
    shape = (*cut(x).shape[:-1], 5)
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, cut(x).shape[-1], shape, generator=g).to(DEV)
    z = torch.randn(shape, generator=g).to(DEV)

    def grads():
        rows = mec.TopKDistillationLoss(1.5, "none")(cut(x), tokens, z)
        yield torch.autograd.grad(rows.sum(), x)[0]
        loss = mec.TopKDistillationLoss(1.5)(cut(x), tokens, z)
        yield torch.autograd.grad(3.0 * loss, x, retain_graph=True)[0]
        yield torch.autograd.grad(loss, x)[0]

    want = list(grads())
    with save_on_cpu(pin_memory=pin):
        got = list(grads())
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))

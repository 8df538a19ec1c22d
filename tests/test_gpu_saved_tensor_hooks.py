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

"""Gradients under saved-tensor hooks are the gradients without them, bit for bit:
the kernels read what came back, wherever and in whatever strides it lies."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu
from torch.utils.checkpoint import checkpoint

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


@pytest.mark.parametrize("dtype,n", [(torch.float32, 200), (torch.float32, 2300), (torch.bfloat16, 300)], ids=str)
@pytest.mark.parametrize("loss", [mec.MemoryEfficientCLIPLoss(), mec.MemoryEfficientLiTLoss()], ids=["clip", "lit"])
@pytest.mark.parametrize("cut", [lambda x: x[:, :96], lambda x: x[:, 4:101], lambda x: x[::2], lambda x: x.t()[:96]])
def test_contrastive_losses(cut, loss, dtype, n):
    g = torch.Generator().manual_seed(3)
    x, y = (torch.randn(2 * n, 128, generator=g).to(dtype).to(DEV).requires_grad_(True) for _ in range(2))

    def grads():
        return torch.autograd.grad(loss(cut(x), cut(y)), (x, y), allow_unused=True)

    torch.use_deterministic_algorithms(True)
    try:
        want = grads()
        with save_on_cpu():
            got = grads()
    finally:
        torch.use_deterministic_algorithms(False)
    # Other strides may be read by other loads, in another order of the fp32 sums (d terms for a
    # similarity, 2 n for a gradient), before the rounding to the type on each side.
    bound = 2.0 ** -24 * (2 * n + 128) + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23)
    for a, b in zip(got, want):
        assert (a is None and b is None) or ((a - b).abs().max() <= bound * b.abs().max()).item()


def distillation(dtype):
    x = logits(dtype)
    g = torch.Generator().manual_seed(4)
    tokens = torch.randint(0, 1003, (4, 6, 5), generator=g).to(DEV)
    z = torch.randn(4, 6, 5, generator=g).to(DEV)
    return x, lambda x: mec.TopKDistillationLoss(1.5)(x * 1.0, tokens, z)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_the_forwards_gradient(dtype):
    x, loss = distillation(dtype)
    want, = torch.autograd.grad(loss(x), x)
    with save_on_cpu():
        got, = torch.autograd.grad(loss(x), x)
    assert torch.equal(got, want)
    got, = torch.autograd.grad(checkpoint(loss, x, use_reentrant=False), x)
    assert torch.equal(got, want)
    # summed with another gradient of the same logits, twice over a graph that is kept
    y = x * 1.0
    total = loss(y) + y.float().square().sum()
    a, = torch.autograd.grad(total, x, retain_graph=True)
    kept = a.clone()
    a.zero_()
    b, = torch.autograd.grad(total, x)
    torch.testing.assert_close(b, kept, rtol=2.0 ** -6 if dtype == torch.bfloat16 else 4e-6, atol=1e-6)


def test_a_checkpointed_region_keeps_no_gradient():
    rows, vocab = 64, 50001
    x = torch.randn(rows, vocab, device=DEV, requires_grad=True)
    tokens, z = torch.zeros(rows, 2, dtype=torch.int64, device=DEV), torch.zeros(rows, 2, device=DEV)
    before = torch.cuda.memory_allocated()
    loss = checkpoint(lambda x: mec.TopKDistillationLoss()(x, tokens, z), x, use_reentrant=False)
    assert torch.cuda.memory_allocated() - before < rows * vocab
    loss.backward()
    assert x.grad.shape == x.shape

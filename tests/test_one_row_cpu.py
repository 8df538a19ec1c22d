"""A matrix of one row may have any row stride, since nothing is ever that far from it:
smaller than the row for a transposed column or a view of one dimension."""
import pytest
import torch

import library_stub as stub
import memoryefficientclip_amd as mec

ROWS = [torch.randn(8, 1).t(), torch.randn(8).as_strided((1, 8), (0, 1)), torch.randn(8)[None], torch.randn(1, 20)[:, 3:11],
        torch.randn(8, 3)[:, :1].t()]


@pytest.fixture
def lib(monkeypatch):
    return stub.install(monkeypatch)


@pytest.mark.parametrize("x", ROWS)
def test_embedding(lib, x):
    w = x.detach().requires_grad_(True)
    mec.scaled_embedding(torch.tensor([0]), w).backward(x)
    (forward,), (backward,) = lib.calls["mec_embedding"], lib.calls["mec_embedding_backward"]
    assert forward[4] >= 8 and backward[4] >= 8


@pytest.mark.parametrize("x", ROWS)
def test_contrastive_loss(lib, x):
    a, b = x.detach().requires_grad_(True), x.clone().requires_grad_(True)
    mec.MemoryEfficientCLIPLoss()(a, b).backward()
    for name in ("mec_forward", "mec_backward"):
        (args,) = lib.calls[name]
        assert args[1] >= 8 and args[3] >= 8

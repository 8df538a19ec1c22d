"""A derivative through a gradient of the operators over a vocabulary raises, however it
is asked for: none of them may be taken for zero."""
import pytest
import torch
from torch.autograd import functional

import library_stub as stub
import memoryefficientclip_amd as mec


@pytest.fixture(autouse=True)
def lib(monkeypatch):
    return stub.install(monkeypatch)


TOKENS = torch.tensor([1, 2, 0])
LOSSES = [lambda x: mec.token_log_probs(x, TOKENS).log_probs.sum(),
          lambda x: mec.token_log_probs(x, TOKENS).entropy.sum(),
          lambda x: mec.TopKDistillationLoss()(x, TOKENS[:, None], torch.zeros(3, 1)),
          lambda x: mec.TopKDistillationLoss(reduction="none")(x, TOKENS[:, None], torch.zeros(3, 1)).sum(),
          lambda x: mec.scaled_embedding(TOKENS, x, 2.0).square().sum()]
# as they are, a slice that is read in place, columns that are copied
VIEWS = [lambda x: x, lambda x: torch.cat([x, x], 1)[:, 5:], lambda x: torch.cat([x, x], 1)[:, ::2]]


def penalty(f, x):
    leaf = x.clone().requires_grad_(True)
    loss = f(leaf)
    first, = torch.autograd.grad(loss, leaf, create_graph=True)
    return torch.autograd.grad(loss + first.square().sum(), leaf)


ASKED = [functional.hessian, lambda f, x: functional.hvp(f, x, x), lambda f, x: functional.vhp(f, x, x),
         lambda f, x: functional.jvp(f, x, x), penalty]


@pytest.mark.parametrize("asked", ASKED)
@pytest.mark.parametrize("view", VIEWS)
@pytest.mark.parametrize("loss", LOSSES)
def test_refused(loss, view, asked):
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        asked(lambda t: loss(view(t)), torch.randn(3, 5))


@pytest.mark.parametrize("loss", LOSSES)
def test_the_first_derivative_is_given_under_create_graph(loss):
    x = torch.randn(3, 5).requires_grad_(True)
    first, = torch.autograd.grad(loss(x), x, create_graph=True)
    assert first.shape == x.shape
    assert functional.jacobian(loss, x.detach()).shape == x.shape


def test_the_embedding_is_linear():
    """Its gradient depends on what arrives from above alone: none arrives here that depends on the weight."""
    assert (functional.hessian(lambda w: mec.scaled_embedding(TOKENS, w, 2.0).sum(), torch.randn(3, 5)) == 0).all()

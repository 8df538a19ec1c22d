"""How the operators over a vocabulary stand in autograd: refused second
derivatives, deterministic mode, gradients that are not asked for, leaves with
strides, and losses added to one another."""
import pytest
import torch

import memoryefficientclip_amd as mec
import vocab_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def inputs(seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(6, 900, generator=g)
    tok = torch.randint(0, 900, (6,), generator=g)
    tt = torch.randint(0, 900, (6, 4), generator=g)
    tz = torch.randn(6, 4, generator=g)
    return x, tok, tt, tz


def losses(x, tok, tt, tz):
    return [mec.token_log_probs(x, tok).log_probs.sum(), mec.TopKDistillationLoss()(x, tt, tz),
            mec.TopKDistillationLoss(reduction="none")(x, tt, tz).sum(), mec.scaled_embedding(tok % 6, x).square().sum()]


def test_second_derivatives_are_refused():
    x, tok, tt, tz = (v.to(DEV) for v in inputs())
    for i in range(4):
        leaf = x.clone().requires_grad_(True)
        first, = torch.autograd.grad(losses(leaf, tok, tt, tz)[i], leaf, create_graph=True)
        assert torch.isfinite(first).all()
        with pytest.raises(RuntimeError, match="differentiate"):
            first.square().sum().backward()


def test_deterministic_mode_changes_nothing():
    x, tok, tt, tz = (v.to(DEV) for v in inputs(1))
    got = []
    for on in (False, True):
        torch.use_deterministic_algorithms(on)
        try:
            leaf = x.clone().requires_grad_(True)
            r = losses(leaf, tok, tt, tz)
            sum(r).backward()
            got.append([*(v.detach() for v in r), leaf.grad])
        finally:
            torch.use_deterministic_algorithms(False)
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_losses_on_the_same_logits_add_up():
    """One leaf, two losses, as in a step that distils and learns from the tokens."""
    x, tok, tt, tz = inputs(2)
    leaf = x.to(DEV).requires_grad_(True)
    loss = mec.TopKDistillationLoss(reduction="sum")(leaf, tt.to(DEV), tz.to(DEV))
    loss = loss - mec.token_log_probs(leaf, tok.to(DEV)).log_probs.sum()
    loss.backward()
    rows, _, dx = ref.distill(x, tt, tz)
    lp, _, _, _ = ref.token_scores(x, tok, 0)
    want = dx - ref.token_scores_grad(x, tok, torch.ones(6), torch.zeros(6))
    tol = ref.score_tolerance(x, 1.0)
    ref.assert_close("loss", loss, rows.sum() - lp.sum(), torch.float32, 12 * 3 * tol)
    ref.assert_close("dx", leaf.grad, want, torch.float32, 4 * tol)


def test_strided_and_frozen_leaves():
    x, tok, tt, tz = inputs(3)
    wide = torch.zeros(6, 1000, device=DEV)
    wide[:, 50:950] = x.to(DEV)
    leaf = wide[:, 50:950].detach().requires_grad_(True)
    assert leaf.stride(0) == 1000
    mec.TopKDistillationLoss(reduction="sum")(leaf, tt.to(DEV), tz.to(DEV)).backward()
    _, _, dx = ref.distill(x, tt, tz)
    ref.assert_close("dx", leaf.grad, dx, torch.float32, 2 * ref.score_tolerance(x, 1.0))
    # frozen inputs, and a teacher that would like a gradient and gets none
    z = tz.to(DEV).requires_grad_(True)
    assert not mec.TopKDistillationLoss()(x.to(DEV), tt.to(DEV), z).requires_grad
    loss = mec.TopKDistillationLoss()(leaf, tt.to(DEV), z)
    loss.backward()
    assert z.grad is None
    r = mec.token_log_probs(leaf, tok.to(DEV), top_k=3)
    assert r.log_probs.requires_grad and r.entropy.requires_grad and not r.top_log_probs.requires_grad


def test_logits_changed_before_the_backward_are_noticed():
    x, tok, tt, tz = (v.to(DEV) for v in inputs(4))
    for i in range(3):
        base = x.clone().requires_grad_(True)
        logits = base * 1.0
        loss = losses(logits, tok, tt, tz)[i]
        logits.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()

"""The entropy does not depend on the tokens: its gradient is its own also where a token
lies outside the vocabulary, whose log probability is NaN."""
import pytest
import torch

import memoryefficientclip_amd as mec
import vocab_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("vocab", [1, 70, 5001, 70000])
def test_gradient_of_the_entropy(vocab, dtype):
    g = torch.Generator().manual_seed(vocab)
    x = (2.0 * torch.randn(6, vocab, generator=g)).to(dtype)
    tokens = torch.tensor([vocab, -1, -100, 0, -(1 << 40), vocab - 1])
    inside = torch.where(tokens == -100, -100, tokens.clamp(0, vocab - 1))
    gh = torch.tensor([0.5, -1.0, 2.0, 1.0, -0.25, 3.0])
    want = ref.token_scores_grad(x, inside, torch.zeros(6), gh)
    # p (log p + H) carries the score's error at the size of p, the entropy's once more; |g| <= 3
    tol = 3 * 3 * ref.score_tolerance(x, 1.0) * max(1.0, float(torch.log(torch.tensor(float(vocab)))))
    leaf = x.to(DEV).requires_grad_(True)
    r = mec.token_log_probs(leaf, tokens.to(DEV))
    dx, = torch.autograd.grad(r.entropy, leaf, gh.to(DEV), retain_graph=True)
    ref.assert_close("entropy alone", dx, want, dtype, tol)
    # log probabilities that are left out of the loss as torch.where leaves them out
    used = torch.tensor([False, False, True, True, False, True])
    lp = torch.where(used.to(DEV), r.log_probs, 0.0)
    dx, = torch.autograd.grad(lp.sum() + (r.entropy * gh.to(DEV)).sum(), leaf, retain_graph=True)
    want = ref.token_scores_grad(x, inside, used.float(), gh)
    ref.assert_close("log probabilities left out", dx, want, dtype, 2 * tol)
    # one that is asked for is NaN, and its row alone
    dx, = torch.autograd.grad(r.log_probs[1] + r.entropy.sum(), leaf)
    assert torch.isnan(dx[1]).all() and torch.isfinite(dx[[0, 2, 3, 4, 5]]).all()

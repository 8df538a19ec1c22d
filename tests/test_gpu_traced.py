"""Functions recorded by torch.jit.trace give what the operators give, on inputs other
than they were traced with, with and without a gradient."""
import pytest
import torch

import memoryefficientclip_amd as mec

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning"),
              pytest.mark.filterwarnings("ignore::DeprecationWarning")]
DEV = "cuda:0"


def inputs(rows, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g).to(DEV), torch.randint(0, vocab, (rows,), generator=g).to(DEV),
            torch.randint(0, vocab, (rows, 4), generator=g).to(DEV), torch.randn(rows, 4, generator=g).to(DEV))


def scores(x, tok, tt, tz):
    r = mec.token_log_probs(x, tok, top_k=3, temperature=0.7)
    return r.log_probs, r.entropy, r.top_tokens, r.top_log_probs


OPERATORS = [scores, lambda x, tok, tt, tz: (mec.TopKDistillationLoss(2.0)(x, tt, tz),),
             lambda x, tok, tt, tz: (mec.scaled_embedding(tok % x.shape[0], x, 1.5),)]


@pytest.mark.parametrize("wanted", [False, True])
@pytest.mark.parametrize("op", OPERATORS)
def test_traced(op, wanted):
    x, *others = inputs(6, 900, 0)
    traced = torch.jit.trace(op, (x.requires_grad_(wanted), *others))
    for seed, rows, vocab in ((1, 6, 900), (2, 11, 50001)):
        x, *others = inputs(rows, vocab, seed)
        with torch.no_grad():
            assert all(torch.equal(a, b) for a, b in zip(traced(x, *others), op(x, *others), strict=True))
        grads = []
        for f in (traced, op):
            leaf = x.clone().requires_grad_(True)
            sum(r.sum() for r in f(leaf, *others) if r.requires_grad).backward()
            grads.append(leaf.grad)
        assert torch.equal(*grads)

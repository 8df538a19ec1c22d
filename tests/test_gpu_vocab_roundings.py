"""Gradients in 16 bits are rounded once: those that the distillation's forward makes and
those that its backward makes anew.  And the embedding's gradient just past the tiles that
one launch of its sort looks through."""
import pytest
import torch

import memoryefficientclip_amd as mec
import vocab_reference as ref
from test_gpu_embedding import check as check_embedding
from test_gpu_embedding import make as make_embedding

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("vocab", [48, 300])
def test_the_distillation_s_gradient_is_rounded_once(vocab, dtype):
    rows, factor = 64, 0.7  # (not a power of two: times it, what was rounded is rounded again)
    g = torch.Generator().manual_seed(vocab)
    x = (2.0 * torch.randn(rows, vocab, generator=g)).to(dtype)
    tok = torch.stack([torch.randperm(vocab, generator=g)[:6] for _ in range(rows)])
    z = torch.randn(rows, 6, generator=g)
    _, _, grad = ref.distill(x, tok, z)
    half = torch.finfo(dtype).eps / 2  # of a unit in the last place, at the value's size or below it
    # p and q each carry the score's absolute error as a relative one, at most 1 in size
    atol = 2 * ref.score_tolerance(x, 1.0) + ref.ROUNDING[dtype][1]

    def within(got, want):
        return (got.cpu().double() - want).abs() <= half * want.abs() + atol

    twice = (grad.to(dtype).float() * factor).to(dtype)
    assert not within(twice, grad * factor).all()  # the bound tells the two apart
    loss = mec.TopKDistillationLoss(reduction="sum")
    for go in (1.0, factor):
        leaf = x.to(DEV).requires_grad_(True)
        loss(leaf, tok.to(DEV), z.to(DEV)).backward(torch.tensor(go, device=DEV))
        # (0.7 in fp32)
        assert within(leaf.grad, grad * float(torch.tensor(go))).all()


def test_one_tile_more_than_a_launch_looks_through():
    check_embedding(*make_embedding(524289, 5000, 8, torch.bfloat16, seed=12))

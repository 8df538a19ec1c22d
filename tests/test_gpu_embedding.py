"""Scaled token embedding on the GPU: the lookup bit for bit, the gradient
against the sum in 64 bits at sizes around the kernels' tiles, with tokens that
occur once, often and always."""
import math

import pytest
import torch

import memoryefficientclip_amd as mec
import vocab_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(n, vocab, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed * 1000003 + n * 131 + vocab * 7 + d)
    w = torch.randn(vocab, d, generator=g).to(dtype)
    tok = torch.randint(0, vocab, (n,), generator=g)
    dy = torch.randn(n, d, generator=g).to(dtype)
    return tok, w, dy


def check(tok, w, dy, scale=1.7, padding_idx=None, gpu_tokens=None, gpu_dy=None):
    leaf = w.to(DEV).requires_grad_(True)
    y = mec.scaled_embedding(tok.to(DEV) if gpu_tokens is None else gpu_tokens, leaf, scale, padding_idx)
    ok = (tok >= 0) & (tok < w.shape[0])
    want = (w[tok.clamp(0, w.shape[0] - 1)].float() * torch.tensor(scale, dtype=torch.float32)).to(w.dtype)
    want[~ok] = math.nan
    assert torch.equal(torch.isnan(y.cpu()), torch.isnan(want))
    assert torch.equal(y.cpu()[ok], want[ok])
    y.backward(dy.to(DEV) if gpu_dy is None else gpu_dy)
    grad = ref.embedding_grad(tok, dy, w.shape[0], scale, padding_idx)
    # sums of c rows in 32 bits, in runs and trees: at most sqrt-like growth, bounded here by
    # (64 + log2 c) roundings of the sum of the sizes
    count = torch.bincount(tok[ok].reshape(-1), minlength=w.shape[0]).double()[:, None]
    size = ref.embedding_grad(tok, dy.abs(), w.shape[0], abs(scale))
    atol = 2.0 ** -24 * (64 + torch.log2(count.clamp_min(1))) * size
    rel, tiny = ref.ROUNDING[w.dtype]
    got = leaf.grad.cpu().double()
    assert leaf.grad.dtype == w.dtype and got.shape == grad.shape
    assert ((got - grad).abs() <= atol + 2 * rel * grad.abs() + tiny).all()
    assert (got[count[:, 0] == 0] == 0).all()
    return leaf.grad


SIZES = [(1, 1, 1), (1, 1000, 64), (2, 3, 7), (63, 10, 65), (64, 64, 128), (65, 5000, 8), (257, 300, 513),
         (1000, 100, 96), (1025, 2, 40), (4096, 9000, 48), (4097, 513, 33), (8193, 70000, 24), (20000, 1, 16),
         (30000, 30000, 64), (3000, 300000, 8), (70000, 4000, 40), (300, 600, 2050), (5000, 20, 1536),
         (20000, 400000, 4), (9000, 1, 3), (511, 3, 40), (512, 1, 600), (513, 2, 1030), (512, 90, 136)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,vocab,d", SIZES)
def test_sizes(n, vocab, d, dtype):
    check(*make(n, vocab, d, dtype))


@pytest.mark.parametrize("n,vocab,d", [(524288, 5000, 8), (600001, 70000, 12), (700000, 3, 4)])
def test_many_tokens(n, vocab, d):
    """More than 128 tiles of the sort."""
    check(*make(n, vocab, d, torch.bfloat16, seed=10))


@pytest.mark.parametrize("n", [17, 40, 70, 300, 2000])
def test_runs_of_every_length(n):
    """Token v occurs v times, in a random order: runs that end inside and at the
    ends of pieces and blocks, at every offset."""
    lengths = torch.arange(n % 7, 400)
    tok = torch.repeat_interleave(lengths, lengths)
    g = torch.Generator().manual_seed(n)
    tok = tok[torch.randperm(tok.numel(), generator=g)][: n * 40]
    _, w, dy = make(tok.numel(), 400, 20, torch.float32, seed=11)
    check(tok, w, dy)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("n", [500, 5000, 60000])
def test_tokens_that_occur_often(n, dtype):
    tok, w, dy = make(n, 2000, 72, dtype, seed=1)
    g = torch.Generator().manual_seed(2)
    tok[torch.rand(n, generator=g) < 0.5] = 1999     # half of all, the last token
    tok[::3] = 0                                     # a third, the first one
    tok[n // 2: n // 2 + 130] = 77                   # a run of neighbours
    check(tok, w, dy)
    check(tok, w, dy, padding_idx=1999)
    check(tok, w, dy, padding_idx=0)
    tok[:] = 5                                       # nothing else
    check(tok, w, dy)
    assert (check(tok, w, dy, padding_idx=5) == 0).all()


@pytest.mark.parametrize("n", [40, 9000])
def test_tokens_outside_the_vocabulary(n):
    tok, w, dy = make(n, 50, 24, torch.float32, seed=3)
    tok[3], tok[7], tok[20] = 50, -1, -(1 << 40)
    tok[30] = 1 << 40
    check(tok, w, dy)
    tok[:] = 51
    assert (check(tok, w, dy) == 0).all()


def test_padding_row_is_looked_up():
    tok, w, _ = make(10, 6, 8, torch.float32)
    tok[4] = 2
    y = mec.scaled_embedding(tok.to(DEV), w.to(DEV), 2.0, padding_idx=2)
    assert torch.equal(y[4].cpu(), 2.0 * w[2])
    y = mec.scaled_embedding(tok.to(DEV), w.to(DEV), 2.0, padding_idx=-4)
    assert torch.equal(y[4].cpu(), 2.0 * w[2])


def test_layouts():
    tok, w, _ = make(60, 40, 100, torch.bfloat16, seed=4)
    g = torch.Generator().manual_seed(5)
    dy = torch.randn(5, 12, 100, generator=g).to(torch.bfloat16)
    tok = tok.reshape(5, 12)
    check(tok, w, dy)
    check(tok.int(), w, dy)
    # tokens and gradients with strides
    wide = torch.zeros(5, 24, dtype=torch.int64, device=DEV)
    wide[:, ::2] = tok.to(DEV)
    gdy = torch.zeros(5, 12, 130, dtype=torch.bfloat16, device=DEV)
    gdy[..., 7:107] = dy.to(DEV)
    check(tok, w, dy, gpu_tokens=wide[:, ::2], gpu_dy=gdy[..., 7:107])
    check(tok, w, dy, gpu_dy=dy.to(DEV).transpose(0, 1).contiguous().transpose(0, 1))
    ones = torch.ones((), dtype=torch.bfloat16, device=DEV).expand(5, 12, 100)
    check(tok, w, torch.ones(5, 12, 100, dtype=torch.bfloat16), gpu_dy=ones)
    # a weight of strided rows
    big = torch.zeros(40, 150, dtype=torch.bfloat16, device=DEV)
    big[:, 3:103] = w.to(DEV)
    y = mec.scaled_embedding(tok.to(DEV), big[:, 3:103], 1.0)
    assert torch.equal(y.cpu(), w[tok])
    y = mec.scaled_embedding(tok.to(DEV)[0, 0], w.to(DEV))
    assert torch.equal(y.cpu(), w[tok[0, 0]])


def test_non_finite_gradients_stay_in_their_row():
    tok, w, dy = make(5000, 300, 16, torch.float32, seed=6)
    dy[17, 3] = math.nan
    dy[4000, 5] = math.inf
    leaf = w.to(DEV).requires_grad_(True)
    mec.scaled_embedding(tok.to(DEV), leaf, 1.0).backward(dy.to(DEV))
    got = leaf.grad.cpu()
    assert torch.isnan(got[tok[17], 3]) and not torch.isfinite(got[tok[4000], 5])
    bad = (~torch.isfinite(got)).nonzero().tolist()
    assert sorted(bad) == sorted([[int(tok[17]), 3], [int(tok[4000]), 5]])


def test_gradient_against_differences():
    """Linear in the weight: the difference of <y, g> for a step of one entry is the gradient."""
    tok, w, dy = make(50, 4, 3, torch.float32, seed=7)
    dw = check(tok, w, dy, scale=0.5).cpu().double()
    for v in range(4):
        for j in range(3):
            diff = 0.0
            for sign in (1, -1):
                u = w.clone()
                u[v, j] += sign * 0.5
                y = mec.scaled_embedding(tok.to(DEV), u.to(DEV), 0.5).cpu().double()
                diff += sign * (y * dy.double()).sum().item()
            assert abs(diff - dw[v, j].item()) <= 1e-4


def test_results_repeat_bit_for_bit():
    tok, w, dy = make(50000, 3000, 40, torch.bfloat16, seed=8)
    tok[::2] = 7
    a = check(tok, w, dy)
    for _ in range(2):
        assert torch.equal(a, check(tok, w, dy))


def test_module():
    m = mec.ScaledTokenEmbedding(30, 16, padding_idx=3, device=DEV)
    assert m.scale == 4.0 and (m.weight[3] == 0).all() and list(m.state_dict()) == ["weight"]
    tok = torch.randint(0, 30, (4, 5), device=DEV)
    y = m(tok)
    assert torch.equal(y, 4.0 * m.weight[tok])
    y.sum().backward()
    want = 4.0 * torch.bincount(tok.reshape(-1), minlength=30).float()
    want[3] = 0
    assert torch.equal(m.weight.grad, want[:, None].expand(30, 16))


def test_no_tokens():
    w = torch.randn(6, 4, device=DEV, requires_grad=True)
    y = mec.scaled_embedding(torch.zeros(2, 0, dtype=torch.int64, device=DEV), w)
    assert y.shape == (2, 0, 4)
    y.sum().backward()
    assert (w.grad == 0).all()


def test_another_stream():
    tok, w, dy = make(9000, 700, 64, torch.bfloat16, seed=9)
    leaf, tg, dg = w.to(DEV).requires_grad_(True), tok.to(DEV), dy.to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        mec.scaled_embedding(tg, leaf, 1.7).backward(dg)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(leaf.grad, check(tok, w, dy))

"""Distillation from a teacher's top logits on the GPU against its definition in
64 bits: sizes, teachers with few, repeated or no entries, masks, reductions,
gradients against the formula and against differences, and the gradient that the
forward makes against the one that the backward makes."""
import math

import pytest
import torch

import memoryefficientclip_amd as mec
import vocab_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(rows, vocab, k, dtype, seed=0, repeated=False):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 131 + vocab * 7 + k)
    x = (3.0 * torch.randn(rows, vocab, generator=g)).to(dtype)
    if repeated or k > vocab:
        tok = torch.randint(0, vocab, (rows, k), generator=g)
    else:
        tok = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)])
    z = 2.0 * torch.randn(rows, k, generator=g)
    return x, tok, z


def run(x, tok, z, temperature=1.0, weight=1.0, reduction="mean", grad_output=None, leaf=None):
    leaf = (x.to(DEV) if leaf is None else leaf).detach().requires_grad_(True)
    loss = mec.TopKDistillationLoss(temperature, reduction, weight)(leaf, tok.to(DEV), z.to(DEV))
    assert loss.dtype == torch.float32
    if grad_output is None and reduction != "none":
        loss.backward()
    else:
        loss.backward(torch.as_tensor(grad_output, dtype=torch.float32).to(DEV).expand(loss.shape))
    return loss.detach(), leaf.grad


def check(x, tok, z, temperature=1.0, weight=1.0, reduction="mean", grad_output=None, leaf=None):
    loss, dx = run(x, tok, z, temperature, weight, reduction, grad_output, leaf)
    rows, some, grad = ref.distill(x.reshape(-1, x.shape[-1]), tok.reshape(-1, tok.shape[-1]),
                                   z.reshape(-1, z.shape[-1]), temperature, weight)
    tol = ref.score_tolerance(x, temperature) * abs(weight)
    g = torch.ones(()) if grad_output is None else torch.as_tensor(grad_output)
    if reduction == "none":
        ref.assert_close("loss", loss.reshape(-1), rows, torch.float32, tol * temperature ** 2 * 2)
        grad = grad * g.reshape(-1).double()[:, None] if g.dim() else grad * g.double()
        scale = float(g.abs().max())
    else:
        n = max(1, int(some.sum())) if reduction == "mean" else 1
        ref.assert_close("loss", loss, rows.sum() / n, torch.float32,
                         tol * temperature ** 2 * 2 * (1 if reduction == "mean" else max(1, int(some.sum()))))
        grad = grad * (g.double() / n)
        scale = float(g.abs()) / n
    # p and q carry about the score's absolute error as a relative one
    ref.assert_close("dx", dx.reshape(grad.shape), grad, x.dtype, 2 * tol * temperature * scale)
    return loss, dx


SIZES = [(1, 1, 1), (1, 2, 2), (3, 7, 3), (5, 63, 8), (4, 64, 64), (2, 65, 5), (7, 1000, 10), (2, 2048, 1),
         (3, 4097, 32), (2, 8192, 7), (2, 16385, 20), (3, 32001, 10), (2, 50001, 64), (2, 65536, 16), (1, 65544, 16),
         (1, 131072, 128), (300, 517, 10), (2, 200003, 64), (3, 700, 700), (2, 5000, 1024), (1, 524288, 9),
         (2, 70000, 1024), (1, 140001, 700), (2, 300001, 33)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,k", SIZES)
def test_sizes(rows, vocab, k, dtype):
    x, tok, z = make(rows, vocab, k, dtype)
    check(x, tok, z, temperature=2.0, weight=0.5)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions_and_grad_output(dtype, reduction):
    x, tok, z = make(37, 3001, 12, dtype, seed=1)
    for go in (1.0, 1024.0, 0.0, -0.37):
        check(x, tok, z, 1.5, 1.0, reduction, grad_output=go)
    if reduction == "none":
        check(x, tok, z, 1.5, 1.0, reduction, grad_output=torch.linspace(-2, 2, 37))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("vocab", [300, 5000, 70001])
def test_teachers_with_few_or_no_entries(dtype, vocab):
    x, tok, z = make(9, vocab, 6, dtype, seed=2)
    tok[0] = -1                          # padding
    tok[1, 2:] = -1
    z[2, 1] = -math.inf                  # an entry that the teacher rules out
    z[3] = -math.inf                     # all of them
    z[4, 0] = 200.0                      # one that takes everything
    tok[5, 3] = -7
    z[6] = torch.finfo(torch.float32).min
    for reduction in ("mean", "sum", "none"):
        loss, dx = check(x, tok, z, 2.0, reduction=reduction, grad_output=1.0)
        assert (dx[[0, 3]] == 0).all()
    tok[:] = -1
    loss, dx = check(x, tok, z)
    assert loss == 0 and (dx == 0).all()


@pytest.mark.parametrize("vocab", [5, 900, 33000])
def test_repeated_entries_add_up(vocab):
    x, tok, z = make(6, vocab, 40, torch.float32, seed=3, repeated=True)
    tok[0] = vocab - 1
    tok[1, ::2] = tok[1, 0]
    check(x, tok, z, 0.7)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [200, 5000, 70001])
def test_masked_students(dtype, vocab):
    x, tok, z = make(6, vocab, 8, dtype, seed=4)
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(1)
    keep = x.clone()
    for row, mask in ((0, -math.inf), (1, low)):
        x[row, torch.rand(vocab, generator=g) < 0.9] = mask
        x[row].scatter_(0, tok[row], keep[row].gather(0, tok[row]))
    x[2] = low
    check(x, tok, z, grad_output=1.0)
    # the teacher's tokens ruled out by the student: an infinite loss, and the gradient of the rest
    x[3, tok[3, 0]] = -math.inf
    x[4] = -math.inf
    loss, dx = run(x, tok, z, reduction="none", grad_output=1.0)
    rows, some, grad = ref.distill(x, tok, z)
    assert torch.isposinf(loss[[3, 4]]).all() and torch.isfinite(loss[[0, 1, 2, 5]]).all()
    assert (dx[4] == 0).all()
    ref.assert_close("dx", dx, grad, dtype, 2 * ref.score_tolerance(x, 1.0))


@pytest.mark.parametrize("offset", [3e4, -3e6])
@pytest.mark.parametrize("vocab", [300, 50001, 150000])
def test_common_offset(vocab, offset):
    x, tok, z = make(3, vocab, 12, torch.float32, seed=13)
    x = (x + offset).float()
    x[:, : vocab // 3] -= 40.0
    for go in (1.0, 2.0):
        check(x, tok, z + offset, 0.7, grad_output=go)


def test_nan_spreads_over_its_row_alone():
    x, tok, z = make(5, 2500, 8, torch.float32, seed=5)
    x[0, 7] = math.nan
    z[1, 2] = math.nan
    tok[2, 3] = 2500                     # past the vocabulary
    x[3, 100] = math.inf
    loss, dx = run(x, tok, z, reduction="none", grad_output=1.0)
    assert torch.isnan(loss[:4]).all() and torch.isfinite(loss[4])
    assert torch.isfinite(dx[4]).all() and torch.isnan(dx[[0, 2]]).all()
    loss, dx = run(x, tok, z)
    assert torch.isnan(loss) and torch.isfinite(dx[4]).all()


@pytest.mark.parametrize("vocab", [1000, 30000, 140000])
def test_the_forward_s_gradient_is_the_backward_s(vocab):
    """grad_output 1 takes the gradient made in the forward; 2 makes it anew: twice it, in every bit."""
    for dtype in (torch.float32, torch.bfloat16):
        x, tok, z = make(5, vocab, 10, dtype, seed=6)
        _, a = run(x, tok, z, 2.0)
        _, b = run(x, tok, z, 2.0, grad_output=2.0)
        torch.testing.assert_close(a * 2, b, rtol=2.0 ** -7 if dtype == torch.bfloat16 else 4e-6, atol=0)


def test_backward_twice():
    x, tok, z = make(4, 600, 5, torch.float32, seed=7)
    leaf = x.to(DEV).requires_grad_(True)
    loss = mec.TopKDistillationLoss()(leaf, tok.to(DEV), z.to(DEV))
    a, = torch.autograd.grad(loss, leaf, retain_graph=True)
    kept = a.clone()
    a.zero_()
    b, = torch.autograd.grad(loss, leaf, retain_graph=True)
    c, = torch.autograd.grad(loss * 3, leaf)
    torch.testing.assert_close(b, kept, rtol=1e-6, atol=1e-9)
    torch.testing.assert_close(c, kept * 3, rtol=1e-6, atol=1e-9)


def test_no_gradient_wanted():
    x, tok, z = make(4, 600, 5, torch.float32, seed=8)
    with torch.no_grad():
        loss = mec.TopKDistillationLoss(2.0)(x.to(DEV).requires_grad_(True), tok.to(DEV), z.to(DEV))
    rows, _, _ = ref.distill(x, tok, z, 2.0)
    ref.assert_close("loss", loss, rows.mean(), torch.float32, ref.score_tolerance(x, 2.0) * 8)
    assert not loss.requires_grad


def test_gradient_against_differences():
    """Central differences of the kernels' own loss, as for the log probabilities."""
    x, tok, z = make(3, 9, 4, torch.float32, seed=9)
    x = x / 3
    _, dx = run(x, tok, z, 1.4, reduction="none", grad_output=1.0)
    step = 2.0 ** -6
    for v in range(9):
        diff = 0.0
        for sign in (1, -1):
            y = x.clone()
            y[:, v] += sign * step
            loss = mec.TopKDistillationLoss(1.4, "none")(y.to(DEV), tok.to(DEV), z.to(DEV))
            diff = diff + sign * loss.cpu().double() / (2 * step)
        assert ((dx[:, v].cpu().double() - diff).abs() <= 1.4 * (step ** 2 / 3 + 2.0 ** -20 / step)).all()


@pytest.mark.parametrize("tz", DTYPES, ids=str)
def test_layouts_and_teacher_types(tz):
    g = torch.Generator().manual_seed(10)
    base = torch.randn(4, 7, 1001, generator=g)
    tok = torch.randint(0, 999, (4, 7, 6), generator=g)
    z = torch.randn(4, 7, 6, generator=g).to(tz)
    check(base, tok, z, leaf=base.to(DEV))
    check(base, tok.int(), z, leaf=base.to(DEV))
    for cut in (lambda t: t[:, :-1], lambda t: t[:, 1:], lambda t: t.transpose(0, 1), lambda t: t[1, 2:3]):
        leaf = base.to(DEV).requires_grad_(True)
        loss = mec.TopKDistillationLoss()(cut(leaf), cut(tok.to(DEV)), cut(z.to(DEV)))
        loss.backward()
        x = cut(base)
        rows, some, grad = ref.distill(x.reshape(-1, 1001), cut(tok).reshape(-1, 6), cut(z).reshape(-1, 6))
        full = torch.zeros(base.shape, dtype=torch.float64)
        cut(full).copy_(grad.reshape(x.shape) / rows.numel())
        ref.assert_close("loss", loss, rows.mean(), torch.float32, 2 * ref.score_tolerance(base, 1.0))
        ref.assert_close("dx", leaf.grad, full, torch.float32, 2 * ref.score_tolerance(base, 1.0))
    # column slices at every alignment
    for off in range(5):
        leaf = base.to(DEV)[..., off:off + 990]
        check(base[..., off:off + 990], tok % 990, z, leaf=leaf)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("vocab", [8191, 8192, 16384, 16385, 32768, 65535, 65536, 65537, 131071, 131072, 131073])
def test_full_segments_at_odd_addresses(dtype, vocab):
    g = torch.Generator().manual_seed(16)
    base = torch.randn(3 * (vocab + 1) + 8, generator=g).to(dtype)
    dev = base.to(DEV)
    tok = torch.randint(0, vocab, (3, 7), generator=g)
    tok[0, :2] = torch.tensor([0, vocab - 1])
    z = torch.randn(3, 7, generator=g)
    for off, ld in ((0, vocab), (1, vocab), (1, vocab + 1), (3, vocab + 1)):
        for go in (1.0, 2.0):
            check(base.as_strided((3, vocab), (ld, 1), off), tok, z, grad_output=go,
                  leaf=dev.as_strided((3, vocab), (ld, 1), off))


def test_gradient_past_32_bits():
    """A gradient of more than 2^32 elements (8.6 GB): all rows of the logits are one in memory."""
    rows, vocab = 66001, 65600
    x, tok, z = make(1, vocab, 5, torch.bfloat16, seed=18)
    leaf = x.to(DEV).expand(rows, vocab).detach().requires_grad_(True)
    tok_all, z_all = tok.to(DEV).repeat(rows, 1), z.to(DEV).repeat(rows, 1)
    tok_all[-1], z_all[-2] = -1, 0.0
    loss = mec.TopKDistillationLoss(reduction="sum")(leaf, tok_all, z_all)
    dx, = torch.autograd.grad(loss, leaf)
    one, _, grad = ref.distill(x, tok, z)
    other, _, grad0 = ref.distill(x, tok, z * 0)
    ref.assert_close("loss", loss, (one * (rows - 2) + other)[0], torch.float32, 2 * rows * ref.score_tolerance(x, 1.0))
    for r in (0, 65471, 65472, rows - 3):   # 2^32 / vocab lies between
        ref.assert_close("dx", dx[r], grad[0], torch.bfloat16, 2 * ref.score_tolerance(x, 1.0))
    ref.assert_close("dx", dx[-2], grad0[0], torch.bfloat16, 2 * ref.score_tolerance(x, 1.0))
    assert (dx[-1] == 0).all()


def test_many_rows_and_repeats_bit_for_bit():
    x, tok, z = make(2000, 777, 9, torch.bfloat16, seed=11)
    tok[::3] = -1
    a = check(x, tok, z, 2.0)
    for _ in range(2):
        b = run(x, tok, z, 2.0)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_student_from_a_scored_teacher():
    """token_log_probs gives what the loss takes, padding included: a student that
    is its teacher has the loss of the tail that the top logits leave out."""
    x, _, _ = make(6, 4000, 1, torch.float32, seed=12)
    tokens = torch.tensor([1, -100, 3, 4, -100, 6]).to(DEV)
    t = mec.token_log_probs(x.to(DEV), tokens, top_k=16)
    loss = mec.TopKDistillationLoss(reduction="none")(x.to(DEV), t.top_tokens, t.top_log_probs)
    tail = torch.logsumexp(t.top_log_probs.double(), 1)
    want = torch.where(tokens == -100, 0.0, -tail)
    assert (loss.double() - want).abs().max().item() <= 2 * ref.score_tolerance(x, 1.0)


def test_no_positions():
    x = torch.zeros(2, 0, 9, device=DEV, requires_grad=True)
    tok, z = torch.zeros(2, 0, 3, dtype=torch.int64, device=DEV), torch.zeros(2, 0, 3, device=DEV)
    for reduction, shape in (("mean", ()), ("sum", ()), ("none", (2, 0))):
        loss = mec.TopKDistillationLoss(reduction=reduction)(x, tok, z)
        assert loss.shape == shape and loss.sum() == 0
        loss.sum().backward()

"""Token log probabilities, entropy and top alternatives on the GPU against
their definition in 64 bits: sizes around the kernels' vectors and workgroups,
masks, ties, infinities and NaN, strides, and the gradient against its formula
and against differences."""
import math

import pytest
import torch

import memoryefficientclip_amd as mec
import vocab_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(rows, vocab, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 131 + vocab)
    x = (scale * torch.randn(rows, vocab, generator=g)).to(dtype)
    tok = torch.randint(0, vocab, (rows,), generator=g)
    return x, tok, g


def check(x, tok, k, temperature=1.0, atol=None, gpu_logits=None, gpu_tokens=None):
    """x [R, V] and tok [R] on the CPU; gpu_*: the same values laid out otherwise."""
    xg = x.to(DEV) if gpu_logits is None else gpu_logits
    tg = tok.to(DEV) if gpu_tokens is None else gpu_tokens
    r = mec.token_log_probs(xg, tg, top_k=k, temperature=temperature)
    lp, h, tt, tlp = ref.token_scores(x, tok, k, temperature)
    atol = ref.score_tolerance(x, temperature) if atol is None else atol
    ref.assert_close("log_probs", r.log_probs.reshape(-1), lp, torch.float32, atol)
    ref.assert_close("entropy", r.entropy.reshape(-1), h, torch.float32, atol)
    if k == 0:
        assert r.top_tokens is None and r.top_log_probs is None
    else:
        assert torch.equal(r.top_tokens.reshape(-1, k).cpu(), tt)
        ref.assert_close("top_log_probs", r.top_log_probs.reshape(-1, k), tlp, torch.float32, atol)
    return r


SIZES = [(1, 1), (1, 2), (3, 7), (5, 63), (4, 64), (2, 65), (3, 255), (7, 1000), (2, 2048), (3, 2051), (3, 4097),
         (2, 8192), (2, 8200), (2, 16384), (2, 16385), (3, 32001), (2, 50001), (1, 131072), (300, 517), (70, 9000),
         (2, 524288)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_sizes(rows, vocab, dtype):
    x, tok, _ = make(rows, vocab, dtype)
    for k in sorted({0, 1, min(5, vocab), min(20, vocab), min(128, vocab)}):
        check(x, tok, k, temperature=0.8)


@pytest.mark.parametrize("rows", [600, 5000])
def test_many_rows(rows):
    x, tok, g = make(rows, 1531, torch.bfloat16)
    tok[torch.rand(rows, generator=g) < 0.3] = -100
    check(x, tok, 7, temperature=2.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [130, 5000, 40000])
def test_masks(dtype, vocab):
    x, tok, g = make(8, vocab, dtype, seed=1)
    low = torch.finfo(dtype).min
    x[0, torch.rand(vocab, generator=g) < 0.95] = -math.inf
    x[1] = -math.inf                       # nothing can occur
    x[2] = -math.inf
    x[2, vocab - 3] = 1.0                  # one token can
    x[3, torch.rand(vocab, generator=g) < 0.95] = low
    x[4] = low                             # all equal, at the type's lowest value
    x[5] = low
    x[5, 3] = 0.0
    x[6, : vocab // 2] = -math.inf         # a whole stretch
    tok[0] = int(x[0].argmax())
    tok[7] = -100
    for k in (1, 20, 128):
        for temperature in (1.0, 0.25):
            check(x, tok, k, temperature)


def test_log_probability_of_a_masked_token():
    x, tok, _ = make(2, 300, torch.float32)
    x[0, 5] = -math.inf
    tok[0] = 5
    x[1] = -math.inf
    r = check(x, tok, 0)
    assert torch.isneginf(r.log_probs).all() and r.entropy[1] == 0.0


@pytest.mark.parametrize("vocab", [100, 5000, 70000])
def test_nan_and_infinity_spread_over_their_row_alone(vocab):
    x, tok, _ = make(6, vocab, torch.float32, seed=2)
    x[0, vocab // 3] = math.nan
    x[2, vocab // 2] = math.inf
    x[4] = math.nan
    r = mec.token_log_probs(x.to(DEV), tok.to(DEV), top_k=3)
    for row in (0, 2, 4):
        assert torch.isnan(r.log_probs[row]) and torch.isnan(r.entropy[row])
    assert r.top_tokens[0, 0].item() == vocab // 3 and r.top_tokens[2, 0].item() == vocab // 2
    assert r.top_tokens[4].tolist() == [0, 1, 2]
    keep = [1, 3, 5]
    lp, h, tt, tlp = ref.token_scores(x[keep], tok[keep], 3)
    atol = ref.score_tolerance(x[keep], 1.0)
    ref.assert_close("log_probs", r.log_probs[keep], lp, torch.float32, atol)
    ref.assert_close("entropy", r.entropy[keep], h, torch.float32, atol)
    assert torch.equal(r.top_tokens[keep].cpu(), tt)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [129, 4096, 5003, 66000])
def test_ties_go_to_the_lower_token(dtype, vocab):
    x, tok, g = make(9, vocab, dtype, seed=3)
    x[0] = 0.0                                             # all equal
    x[1] = torch.randint(0, 3, (vocab,), generator=g).to(dtype)
    x[2] = torch.arange(vocab).div(4, rounding_mode="floor").clamp(max=2000).to(dtype) / 64
    x[3] = -torch.arange(vocab).clamp(max=2000).to(dtype) / 64   # falling: the first tokens lead
    x[4] = torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0).to(dtype)
    x[5] = 0.0
    x[5, vocab - 1] = 1.0
    x[6] = -1.0
    x[6, ::8] = 0.0
    x[7] = torch.arange(vocab).clamp(max=2000).to(dtype) / 64
    for k in (1, 8, 64, 128):
        check(x, tok, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_a_few_columns_hold_all_large_values(dtype):
    """The largest values sit where one thread after another would find them all."""
    vocab = 65536
    x, tok, g = make(4, vocab, dtype, seed=4)
    for row, step in enumerate((1024, 2048, 4096, 8192)):
        x[row, ::step] += 40.0
        for i in range(1, 8):
            x[row, i::step] += 35.0
    for k in (20, 128):
        check(x, tok, k)


def test_large_values():
    """Values near the ends of fp32: differences and scaled references overflow."""
    x = torch.tensor([[3e38, 2.9e38, -3e38, 0.0], [-3e38, -3.2e38, -3.3e38, -3.4e38], [1e30, 1e30, 1e30, -1e30],
                      [-3.4028235e38] * 4, [1e4, 1e4 + 1, 1e4 - 2, -1e4]])
    tok = torch.tensor([0, 0, 1, 2, 1])
    for temperature in (1.0, 0.1, 10.0):
        check(x, tok, 4, temperature, atol=3e-6 * max(1.0, 3.0 / temperature))


@pytest.mark.parametrize("offset", [3e4, -3e4, 3e6, -3e7])
@pytest.mark.parametrize("vocab", [300, 50001, 131072])
def test_common_offset(vocab, offset):
    """Logits far from zero: their differences are exact in fp32, and so must the
    results be, though scaled logits are rounded by far more than the tolerance."""
    x, tok, g = make(3, vocab, torch.float32, seed=14)
    x = (x + offset).float()
    x[:, : vocab // 3] -= 40.0     # segments with other maxima
    for temperature in (1.0, 0.7):
        check(x, tok, 5, temperature)
    gl, gh = torch.randn(3, generator=g), torch.randn(3, generator=g)
    want = ref.token_scores_grad(x, tok, gl, gh, 0.7)
    atol = ref.score_tolerance(x, 0.7) / 0.7 * (gl.abs().max() + gh.abs().max() * (1 + ref.spread(x, 0.7))).item()
    ref.assert_close("dx", gradient(x, tok, gl, gh, 0.7), want, torch.float32, atol)


def test_layouts():
    g = torch.Generator().manual_seed(5)
    base = torch.randn(4, 9, 1003, generator=g)
    tok = torch.randint(0, 1003, (4, 9), generator=g)
    big = base.to(DEV)
    # rows next to each other, slices along the positions (the usual shift by one), column slices
    check(base.reshape(36, 1003), tok.reshape(-1), 5, gpu_logits=big, gpu_tokens=tok.to(DEV))
    for a, b in ((slice(0, 8), slice(1, 9)), (slice(1, 9), slice(0, 8))):
        x = big[:, a]
        assert not x.is_contiguous()
        check(base[:, a].reshape(32, 1003), tok[:, b].reshape(-1), 5, gpu_logits=x, gpu_tokens=tok[:, b].to(DEV))
    check(base[..., 3:900].reshape(36, 897), tok.reshape(-1) % 897, 5, gpu_logits=big[..., 3:900],
          gpu_tokens=(tok % 897).to(DEV))
    # positions in front of texts, every other text, column stride 2, one row for all
    check(base.transpose(0, 1).reshape(36, 1003), tok.t().reshape(-1), 5, gpu_logits=big.transpose(0, 1),
          gpu_tokens=tok.t().to(DEV))
    check(base[::2].reshape(18, 1003), tok[::2].reshape(-1), 5, gpu_logits=big[::2], gpu_tokens=tok[::2].to(DEV))
    check(base[..., ::2].reshape(36, 502), tok.reshape(-1) % 502, 5, gpu_logits=big[..., ::2],
          gpu_tokens=(tok % 502).to(DEV))
    check(base[0, :1].expand(9, -1), tok[0], 5, gpu_logits=big[0, :1].expand(9, -1), gpu_tokens=tok[0].to(DEV))
    # one row, no leading dimension; int32 tokens; four dimensions
    check(base[0, :1], tok[0, :1], 5, gpu_logits=big[0, 0], gpu_tokens=tok[0, 0].to(DEV))
    check(base.reshape(36, 1003), tok.reshape(-1), 5, gpu_logits=big, gpu_tokens=tok.to(DEV).int())
    x4 = big.reshape(2, 2, 9, 1003)[:, :, 1:, :]
    check(base[:, 1:].reshape(32, 1003), tok[:, 1:].reshape(-1), 5, gpu_logits=x4,
          gpu_tokens=tok.reshape(2, 2, 9)[..., 1:].to(DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_every_alignment(dtype):
    g = torch.Generator().manual_seed(6)
    base = torch.randn(40000, generator=g).to(dtype)
    dev = base.to(DEV)
    for off in range(9):
        for vocab, ld in ((1001, 1001), (1000, 1007), (9000, 9001)):
            x = base.as_strided((3, vocab), (ld, 1), off)
            check(x, torch.tensor([0, vocab - 1, 17]), 9, gpu_logits=dev.as_strided((3, vocab), (ld, 1), off))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("vocab", [2047, 2048, 2049, 16383, 16384, 16385, 32767, 32768, 65535, 65536, 65537, 131072])
def test_full_segments_at_odd_addresses(dtype, vocab):
    """Rows that fill their segments and begin off the boundaries of the vectors."""
    g = torch.Generator().manual_seed(15)
    base = torch.randn(3 * (vocab + 1) + 8, generator=g).to(dtype)
    dev = base.to(DEV)
    tok = torch.tensor([0, vocab - 1, vocab // 2])
    gl, gh = torch.ones(3), torch.ones(3)
    for off, ld in ((0, vocab), (1, vocab), (1, vocab + 1), (3, vocab + 1)):
        x = base.as_strided((3, vocab), (ld, 1), off)
        leaf = dev.as_strided((3, vocab), (ld, 1), off)
        check(x, tok, 6, gpu_logits=leaf)
        want = ref.token_scores_grad(x, tok, gl, gh)
        ref.assert_close("dx", gradient(x, tok, gl, gh, leaf=leaf), want, dtype,
                         ref.score_tolerance(x, 1.0) * (2 + ref.spread(x, 1.0)))


def test_tokens_outside_the_vocabulary():
    x, tok, _ = make(5, 70, torch.float32)
    tok[1], tok[2], tok[3] = 70, -1, -100
    r = mec.token_log_probs(x.to(DEV), tok.to(DEV), top_k=2)
    assert torch.isnan(r.log_probs[[1, 2]]).all() and torch.isfinite(r.entropy).all()
    assert r.log_probs[3] == 0 and r.entropy[3] == 0 and r.top_tokens[3].tolist() == [-1, -1]
    r = mec.token_log_probs(x.to(DEV), tok.to(DEV), top_k=2, ignore_index=70)
    assert r.log_probs[1] == 0 and torch.isnan(r.log_probs[[2, 3]]).all()


def test_past_32_bits():
    """Rows whose elements lie beyond 2^32: 9 of them over 4.3e9 elements, of an allocation of 8.6 GB."""
    ld = (1 << 32) // 8 + 7
    flat = torch.zeros(8 * ld + 1000, dtype=torch.bfloat16, device=DEV)
    x = flat.as_strided((9, 1000), (ld, 1))
    vals, tok, _ = make(9, 1000, torch.bfloat16, seed=7)
    x.copy_(vals.to(DEV))
    check(vals, tok, 4, gpu_logits=x)
    leaf = x.detach().requires_grad_(True)
    mec.token_log_probs(leaf, tok.to(DEV)).log_probs.sum().backward()
    want = ref.token_scores_grad(vals, tok, torch.ones(9), torch.zeros(9))
    ref.assert_close("dx", leaf.grad, want, torch.bfloat16, 1e-6)


def test_gradient_past_32_bits():
    """A gradient of more than 2^32 elements (8.6 GB): all rows of the logits are one in memory."""
    rows, vocab = 66001, 65600
    x, tok, _ = make(1, vocab, torch.bfloat16, seed=18)
    leaf = x.to(DEV).expand(rows, vocab).detach().requires_grad_(True)
    tok_all = tok.to(DEV).repeat(rows)
    tok_all[-1] = -100
    r = mec.token_log_probs(leaf, tok_all)
    dx, = torch.autograd.grad(r.log_probs, leaf, torch.ones(rows, device=DEV))
    want = ref.token_scores_grad(x, tok, torch.ones(1), torch.zeros(1))[0]
    for row in (0, 65471, 65472, rows - 2):   # 2^32 / vocab lies between
        ref.assert_close("dx", dx[row], want, torch.bfloat16, 2 * ref.score_tolerance(x, 1.0))
    assert (dx[-1] == 0).all()


def gradient(x, tok, gl, gh, temperature=1.0, leaf=None):
    leaf = x.to(DEV) if leaf is None else leaf
    leaf = leaf.detach().requires_grad_(True)
    r = mec.token_log_probs(leaf, tok.to(DEV), temperature=temperature)
    outs, grads = [], []
    for o, gr in ((r.log_probs, gl), (r.entropy, gh)):
        if gr is not None:
            outs.append(o), grads.append(gr.to(DEV))
    torch.autograd.backward(outs, grads)
    return leaf.grad


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (2, 65), (5, 1000), (3, 4097), (2, 16385), (2, 50001),
                                        (300, 517), (1, 200001)])
def test_gradient_against_the_formula(rows, vocab, dtype):
    x, tok, g = make(rows, vocab, dtype, seed=8)
    gl, gh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    if rows > 2:
        tok[1] = -100
        x[2, : vocab // 2] = -math.inf
        tok[2] = vocab - 1
    # p carries about the score's absolute error as a relative one; p <= 1, |log p + H| <= the spread
    t = 0.7
    atol = ref.score_tolerance(x, t) / t * (gl.abs().max() + gh.abs().max() * (1 + ref.spread(x, t))).item()
    for a, b in ((gl, gh), (gl, None), (None, gh)):
        want = ref.token_scores_grad(x, tok, gl if a is not None else gl * 0, gh if b is not None else gh * 0, t)
        ref.assert_close("dx", gradient(x, tok, a, b, t), want, dtype, atol)


def test_gradient_of_masked_rows():
    x, tok, g = make(6, 3000, torch.float32, seed=9)
    x[0] = -math.inf
    x[1, 0] = math.nan
    x[2] = torch.finfo(torch.float32).min
    tok[3], tok[4] = 3000, -100
    x[5] = -math.inf
    x[5, 9] = 2.0
    gl, gh = torch.ones(6), torch.ones(6)
    dx = gradient(x, tok, gl, gh).cpu()
    assert (dx[0] == 0).all() and torch.isnan(dx[1]).all() and torch.isnan(dx[3]).all() and (dx[4] == 0).all()
    want = ref.token_scores_grad(x, tok, gl, gh)
    ref.assert_close("dx", dx[[2, 5]], want[[2, 5]], torch.float32, 1e-5)


def test_gradient_against_differences():
    """Central differences of the kernels' own results, step 2^-6: h^2 / 6 times a
    third derivative below 2, and rounding 2 * 2^-21 / (2 h)."""
    x, tok, g = make(3, 11, torch.float32, seed=10, scale=1.0)
    gl, gh = torch.randn(3, generator=g), torch.randn(3, generator=g)
    dx = gradient(x, tok, gl, gh, temperature=1.3).cpu().double()
    step = 2.0 ** -6
    for v in range(11):
        diff = 0.0
        for sign in (1, -1):
            y = x.clone()
            y[:, v] += sign * step
            r = mec.token_log_probs(y.to(DEV), tok.to(DEV), temperature=1.3)
            diff = diff + sign * (gl * r.log_probs.cpu() + gh * r.entropy.cpu()).double() / (2 * step)
        bound = (gl.abs() + 3 * gh.abs()).double() * (step ** 2 / 3 + 2.0 ** -21 / step)
        assert ((dx[:, v] - diff).abs() <= bound).all()


def test_gradient_layouts():
    g = torch.Generator().manual_seed(11)
    base = torch.randn(3, 6, 501, generator=g).to(torch.bfloat16)
    tok = torch.randint(0, 501, (3, 6), generator=g)
    for cut in (lambda t: t[:, :-1], lambda t: t[:, 1:], lambda t: t.transpose(0, 1), lambda t: t[..., 0:501:2]):
        x = cut(base)
        tk = (cut(tok[..., None].expand(3, 6, 501))[..., 0] % x.shape[-1]).contiguous()
        leaf = base.to(DEV).requires_grad_(True)
        mec.token_log_probs(cut(leaf), tk.to(DEV)).log_probs.sum().backward()
        n = x.shape[0] * x.shape[1]
        want = ref.token_scores_grad(x.reshape(n, -1), tk.reshape(-1), torch.ones(n), torch.zeros(n))
        full = torch.zeros(base.shape, dtype=torch.float64)
        cut(full).copy_(want.reshape(x.shape))
        ref.assert_close("dx", leaf.grad, full, torch.bfloat16, 1e-5)


def test_c_abi_row_map():
    """Rows on two strides through the C ABI; an `inner` beyond the rows is one stride."""
    from memoryefficientclip_amd import _lib
    x, tok, _ = make(6, 700, torch.float32, seed=17)
    flat, tg = x.to(DEV), tok.to(DEV)
    lp, _, _, _ = ref.token_scores(x, tok, 0)
    st = torch.cuda.current_stream().cuda_stream
    ws = torch.empty(_lib.load().mec_token_scores_workspace_bytes(6, 700, 0, _lib.DTYPE_F32), dtype=torch.uint8,
                     device=DEV)
    for inner, outer, step in ((1, 700, 0), (2, 1400, 700), (6, 0, 700), (1 << 32, 12345, 700), (7, 1, 700)):
        out, h = torch.empty(6, device=DEV), torch.empty(6, device=DEV)
        _lib.call("mec_token_scores", flat.data_ptr(), 6, inner, outer, step, 700, _lib.DTYPE_F32, tg.data_ptr(), 8, -100,
                  1.0, 0, out.data_ptr(), h.data_ptr(), None, None, None, ws.data_ptr(), ws.numel(), st)
        ref.assert_close("log_probs", out, lp, torch.float32, ref.score_tolerance(x, 1.0))


def test_results_repeat_bit_for_bit():
    x, tok, _ = make(70, 50001, torch.bfloat16, seed=12)
    x, tok = x.to(DEV), tok.to(DEV)
    a = mec.token_log_probs(x, tok, top_k=20)
    for _ in range(3):
        b = mec.token_log_probs(x, tok, top_k=20)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_another_stream():
    x, tok, _ = make(300, 5000, torch.bfloat16, seed=13)
    s = torch.cuda.Stream()
    xg, tg = x.to(DEV), tok.to(DEV)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaf = xg.detach().requires_grad_(True)
        r = mec.token_log_probs(leaf, tg, top_k=4)
        r.log_probs.sum().backward()
    torch.cuda.current_stream().wait_stream(s)
    lp, h, tt, tlp = ref.token_scores(x, tok, 4)
    ref.assert_close("log_probs", r.log_probs, lp, torch.float32, ref.score_tolerance(x, 1.0))
    assert torch.equal(r.top_tokens.cpu(), tt)
    want = ref.token_scores_grad(x, tok, torch.ones(300), torch.zeros(300))
    ref.assert_close("dx", leaf.grad, want, torch.bfloat16, 1e-5)


def test_no_positions():
    x = torch.zeros(0, 9, device=DEV, requires_grad=True)
    r = mec.token_log_probs(x, torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    assert r.log_probs.shape == (0,) and r.top_tokens.shape == (0, 2) and r.top_log_probs.shape == (0, 2)
    (r.log_probs.sum() + r.entropy.sum()).backward()
    assert x.grad.shape == (0, 9)

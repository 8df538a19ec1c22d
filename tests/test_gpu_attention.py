"""Attention and its gradients against their definition in 64 bits."""
import math

import pytest
import torch

import memoryefficientclip_amd as mec
import tower_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(b, nq, nk, h, hk, d, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(b, nq, h, d, generator=g) * spread).to(dtype)
    k, v = (torch.randn(b, nk, hk, d, generator=g).to(dtype) for _ in "kv")
    return q, k, v, torch.randn(b, nq, h, d, generator=g).to(dtype)


def lengths(*n, dtype=torch.int32):
    return torch.tensor(n, dtype=dtype)


def check(q, k, v, do, train=True, device=DEV, finite=False, **how):
    """`finite`: what is inf in one may be NaN in the other."""
    want = ref.attention(q, k, v, do if train else None, **how)
    leaves = [t.to(device).requires_grad_(train) for t in (q, k, v)]
    on = {n: t.to(device) if isinstance(t, torch.Tensor) else t for n, t in how.items()}
    out = mec.attention(*leaves, **on)
    got = {"out": out}
    if train:
        out.backward(do.to(device))
        got.update(zip(("dq", "dk", "dv"), (t.grad for t in leaves)))
    for name, (value, tolerance) in want.items():
        assert got[name].dtype == q.dtype and got[name].is_contiguous()
        x = got[name]
        if finite:
            x, value = (torch.where(torch.isfinite(y), y, math.nan) for y in (x, value))
        ref.close(name, x, value, tolerance)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n,m", [(1, 1), (1, 2), (31, 33), (33, 31), (64, 64), (65, 129), (130, 70), (257, 257)])
def test_lengths_of_tokens(n, m, causal, dtype):
    check(*inputs(2, n, m, 2, 2, 64, dtype, seed=n + m), causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 2, 7, 8, 16, 31, 32, 40, 63, 64, 65, 72, 80, 81, 96, 100, 127, 128])
def test_head_dims(d, dtype):
    check(*inputs(1, 45, 70, 2, 1, d, dtype, seed=d), causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("h,hk", [(1, 1), (3, 1), (8, 2), (6, 6), (7, 7), (40, 1)])
@pytest.mark.parametrize("n", [1, 3, 50])
def test_shared_heads(n, h, hk, dtype):
    check(*inputs(2, n, 67, h, hk, 32, dtype, seed=h), causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_batches(causal, kind, dtype):
    """Lengths of none, one, some and all, and beyond the ends; rows that see nothing."""
    n = lengths(0, 1, 40, 77, 90, -5, 77, 3, dtype=kind)
    m = lengths(5, 1, 39, 100, 200, 9, 0, 64, dtype=kind)
    q, k, v, do = inputs(8, 77, 100, 4, 2, 64, dtype, seed=3)
    check(q, k, v, do, causal=causal, query_lengths=n, key_lengths=m)
    check(q, k, v, do, causal=causal, key_lengths=m)
    check(q, k, v, do, causal=causal, query_lengths=n)
    # fewer keys than queries: the first queries see none
    check(*inputs(2, 77, 20, 4, 2, 64, dtype, seed=4), causal=causal, key_lengths=lengths(20, 7, dtype=kind))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_padding_is_not_read(bad, dtype):
    q, k, v, do = inputs(3, 70, 90, 2, 1, 40, dtype, seed=5)
    n, m = lengths(70, 33, 0), lengths(65, 90, 7)
    for b in range(3):
        for t, length in ((q, n), (do, n), (k, m), (v, m)):
            t[b, length[b]:] = bad
    got = check(q, k, v, do, query_lengths=n, key_lengths=m)
    assert all(torch.isfinite(t).all() for t in got.values())


# Sizes at which each of the forms runs: all tokens of a head in LDS; 32 rows or keys a workgroup; 128 of them; keys or
# queries split over workgroups.
FORMS = [(2, 77, 77, 2, 2), (1, 300, 420, 2, 1), (11, 300, 420, 8, 8), (1, 1300, 1300, 2, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what,bad", [("q", math.nan), ("k", math.nan), ("v", math.nan), ("v", math.inf),
                                      ("do", math.nan), ("do", -math.inf)])
@pytest.mark.parametrize("b,n,m,h,hk", FORMS[:3])
def test_what_is_not_seen_has_no_part(b, n, m, h, hk, what, bad, dtype):
    """An inf or a NaN in the middle of a causal sequence: earlier tokens do not see it."""
    q, k, v, do = inputs(b, n, m, h, hk, 24, dtype, seed=n)
    at = {"q": q, "k": k, "v": v, "do": do}[what]
    at[0, at.shape[1] // 2, 0, 5] = bad
    at[-1, at.shape[1] // 3, -1, :] = bad
    # Through an inf the gradients are sums of infs of both signs and products of 0 and inf, NaN or inf by the order
    # that they are formed in (do . o and sum_j p_ij do . v_j are the same number only while both are finite): they
    # must not be finite where the formula's are not, nor the other way round.
    check(q, k, v, do, finite=math.isinf(bad), causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,n,m,h,hk,d", [(*form, d) for form in FORMS for d in (16, 40, 64, 72, 96, 121, 128)
                                          if form[0] * form[1] * d <= 11 * 300 * 72])
def test_forms(b, n, m, h, hk, d, causal, dtype):
    check(*inputs(b, n, m, h, hk, d, dtype, seed=d), causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,n,m,h,hk", FORMS)
def test_forms_of_padded_batches(b, n, m, h, hk, dtype):
    g = torch.Generator().manual_seed(m)
    nq, nk = (torch.randint(0, x + 1, (b,), generator=g, dtype=torch.int32) for x in (n, m))
    check(*inputs(b, n, m, h, hk, 32, dtype, seed=b), causal=True, query_lengths=nq, key_lengths=nk)
    check(*inputs(b, n, m, h, hk, 32, dtype, seed=b), query_lengths=nq, key_lengths=nk)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,m", [(2500, 20), (20, 2500), (3, 700)])
def test_many_queries_of_few_keys_and_few_of_many(n, m, dtype):
    check(*inputs(1, n, m, 2, 1, 64, dtype, seed=n))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 72, 128])
@pytest.mark.parametrize("b,m", [(1, 300), (3, 5000), (20, 129)])
def test_single_tokens(b, m, d, dtype):
    """The form for serving: one query, keys of different lengths, with and without shared heads."""
    g = torch.Generator().manual_seed(m)
    n = torch.randint(0, m + 1, (b,), generator=g, dtype=torch.int32)
    n[0] = m
    for h, hk in ((4, 4), (16, 2)):
        check(*inputs(b, 1, m, h, hk, d, dtype, seed=b), train=False, causal=True, key_lengths=n)
    check(*inputs(b, 1, m, 2, 2, d, dtype, seed=b), key_lengths=n)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dtype):
    """One key takes everything, and the running maximum grows along the keys."""
    q, k, v, do = inputs(1, 40, 300, 2, 2, 64, dtype, seed=6, spread=8.0)
    check(q, k, v, do, scale=1.0)
    ramp = (torch.arange(300) / 10)[None, :, None, None]
    k = (q[:, :1].float() * 0.05 * ramp).to(dtype)
    check(q, k, v, do, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    """Slices of one projection, heads before tokens, odd addresses, one row for all, and a broadcast gradient."""
    g = torch.Generator().manual_seed(7)
    want = None
    whole = torch.randn(2, 50, 8, 64, generator=g).to(dtype)
    do = torch.randn(2, 50, 4, 64, generator=g).to(dtype)
    q, k, v = whole.split([4, 2, 2], 2)
    want = ref.attention(q, k, v, do, causal=True)
    odd = torch.zeros(2 * 50 * 8 * 67 + 1, dtype=dtype, device=DEV)[1:].view(2, 50, 8, 67)[..., 1:65]
    for layout in ("slices", "heads first", "odd", "columns"):
        on = whole.to(DEV)
        if layout == "odd":
            on = odd.copy_(on)
        leaves = [t.detach() for t in on.split([4, 2, 2], 2)]
        if layout == "heads first":
            leaves = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in leaves]
        if layout == "columns":
            leaves = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in leaves]
        leaves = [t.requires_grad_(True) for t in leaves]
        gd = do.to(DEV)
        if layout == "heads first":
            gd = gd.transpose(1, 3).contiguous().transpose(1, 3)
        out = mec.attention(*leaves, causal=True)
        out.backward(gd)
        for name, t in zip(("out", "dq", "dk", "dv"), (out, *(t.grad for t in leaves))):
            ref.close(f"{layout} {name}", t, *want[name])
    # one row for all tokens
    k1, v1 = (t[:, :1].expand(2, 50, 2, 64) for t in (k, v))
    q1 = q[:1, :1, :1].expand(2, 50, 4, 64)
    want = ref.attention(q1, k1, v1, torch.ones(2, 50, 4, 64, dtype=dtype))
    leaves = [t.to(DEV)[:, :1].expand(2, 50, 2, 64) for t in (k, v)]
    ql = q[:1, :1, :1].to(DEV).requires_grad_(True)
    out = mec.attention(ql.expand(2, 50, 4, 64), *leaves)
    out.sum().backward()
    ref.close("expanded", out, *want["out"])
    dq, tol = (t.sum((0, 1, 2))[None, None, None] for t in want["dq"])
    ref.close("expanded dq", ql.grad, dq, tol + 400 * ref.half_step(dtype) * want["dq"][0].abs().sum((0, 1, 2)))


def test_gradients_are_differences():
    q, k, v, do = (t.to(DEV) for t in inputs(1, 20, 24, 2, 1, 16, torch.float32, seed=8))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = mec.attention(*leaves, causal=True)
    grads = torch.autograd.grad(out, leaves, do)
    g = torch.Generator().manual_seed(9)
    with torch.no_grad():
        for i in range(3):
            step = torch.randn(leaves[i].shape, generator=g).to(DEV)
            h = 2.0 ** -7
            ends = []
            for sign in (1, -1):
                moved = list(leaves)
                moved[i] = leaves[i] + sign * h * step
                ends.append((mec.attention(*moved, causal=True).double() * do.double()).sum())
            diff = (ends[0] - ends[1]) / (2 * h)
            want = (grads[i].double() * step.double()).sum()
            # h^2 / 6 of the third derivative along the step, and the two results' errors over 2 h
            size = (out.double().abs() * do.double().abs()).sum()
            assert abs(diff - want) <= h * h * 20 * size + 64 * ref.E * size / h


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_bits_again(dtype):
    q, k, v, do = (t.to(DEV) for t in inputs(2, 200, 333, 6, 3, 72, dtype, seed=10))
    runs = []
    for _ in range(3):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = mec.attention(*leaves, causal=True)
        out.backward(do)
        runs.append([out.detach(), *(t.grad for t in leaves)])
    assert all(torch.equal(a, b) for run in runs[1:] for a, b in zip(runs[0], run))


def test_no_tokens():
    q, k = torch.zeros(2, 3, 4, 8, device=DEV, requires_grad=True), torch.zeros(2, 0, 2, 8, device=DEV, requires_grad=True)
    out = mec.attention(q, k, k)
    out.sum().backward()
    assert out.shape == q.shape and not out.any() and not q.grad.any() and k.grad.shape == k.shape
    assert mec.attention(q[:, :0], k, k).shape == (2, 0, 4, 8)
    assert mec.attention(q[:0], q[:0], q[:0]).shape == (0, 3, 4, 8)


def test_frozen_inputs():
    q, k, v, do = (t.to(DEV) for t in inputs(1, 40, 40, 2, 2, 32, torch.float32, seed=11))
    want = ref.attention(q, k, v, do)
    for wanted in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        leaves = [t.clone().requires_grad_(w) for t, w in zip((q, k, v), wanted)]
        mec.attention(*leaves).backward(do)
        for name, t, w in zip(("dq", "dk", "dv"), leaves, wanted):
            if w:
                ref.close(name, t.grad, *want[name])
            else:
                assert t.grad is None


def test_another_stream():
    q, k, v, do = inputs(2, 100, 150, 4, 2, 64, torch.bfloat16, seed=12)
    want = ref.attention(q, k, v, do)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
        out = mec.attention(*leaves)
        out.backward(do.to(DEV))
    stream.synchronize()
    for name, t in zip(("out", "dq", "dk", "dv"), (out, *(t.grad for t in leaves))):
        ref.close(name, t, *want[name])


def test_a_cache_beyond_32_bits():
    """A long cache of two texts, the second beyond 2^31 bytes, its end beyond 2^31 elements: one new token of each."""
    n, hk, d = 1_100_000, 8, 128
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v = (torch.empty(2, n, hk, d, device=DEV, dtype=torch.bfloat16) for _ in "kv")
    for t, mean in ((k, 0.0), (v, 1.0)):
        for b in range(2):
            t[b].normal_(mean, 1.0, generator=g)
    assert k.stride(0) * k.element_size() > 1 << 31 and k.numel() > 1 << 31
    q = torch.randn(2, 1, 2 * hk, d, device=DEV, generator=g).bfloat16()
    lengths = torch.tensor([n, n - 77], device=DEV)
    out = mec.attention(q, k, v, causal=True, key_lengths=lengths)
    for b in range(2):
        for h in range(2 * hk):
            m = lengths[b].item()
            kd, vd = k[b, :m, h // 2].double(), v[b, :m, h // 2].double()
            p = torch.softmax(kd @ q[b, 0, h].double() / d ** 0.5, 0)
            want = p @ vd
            # A score is off by (d + 2) E times the sizes of its terms, here 20 at most.  A lane adds up less than 10000
            # probabilities, and its products; 32 parts are joined.  Probabilities and result are rounded to bf16.
            u = ref.half_step(torch.bfloat16)
            tolerance = (u + 2 * (d + 2) * ref.E * 20 + 10100 * ref.E) * (p @ vd.abs()) + u * want.abs()
            ref.close(f"{b} {h}", out[b, 0, h], want.cpu(), tolerance.cpu())

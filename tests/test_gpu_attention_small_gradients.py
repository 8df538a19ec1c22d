"""fp16 gradients of the scores that fp16 itself would flush to 0, or could not hold: a score's gradient falls with the
number of keys, but dq and dk are sums of thousands of them, and well within fp16."""
import math

import pytest
import torch

import memoryefficientclip_amd as mec
import tower_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = torch.float16


def largest_score_gradient(q, k, v, do, causal):
    h, hk = q.shape[2], k.shape[2]
    head = lambda t: t.double().transpose(1, 2)  # noqa: E731
    many = lambda t: head(t).repeat_interleave(h // hk, 1)  # noqa: E731
    see = ref.sees(q.shape[0], q.shape[1], k.shape[1], causal, None, None)[:, None]
    s = (head(q) @ many(k).transpose(2, 3) / math.sqrt(q.shape[3])).masked_fill(~see, -math.inf)
    p = torch.softmax(s, 3).nan_to_num(0.0)
    dp = head(do) @ many(v).transpose(2, 3)
    return (p * (dp - (p * dp).sum(3, keepdim=True))).abs().max().item()


def check(b, q, k, v, do, causal):
    """The kernels hold the ds_ij in units of a power of two for each row (dq) or key (dk), in which the largest so far
    is 2^10 or more: each is off by half of fp16's least step, 2^-25 of such a unit, beside its rounding.  That is what
    the reference allows ds of up to 2^10: it is given do times the power of two that makes them so large, which scales
    all gradients alike.  What they come out in has steps of 2^-24 at least."""
    up = 2.0 ** math.floor(math.log2(2.0 ** 10 / largest_score_gradient(q, k, v, do, causal)))
    want = ref.attention(q, k, v, do.double() * up, causal=causal)
    times = b // q.shape[0]
    leaves = [t.to(DEV).repeat(times, 1, 1, 1).requires_grad_(True) for t in (q, k, v)]
    out = mec.attention(*leaves, causal=causal)
    out.backward(do.to(DEV).repeat(times, 1, 1, 1))
    got = dict(zip(("dq", "dk", "dv"), (t.grad for t in leaves)), out=out)
    for name, (value, tolerance) in want.items():
        if name != "out":
            value, tolerance = value / up, tolerance / up + 2.0 ** -25
        for x in (got[name][:q.shape[0]], got[name][-q.shape[0]:]):
            ref.close(name, x, value, tolerance)


# a head in LDS; 32 rows or keys a workgroup, up to 512 keys and beyond; 128 of them; queries split over workgroups; few
# queries of many keys, many of few
FORMS = [(2, 77, 77, 2, 2), (2, 250, 250, 2, 2), (1, 300, 420, 2, 1), (1, 1300, 1300, 2, 1), (64, 70, 200, 12, 2),
         (64, 200, 129, 8, 2), (16, 700, 900, 2, 2), (1, 3, 4096, 2, 2), (1, 2500, 20, 2, 1)]


@pytest.mark.parametrize("large", ["q", "k"])
@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-5])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [32, 64, 72, 128])
@pytest.mark.parametrize("b,n,m,h,hk", FORMS)
def test_small_gradients(b, n, m, h, hk, d, causal, size, large):
    """Scores of the size of 1, from large queries and small keys (so that dk is large beside ds) or the other way round."""
    g = torch.Generator().manual_seed(n + d)
    q, do = (torch.randn(1, n, h, d, generator=g) for _ in "qd")
    k, v = (torch.randn(1, m, hk, d, generator=g) for _ in "kv")
    scale = 32.0 if large == "q" else 1 / 32.0
    check(b, (q * scale).to(HALF), (k / scale).to(HALF), v.to(HALF), (do * size).to(HALF), causal)


@pytest.mark.parametrize("d", [32, 64, 72, 128])
@pytest.mark.parametrize("b,n,m,h,hk", [(2, 5, 5, 2, 2), (1, 5, 7, 2, 1), (64, 40, 129, 8, 2)])
def test_gradients_of_scores_beyond_fp16(b, n, m, h, hk, d):
    """ds of 10^5 and more; queries and keys so small that dq and dk are within fp16."""
    g = torch.Generator().manual_seed(d)
    q, do = (torch.randn(1, n, h, d, generator=g) for _ in "qd")
    k, v = (torch.randn(1, m, hk, d, generator=g) for _ in "kv")
    q, k, v, do = ((t * s).to(HALF) for t, s in ((q, 1 / 256), (k, 1 / 256), (v, 64), (do, 1024 * m ** 0.5)))
    assert largest_score_gradient(q, k, v, do, False) > 65504
    check(b, q, k, v, do, False)


def test_rows_of_very_different_sizes():
    """One query's gradient is 2^30 times another's, and the gradients grow along the keys and along the queries."""
    g = torch.Generator().manual_seed(1)
    for b, n, h, hk, d in ((1, 200, 2, 2, 64), (1, 700, 2, 1, 64), (64, 200, 8, 2, 128)):
        q, do = (torch.randn(1, n, h, d, generator=g) for _ in "qd")
        k, v = (torch.randn(1, n, hk, d, generator=g) for _ in "kv")
        ramp = torch.linspace(-18, 6, n).exp2()[None, :, None, None]
        for v_ramp, do_ramp in ((ramp, 1.0), (1.0, ramp), (ramp.flip(1), 1.0), (1.0, ramp.flip(1)), (ramp, ramp.flip(1))):
            check(b, q.to(HALF), k.to(HALF), (v * v_ramp).to(HALF), (do * do_ramp).to(HALF), True)

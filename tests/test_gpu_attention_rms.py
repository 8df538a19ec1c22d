"""How far 16-bit gradients of attention are off in the mean square, where the kernels correct what 16 bits would cost.

dq and dk are sums of score gradients that are rounded once, and are rounded once themselves.  A rounding is off by up
to u (half a step, relative to the power of two below the value) and evenly so: u / sqrt(3) of the values' size in the
mean square at most, where all lie just above a power of two.  Of two roundings, which know nothing of each other:
sqrt(2 / 3) u, 0.82 u.  (Values spread over their binade: 0.60 u.)

Without the corrections, the roundings of the result in delta = do . o, and the sum of a row's rounded score gradients
times the mean key, would be added.  They grow with what all values, or all keys, have in common, of which the
gradients are free: here that is 8 times as large as what they do not.
"""
import math

import pytest
import torch

import memoryefficientclip_amd as mec
import tower_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16]


def gradients(q, k, v, do):
    """dq, dk of the definition in 64 bits, causal."""
    (_, n, h, d), (m, hk) = q.shape, k.shape[1:3]
    head = lambda t: t.double().transpose(1, 2)  # noqa: E731
    many = lambda t: head(t).repeat_interleave(h // hk, 1)  # noqa: E731
    see = ref.sees(1, n, m, True, None, None)[:, None]
    p = torch.softmax((head(q) @ many(k).transpose(2, 3) / math.sqrt(d)).masked_fill(~see, -math.inf), 3)
    dp = head(do) @ many(v).transpose(2, 3)
    ds = p * (dp - (p * dp).sum(3, keepdim=True)) / math.sqrt(d)
    dk = (ds.transpose(2, 3) @ head(q)).unflatten(1, (hk, h // hk)).sum(2)
    return {"dq": (ds @ many(k)).transpose(1, 2), "dk": dk.transpose(1, 2)}


def check(b, n, m, h, hk, d, dtype, key_mean, value_mean):
    g = torch.Generator().manual_seed(n + d)
    q, do = (torch.randn(1, n, h, d, generator=g).to(dtype) for _ in "qd")
    k, v = ((torch.randn(1, m, hk, d, generator=g) + mean).to(dtype) for mean in (key_mean, value_mean))
    want = gradients(q, k, v, do)
    leaves = [t.to(DEV).repeat(b, 1, 1, 1).requires_grad_(True) for t in (q, k, v)]
    mec.attention(*leaves, causal=True).backward(do.to(DEV).repeat(b, 1, 1, 1))
    for (name, value), t in zip(want.items(), leaves):
        off = ((t.grad[-1:].cpu().double() - value).norm() / value.norm()).item()
        assert off <= math.sqrt(2 / 3) * ref.half_step(dtype), (name, off / ref.half_step(dtype))


# a head in LDS; 32 rows or keys a workgroup; 128 of them
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("means", [(0.0, 0.0), (0.0, 8.0), (8.0, 0.0)])
@pytest.mark.parametrize("b,n,m,h,hk,d", [(2, 77, 77, 4, 4, 64), (2, 250, 250, 4, 4, 40), (1, 600, 600, 4, 2, 16),
                                          (1, 900, 900, 2, 1, 48), (64, 70, 200, 12, 2, 32), (64, 70, 200, 12, 2, 48)])
def test_delta_and_the_mean_key(b, n, m, h, hk, d, means, dtype):
    """Heads whose dq is corrected by the mean key: of up to 64 in LDS, of up to 48 at all lengths."""
    check(b, n, m, h, hk, d, dtype, *means)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value_mean", [0.0, 8.0])
@pytest.mark.parametrize("b,n,m,h,hk,d", [(2, 77, 77, 4, 4, 96), (1, 400, 400, 4, 2, 64), (1, 300, 512, 4, 2, 128),
                                          (64, 70, 200, 12, 2, 64), (64, 70, 200, 12, 2, 128)])
def test_delta(b, n, m, h, hk, d, value_mean, dtype):
    """Heads whose delta alone is whole: wide ones in LDS, and others that see up to 512 keys."""
    check(b, n, m, h, hk, d, dtype, 0.0, value_mean)

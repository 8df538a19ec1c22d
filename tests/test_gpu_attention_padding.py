"""What lies beyond the queries of a tile has no part in the gradients of the keys, whatever these
hold: not causal, with numbers of queries that no tile divides."""
import math

import pytest
import torch

import memoryefficientclip_amd as mec
import tower_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("lengths", [False, True])
@pytest.mark.parametrize("b,n,m,h,hk,d", [(2, 77, 77, 2, 2, 64), (2, 1, 70, 2, 2, 40), (2, 33, 40, 2, 2, 96),
                                          (1, 300, 420, 2, 1, 64), (1, 7, 420, 4, 2, 128), (64, 70, 200, 8, 2, 32),
                                          (64, 70, 200, 8, 2, 72), (64, 1, 200, 4, 4, 72)])
def test_a_key_that_every_query_scores_minus_infinity(b, n, m, h, hk, d, lengths, bad, dtype):
    """A key overflowed: every query's score of it is -inf and its probability 0, exactly.  The result and
    the gradients of keys and values are those of the other keys alone; its own gradients are 0.  (The
    gradient of the queries is 0 times inf in that feature, and of the other keys elsewhere.)"""
    g = torch.Generator().manual_seed(m)
    q, do = (torch.randn(1, n, h, d, generator=g).to(dtype) for _ in "qd")
    k, v = (torch.randn(1, m, hk, d, generator=g).to(dtype) for _ in "kv")
    q[..., 5] = (q[..., 5].abs() + 0.25) * (-1 if bad > 0 else 1)
    at = m // 3
    others = torch.arange(m) != at
    how, on = {}, {}
    if lengths:
        how = dict(query_lengths=torch.tensor([max(1, n - 5)]), key_lengths=torch.tensor([m - 3]))
        on = {name: t.to(DEV).repeat(b) for name, t in how.items()}
        how["key_lengths"] = how["key_lengths"] - 1  # (of the others)
    want = ref.attention(q, k[:, others], v[:, others], do, **how)
    k[:, at, :, 5] = bad
    leaves = [t.to(DEV).repeat(b, 1, 1, 1).requires_grad_(True) for t in (q, k, v)]
    out = mec.attention(*leaves, **on)
    out.backward(do.to(DEV).repeat(b, 1, 1, 1))
    dq, dk, dv = (t.grad.cpu() for t in leaves)
    for i in {0, b - 1}:
        ref.close("out", out[i:i + 1], *want["out"])
        for name, x in (("dk", dk), ("dv", dv)):
            assert not x[i, at].any(), f"{name} of the key itself"
            ref.close(name, x[i:i + 1, others], *want[name])
        rest = torch.arange(d) != 5
        ref.close("dq", dq[i:i + 1, ..., rest], *(t[..., rest] for t in want["dq"]))

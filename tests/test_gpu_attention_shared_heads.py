"""Attention with shared heads in the forms for whole batches: four blocks of 32 rows or keys a
workgroup, and queries split over workgroups beside that.  They run where the device has a
workgroup of 128 rows or keys for each compute unit, so the batches here are a few entries,
repeated: the definition is worked out for those, and all of their copies have to agree with it.
"""
import pytest
import torch

import memoryefficientclip_amd as mec
import tower_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(b, q, k, v, do, layout=None, **how):
    """q, k, v, do of a few entries, repeated to `b`; `layout` lays a tensor on the GPU out."""
    want = ref.attention(q, k, v, do, **how)
    times = b // q.shape[0]
    many = lambda t: t.to(DEV).repeat(times, *(1,) * (t.dim() - 1))  # noqa: E731
    laid = layout or (lambda t: t)
    leaves = [laid(many(t)).requires_grad_(True) for t in (q, k, v)]
    out = mec.attention(*leaves, **{n: many(t) if isinstance(t, torch.Tensor) else t for n, t in how.items()})
    out.backward(laid(many(do)))
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *(t.grad for t in leaves))):
        copies = x.detach().reshape(times, -1, *x.shape[1:])
        ref.close(name, copies[0], *want[name])
        # (NaN in the same places and the same bits elsewhere: no copy differs from the first)
        same = (copies == copies[:1]) | (copies.isnan() & copies[:1].isnan())
        assert same.all(), f"{name}: copies of an entry differ"


def inputs(b, n, m, h, hk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, do = (torch.randn(b, n, h, d, generator=g).to(dtype) for _ in "qd")
    k, v = (torch.randn(b, m, hk, d, generator=g).to(dtype) for _ in "kv")
    return q, k, v, do


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("row", [65, 67, 68, 72])
def test_heads_on_other_boundaries_than_the_first(row, dtype):
    """Heads of 64 in rows of 65, 67 or 68 elements: a token of 8 heads is whole vectors of 16 bytes, a head is not.  72
    are whole vectors."""
    def layout(t):
        room = torch.zeros(*t.shape[:3], row, dtype=t.dtype, device=t.device)[..., :64]
        return room.copy_(t)

    q, k, v, do = inputs(2, 40, 256, 8, 2, 64, dtype, seed=row)
    assert layout(q).stride()[1:3] == (8 * row, row)
    check(64, q, k, v, do, layout=layout)

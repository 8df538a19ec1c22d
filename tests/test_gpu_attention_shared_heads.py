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


# batch, queries, keys, heads, key heads; of 256 compute units: 512 and 896 workgroups of 128 rows, 256 of 128 keys; in the
# second, queries are split in two for each 128 keys
FORMS = [(64, 70, 200, 12, 2), (64, 200, 129, 8, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [16, 40, 64, 72, 100, 128])
@pytest.mark.parametrize("b,n,m,h,hk", FORMS)
def test_forms_of_whole_batches(b, n, m, h, hk, d, causal, dtype):
    check(b, *inputs(2, n, m, h, hk, d, dtype, seed=d), causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [40, 64, 128])
@pytest.mark.parametrize("b,n,m,h,hk", FORMS)
def test_padded_batches(b, n, m, h, hk, d, causal, dtype):
    """Lengths of none, one, some and all; rows that see nothing."""
    nq = torch.tensor([n, 0, 1, n - 31, n // 2, 3, n, 33], dtype=torch.int32)
    nk = torch.tensor([m, 50, m, 65, 0, 1, 7, m - 1], dtype=torch.int32)
    check(b, *inputs(8, n, m, h, hk, d, dtype, seed=d), causal=causal, query_lengths=nq, key_lengths=nk)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("d", [40, 72, 128])
@pytest.mark.parametrize("b,n,m,h,hk", FORMS)
def test_what_is_not_seen_has_no_part(b, n, m, h, hk, d, what, dtype):
    """A NaN in the middle of a causal sequence: earlier tokens do not see it."""
    q, k, v, do = inputs(1, n, m, h, hk, d, dtype, seed=d)
    at = {"q": q, "k": k, "v": v, "do": do}[what]
    at[0, at.shape[1] // 2, -1, 5] = float("nan")
    at[0, at.shape[1] // 3 * 2, 0, :] = float("nan")
    check(b, q, k, v, do, causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 72, 128])
@pytest.mark.parametrize("n,m,h,hk", [(300, 420, 4, 2), (1300, 1300, 2, 1), (40, 700, 2, 1)])
def test_what_is_not_seen_has_no_part_in_long_sequences(n, m, h, hk, d, dtype):
    """The same where a workgroup has 32 rows or keys, or keys and queries are split over workgroups."""
    q, k, v, do = inputs(1, n, m, h, hk, d, dtype, seed=d)
    k[0, m // 2, 0, 5] = v[0, m // 3 * 2, -1, 5] = float("nan")
    q[0, n // 3, 0, 1] = do[0, n // 5, 0, 2] = float("nan")
    check(1, q, k, v, do, causal=True)

"""Distillation of rows longer than one workgroup's registers: lengths where the
number of segments, the place that holds one, or the workgroup's size changes."""
import pytest
import torch

import vocab_reference as ref
from test_gpu_distill import DEV, check, make

pytestmark = pytest.mark.gpu

# Segments of 32768 16-bit (16384 fp32) logits, in vectors of 8 (4); another
# workgroup above 204800 (65536), with segments of twice the length.
LENGTHS = [(torch.float32, n) for n in (32769, 49151, 49152, 49153, 65535, 65536, 65537, 98305, 131071, 163841)]
LENGTHS += [(torch.bfloat16, n) for n in (98303, 98304, 98305, 163841, 196607, 204799, 204800, 204801, 262143, 262145)]
LENGTHS += [(torch.float16, n) for n in (65537, 98311, 204801)]


@pytest.mark.parametrize("dtype,vocab", LENGTHS, ids=str)
def test_lengths_and_addresses(dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    base = (2.0 * torch.randn(2 * (vocab + 1) + 8, generator=g)).to(dtype)
    dev = base.to(DEV)
    tok = torch.randint(0, vocab, (2, 9), generator=g)
    tok[0, :2] = torch.tensor([0, vocab - 1])
    z = torch.randn(2, 9, generator=g)
    for off, ld in ((0, vocab), (1, vocab + 1)):
        check(base.as_strided((2, vocab), (ld, 1), off), tok, z, leaf=dev.as_strided((2, vocab), (ld, 1), off))


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 50001), (torch.bfloat16, 170001), (torch.bfloat16, 280001)], ids=str)
def test_the_largest_in_each_part(dtype, vocab):
    """The largest logits in one part of a row after another, masked parts, and a row without a teacher."""
    parts = 9
    x, tok, z = make(parts + 1, vocab, 12, dtype, seed=31)
    step = vocab // parts
    for i in range(parts):
        x[i, i * step:i * step + 3] += 60.0
        x[i, ((i + 1) % parts) * step:((i + 1) % parts) * step + step // 2] = -float("inf")
        tok[i, 0] = i * step
    tok[parts] = -1
    # (a teacher's token that cannot occur is an infinite loss: none here)
    tok[torch.isinf(torch.gather(x.float(), 1, tok.clamp(min=0)))] = -1
    check(x, tok, z, temperature=1.5, reduction="sum")


def test_more_rows_than_the_chip_holds():
    x, tok, z = make(4, 70001, 6, torch.bfloat16, seed=32)
    n = 150
    leaf = x.to(DEV).repeat(n, 1)
    loss, dx = check(x.repeat(n, 1), tok.repeat(n, 1), z.repeat(n, 1), leaf=leaf)
    assert all(torch.equal(dx[:4], dx[4 * i:4 * i + 4]) for i in range(n))

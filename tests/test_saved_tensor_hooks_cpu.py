"""Saved-tensor hooks may bring the values that a backward needs back in other memory
and other strides: what the kernels are told has to be of the tensor that came back."""
import ctypes
import gc

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import library_stub as stub
import memoryefficientclip_amd as mec

CUTS = [lambda x: x[:, :-1], lambda x: x[:, 1:], lambda x: x[..., 3:40], lambda x: x.transpose(0, 1),
        lambda x: x[:, :1].expand(4, 5, 50), lambda x: x[..., ::2], lambda x: x]


@pytest.fixture
def lib(monkeypatch):
    return stub.install(monkeypatch)


def logits(cut):
    g = torch.Generator().manual_seed(1)
    leaf = torch.randn(4, 6, 50, generator=g).requires_grad_(True)
    return cut(leaf)


@pytest.mark.parametrize("cut", CUTS)
def test_token_scores_backward(lib, cut):
    x = logits(cut)
    tokens = torch.arange(x[..., 0].numel()).reshape(x.shape[:-1]) % x.shape[-1]
    with stub.copying_hooks() as back:
        r = mec.token_log_probs(x, tokens)
        (r.log_probs.sum() + r.entropy.sum()).backward()
    (args,), v = lib.calls["mec_token_scores_backward"], x.shape[-1]
    assert args[5] == v
    assert torch.equal(stub.rows_at(back, *args[:5], v), x.detach().reshape(-1, v))
    assert torch.equal(stub.rows_at(back, args[7], 1, 1, 0, 0, tokens.numel())[0], tokens.reshape(-1))


@pytest.mark.parametrize("unpack", [lambda t: t.half(), lambda t: t[..., :-1], lambda t: t.to("meta")])
def test_other_values_than_were_saved_are_refused(lib, unpack):
    x = logits(lambda x: x)
    with pytest.raises(RuntimeError, match="saved-tensor hook returned"):
        with stub.copying_hooks(unpack):
            mec.token_log_probs(x, torch.zeros(4, 6, dtype=torch.int64)).log_probs.sum().backward()
    assert "mec_token_scores_backward" not in lib.calls


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("cut", CUTS)
def test_distillation_backward(lib, cut, reduction):
    x = logits(cut)
    v, shape = x.shape[-1], (*x.shape[:-1], 3)
    g = torch.Generator().manual_seed(2)
    tokens, z = torch.randint(0, v, shape, generator=g), torch.randn(shape, generator=g)
    with stub.copying_hooks() as back:
        loss = mec.TopKDistillationLoss(reduction=reduction)(x, tokens, z)
        loss.sum().backward(torch.tensor(3.0))
    (args,) = lib.calls["mec_distill_backward"]
    assert args[5] == v
    assert torch.equal(stub.rows_at(back, *args[:5], v), x.detach().reshape(-1, v))
    for at, want in ((7, tokens), (9, z)):
        assert torch.equal(stub.rows_at(back, args[at], 1, 1, 0, 0, want.numel())[0], want.reshape(-1))


def test_distillation_refuses_other_values(lib):
    x = logits(lambda x: x)
    with pytest.raises(RuntimeError, match="saved-tensor hook returned"):
        with stub.copying_hooks(lambda t: t.half()):
            mec.TopKDistillationLoss()(x, torch.zeros(4, 6, 2, dtype=torch.int64), torch.zeros(4, 6, 2)).backward()
    assert "mec_distill_backward" not in lib.calls


@pytest.mark.parametrize("cut", [lambda x: x[:, 2:8], lambda x: x[:, 1:], lambda x: x[::2], lambda x: x.t()[:6],
                                 lambda x: x[:, ::2], lambda x: x[1:2], lambda x: x])
def test_contrastive_backward(lib, cut):
    g = torch.Generator().manual_seed(3)
    x, y = (torch.randn(10, 10, generator=g).requires_grad_(True) for _ in range(2))
    with stub.copying_hooks() as back:
        mec.MemoryEfficientCLIPLoss()(cut(x), cut(y)).backward()
    (args,), (n, d) = lib.calls["mec_backward"], cut(x).shape
    assert args[4:6] == (n, d)
    for at, want in ((0, cut(x)), (2, cut(y))):
        assert torch.equal(stub.rows_at(back, args[at], n, 1, args[at + 1], 0, d), want.detach())


def test_contrastive_refuses_other_values(lib):
    x = torch.randn(10, 10).requires_grad_(True)
    with pytest.raises(RuntimeError, match="saved-tensor hook returned"):
        with stub.copying_hooks(lambda t: t.half()):
            mec.MemoryEfficientCLIPLoss()(x, x).backward()
    assert "mec_backward" not in lib.calls


def test_the_forwards_gradient_is_a_saved_tensor(lib):
    """It is the largest thing from forward to backward: offloading and checkpointing have to see it."""
    x = logits(lambda x: x)
    tokens, z = torch.zeros(4, 6, 2, dtype=torch.int64), torch.zeros(4, 6, 2)
    with stub.copying_hooks() as back:
        loss = mec.TopKDistillationLoss()(x, tokens, z)
        loss.backward()
    (forward,), (backward,) = lib.calls["mec_distill_forward"], lib.calls["mec_distill_backward"]
    pointers = [t.data_ptr() for t in back]
    assert forward[17] is not None and forward[17] not in pointers
    # what came back is what is handed out
    assert backward[17] == 1 and backward[18] in pointers


def test_a_checkpointed_region_keeps_no_gradient(lib):
    x = logits(lambda x: x)
    tokens, z = torch.zeros(4, 6, 2, dtype=torch.int64), torch.zeros(4, 6, 2)
    loss = checkpoint(lambda x: mec.TopKDistillationLoss()(x * 1.0, tokens, z), x, use_reentrant=False)
    gc.collect()
    assert [t for t in gc.get_objects() if type(t) is torch.Tensor and t.shape == x.shape and t is not x] == []
    loss.backward()
    first, again = lib.calls["mec_distill_forward"]
    (backward,) = lib.calls["mec_distill_backward"]
    assert backward[17] == 1 and backward[18] == again[17]


def test_the_forwards_gradient_is_handed_out_once(lib):
    x = logits(lambda x: x)
    loss = mec.TopKDistillationLoss()(x, torch.zeros(4, 6, 2, dtype=torch.int64), torch.zeros(4, 6, 2))
    first, = torch.autograd.grad(loss, x, retain_graph=True)
    (forward,) = lib.calls["mec_distill_forward"]
    assert first.data_ptr() == forward[17]  # (no copy)
    first.zero_()
    second, = torch.autograd.grad(loss, x)
    assert second.data_ptr() != first.data_ptr()
    assert [(args[17], args[18]) for args in lib.calls["mec_distill_backward"]] == [(1, first.data_ptr()),
                                                                                   (0, second.data_ptr())]


def test_the_forwards_gradient_becomes_the_leafs(lib):
    """AccumulateGrad takes it over without a copy."""
    x = logits(lambda x: x)
    mec.TopKDistillationLoss()(x, torch.zeros(4, 6, 2, dtype=torch.int64), torch.zeros(4, 6, 2)).backward()
    assert x.grad.data_ptr() == lib.calls["mec_distill_forward"][0][17]


def test_embedding_backward(lib):
    tokens = torch.arange(12).reshape(3, 4)
    w = torch.randn(12, 5).requires_grad_(True)
    read = []

    def backward(*args):
        read.append(torch.frombuffer(bytearray(ctypes.string_at(args[0], 12 * args[1])), dtype=torch.int64))
        return 0

    lib.mec_embedding_backward = backward
    with stub.copying_hooks(lambda t: t.t().contiguous().t()):
        mec.scaled_embedding(tokens, w).sum().backward()
    assert torch.equal(read[0], tokens.reshape(-1))
    for unpack in (lambda t: t.int(), lambda t: t[:2]):
        with pytest.raises(RuntimeError, match="saved-tensor hook returned"):
            with stub.copying_hooks(unpack):
                mec.scaled_embedding(tokens, w).sum().backward()
    assert len(read) == 1


def narrow(t):
    """What is held in 32 bits or more comes back in half of them."""
    return t.to({torch.float32: torch.float16, torch.int64: torch.int32}.get(t.dtype, t.dtype))


@pytest.mark.parametrize("kinds", [{torch.float32}, {torch.int64}])
def test_other_tensors_than_the_logits_are_refused_too(lib, kinds):
    """bf16 logits come back as they were, and what is saved beside them in fewer bytes than the kernels read."""
    x = torch.randn(4, 6, 50).bfloat16().requires_grad_(True)
    tokens, z = torch.zeros(4, 6, 2, dtype=torch.int64), torch.zeros(4, 6, 2)
    calls = [lambda: mec.token_log_probs(x, tokens[..., 0]).entropy, lambda: mec.TopKDistillationLoss()(x, tokens, z),
             lambda: mec.TopKDistillationLoss(reduction="none")(x, tokens, z)]
    if torch.float32 in kinds:
        y = torch.randn(10, 8).bfloat16().requires_grad_(True)
        calls.append(lambda: mec.MemoryEfficientCLIPLoss()(y, y))
    for call in calls:
        with pytest.raises(RuntimeError, match="saved-tensor hook returned"):
            with stub.copying_hooks(lambda t: narrow(t) if t.dtype in kinds else t):
                call().sum().backward()
    assert not any(name.endswith("_backward") for name in lib.calls)

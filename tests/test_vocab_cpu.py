"""Host-side behaviour of the operators over a vocabulary that needs no GPU:
the refusals of the Python entry points and of the C ABI (all before any launch),
and how logits are laid out for the kernels."""
import ctypes
import math

import pytest
import torch

import memoryefficientclip_amd as mec
from memoryefficientclip_amd import _lib, _vocab


class FakeCuda(torch.Tensor):
    @property
    def is_cuda(self):
        return True


def fake(shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(FakeCuda)


def ids(*shape, dtype=torch.int64):
    return fake(shape, dtype)


@pytest.fixture(autouse=True)
def no_capture(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def test_cpu_tensors_raise():
    x, t = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(AssertionError, match="GPU"):
        mec.token_log_probs(x, t)
    with pytest.raises(AssertionError, match="GPU"):
        mec.TopKDistillationLoss()(x, t[:, None], x[:, :1])
    with pytest.raises(AssertionError, match="GPU"):
        mec.scaled_embedding(t, x)
    with pytest.raises(AssertionError, match="GPU"):
        mec.token_log_probs(fake((3, 5)), t)
    with pytest.raises(TypeError, match="Tensor"):
        mec.token_log_probs([[1.0]], t)


def test_token_log_probs_refuses():
    with pytest.raises(ValueError, match="one row for each"):
        mec.token_log_probs(fake((3, 5)), ids(4))
    with pytest.raises(ValueError, match="one row for each"):
        mec.token_log_probs(fake((3, 5)), ids(3, 1))
    with pytest.raises(TypeError, match="dtype"):
        mec.token_log_probs(fake((3, 5), torch.float64), ids(3))
    with pytest.raises(TypeError, match="dtype"):
        mec.token_log_probs(fake((3, 5)), ids(3, dtype=torch.int16))
    with pytest.raises(ValueError, match="vocabulary"):
        mec.token_log_probs(fake((3, 0)), ids(3))
    with pytest.raises(ValueError, match="vocabulary"):
        mec.token_log_probs(fake((1, 1)).expand(1, (1 << 19) + 1), ids(1))
    for k in (-1, 6):
        with pytest.raises(ValueError, match="top_k"):
            mec.token_log_probs(fake((3, 5)), ids(3), top_k=k)
    with pytest.raises(ValueError, match="top_k"):
        mec.token_log_probs(fake((3, 500)), ids(3), top_k=129)
    for t in (0.0, -1.0, math.nan, math.inf, 1e-9):
        with pytest.raises(ValueError, match="temperature"):
            mec.token_log_probs(fake((3, 5)), ids(3), temperature=t)


def test_distillation_refuses():
    loss = mec.TopKDistillationLoss()
    with pytest.raises(ValueError, match="reduction"):
        mec.TopKDistillationLoss(reduction="batchmean")
    with pytest.raises(ValueError, match="temperature"):
        mec.TopKDistillationLoss(temperature=0.0)
    with pytest.raises(ValueError, match="weight"):
        mec.TopKDistillationLoss(weight=math.inf)
    with pytest.raises(ValueError, match="same positions"):
        loss(fake((3, 5)), ids(4, 2), fake((4, 2)))
    with pytest.raises(ValueError, match="differ in shape"):
        loss(fake((3, 5)), ids(3, 2), fake((3, 3)))
    with pytest.raises(ValueError, match="teacher entries"):
        loss(fake((3, 5)), ids(3, 0), fake((3, 0)))
    with pytest.raises(ValueError, match="teacher entries"):
        loss(fake((3, 5)), ids(3, 1025), fake((3, 1025)))
    with pytest.raises(TypeError, match="dtype"):
        loss(fake((3, 5)), ids(3, 2), fake((3, 2), torch.float64))
    with pytest.raises(TypeError, match="dtype"):
        loss(fake((3, 5)), fake((3, 2)), fake((3, 2)))
    assert loss.state_dict() == {}


def test_embedding_refuses():
    w = fake((6, 4))
    with pytest.raises(ValueError, match=r"\[V, D\]"):
        mec.scaled_embedding(ids(3), fake((6,)))
    with pytest.raises(ValueError, match=r"\[V, D\]"):
        mec.scaled_embedding(ids(3), fake((6, 0)))
    with pytest.raises(TypeError, match="dtype"):
        mec.scaled_embedding(fake((3,)), w)
    with pytest.raises(TypeError, match="dtype"):
        mec.scaled_embedding(ids(3), fake((6, 4), torch.float64))
    for p in (6, -7):
        with pytest.raises(ValueError, match="padding_idx"):
            mec.scaled_embedding(ids(3), w, padding_idx=p)
        with pytest.raises(ValueError, match="padding_idx"):
            mec.ScaledTokenEmbedding(6, 4, padding_idx=p)
    with pytest.raises(ValueError, match="scale"):
        mec.scaled_embedding(ids(3), w, scale=math.nan)
    with pytest.raises(ValueError, match="maxima"):
        mec.scaled_embedding(ids(3), fake((1, 1)).expand(6, (1 << 16) + 1))
    m = mec.ScaledTokenEmbedding(8, 16)
    assert m.scale == 4.0 and m.weight.shape == (8, 16)
    assert "scale=4" in repr(m)


def test_graph_capture_is_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="graph capture"):
        mec.token_log_probs(fake((3, 5)), ids(3))
    with pytest.raises(RuntimeError, match="graph capture"):
        mec.TopKDistillationLoss()(fake((3, 5)), ids(3, 2), fake((3, 2)))
    with pytest.raises(RuntimeError, match="graph capture"):
        mec.scaled_embedding(ids(3), fake((6, 4)))


@pytest.mark.parametrize("make,want", [
    (lambda x: x, (24, 1, 30, 0)),
    (lambda x: x[:, :-1], (20, 5, 180, 30)),
    (lambda x: x[..., 3:9], (24, 1, 30, 0)),
    (lambda x: x.transpose(0, 1), (24, 4, 30, 180)),
    (lambda x: x[0, 0], (1, 1, 0, 0)),
    (lambda x: x[:1, :1], (1, 1, 0, 0)),
    (lambda x: x[:, 2:3], (4, 1, 180, 0)),
    (lambda x: x[:1, :1].expand(3, 5, 30), (15, 1, 0, 0)),
    (lambda x: x.reshape(2, 2, 6, 30)[:, :, 1:], (20, 5, 180, 30)),
    (lambda x: x.reshape(2, 2, 6, 30)[:, :1, 1:], (10, 5, 360, 30)),
])
def test_rows_are_read_in_place(make, want):
    x = torch.arange(4 * 6 * 30.0).reshape(4, 6, 30)
    view = make(x)
    held, ptr, rows = _vocab.rows_of(view)
    assert rows == want and ptr == view.data_ptr() and held is view
    n, inner, so, si = rows
    flat = view.reshape(-1, view.shape[-1])
    base = view.storage_offset()
    for r in range(n):
        at = base + (r // inner) * so + (r % inner) * si
        assert torch.equal(x.reshape(-1)[at:at + view.shape[-1]], flat[r])


def test_rows_that_lie_on_no_grid_are_copied():
    x = torch.arange(4 * 6 * 30.0).reshape(4, 6, 30)
    held, ptr, rows = _vocab.rows_of(x[..., ::2])
    assert held.is_contiguous() and rows == (24, 1, 15, 0)
    y = torch.arange(2 * 3 * 4 * 10.0).reshape(2, 3, 4, 10)[:, :2, :3]
    held, ptr, rows = _vocab.rows_of(y)
    assert held.is_contiguous() and rows == (12, 1, 10, 0)


P = ctypes.c_void_p(1 << 12)  # never dereferenced: every call below is refused before a launch


def refused(code, name, *args):
    assert getattr(_lib.load(), name)(*args) == code
    assert _lib.last_error()


SCORES = [P, 8, 1, 100, 0, 100, 0, P, 8, -100, 1.0, 4, P, P, P, P, P, None, 0, None]
SCORES_BACK = [P, 8, 1, 100, 0, 100, 0, P, 8, -100, 1.0, P, P, P, P, P, None]
DISTILL = [P, 8, 1, 100, 0, 100, 0, P, 8, P, 0, 4, 1.0, 1.0, 2, P, P, None, P, 1 << 20, None]
DISTILL_BACK = [P, 8, 1, 100, 0, 100, 0, P, 8, P, 0, 4, 1.0, 1.0, 2, P, P, 0, P, None]
LOGITS_BAD = [(0, None, -1), (1, 0, -1), (1, 1 << 24, -2), (2, 0, -1), (3, -1, -1), (4, -1, -1), (3, 1 << 50, -1),
              (5, 0, -1), (5, (1 << 19) + 1, -2), (6, 3, -1), (6, 6, -1), (7, None, -1), (8, 2, -1)]


@pytest.mark.parametrize("name,good,more", [
    ("mec_token_scores", SCORES, [(10, 0.0, -1), (10, math.nan, -1), (11, -1, -1), (11, 101, -1), (12, None, -1),
                                  (13, None, -1), (14, None, -1), (15, None, -1)]),
    ("mec_token_scores_backward", SCORES_BACK, [(10, 0.0, -1), (11, None, -1), (12, None, -1), (15, None, -1)]),
    ("mec_distill_forward", DISTILL, [(9, None, -1), (10, 4, -1), (11, 0, -1), (11, 1025, -2), (12, -1.0, -1),
                                      (13, math.inf, -1), (14, 3, -1), (15, None, -1), (16, None, -1), (18, None, -1),
                                      (18, ctypes.c_void_p((1 << 12) + 4), -1), (19, 3, -1)]),
    ("mec_distill_backward", DISTILL_BACK, [(9, None, -1), (10, 4, -1), (11, 0, -1), (12, 0.0, -1), (14, -1, -1),
                                            (15, None, -1), (16, None, -1), (18, None, -1)]),
])
def test_c_abi_refuses(name, good, more):
    for at, value, code in LOGITS_BAD + more:
        args = list(good)
        args[at] = value
        refused(code, name, *args)


def test_c_abi_refuses_top_k_and_made():
    args = list(SCORES)
    args[5], args[3], args[11] = 1000, 1000, 129
    refused(-2, "mec_token_scores", *args)
    args = list(DISTILL)
    args[14], args[17] = 0, P  # the gradient of each row's loss has no common grad_output
    refused(-1, "mec_distill_forward", *args)
    args = list(DISTILL_BACK)
    args[14], args[17] = 0, 1
    refused(-1, "mec_distill_backward", *args)


EMBED = [P, 8, 9, P, 16, 30, 16, 0, 1.0, P, None]
EMBED_BACK = [P, 8, 9, P, 16, 30, 16, 0, 1.0, -1, P, P, 1 << 24, None]


@pytest.mark.parametrize("at,value,code", [(0, None, -1), (1, 3, -1), (2, 0, -1), (2, (1 << 23) + 1, -2),
                                           (3, None, -1), (4, 15, -1), (5, 0, -1), (5, (1 << 22) + 1, -2), (6, 0, -1),
                                           (6, (1 << 16) + 1, -2), (7, 3, -1), (8, math.inf, -1)])
def test_c_abi_embedding_refuses(at, value, code):
    for name, good in (("mec_embedding", EMBED), ("mec_embedding_backward", EMBED_BACK)):
        args = list(good)
        args[at] = value
        if at == 6 and value > 16:  # (the row strides go with it)
            args[4] = value
        refused(code, name, *args)


def test_c_abi_embedding_refuses_outputs_and_padding():
    refused(-1, "mec_embedding", *EMBED[:9], None, None)
    for at, value in ((9, 30), (9, -2), (10, None)):
        args = list(EMBED_BACK)
        args[at] = value
        refused(-1, "mec_embedding_backward", *args)


def test_c_abi_refuses_a_capture(monkeypatch):
    monkeypatch.setenv("MEC_TEST_ASSUME_CAPTURING", "1")
    for name, args in (("mec_token_scores", SCORES), ("mec_token_scores_backward", SCORES_BACK),
                       ("mec_distill_forward", DISTILL), ("mec_distill_backward", DISTILL_BACK),
                       ("mec_embedding", EMBED), ("mec_embedding_backward", EMBED_BACK)):
        args = list(args)
        if name == "mec_token_scores":
            args[17], args[18] = P, 1 << 24
        refused(-2, name, *args)
        assert "captur" in _lib.last_error()


def test_size_queries():
    lib = _lib.load()
    assert lib.mec_token_scores_workspace_bytes(8, 100, 4, 0) >= 0
    assert lib.mec_token_scores_workspace_bytes(8, 100, 101, 0) == -1
    assert lib.mec_token_scores_workspace_bytes(0, 100, 4, 0) == -1
    assert lib.mec_token_scores_workspace_bytes(8, 1 << 20, 4, 0) == -2
    assert lib.mec_distill_workspace_bytes(8, 100, 4, 0, 1) >= 0
    assert lib.mec_distill_workspace_bytes(8, 100, 0, 0, 1) == -1
    assert lib.mec_embedding_workspace_bytes(9, 30, 16, 0) >= 0
    assert lib.mec_embedding_workspace_bytes(9, 30, 0, 0) == -1

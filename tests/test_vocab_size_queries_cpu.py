"""A size query answers an argument as the operator that takes the workspace does."""
import ctypes

import pytest

from memoryefficientclip_amd import _lib

P = ctypes.c_void_p(1 << 12)  # never dereferenced: every call below is refused before a launch


@pytest.mark.parametrize("k", [-1, 0, 1025, 1 << 40])
def test_distillation_s_entries(k):
    lib = _lib.load()
    want = lib.mec_distill_forward(P, 8, 1, 100, 0, 100, 0, P, 8, P, 0, k, 1.0, 1.0, 2, P, P, None, P, 1 << 20, None)
    text = _lib.last_error()
    assert want == (-1 if k < 1 else -2)
    for with_grad in (0, 1):
        assert lib.mec_distill_workspace_bytes(8, 100, k, 0, with_grad) == want
        assert _lib.last_error() == text


@pytest.mark.parametrize("rows,vocab,k", [(0, 100, 4), (1 << 24, 100, 4), (8, 0, 1), (8, (1 << 19) + 1, 4), (8, 100, 101),
                                          (8, 1000, 129), (8, 100, -1)])
def test_token_scores(rows, vocab, k):
    lib = _lib.load()
    want = lib.mec_token_scores(P, rows, 1, vocab, 0, vocab, 0, P, 8, -100, 1.0, k, P, P, P, P, P, P, 1 << 40, None)
    text = _lib.last_error()
    assert want < 0 and lib.mec_token_scores_workspace_bytes(rows, vocab, k, 0) == want
    assert _lib.last_error() == text


@pytest.mark.parametrize("n,vocab,d,dtype", [(0, 30, 16, 0), (9, 0, 16, 0), (9, 30, 0, 0), ((1 << 23) + 1, 30, 16, 0),
                                             (9, (1 << 22) + 1, 16, 0), (9, 30, (1 << 16) + 1, 0), (9, 30, 16, 3)])
def test_embedding(n, vocab, d, dtype):
    lib = _lib.load()
    want = lib.mec_embedding_backward(P, 8, n, P, max(d, 16), vocab, d, dtype, 1.0, -1, P, P, 1 << 40, None)
    text = _lib.last_error()
    assert want < 0 and lib.mec_embedding_workspace_bytes(n, vocab, d, dtype) == want
    assert _lib.last_error() == text

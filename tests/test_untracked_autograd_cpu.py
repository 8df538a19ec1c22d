"""Where no input asks for a gradient the operators are called without autograd; what
autograd sees in such calls all the same, tangents and traces, is not lost without an error."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import library_stub as stub
import memoryefficientclip_amd as mec


@pytest.fixture(autouse=True)
def lib(monkeypatch):
    return stub.install(monkeypatch)


TOKENS = torch.tensor([1, 2, 0])
OPERATORS = [lambda x: mec.token_log_probs(x, TOKENS).log_probs,
             lambda x: mec.TopKDistillationLoss()(x, TOKENS[:, None], torch.zeros(3, 1)),
             lambda x: mec.scaled_embedding(TOKENS, x, 2.0)]


@pytest.mark.parametrize("wanted", [False, True])
@pytest.mark.parametrize("op", OPERATORS)
def test_forward_mode_is_refused(op, wanted):
    x = torch.randn(3, 5).requires_grad_(wanted)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward mode"):
            op(fwd.make_dual(x, torch.ones(3, 5)))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward mode"):
            op(fwd.make_dual(x, torch.ones(3, 5)))
        # a level alone, or no gradient of any kind, is no reason
        assert fwd.unpack_dual(op(x)).tangent is None
        with torch.no_grad(), fwd._set_fwd_grad_enabled(False):
            op(fwd.make_dual(x, torch.ones(3, 5)))

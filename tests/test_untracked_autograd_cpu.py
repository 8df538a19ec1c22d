"""Where no input asks for a gradient the operators are called without autograd; what
autograd sees in such calls all the same, tangents and traces, is not lost without an error."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import library_stub as stub
import memoryefficientclip_amd as mec

pytestmark = [pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning"),
              pytest.mark.filterwarnings("ignore::DeprecationWarning")]


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


CALLS = ["mec_token_scores", "mec_distill_forward", "mec_embedding"]
WRONG = [(OPERATORS[0], torch.randn(4, 5), "one row for each"), (OPERATORS[1], torch.randn(4, 5), "same positions"),
         (OPERATORS[2], torch.randn(5), r"\[V, D\]"), (OPERATORS[2], torch.randn(0, 5), r"\[V, D\]"),
         (OPERATORS[0], torch.randn(3, 0), "vocabulary"), (OPERATORS[1], torch.randn(3, 0), "vocabulary"),
         *((op, torch.randn(3, 5).double(), "dtype") for op in OPERATORS)]


def check_trace(lib, op, example, wrong, message):
    traced = torch.jit.trace(op, example, check_trace=False)
    lib.calls.clear()
    with pytest.raises(Exception, match=message):
        traced(wrong)
    assert not any(call in lib.calls for call in CALLS)


@pytest.mark.parametrize("op,wrong,message", WRONG)
def test_a_traced_function_checks_its_inputs(lib, op, wrong, message):
    """Traced with a gradient; other inputs than were traced, which no kernel may be started on."""
    check_trace(lib, op, torch.randn(3, 5).requires_grad_(True), wrong, message)

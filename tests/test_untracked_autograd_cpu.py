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


@pytest.mark.parametrize("op,wrong,message", WRONG)
def test_a_function_traced_without_a_gradient_checks_its_inputs(lib, op, wrong, message):
    check_trace(lib, op, torch.randn(3, 5), wrong, message)


@pytest.mark.parametrize("wanted", [False, True])
@pytest.mark.parametrize("op,call", zip(OPERATORS, CALLS))
def test_a_traced_function_calls_the_library(lib, op, call, wanted):
    x = torch.randn(3, 5).requires_grad_(wanted)
    traced = torch.jit.trace(op, x, check_trace=False)
    lib.calls.clear()
    y = torch.randn(3, 5)
    assert traced(y).shape == op(y).shape
    got, want = lib.calls[call]
    # the operator's numbers, and the tensor that the trace was called with
    numbers = [[a for a in args if isinstance(a, (int, float)) and abs(a) < 1 << 30] for args in (got, want)]
    assert numbers[0] == numbers[1] and y.data_ptr() in got


@pytest.mark.parametrize("op", OPERATORS)
def test_a_gradient_through_a_traced_function(lib, op):
    traced = torch.jit.trace(op, torch.randn(3, 5), check_trace=False)
    x = torch.randn(3, 5).requires_grad_(True)
    traced(x).sum().backward()
    assert x.grad.shape == x.shape and any(name.endswith("_backward") for name in lib.calls)


@pytest.mark.parametrize("wanted", [False, True])
@pytest.mark.parametrize("op", [*OPERATORS, lambda x: mec.MemoryEfficientCLIPLoss()(x, x)])
def test_make_fx_is_refused(lib, op, wanted):
    """It records tensor operations alone: of these calls, the empty results."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn(3, 5).requires_grad_(wanted)
    op(x)
    lib.calls.clear()
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(op)(x)
    assert not lib.calls
    op(x)

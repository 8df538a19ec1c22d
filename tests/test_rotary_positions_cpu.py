"""Positions and frequencies that ask for a gradient, which norm_rotary does not have (the library
stubbed): refused, where None would be taken for zero."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import library_stub as stub
import memoryefficientclip_amd as mec


@pytest.fixture
def lib(monkeypatch):
    return stub.install(monkeypatch)


def call(x, positions=None, frequencies=None):
    positions = torch.arange(5.0)[:, None] if positions is None else positions
    return mec.norm_rotary(x, x, positions, (4,), frequencies=frequencies)


@pytest.mark.parametrize("wanted", [False, True])
@pytest.mark.parametrize("kind", [torch.float64, torch.float32])
def test_a_gradient_of_frequencies_is_refused(lib, kind, wanted):
    x, f = torch.randn(2, 5, 4, 8, requires_grad=wanted), torch.rand(4, dtype=kind, requires_grad=True)
    with pytest.raises(RuntimeError, match="positions and frequencies"):
        call(x, frequencies=f)
    assert not lib.calls
    with torch.no_grad():
        call(x, frequencies=f)
    y, _ = call(x, frequencies=f.detach())
    assert y.requires_grad == wanted and len(lib.calls["mec_norm_rotary"]) == 2


@pytest.mark.parametrize("wanted", [False, True])
def test_a_gradient_of_positions_is_refused(lib, wanted):
    x, p = torch.randn(2, 5, 4, 8, requires_grad=wanted), torch.rand(5, 1, requires_grad=True)
    with pytest.raises(RuntimeError, match="positions and frequencies"):
        call(x, positions=p)
    assert not lib.calls
    call(x, positions=p.detach())


def test_a_tangent_of_either_is_refused(lib):
    x, p, f = torch.randn(2, 5, 4, 8), torch.rand(5, 1), torch.rand(4)
    with fwd.dual_level():
        for how in (dict(positions=fwd.make_dual(p, torch.ones(5, 1))), dict(frequencies=fwd.make_dual(f, torch.ones(4)))):
            with pytest.raises(NotImplementedError, match="forward mode"):
                call(x, **how)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_a_trace_refuses_them_too(lib):
    traced = torch.jit.trace(lambda x, f: call(x, frequencies=f)[0], (torch.randn(2, 5, 4, 8), torch.rand(4)),
                             check_trace=False)
    traced(torch.randn(2, 5, 4, 8), torch.rand(4))
    with pytest.raises(RuntimeError, match="positions and frequencies"):
        traced(torch.randn(2, 5, 4, 8), torch.rand(4, requires_grad=True))

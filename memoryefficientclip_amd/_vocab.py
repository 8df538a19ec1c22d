"""Host side shared by the operators over a vocabulary: argument checks, the
layout of logits, scratch and the calls into the HIP library
(``include/mec.h``)."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _function as _f
from . import _lib


def refuse_graph_capture() -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("memoryefficientclip_amd: the operators over a vocabulary do not support CUDA/HIP graph "
                           "capture; call them outside the captured region")


refuse_make_fx = _f.refuse_make_fx


def check_gpu(name: str, t: torch.Tensor, device: torch.device | None = None) -> None:
    """`t` is a tensor on the GPU (AssertionError else, as the losses raise it), on `device` if given."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise AssertionError(f"{name} must be a GPU tensor ({name}.is_cuda)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other inputs on {device}")


def check_float(name: str, t: torch.Tensor) -> None:
    if t.dtype not in _f._DTYPES:
        raise TypeError(f"unsupported dtype {t.dtype} of {name}; supported: float32, bfloat16, float16")


def code_of(t: torch.Tensor) -> int:
    """The C-ABI dtype code of a tensor that passed check_float."""
    return _f._DTYPES[t.dtype]


def check_tokens(name: str, t: torch.Tensor) -> None:
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"unsupported dtype {t.dtype} of {name}; supported: int64, int32")


def check_temperature(temperature: float) -> float:
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must be in [1e-6, 1e6], got {temperature}")
    return temperature


def rows_of(logits: torch.Tensor) -> tuple[torch.Tensor, int, tuple[int, int, int, int]]:
    """(tensor to hold, data pointer, (rows, inner, outer stride, inner stride)) of
    logits [..., V]: read in place where the rows lie on a grid of two strides (any
    2-d tensor with unit column stride, slices of a 3-d one), else copied."""
    if logits.is_contiguous():
        vocab = logits.shape[-1]
        rows = logits.numel() // vocab
        return logits, logits.data_ptr(), (rows, 1, vocab if rows > 1 else 0, 0)
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        return rows_of(logits.contiguous())
    dims = [(n, s) for n, s in zip(logits.shape[:-1], logits.stride()[:-1]) if n != 1]
    # neighbouring dimensions that are one
    merged: list[tuple[int, int]] = []
    for n, s in dims:
        if merged and merged[-1][1] == n * s:
            merged[-1] = (merged[-1][0] * n, s)
        else:
            merged.append((n, s))
    if len(merged) > 2:
        return rows_of(logits.contiguous())
    if not merged:
        return logits, logits.data_ptr(), (1, 1, 0, 0)
    if len(merged) == 1:
        return logits, logits.data_ptr(), (merged[0][0], 1, merged[0][1], 0)
    (n0, s0), (n1, s1) = merged
    return logits, logits.data_ptr(), (n0 * n1, n1, s0, s1)


# (torch.jit.is_tracing, in half of its time)
is_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)


def wants_autograd(t: torch.Tensor) -> bool:
    """Whether a call on `t` has to go through its autograd function: where a gradient
    is asked for, where `t` has a tangent, which the function refuses, and in a trace,
    which records the function (of a direct call it records the empty results).
    Otherwise the call is made directly, for less host time."""
    return ((t.requires_grad and torch.is_grad_enabled()) or is_tracing()
            or (getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None))


def save_logits(ctx, held: torch.Tensor, rows: tuple[int, int, int, int], *others: torch.Tensor) -> None:
    """Saves what ``rows_of`` returned for the logits, and other tensors (contiguous)."""
    ctx.save_for_backward(held, *others)
    ctx.mec_logits = rows, _f.layout(held), held.shape, [t.nbytes for t in others]


def saved_logits(ctx) -> list:
    """[held, rows, *others] as save_logits had them; the rows are those of the tensor
    that came back."""
    held, *others = ctx.saved_tensors
    rows, saved, shape, nbytes = ctx.mec_logits
    if _f.layout(held) != saved:
        _f.check_unpacked(held, saved, shape)
        held, _, rows = rows_of(held)
    if [t.nbytes for t in others] != nbytes:
        for t, n in zip(others, nbytes):
            _f.check_unpacked_bytes(t, n)
    return [held, rows, *[t.contiguous() for t in others]]


class _Once(torch.autograd.Function):
    """Passes a gradient on that depends on other tensors; a derivative through it is refused."""

    @staticmethod
    def forward(ctx, grad, *others):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("memoryefficientclip_amd: the operators over a vocabulary cannot be differentiated twice")


def backward_of(grad):
    """``Function.backward`` from `grad(ctx, *grad_outputs)`, which is differentiable once.

    Under ``create_graph`` the gradients depend on the saved inputs and on what
    arrived from above, and are tied to them: a derivative through them would
    otherwise be taken for zero without a word.  Otherwise nothing is added, since
    autograd runs this on a thread of its own, where Python code is several times
    slower than on the caller's."""

    def backward(ctx, *grad_outputs):
        if not torch.is_grad_enabled():
            return grad(ctx, *grad_outputs)
        with torch.no_grad():
            found = grad(ctx, *grad_outputs)
        return tuple(g if g is None else _Once.apply(g.requires_grad_(), *grad_outputs, *ctx.saved_tensors)
                     for g in (found if isinstance(found, tuple) else (found,)))

    return staticmethod(backward)


def launch(index: int, nbytes: int, call) -> int:
    """``call(workspace, stream)``, a C-ABI call, on device `index` with `nbytes` of
    the caching allocator's memory in the order of the current stream (< 0: a
    size query's error code).  Returns its status."""
    if nbytes < 0:
        raise _lib.error("size query", nbytes)
    # (the C-ABI calls launch on the current device)
    cur = torch.cuda.current_device()
    if cur != index:
        torch.cuda.set_device(index)
    ws = None
    try:
        if nbytes:
            ws = _f._alloc(nbytes, index)
        return call(ws, _f._stream(index))
    finally:
        if ws is not None:
            torch.cuda.caching_allocator_delete(ws)
        if cur != index:
            torch.cuda.set_device(cur)

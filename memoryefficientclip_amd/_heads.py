"""Host side shared by the operators of a tower's attention: heads as the HIP
library (``include/mec.h``) reads them, and what comes back of them in a backward
pass."""
from __future__ import annotations

import ctypes

import torch

from . import _function as _f
from . import _lib
from . import _vocab as _v


def refuse_graph_capture() -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("memoryefficientclip_amd: the operators of a tower's attention do not support CUDA/HIP graph "
                           "capture; call them outside the captured region")


def check(name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> None:
    """`t` is heads [batch, tokens, heads, head_dim] on the GPU, of the type and on the device of `like`."""
    _v.check_gpu(name, t, None if like is None else like.device)
    _v.check_float(name, t)
    if t.dim() != 4:
        raise ValueError(f"{name} must be [batch, tokens, heads, head_dim], got {tuple(t.shape)}")
    if like is not None and t.dtype != like.dtype:
        raise TypeError(f"dtype mismatch {like.dtype} vs {t.dtype} of {name}")


def of(t: torch.Tensor) -> tuple[torch.Tensor, _lib.Heads]:
    """(tensor to hold, its heads): read in place for any strides but that of the features."""
    s = t.stride()
    if s[3] != 1 and t.shape[3] > 1:
        t = t.contiguous()
        s = t.stride()
    return t, _lib.Heads(t.data_ptr(), s[0], s[1], s[2])


def wants_autograd(*tensors: torch.Tensor | None) -> bool:
    return any(_v.wants_autograd(t) for t in tensors if t is not None)


def save(ctx, *tensors: torch.Tensor | None) -> None:
    ctx.save_for_backward(*tensors)
    ctx.mec_tensors = [None if t is None else (_f.layout(t), t.shape) for t in tensors]


def saved(ctx) -> list[torch.Tensor | None]:
    """What ``save`` saved; a saved-tensor hook may have changed its strides, and nothing else."""
    tensors = list(ctx.saved_tensors)
    for t, had in zip(tensors, ctx.mec_tensors):
        if t is not None and _f.layout(t) != had[0]:
            _f.check_unpacked(t, *had)
    return tensors


def pointer(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


by_reference = ctypes.byref

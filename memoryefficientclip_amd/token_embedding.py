"""Token embedding with a scale, and its gradient summed by sorted tokens: in
32 bits, in a fixed order, without atomics.

    from memoryefficientclip_amd import ScaledTokenEmbedding
    features = ScaledTokenEmbedding(49408, 768, padding_idx=0)(tokens)    # sqrt(768) * weight[tokens]
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _function as _f
from . import _lib
from . import _vocab as _v

_MAX_TOKENS, _MAX_VOCAB, _MAX_DIM = 1 << 23, 1 << 22, 1 << 16


def _check(tokens, weight):
    _v.check_gpu("weight", weight)
    _v.check_gpu("tokens", tokens, weight.device)
    _v.refuse_graph_capture()
    _v.refuse_make_fx()
    _v.check_float("weight", weight)
    _v.check_tokens("tokens", tokens)
    shape, n = weight.shape, tokens.numel()
    if len(shape) != 2 or shape[0] < 1 or shape[1] < 1:
        raise ValueError(f"weight must be [V, D] with V, D >= 1, got {tuple(shape)}")
    vocab, d = shape
    if vocab > _MAX_VOCAB or d > _MAX_DIM or n > _MAX_TOKENS:
        raise ValueError(f"{n} tokens of {vocab} x {d} exceed the maxima {_MAX_TOKENS}, {_MAX_VOCAB} x {_MAX_DIM}")
    return vocab, d, n


def _lookup(tokens, weight, scale):
    w, ldw = _f._rows(weight)
    vocab, d = w.shape
    out = torch.empty((*tokens.shape, d), dtype=w.dtype, device=w.device)
    lib = _lib.load()
    rc = _v.launch(w.device.index, 0, lambda ws, stream: lib.mec_embedding(
        tokens.data_ptr(), tokens.element_size(), tokens.numel(), w.data_ptr(), ldw, vocab, d, _v.code_of(w), scale,
        out.data_ptr(), stream))
    if rc:
        raise _lib.error("mec_embedding", rc)
    return out


def _weight_grad(ctx, grad_output):
    tokens, = ctx.saved_tensors
    saved, shape = ctx.mec_tokens
    if _f.layout(tokens) != saved:
        _f.check_unpacked(tokens, saved, shape)
        tokens = tokens.contiguous()
    vocab, d, n, code, index, scale, padding_idx, nbytes = ctx.mec
    dy, ldg = (grad_output, d) if grad_output.is_contiguous() else _f._rows(grad_output.reshape(-1, d))
    dw = dy.new_empty((vocab, d))
    lib = _lib.load()
    rc = _v.launch(index, nbytes, lambda ws, stream: lib.mec_embedding_backward(
        tokens.data_ptr(), tokens.element_size(), n, dy.data_ptr(), ldg, vocab, d, code, scale, padding_idx,
        dw.data_ptr(), ws, nbytes, stream))
    if rc:
        raise _lib.error("mec_embedding_backward", rc)
    return None, dw, None, None, None


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx, traced):
        if traced:
            _check(tokens, weight)
            tokens = tokens.contiguous()
        out = _lookup(tokens, weight, scale)
        ctx.save_for_backward(tokens)
        ctx.mec_tokens = _f.layout(tokens), tokens.shape
        (vocab, d), n, code = weight.shape, tokens.numel(), _v.code_of(weight)
        ctx.mec = (vocab, d, n, code, weight.device.index, scale, padding_idx,
                   _lib.load().mec_embedding_workspace_bytes(n, vocab, d, code))
        return out

    backward = _v.backward_of(_weight_grad)


def scaled_embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                     padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[tokens]``, [..., D] in the weight's type, rounded once.

    ``tokens`` [...] int64 or int32; ``weight`` [V, D] fp32, bf16 or fp16.  The
    gradient of the weight is dense: ``scale`` times the sum of a token's rows,
    zero for tokens that do not occur and for ``padding_idx`` (whose row is
    looked up like any other).  A token outside [0, V) gives a row of NaN and
    has no part in the gradient.  Up to 2^23 tokens, V up to 2^22, D up to 2^16.
    """
    vocab, d, n = _check(tokens, weight)
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    if padding_idx is None:
        padding_idx = -1
    elif not -vocab <= padding_idx < vocab:
        raise ValueError(f"padding_idx must be in [{-vocab}, {vocab}), got {padding_idx}")
    elif padding_idx < 0:
        padding_idx += vocab
    if n == 0:
        return weight[:0].sum() * scale + torch.empty((*tokens.shape, d), dtype=weight.dtype, device=weight.device)
    tokens = tokens.contiguous()
    if _v.wants_autograd(weight):
        return _EmbeddingFn.apply(tokens, weight, scale, int(padding_idx), _v.is_tracing())
    return _lookup(tokens, weight, scale)


class ScaledTokenEmbedding(nn.Module):
    """``forward(tokens)``: :func:`scaled_embedding` of a weight of its own.

    ``scale`` defaults to sqrt(embedding_dim); the weight starts normal with
    standard deviation 1 / sqrt(embedding_dim), so that the default scale gives
    features of variance 1; the row of ``padding_idx`` starts at zero.
    """

    def __init__(self, num_embeddings, embedding_dim, scale=None, padding_idx=None, device=None, dtype=None):
        super().__init__()
        self.num_embeddings = num_embeddings
        self.embedding_dim = embedding_dim
        self.scale = math.sqrt(embedding_dim) if scale is None else float(scale)
        if padding_idx is not None and not -num_embeddings <= padding_idx < num_embeddings:
            raise ValueError(f"padding_idx must be in [{-num_embeddings}, {num_embeddings}), got {padding_idx}")
        self.padding_idx = padding_idx
        self.weight = nn.Parameter(torch.empty((num_embeddings, embedding_dim), device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.normal_(self.weight, std=1.0 / math.sqrt(self.embedding_dim))
        if self.padding_idx is not None:
            with torch.no_grad():
                self.weight[self.padding_idx].zero_()

    def forward(self, tokens):
        return scaled_embedding(tokens, self.weight, self.scale, self.padding_idx)

    def extra_repr(self):
        pad = "" if self.padding_idx is None else f", padding_idx={self.padding_idx}"
        return f"{self.num_embeddings}, {self.embedding_dim}, scale={self.scale:g}{pad}"


__all__ = ["ScaledTokenEmbedding", "scaled_embedding"]

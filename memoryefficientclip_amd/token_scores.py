"""Log probabilities of given tokens under a model's logits, with the entropy of
the distribution and its most probable tokens, in one pass over the logits and
differentiable in the first two.

    from memoryefficientclip_amd import token_log_probs
    r = token_log_probs(logits, tokens, top_k=32)
    r.log_probs, r.entropy, r.top_tokens, r.top_log_probs

No probability of a token that was not asked for is kept: beside the logits the
forward holds two floats per position for the backward.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from . import _vocab as _v


class TokenScores(NamedTuple):
    """Results of :func:`token_log_probs`, shaped like its tokens."""
    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_tokens: torch.Tensor | None
    top_log_probs: torch.Tensor | None


class _TokenScoresFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature, ignore_index):
        code, token_bytes = _v.check_float("logits", logits), _v.check_tokens("tokens", tokens)
        held, px, rows = _v.rows_of(logits)
        tokens = tokens.contiguous()
        vocab, dev = logits.shape[-1], logits.device
        di = dev.index
        log_probs = torch.empty(tokens.shape, dtype=torch.float32, device=dev)
        entropy = torch.empty(tokens.shape, dtype=torch.float32, device=dev)
        top_tokens = torch.empty((*tokens.shape, top_k), dtype=torch.int64, device=dev)
        top_log_probs = torch.empty((*tokens.shape, top_k), dtype=torch.float32, device=dev)
        state = torch.empty(2 * rows[0], dtype=torch.float32, device=dev)
        lib = _lib.load()
        with _v.on_device(di) as stream:
            nbytes = lib.mec_token_scores_workspace_bytes(rows[0], vocab, top_k, code)
            with _v.scratch(nbytes, di) as ws:
                rc = lib.mec_token_scores(px, *rows, vocab, code, tokens.data_ptr(), token_bytes, ignore_index,
                                          temperature, top_k, log_probs.data_ptr(), entropy.data_ptr(),
                                          top_tokens.data_ptr(), top_log_probs.data_ptr(), state.data_ptr(), ws,
                                          nbytes, stream)
        if rc:
            raise _lib.error("mec_token_scores", rc)
        ctx.mark_non_differentiable(top_tokens, top_log_probs)
        ctx.set_materialize_grads(False)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(held, tokens, entropy, state)
            ctx.mec = (rows, vocab, code, token_bytes, ignore_index, temperature, logits.shape)
        return log_probs, entropy, top_tokens, top_log_probs

    @staticmethod
    @once_differentiable
    def backward(ctx, g_log_probs, g_entropy, _g_tokens, _g_top):
        if not ctx.needs_input_grad[0] or (g_log_probs is None and g_entropy is None):
            return None, None, None, None, None
        _v.refuse_graph_capture()
        held, tokens, entropy, state = ctx.saved_tensors
        rows, vocab, code, token_bytes, ignore_index, temperature, shape = ctx.mec
        gl = None if g_log_probs is None else g_log_probs.to(torch.float32).contiguous()
        gh = None if g_entropy is None else g_entropy.to(torch.float32).contiguous()
        dx = torch.empty(shape, dtype=held.dtype, device=held.device)
        with _v.on_device(held.device.index) as stream:
            _lib.call("mec_token_scores_backward", held.data_ptr(), *rows, vocab, code, tokens.data_ptr(), token_bytes,
                      ignore_index, temperature, state.data_ptr(), entropy.data_ptr(),
                      None if gl is None else gl.data_ptr(), None if gh is None else gh.data_ptr(), dx.data_ptr(),
                      stream)
        return dx, None, None, None, None


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0, temperature: float = 1.0,
                    ignore_index: int = -100) -> TokenScores:
    """Scores of ``tokens`` [...] under ``softmax(logits / temperature)``, logits [..., V].

    * ``log_probs``, ``entropy``: fp32, shaped like ``tokens``; gradients flow to
      the logits through both.
    * ``top_tokens`` (int64), ``top_log_probs`` (fp32, no gradient): [..., top_k],
      the most probable tokens in order, the lower token first among equals, NaN
      before everything; ``None`` for ``top_k=0``.

    Positions whose token is ``ignore_index`` score 0, with top tokens -1, and
    have no gradient; other tokens outside [0, V) score NaN.  Logits of -inf are
    tokens that cannot occur; where none can, every log probability is -inf, the
    entropy 0 and the gradient 0.

    fp32, bf16 and fp16 logits, read in place (any row strides), V up to 2^19 and
    ``top_k`` up to 128; int64 or int32 tokens.
    """
    _v.check_gpu("logits", logits)
    _v.check_gpu("tokens", tokens, logits.device)
    _v.refuse_graph_capture()
    _v.check_float("logits", logits)
    _v.check_tokens("tokens", tokens)
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape:
        raise ValueError(f"logits {tuple(logits.shape)} need one row for each of the tokens {tuple(tokens.shape)}")
    vocab, top_k = logits.shape[-1], int(top_k)
    if not 1 <= vocab <= _lib.MAX_VOCAB:
        raise ValueError(f"the vocabulary must have 1 to {_lib.MAX_VOCAB} tokens, got {vocab}")
    if not 0 <= top_k <= min(vocab, _lib.MAX_TOP_K):
        raise ValueError(f"top_k must be in [0, {min(vocab, _lib.MAX_TOP_K)}], got {top_k}")
    temperature = _v.check_temperature(temperature)
    if tokens.numel() == 0:
        zero = logits.sum(-1, dtype=torch.float32)  # (no element: the graph's link to the logits)
        return TokenScores(zero, zero.clone(),
                           torch.empty((*tokens.shape, top_k), dtype=torch.int64, device=logits.device) if top_k else None,
                           zero.detach()[..., None].expand(*tokens.shape, top_k) if top_k else None)
    lp, h, tt, tlp = _TokenScoresFn.apply(logits, tokens, top_k, temperature, int(ignore_index))
    return TokenScores(lp, h, tt if top_k else None, tlp if top_k else None)


__all__ = ["TokenScores", "token_log_probs"]

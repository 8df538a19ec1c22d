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

from . import _lib
from . import _vocab as _v


class TokenScores(NamedTuple):
    """Results of :func:`token_log_probs`, shaped like its tokens."""
    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_tokens: torch.Tensor | None
    top_log_probs: torch.Tensor | None


def _check(logits, tokens, top_k):
    _v.check_gpu("logits", logits)
    _v.check_gpu("tokens", tokens, logits.device)
    _v.refuse_graph_capture()
    _v.refuse_make_fx()
    shape = logits.shape
    if len(shape) < 1 or shape[:-1] != tokens.shape:
        raise ValueError(f"logits {tuple(shape)} need one row for each of the tokens {tuple(tokens.shape)}")
    _v.check_float("logits", logits)
    _v.check_tokens("tokens", tokens)
    vocab, top_k = shape[-1], int(top_k)
    if not 1 <= vocab <= _lib.MAX_VOCAB:
        raise ValueError(f"the vocabulary must have 1 to {_lib.MAX_VOCAB} tokens, got {vocab}")
    if not 0 <= top_k <= min(vocab, _lib.MAX_TOP_K):
        raise ValueError(f"top_k must be in [0, {min(vocab, _lib.MAX_TOP_K)}], got {top_k}")


def _scores(logits, rows, tokens, top_k, temperature, ignore_index, keep):
    """Results, and with `keep` what the backward needs of them; logits and their rows as ``rows_of`` has them."""
    code, token_bytes = _v.code_of(logits), tokens.element_size()
    tokens = tokens.contiguous()
    vocab, dev, shape = logits.shape[-1], logits.device, tokens.shape
    log_probs = torch.empty(shape, dtype=torch.float32, device=dev)
    entropy = torch.empty(shape, dtype=torch.float32, device=dev)
    top_tokens = top_log_probs = state = None
    if top_k:
        top_tokens = torch.empty((*shape, top_k), dtype=torch.int64, device=dev)
        top_log_probs = torch.empty((*shape, top_k), dtype=torch.float32, device=dev)
    if keep:
        state = torch.empty(2 * rows[0], dtype=torch.float32, device=dev)
    lib = _lib.load()
    nbytes = lib.mec_token_scores_workspace_bytes(rows[0], vocab, top_k, code)
    rc = _v.launch(dev.index, nbytes, lambda ws, stream: lib.mec_token_scores(
        logits.data_ptr(), *rows, vocab, code, tokens.data_ptr(), token_bytes, ignore_index, temperature, top_k,
        log_probs.data_ptr(), entropy.data_ptr(), top_tokens.data_ptr() if top_k else None,
        top_log_probs.data_ptr() if top_k else None, state.data_ptr() if keep else None, ws, nbytes, stream))
    if rc:
        raise _lib.error("mec_token_scores", rc)
    kept = (logits, rows, tokens, entropy, state), (vocab, code, token_bytes, ignore_index, temperature)
    return (log_probs, entropy, top_tokens, top_log_probs), kept


def _logits_grad(ctx, g_log_probs, g_entropy, _g_tokens, _g_top):
    if g_log_probs is None and g_entropy is None:
        return None, None, None, None, None, None
    held, rows, tokens, entropy, state = _v.saved_logits(ctx)
    vocab, code, token_bytes, ignore_index, temperature = ctx.mec
    gl = None if g_log_probs is None else g_log_probs.contiguous()
    gh = None if g_entropy is None else g_entropy.contiguous()
    dx = held.new_empty(held.shape)
    lib = _lib.load()
    rc = _v.launch(held.device.index, 0, lambda ws, stream: lib.mec_token_scores_backward(
        held.data_ptr(), *rows, vocab, code, tokens.data_ptr(), token_bytes, ignore_index, temperature,
        state.data_ptr(), entropy.data_ptr(), None if gl is None else gl.data_ptr(),
        None if gh is None else gh.data_ptr(), dx.data_ptr(), stream))
    if rc:
        raise _lib.error("mec_token_scores_backward", rc)
    return dx, None, None, None, None, None


class _TokenScoresFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rows, tokens, top_k, temperature, ignore_index):
        if rows is None:
            _check(logits, tokens, top_k)
            logits, _, rows = _v.rows_of(logits)
        out, kept = _scores(logits, rows, tokens, top_k, temperature, ignore_index, True)
        if top_k:
            ctx.mark_non_differentiable(out[2], out[3])
        ctx.set_materialize_grads(False)
        _v.save_logits(ctx, *kept[0])
        ctx.mec = kept[1]
        return out

    backward = _v.backward_of(_logits_grad)


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0, temperature: float = 1.0,
                    ignore_index: int = -100) -> TokenScores:
    """Scores of ``tokens`` [...] under ``softmax(logits / temperature)``, logits [..., V].

    * ``log_probs``, ``entropy``: fp32, shaped like ``tokens``; gradients flow to
      the logits through both.
    * ``top_tokens`` (int64), ``top_log_probs`` (fp32, no gradient): [..., top_k],
      the most probable tokens in order, the lower token first among equals, NaN
      before everything; ``None`` for ``top_k=0``.

    Positions whose token is ``ignore_index`` score 0, with top tokens -1, and
    have no gradient; other tokens outside [0, V) score NaN (the entropy of their
    position and its gradient do not depend on them).  Logits of -inf are tokens
    that cannot occur; where none can, every log probability is -inf, the
    entropy 0 and the gradient 0.

    fp32, bf16 and fp16 logits, read in place (any row strides), V up to 2^19 and
    ``top_k`` up to 128; int64 or int32 tokens.
    """
    _check(logits, tokens, top_k)
    top_k = int(top_k)
    temperature = _v.check_temperature(temperature)
    if tokens.numel() == 0:
        zero = logits.sum(-1, dtype=torch.float32)  # (no element: the graph's link to the logits)
        none = torch.empty((*tokens.shape, top_k), dtype=torch.int64, device=logits.device)
        return TokenScores(zero, zero.clone(), none if top_k else None, none.float() if top_k else None)
    logits, _, rows = _v.rows_of(logits)
    if _v.wants_autograd(logits):
        # (a trace calls this again, with other inputs)
        rows = None if _v.is_tracing() else rows
        return TokenScores(*_TokenScoresFn.apply(logits, rows, tokens, top_k, temperature, int(ignore_index)))
    return TokenScores(*_scores(logits, rows, tokens, top_k, temperature, int(ignore_index), False)[0])


__all__ = ["TokenScores", "token_log_probs"]

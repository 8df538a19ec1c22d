"""Attention of a tower's heads, forward and backward, without a matrix of scores
in memory: the forward keeps one number a query and head, from which the backward
makes the probabilities anew.

    from memoryefficientclip_amd import attention, norm_rotary
    q, k, v = qkv.split([heads, key_heads, key_heads], 2)       # [batch, tokens, heads, head_dim]
    q, k = norm_rotary(q, k, positions, sections, q_weight, k_weight, eps=1e-6)
    features = attention(q, k, v, causal=True, query_lengths=n, key_lengths=n).flatten(2)
"""
from __future__ import annotations

import math

import torch

from . import _heads as _h
from . import _lib
from . import _vocab as _v

_MAX = 1 << 30


def _check(query, key, value, query_lengths, key_lengths):
    _h.check("query", query)
    _h.check("key", key, query)
    _h.check("value", value, query)
    _h.refuse_graph_capture()
    _v.refuse_make_fx()
    (b, nq, h, d), (bk, nk, hk, dk) = query.shape, key.shape
    if key.shape != value.shape:
        raise ValueError(f"key {tuple(key.shape)} and value {tuple(value.shape)} differ in shape")
    if b != bk or d != dk:
        raise ValueError(f"query {tuple(query.shape)} and key {tuple(key.shape)} need the same batch and head_dim")
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"the {hk} heads of the keys must divide the {h} heads of the queries")
    if not 1 <= d <= _lib.MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be in [1, {_lib.MAX_HEAD_DIM}], got {d}")
    if max(b * hk, nq * (h // hk), nk) > _MAX:
        raise ValueError(f"query {tuple(query.shape)} and key {tuple(key.shape)} exceed the maximum 2^30 of batch * key "
                         f"heads, queries * heads / key heads, or keys")
    for name, n in (("query_lengths", query_lengths), ("key_lengths", key_lengths)):
        if n is not None:
            _v.check_gpu(name, n, query.device)
            _v.check_tokens(name, n)
            if n.shape != (b,):
                raise ValueError(f"{name} must be [{b}], got {tuple(n.shape)}")
    if query_lengths is not None and key_lengths is not None and query_lengths.dtype != key_lengths.dtype:
        raise TypeError(f"dtype mismatch {query_lengths.dtype} vs {key_lengths.dtype} of the lengths")


def _problem(q, k, causal, scale, query_lengths, key_lengths):
    (b, nq, h, d), (_, nk, hk, _) = q.shape, k.shape
    some = key_lengths if query_lengths is None else query_lengths
    return _lib.Attention(b, nq, nk, h, hk, d, _v.code_of(q), causal, scale, 0 if some is None else some.element_size(),
                          _h.pointer(query_lengths), _h.pointer(key_lengths))


def _attend(q, k, v, causal, scale, query_lengths, key_lengths, keep):
    q, heads_q = _h.of(q)
    k, heads_k = _h.of(k)
    v, heads_v = _h.of(v)
    problem = _h.by_reference(_problem(q, k, causal, scale, query_lengths, key_lengths))
    b, nq, h, _ = q.shape
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((b, h, nq), dtype=torch.float32, device=q.device) if keep else None
    lib = _lib.load()
    # (the size depends on the current device's compute units)
    rc = _v.launch_sized(q.device.index, lambda: lib.mec_attention_workspace_bytes(problem),
                         lambda ws, nbytes, stream: lib.mec_attention(
                             problem, _h.by_reference(heads_q), _h.by_reference(heads_k), _h.by_reference(heads_v),
                             out.data_ptr(), _h.pointer(lse), ws, nbytes, stream))
    if rc:
        raise _lib.error("mec_attention", rc)
    return out, (q, k, v, lse)


def _grads(ctx, grad_out):
    q, k, v, out, lse, query_lengths, key_lengths = _h.saved(ctx)
    causal, scale = ctx.mec
    (q, heads_q), (k, heads_k), (v, heads_v), (grad_out, heads_g) = _h.of(q), _h.of(k), _h.of(v), _h.of(grad_out)
    out, lse = out.contiguous(), lse.contiguous()
    query_lengths, key_lengths = (n if n is None else n.contiguous() for n in (query_lengths, key_lengths))
    problem = _h.by_reference(_problem(q, k, causal, scale, query_lengths, key_lengths))
    need = ctx.needs_input_grad
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device) if need[0] else None
    dk, dv = (torch.empty(k.shape, dtype=k.dtype, device=k.device) if need[1] or need[2] else None for _ in "kv")
    lib = _lib.load()
    rc = _v.launch_sized(q.device.index, lambda: lib.mec_attention_backward_workspace_bytes(problem),
                         lambda ws, nbytes, stream: lib.mec_attention_backward(
                             problem, _h.by_reference(heads_q), _h.by_reference(heads_k), _h.by_reference(heads_v),
                             out.data_ptr(), lse.data_ptr(), _h.by_reference(heads_g), _h.pointer(dq), _h.pointer(dk),
                             _h.pointer(dv), ws, nbytes, stream))
    if rc:
        raise _lib.error("mec_attention_backward", rc)
    return dq, dk if need[1] else None, dv if need[2] else None, None, None, None, None, None


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, causal, scale, query_lengths, key_lengths, traced):
        if traced:
            _check(query, key, value, query_lengths, key_lengths)
            query_lengths, key_lengths = (n if n is None else n.contiguous() for n in (query_lengths, key_lengths))
        out, (q, k, v, lse) = _attend(query, key, value, causal, scale, query_lengths, key_lengths, True)
        _h.save(ctx, q, k, v, out, lse, query_lengths, key_lengths)
        ctx.mec = causal, scale
        return out

    backward = _v.backward_of(_grads)


def attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, causal: bool = False,
              scale: float | None = None, query_lengths: torch.Tensor | None = None,
              key_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale * query @ key^T) @ value`` for each head, [batch, queries, heads, head_dim].

    ``query`` [batch, queries, heads, head_dim]; ``key``, ``value`` [batch, keys,
    key_heads, head_dim], where ``key_heads`` divides ``heads`` and each key head serves
    ``heads / key_heads`` neighbouring heads.  fp32, bf16 or fp16; any strides (slices of
    a fused projection are read in place).  ``scale`` defaults to 1 / sqrt(head_dim).

    ``query_lengths``, ``key_lengths`` [batch], int64 or int32, on the GPU: what lies at or
    beyond them is padding, which is not read; padded queries give 0, and padding has a
    gradient of 0.  With ``causal`` query i of n sees the keys up to i + m - n of m (the
    lengths, where given): the last query sees the last key, as for new tokens over the
    keys of all tokens so far.  A query that sees no key gives 0 and has no gradient.  What
    a query does not see has no part in its result, not even inf or NaN.

    head_dim up to 128; any lengths.  The result and the gradients are deterministic.
    """
    _check(query, key, value, query_lengths, key_lengths)
    scale = 1.0 / math.sqrt(query.shape[3]) if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"scale must be in [1e-30, 1e30], got {scale}")
    if query.numel() == 0 or key.numel() == 0:
        # nothing to see, or nothing that sees: the graph's link to the inputs
        zero = query[..., :0].sum(-1, keepdim=True) + (key[:, :0].sum() + value[:, :0].sum())
        return zero.expand(query.shape).contiguous()
    query_lengths, key_lengths = (n if n is None else n.contiguous() for n in (query_lengths, key_lengths))
    if _h.wants_autograd(query, key, value):
        return _AttentionFn.apply(query, key, value, bool(causal), scale, query_lengths, key_lengths, _v.is_tracing())
    return _attend(query, key, value, bool(causal), scale, query_lengths, key_lengths, False)[0]


__all__ = ["attention"]

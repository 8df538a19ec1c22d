"""Rotation of queries and keys by positions on several axes, with the norm of each
head in the same pass, and its gradient.

    from memoryefficientclip_amd import norm_rotary
    positions = torch.cartesian_prod(torch.arange(height), torch.arange(width))     # [tokens, 2], on the GPU
    q, k = norm_rotary(q, k, positions, (16, 16), q_weight, k_weight, eps=1e-6)     # heads of 64: 32 pairs
"""
from __future__ import annotations

import math

import torch

from . import _function as _f
from . import _heads as _h
from . import _lib
from . import _vocab as _v

_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}  # MEC_POSITION_*
_MAX_DIM, _MAX_TOKENS, _MAX_HEADS = 256, (1 << 31) - 1, 1 << 16


def _check(query, key, positions, sections, query_weight, key_weight, eps, frequencies):
    _h.check("query", query)
    _h.check("key", key, query)
    _v.check_gpu("positions", positions, query.device)
    _h.refuse_graph_capture()
    _v.refuse_make_fx()
    (b, n, h, d), (bk, nk, hk, dk) = query.shape, key.shape
    if (b, n, d) != (bk, nk, dk):
        raise ValueError(f"query {tuple(query.shape)} and key {tuple(key.shape)} may differ in their heads only")
    if h < 1 or hk < 1 or max(h, hk) > _MAX_HEADS:
        raise ValueError(f"query and key need 1 to {_MAX_HEADS} heads, got {h} and {hk}")
    if d < 2 or d % 2 or d > _MAX_DIM:
        raise ValueError(f"head_dim must be even and in [2, {_MAX_DIM}], got {d}")
    if b * n > _MAX_TOKENS:
        raise ValueError(f"{b} x {n} tokens exceed the maximum 2^31 - 1")
    if not 1 <= len(sections) <= _lib.MAX_AXES or min(sections) < 0 or 2 * sum(sections) != d:
        raise ValueError(f"sections must be the pairs of 1 to {_lib.MAX_AXES} axes, {d // 2} together, got {sections}")
    if positions.dtype not in _POSITIONS:
        raise TypeError(f"unsupported dtype {positions.dtype} of positions; supported: int64, int32, float32")
    axes = len(sections)
    if positions.shape not in ((n, axes), (b, n, axes)):
        raise ValueError(f"positions must be [{n}, {axes}] or [{b}, {n}, {axes}], got {tuple(positions.shape)}")
    for name, w in (("query_weight", query_weight), ("key_weight", key_weight)):
        if w is not None:
            _v.check_gpu(name, w, query.device)
            _v.check_float(name, w)
            if eps is None:
                raise ValueError(f"{name} needs a norm: give eps")
            if w.shape != (d,):
                raise ValueError(f"{name} must be [{d}], got {tuple(w.shape)}")
    if query_weight is not None and key_weight is not None and query_weight.dtype != key_weight.dtype:
        raise TypeError(f"dtype mismatch {query_weight.dtype} vs {key_weight.dtype} of the weights")
    if frequencies is not None:
        _v.check_gpu("frequencies", frequencies, query.device)
        if frequencies.dtype not in (torch.float64, torch.float32):
            raise TypeError(f"unsupported dtype {frequencies.dtype} of frequencies; supported: float64, float32")
        if frequencies.shape != (d // 2,):
            raise ValueError(f"frequencies must be [{d // 2}], got {tuple(frequencies.shape)}")


def _rotary(shape, key_heads, dtype, positions, sections, query_weight, key_weight, eps, theta, frequencies, interleaved):
    b, n, h, d = shape
    w = query_weight if query_weight is not None else key_weight
    return _lib.Rotary(b, n, h, key_heads, d, dtype, _lib.DTYPE_F32 if w is None else _v.code_of(w), int(eps is not None),
                       int(interleaved), 0.0 if eps is None else eps, len(sections), (*sections,),
                       _POSITIONS[positions.dtype], int(positions.dim() == 3), theta, _h.pointer(query_weight),
                       _h.pointer(key_weight), positions.data_ptr(), _h.pointer(frequencies))


def _turn(q, k, positions, query_weight, key_weight, frequencies, sections, eps, theta, interleaved):
    q, heads_q = _h.of(q)
    k, heads_k = _h.of(k)
    rotary = _rotary(q.shape, k.shape[2], _v.code_of(q), positions, sections, query_weight, key_weight, eps, theta,
                     frequencies, interleaved)
    out_q = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    out_k = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    lib = _lib.load()
    rc = _v.launch(q.device.index, 0, lambda ws, stream: lib.mec_norm_rotary(
        _h.by_reference(rotary), _h.by_reference(heads_q), _h.by_reference(heads_k), out_q.data_ptr(),
        out_k.data_ptr(), stream))
    if rc:
        raise _lib.error("mec_norm_rotary", rc)
    return out_q, out_k, q, k


def _grads(ctx, grad_q, grad_k):
    sections, eps, theta, interleaved, shape, key_heads, dtype, device = ctx.mec
    q, k, positions, query_weight, key_weight, frequencies = _h.saved(ctx)
    positions, query_weight, key_weight, frequencies = (
        t if t is None else t.contiguous() for t in (positions, query_weight, key_weight, frequencies))
    need = ctx.needs_input_grad
    # a side whose result was not used, or nothing of which is asked for, has no part
    b, n, h, d = shape
    h = h if grad_q is not None and (need[0] or need[3]) else 0
    key_heads = key_heads if grad_k is not None and (need[1] or need[4]) else 0
    none = (None,) * 10
    if h + key_heads == 0:
        return none
    norm = eps is not None
    code = _f._DTYPES[dtype]
    sides = []
    for x, grad, heads, wanted, w, weight_wanted in ((q, grad_q, h, need[0], query_weight, need[3]),
                                                     (k, grad_k, key_heads, need[1], key_weight, need[4])):
        heads_x = heads_g = dx = dw = None
        if heads:
            grad, heads_g = _h.of(grad)
            if norm:
                x, heads_x = _h.of(x)
            if wanted:
                dx = torch.empty((b, n, heads, d), dtype=dtype, device=device)
            if weight_wanted:
                dw = torch.empty_like(w)
        sides.append((x, grad, heads_x, heads_g, dx, dw))
    (q, grad_q, heads_q, heads_gq, dq, dwq), (k, grad_k, heads_k, heads_gk, dk, dwk) = sides
    rotary = _rotary((b, n, h, d), key_heads, code, positions, sections, query_weight, key_weight, eps, theta,
                     frequencies, interleaved)
    reference = lambda heads: None if heads is None else _h.by_reference(heads)  # noqa: E731
    lib = _lib.load()
    weights = dwq is not None or dwk is not None
    # (the size depends on the current device's compute units)
    rc = _v.launch_sized(device.index,
                         lambda: lib.mec_norm_rotary_workspace_bytes(_h.by_reference(rotary)) if weights else 0,
                         lambda ws, nbytes, stream: lib.mec_norm_rotary_backward(
                             _h.by_reference(rotary), reference(heads_q), reference(heads_k), reference(heads_gq),
                             reference(heads_gk), _h.pointer(dq), _h.pointer(dk), _h.pointer(dwq), _h.pointer(dwk),
                             ws, nbytes, stream))
    if rc:
        raise _lib.error("mec_norm_rotary_backward", rc)
    return dq, dk, None, dwq, dwk, None, None, None, None, None


class _NormRotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, positions, query_weight, key_weight, frequencies, sections, eps, theta, traced):
        theta, interleaved = theta
        if ctx.needs_input_grad[2] or ctx.needs_input_grad[5]:
            # (it would be taken for zero without a word)
            raise RuntimeError("memoryefficientclip_amd: norm_rotary has no gradient for positions and frequencies; detach "
                               "them")
        if traced:
            _check(query, key, positions, sections, query_weight, key_weight, eps, frequencies)
            positions, query_weight, key_weight, frequencies = _plain(positions, query_weight, key_weight, frequencies)
        out_q, out_k, q, k = _turn(query, key, positions, query_weight, key_weight, frequencies, sections, eps, theta,
                                   interleaved)
        norm = eps is not None
        ctx.set_materialize_grads(False)
        # (the turn's gradient needs no inputs)
        _h.save(ctx, q if norm else None, k if norm else None, positions, query_weight, key_weight, frequencies)
        ctx.mec = sections, eps, theta, interleaved, query.shape, key.shape[2], query.dtype, query.device
        return out_q, out_k

    backward = _v.backward_of(_grads)


def _plain(positions, query_weight, key_weight, frequencies):
    return (positions.contiguous(), *(w if w is None else w.contiguous() for w in (query_weight, key_weight)),
            frequencies if frequencies is None else frequencies.double().contiguous())


def norm_rotary(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor, sections,
                query_weight: torch.Tensor | None = None, key_weight: torch.Tensor | None = None,
                eps: float | None = None, theta: float = 10000.0, frequencies: torch.Tensor | None = None,
                interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys, each head normed and turned by its token's positions, rounded once.

    ``query`` [batch, tokens, heads, head_dim], ``key`` [batch, tokens, key_heads, head_dim],
    fp32, bf16 or fp16, any strides (slices of a fused projection are read in place).

    * Norm, where ``eps`` is given: ``x / sqrt(mean(x^2) + eps)`` of each head, times
      ``query_weight`` or ``key_weight`` [head_dim] (``None``: ones; any of the three types).
    * Rotation: ``positions`` [tokens, axes] or [batch, tokens, axes], int64, int32 or
      float32; ``sections`` gives the pairs of features that each axis turns, head_dim / 2
      together.  A pair is (x[p], x[p + head_dim / 2]), or (x[2p], x[2p + 1]) if
      ``interleaved``, and is turned by position * frequency, formed in 64 bits.  The j-th
      pair of an axis's n has the frequency ``theta ** (-j / n)``, or give ``frequencies``
      [head_dim / 2] (float64 or float32; 0 leaves a pair as it is).

    Gradients flow to query, key and the weights; those of the weights are summed in fp32,
    in a fixed order.  Positions or frequencies that ask for one are refused.  head_dim
    even, up to 256; up to 8 axes.
    """
    sections = tuple(int(n) for n in sections)
    _check(query, key, positions, sections, query_weight, key_weight, eps, frequencies)
    theta = float(theta)
    if not (theta > 0.0 and math.isfinite(theta)):
        raise ValueError(f"theta must be finite and > 0, got {theta}")
    if eps is not None:
        eps = float(eps)
        if not 0.0 <= eps <= 3e38:
            raise ValueError(f"eps must be finite and >= 0, got {eps}")
    if query.numel() == 0:
        # no token: the graph's link to the inputs
        links = [w.sum() * 0 for w in (query_weight, key_weight) if w is not None]
        return tuple(x * 1 + sum(links).to(x.dtype) if links else x * 1 for x in (query, key))
    positions, query_weight, key_weight, frequencies = _plain(positions, query_weight, key_weight, frequencies)
    args = (query, key, positions, query_weight, key_weight, frequencies, sections, eps)
    if _h.wants_autograd(query, key, query_weight, key_weight, positions, frequencies):
        return _NormRotaryFn.apply(*args, (theta, bool(interleaved)), _v.is_tracing())
    return _turn(*args, theta, bool(interleaved))[:2]


__all__ = ["norm_rotary"]

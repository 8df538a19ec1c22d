"""Plain definitions, in 64 bits on the CPU, of the operators of a tower's attention,
and the errors that their arithmetic allows.

u is half a step of the type (eps / 2): a result is rounded once, and so are, for
16-bit types, the probabilities and their gradients that the products of the values
take.  Everything else is fp32, half a step of which is E.
"""
import math

import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(name, got, want, tolerance):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    off = torch.where(torch.isnan(want) | (got == want), torch.zeros_like(want), (got - want).abs() - tolerance)
    assert not (off > 0).any(), (f"{name}: {int((off > 0).sum())} of {off.numel()} off, by up to {off.max():.3g} beyond "
                                 f"the tolerance there; first at {(off > 0).nonzero()[0].tolist()}")


def sees(batch, queries, keys, causal, query_lengths, key_lengths):
    """[batch, queries, keys]"""
    nq = torch.full((batch,), queries) if query_lengths is None else query_lengths.cpu().long().clamp(0, queries)
    nk = torch.full((batch,), keys) if key_lengths is None else key_lengths.cpu().long().clamp(0, keys)
    i, j = torch.arange(queries)[:, None], torch.arange(keys)
    see = (i < nq[:, None, None]) & (j < nk[:, None, None])
    if causal:
        see = see & (j <= i + (nk - nq)[:, None, None])
    return see


def attention(q, k, v, do=None, causal=False, scale=None, query_lengths=None, key_lengths=None):
    """{"out": (value, tolerance)} and with `do` "dq", "dk", "dv" too, of tensors [batch, tokens, heads, d].

    Errors.  A score is a sum of d products in fp32, off by (d + 2) E sum |q k| scale at most, where the 2 are the
    scale and the difference to the maximum; so much is a probability off, relative, beside 4 E of the exponential
    and n E of the sum (and as much of the maximum's lag) -> e.  Rounding a probability to T: u.  A sum of n
    products in fp32: n E of the sum of their sizes.
    """
    dtype = q.dtype
    q, k, v = (t.detach().cpu() for t in (q, k, v))
    b, nq, h, d = q.shape
    nk, hk = k.shape[1:3]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    see = sees(b, nq, nk, causal, query_lengths, key_lengths)[:, None]
    heads = lambda t, seen: t.double().permute(0, 2, 1, 3).masked_fill(~seen, 0.0)  # noqa: E731
    # (what nobody sees, or that sees nothing, is not looked at)
    qd, kd, vd = heads(q, see.any(3)[..., None]), heads(k, see.any(2)[..., None]), heads(v, see.any(2)[..., None])
    many = lambda t: t.repeat_interleave(h // hk, 1)  # noqa: E731
    few = lambda t: t.unflatten(1, (hk, h // hk)).sum(2)  # noqa: E731
    back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    kd, vd = many(kd), many(vd)
    at = lambda a, x: _masked_product(a, x, see)  # noqa: E731
    s = qd @ kd.transpose(2, 3) * scale
    es = (d + 2) * E * scale * (qd.abs() @ kd.abs().transpose(2, 3))
    s = s.masked_fill(~see, -math.inf)
    m = s.amax(3, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    es = es.masked_fill(~see, 0.0)
    e = es + es.amax(3, keepdim=True) + (2 * nk + 8) * E
    u = half_step(dtype)
    # (fp32 keeps its probabilities; the fp16 ones lose what lies 2^-30 below the largest; the exponential of
    # fp32 is 0 below its least normal number, 2^-126)
    up = 0.0 if dtype == torch.float32 else u
    lost = (2.0 ** -30 if dtype == torch.float16 else 0.0) * p.amax(3, keepdim=True) * see + 2.0 ** -126 * see
    pe = p * (e + up) + lost
    out = at(p, vd)
    tout = at(pe + p * nk * E, vd.abs()) + u * out.abs()
    # (the least number of the type)
    tiny = torch.finfo(dtype).tiny * u * 2
    found = {"out": (back(out), back(tout + tiny))}
    if do is None:
        return found
    g = heads(do.detach().cpu(), see.any(3)[..., None])
    dv = few(_masked_product(p.transpose(2, 3), g, see.transpose(2, 3)))
    n = nq * (h // hk)
    tdv = few(_masked_product((pe + p * n * E).transpose(2, 3), g.abs(), see.transpose(2, 3))) + u * dv.abs()
    dp, delta = g @ vd.transpose(2, 3), (g * out).sum(3, keepdim=True)
    edp = (d + 1) * E * (g.abs() @ vd.abs().transpose(2, 3))
    # (delta is made from the rounded result)
    edelta = (g.abs() * (tout + d * E * out.abs())).sum(3, keepdim=True)
    ds = (p * (dp - delta)).masked_fill(~see, 0.0)
    # (the backward's probabilities come from lse: the same e, and are not rounded on the way to ds)
    eds = (p * (e + 4 * E) + lost) * (dp - delta).abs() + p * (edp + edelta) + up * ds.abs()
    eds = eds.masked_fill(~see, 0.0)
    if dtype == torch.float16:
        eds = eds + 2.0 ** -25 * see  # half of fp16's smallest step
    if dtype == torch.bfloat16:
        eds = eds + 2.0 ** -134 * see
    dq = scale * _masked_product(ds, kd, see)
    tdq = scale * _masked_product(eds + ds.abs() * nk * E, kd.abs(), see) + 2 * u * dq.abs()
    dk = scale * few(_masked_product(ds.transpose(2, 3), qd, see.transpose(2, 3)))
    tdk = scale * few(_masked_product((eds + ds.abs() * n * E).transpose(2, 3), qd.abs(), see.transpose(2, 3)))
    tdk = tdk + 2 * u * dk.abs()
    found.update(dq=(back(dq), back(tdq + tiny)), dk=(back(dk), back(tdk + tiny)), dv=(back(dv), back(tdv + tiny)))
    return found


def _masked_product(a, x, see):
    """sum_j a_ij x_j over the j that i sees: what it does not see may be inf or NaN."""
    if torch.isfinite(x).all() and torch.isfinite(a).all():
        return a @ x
    out = torch.zeros((*torch.broadcast_shapes(a.shape[:2], x.shape[:2]), a.shape[2], x.shape[3]), dtype=a.dtype)
    a = a.expand(*out.shape[:2], *a.shape[2:])
    for i in range(a.shape[2]):
        seen = see[:, :, i, :, None].expand(*out.shape[:2], -1, 1)
        out[:, :, i] = torch.where(seen, a[:, :, i, :, None] * x, torch.zeros_like(x[..., :1])).sum(2)
    return out


def frequencies(sections, theta):
    return torch.tensor([theta ** (-j / n) for n in sections for j in range(n)], dtype=torch.float64)


def norm_rotary(x, positions, sections, weight=None, eps=None, theta=10000.0, freq=None, interleaved=False, dy=None):
    """{"y": (value, tolerance)} of one side's heads, and with `dy` "dx" and "dw" too.

    Errors.  The angle's cosine and sine are off by a few E; a norm's sum of squares by d E, its root by d E / 2, and
    a few operations more: e = (d / 2 + 12) E of the sizes of the two terms of a turn.
    """
    dtype = x.dtype
    x = x.detach().cpu().double()
    b, n, h, d = x.shape
    freq = frequencies(sections, theta) if freq is None else freq.detach().cpu().double()
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    pos = positions.detach().cpu().double().expand(b, n, len(sections))
    angle = (pos[..., axis] * freq)[:, :, None]
    c, z = torch.cos(angle), torch.sin(angle)
    half = d // 2
    first, second = (slice(0, d, 2), slice(1, d, 2)) if interleaved else (slice(0, half), slice(half, d))

    def turn(t, c, z):
        y = torch.empty_like(t)
        y[..., first] = t[..., first] * c - t[..., second] * z
        y[..., second] = t[..., second] * c + t[..., first] * z
        return y

    size = lambda t: _both(t.abs(), c.abs(), z.abs(), first, second)  # noqa: E731
    u, e = half_step(dtype), (d / 2 + 12) * E
    w = torch.ones(d, dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    r = 1.0 if eps is None else 1.0 / torch.sqrt(x.square().mean(3, keepdim=True) + eps)
    y = turn(x * r * w, c, z)
    tiny = torch.finfo(dtype).tiny * u * 2
    found = {"y": (y, u * y.abs() + e * size(x * r * w) + tiny)}
    if dy is None:
        return found
    dy = dy.detach().cpu().double()
    g = turn(dy, c, -z)
    eg = e * size(dy)
    if eps is None:
        found["dx"] = g, u * g.abs() + eg + tiny
        return found
    xr = x * r
    dw = (g * xr).sum((0, 1, 2))
    rows = b * n * h
    wtype = dtype if weight is None else weight.dtype
    found["dw"] = dw, half_step(wtype) * dw.abs() + ((eg * xr.abs() + (e + rows * E) * (g * xr).abs()).sum((0, 1, 2)))
    hg = g * w
    mean = (hg * xr).mean(3, keepdim=True)
    dx = r * (hg - xr * mean)
    emean = (eg * w.abs() * xr.abs() + 2 * e * (hg * xr).abs()).mean(3, keepdim=True) + e * (hg * xr).abs().mean(3, keepdim=True)
    found["dx"] = dx, u * dx.abs() + r * (eg * w.abs() + 2 * e * (hg.abs() + (xr * mean).abs()) + xr.abs() * emean) + tiny
    return found


def _both(t, c, z, first, second):
    """|a| |cos| + |b| |sin| of each pair, in both places."""
    y = torch.empty_like(t)
    y[..., first] = t[..., first] * c + t[..., second] * z
    y[..., second] = t[..., second] * c + t[..., first] * z
    return y

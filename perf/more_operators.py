"""The operators of a tower's attention whose speed is measured: the rotation of
queries and keys by positions on several axes, with the norm of each head in the
same pass, and attention itself, each with its gradient.

A case is a dict of plain values:

  op         "attend" (no gradient), "attend_train", "rotary" (no gradient), "rotary_train"
  batch      texts, images or clips of a call
  queries    tokens of each that ask
  keys       tokens of each that are looked at
  heads, key_heads   heads of the queries, and of the keys and values (shared by heads / key_heads of the former)
  dim        features of a head
  dtype      "f32", "bf16", "f16"
  causal     a token looks at itself and at what precedes it (the last query at the last key)
  fill       lengths lie between this share of the keys and all of them (1: all full); with as many queries as
             keys the queries have the same lengths
  fused      queries, keys and values are slices of one projection's output
  axes       rotary: positions a token has: 1 (texts), 2 (images), 3 (clips)
  norm       rotary: the heads are normed first
  far        rotary: the first position on the first axis

With ``own`` false every operator is computed in its plain form, in elementary
torch operations in 32 bits (the angles in 64), rounded once at the end; with
``own`` true by this package.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_THETA = 10000.0
_EPS = 1e-6
_ROTARY_OUT = ("q", "k", "dq", "dk", "dwq", "dwk")


def _attend(name, op, batch, queries, keys, heads, key_heads, dim, dtype, causal=False, fill=1.0, fused=False):
    c = {"op": op, "batch": batch, "queries": queries, "keys": keys, "heads": heads, "key_heads": key_heads,
         "dim": dim, "dtype": dtype, "causal": causal, "fill": fill, "fused": fused}
    return {"name": name, **c} if name else c


def _rotary(name, op, batch, tokens, heads, key_heads, dim, dtype, axes, norm=True, far=0, fused=False):
    c = {"op": op, "batch": batch, "queries": tokens, "heads": heads, "key_heads": key_heads, "dim": dim,
         "dtype": dtype, "axes": axes, "norm": norm, "far": far, "fused": fused}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one caption being generated: latency
        _attend("attend_bf16_1x1x300_12h64", "attend", 1, 1, 300, 12, 12, 64, "bf16"),
        # a batch of long texts being generated, of different lengths, heads sharing keys and values
        _attend("attend_bf16_16x1x32768_32h8_128", "attend", 16, 1, 32768, 32, 8, 128, "bf16", causal=True, fill=0.5),
        # images of 27 x 27 patches are embedded; 1152 features in 16 heads
        _attend("attend_f16_64x729_16h72", "attend", 64, 729, 729, 16, 16, 72, "f16", fused=True),
        # a small debugging batch in fp32 with sizes that no tile divides; a head of 40
        _attend("attend_train_f32_3x333_6h40", "attend_train", 3, 333, 333, 6, 6, 40, "f32", causal=True, fill=0.6),
        # the texts of a contrastive batch, padded to 77 tokens
        _attend("attend_train_bf16_1024x77_12h64", "attend_train", 1024, 77, 77, 12, 12, 64, "bf16", causal=True,
                fill=0.1, fused=True),
        # the images of a contrastive batch: 256 patches and a token for the whole
        _attend("attend_train_bf16_256x257_12h64", "attend_train", 256, 257, 257, 12, 12, 64, "bf16", fused=True),
        # one learned query looks at all patches of an image and pools them
        _attend("attend_train_f16_256x1x729_16h72", "attend_train", 256, 1, 729, 16, 16, 72, "f16"),
        # a long document
        _attend("attend_train_bf16_1x16384_16h4_128", "attend_train", 1, 16384, 16384, 16, 4, 128, "bf16", causal=True),
        # the next token of each of 32 texts
        _rotary("rotary_bf16_32x1_32h8_128", "rotary", 32, 1, 32, 8, 128, "bf16", 1, far=100000),
        # odd sizes in fp32, without a norm
        _rotary("rotary_train_f32_5x317_6h6_36", "rotary_train", 5, 317, 6, 6, 36, "f32", 2, norm=False),
        # the images of a batch, 32 x 32 patches
        _rotary("rotary_train_bf16_128x1024_12h12_64", "rotary_train", 128, 1024, 12, 12, 64, "bf16", 2, fused=True),
        # clips: the largest
        _rotary("rotary_train_bf16_4x32768_20h20_128", "rotary_train", 4, 32768, 20, 20, 128, "bf16", 3, fused=True),
    ]


# no drawn case computes or moves more than the largest listed ones
_MOST_FLOPS, _MOST_BYTES = 3.0e12, 4.0e9


def _log_uniform(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend_train", "attend_train", "rotary", "rotary_train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    while True:
        key_heads = rng.choice([1, 2, 4, 8, 12, 16])
        heads = key_heads * rng.choice([1, 1, 1, 2, 4, 7])
        batch = _log_uniform(rng, 1, 512)
        fused = rng.random() < 0.5
        if op.startswith("rotary"):
            axes = rng.choice([1, 2, 3])
            dim = rng.choice([32, 64, 64, 72, 80, 128, 2 * rng.randint(8, 64)])
            c = _rotary(None, op, batch, rng.choice([1, _log_uniform(rng, 2, 16384)]), heads, key_heads, dim, dtype,
                        axes, norm=rng.random() < 0.7, far=rng.choice([0, 0, _log_uniform(rng, 100, 1000000)]),
                        fused=fused)
        else:
            dim = rng.choice([32, 40, 64, 64, 72, 80, 96, 128, 128, rng.randint(16, 128)])
            keys = _log_uniform(rng, 1, 16384)
            queries = rng.choice([keys, keys, 1, min(keys, _log_uniform(rng, 1, 64))])
            c = _attend(None, op, batch, queries, keys, heads, key_heads, dim, dtype, causal=rng.random() < 0.5,
                        fill=rng.choice([1.0, 0.5, 0.0]), fused=fused and queries == keys)
        w = work(c)
        f32 = 8.0 if dtype == "f32" else 1.0
        if w["flops"] * f32 < _MOST_FLOPS and w["bytes"] < _MOST_BYTES and (
                c["op"].startswith("rotary") or batch * heads * c["queries"] * c["keys"] < 4.0e9):
            return c


def _sections(dim, axes):
    """Pairs of features that each axis turns: equal shares, what is left over to the last."""
    share = dim // 2 // axes
    return [share] * (axes - 1) + [dim // 2 - share * (axes - 1)]


def _randn(shape, g, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _projected(case, g, dtype, *more):
    """Queries and keys (and values) [batch, tokens, heads, dim], as a program's projections give them."""
    b, n, h, hk, d = case["batch"], case["queries"], case["heads"], case["key_heads"], case["dim"]
    heads = [h, hk, *more]
    if case["fused"]:
        return list(_randn((b, n, sum(heads), d), g, dtype).split(heads, 2))
    keys = case.get("keys", n)
    return [_randn((b, n if i == 0 else keys, x, d), g, dtype) for i, x in enumerate(heads)]


def _positions(case):
    """Grids of an image or of a clip's frames as nearly square as they come; texts count on."""
    n, axes, far = case["queries"], case["axes"], case["far"]
    i = torch.arange(n, device="cuda")
    if axes == 1:
        return (i + far)[:, None]
    frames = 1 if axes == 2 else max(1, n // 1024)
    width = max(1, math.isqrt(max(1, n // frames)))
    height = -(-n // (frames * width))
    grid = [i // (height * width), i // width % height, i % width][3 - axes:]
    grid[0] = grid[0] + far
    return torch.stack(grid, 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, train = _DTYPES[case["dtype"]], case["op"].endswith("_train")
    state = {"case": case}
    if case["op"].startswith("rotary"):
        q, k = _projected(case, g, dtype)
        state["positions"], state["sections"] = _positions(case), _sections(case["dim"], case["axes"])
        state["weights"] = [None, None]
        if case["norm"]:
            state["weights"] = [_randn((case["dim"],), g, torch.float32, 0.1).add_(1.0).to(dtype) for _ in "qk"]
        leaves = [q, k, *(w for w in state["weights"] if w is not None)]
        if train:
            state["dy"] = [_randn(t.shape, g, dtype) for t in (q, k)]
        state.update(query=q, key=k)
    else:
        q, k, v = _projected(case, g, dtype, case["key_heads"])
        # heads that look at a few tokens more than at the others
        q.mul_(1.5)
        state["lengths"] = None
        if case["fill"] < 1:
            u = torch.rand(case["batch"], generator=g, device="cuda", dtype=torch.float64)
            share = case["fill"] + (1 - case["fill"]) * u
            state["lengths"] = (share * case["keys"]).round().int()
        leaves = [q, k, v]
        if train:
            state["dy"] = _randn(q.shape, g, dtype)
        state.update(query=q, key=k, value=v)
    if train:
        for t in leaves:
            t.requires_grad_(True)
    state["leaves"] = leaves
    return state


def _lengths(s):
    """Lengths of the queries and of the keys; None: full."""
    c = s["case"]
    return s["lengths"] if c["queries"] == c["keys"] else None, s["lengths"]


# ---- plain forms ----


def _sees(s, rows):
    """[rows, 1, 1, queries, keys]: whether a query looks at a key, for a slice of the batch."""
    c = s["case"]
    nq, nk = (torch.full((1, 1, 1), full, device="cuda") if n is None else n[rows, None, None]
              for n, full in zip(_lengths(s), (c["queries"], c["keys"])))
    i = torch.arange(c["queries"], device="cuda")[:, None]
    j = torch.arange(c["keys"], device="cuda")
    see = (i < nq) & (j < nk)
    if c["causal"]:
        see = see & (j <= i + (nk - nq))
    return see[:, None, None]


def _plain_attend(s):
    c = s["case"]
    b, nq, nk, h, hk, d = (c[x] for x in ("batch", "queries", "keys", "heads", "key_heads", "dim"))
    train, scale = c["op"] == "attend_train", 1.0 / math.sqrt(d)
    dtype = s["query"].dtype
    out = torch.empty((b, nq, h, d), device="cuda", dtype=dtype)
    grads = [torch.empty(t.shape, device="cuda", dtype=dtype) for t in s["leaves"]] if train else []
    # parts of the batch, and of the heads, whose scores fit well into memory
    most = 1 << 30
    rows = max(1, min(b, most // (h * nq * nk)))
    some = hk if rows > 1 else max(1, min(hk, most // (h // hk * nq * nk)))
    group = h // hk
    for r in range(0, b, rows):
        at = slice(r, min(b, r + rows))
        see = _sees(s, at)
        for first in range(0, hk, some):
            kh = slice(first, min(hk, first + some))
            qh = slice(first * group, kh.stop * group)

            def by_head(t, heads, groups):
                t = t.detach()[at, :, heads].float().transpose(1, 2)
                return t.reshape(t.shape[0], -1, groups, *t.shape[2:]).contiguous()

            q, k, v = by_head(s["query"], qh, group), by_head(s["key"], kh, 1), by_head(s["value"], kh, 1)
            x = torch.matmul(q, k.transpose(-1, -2)) * scale
            x = torch.where(see, x, torch.full((), -math.inf, device="cuda"))
            m = x.amax(-1, keepdim=True)
            p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
            del x
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, torch.ones_like(total), total)
            o = torch.matmul(p, v)

            def put(into, heads, t):
                t = t.reshape(t.shape[0], -1, *t.shape[3:])
                into[at, :, heads] = t.transpose(1, 2).to(dtype)

            put(out, qh, o)
            if train:
                do = by_head(s["dy"], qh, group)
                dv = torch.matmul(p.transpose(-1, -2), do).sum(2, keepdim=True)
                dp = torch.matmul(do, v.transpose(-1, -2))
                ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
                del dp, p
                put(grads[0], qh, torch.matmul(ds, k))
                put(grads[1], kh, torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True))
                put(grads[2], kh, dv)
    return {"out": out, **dict(zip(("dq", "dk", "dv"), grads))}


def _angles(s):
    """cos and sin [tokens, 1, pairs], the angles in 64 bits."""
    parts = [s["positions"][:, a, None].double() * _THETA ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)
             for a, n in enumerate(s["sections"])]
    angle = torch.cat(parts, 1)[:, None]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _turn(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_rotary(s):
    cos, sin = _angles(s)
    out = {}
    for i, (name, x, w) in enumerate(zip("qk", (s["query"], s["key"]), s["weights"])):
        dtype, x = x.dtype, x.detach().float()
        norm = w is not None
        if norm:
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
            x, wf = x * r, w.detach().float()
        out[name] = _turn(x * wf if norm else x, cos, sin).to(dtype)
        if "dy" in s:
            dx = _turn(s["dy"][i].float(), cos, -sin)
            if norm:
                out["dw" + name] = (dx * x).sum((0, 1, 2)).to(dtype)
                dx = dx * wf
                dx = r * (dx - x * (dx * x).mean(-1, keepdim=True))
            out["d" + name] = dx.to(dtype)
    return {n: out[n] for n in _ROTARY_OUT if n in out}


# ---- the framework's operators ----


def _own(s):
    import memoryefficientclip_amd as mec

    c = s["case"]
    train = c["op"].endswith("_train")
    for t in s["leaves"]:
        t.grad = None
    if c["op"].startswith("rotary"):
        with torch.set_grad_enabled(train):
            q, k = mec.norm_rotary(s["query"], s["key"], s["positions"], s["sections"], *s["weights"],
                                   eps=_EPS if c["norm"] else None, theta=_THETA)
        out = {"q": q.detach(), "k": k.detach()}
        if train:
            torch.autograd.backward([q, k], s["dy"])
            out.update(dq=s["query"].grad, dk=s["key"].grad)
            if c["norm"]:
                out.update(dwq=s["weights"][0].grad, dwk=s["weights"][1].grad)
        return out
    query_lengths, key_lengths = _lengths(s)
    with torch.set_grad_enabled(train):
        o = mec.attention(s["query"], s["key"], s["value"], causal=c["causal"], query_lengths=query_lengths,
                          key_lengths=key_lengths)
    if not train:
        return {"out": o}
    o.backward(s["dy"])
    return {"out": o.detach(), "dq": s["query"].grad, "dk": s["key"].grad, "dv": s["value"].grad}


def run(state):
    if own:
        return _own(state)
    return _plain_rotary(state) if state["case"]["op"].startswith("rotary") else _plain_attend(state)


def work(case):
    """Each input read once and each output written once; tokens beyond the lengths need no read, and pairs of
    tokens that do not see one another no products."""
    b, nq, h, hk, d, size = (*(case[x] for x in ("batch", "queries", "heads", "key_heads", "dim")),
                             _SIZE[case["dtype"]])
    train = case["op"].endswith("_train")
    if case["op"].startswith("rotary"):
        x = b * nq * (h + hk) * d
        w = 2 * d * size if case["norm"] else 0
        n = 2 * x * size + w + 8 * nq * case["axes"]
        f = (7.0 if case["norm"] else 3.0) * x
        if train:
            # the gradients; a norm's need the inputs, which were read for the results
            n += 2 * x * size + w
            f += (14.0 if case["norm"] else 3.0) * x
        return {"bytes": float(n), "flops": f}
    nk, fill = case["keys"], case["fill"]
    mean = (1.0 + fill) / 2
    if nq == nk:
        square = (1.0 + fill + fill * fill) / 3
        pairs = nq * nk * square / 2 + nq * mean / 2 if case["causal"] else nq * nk * square
        asked = nq * mean
    else:
        pairs = nq * nk * mean - (nq * (nq - 1) / 2 if case["causal"] else 0.0)
        asked = nq
    seen = nk * mean
    # read: what the lengths leave; written: everything
    n = b * d * size * (asked * h + 2 * seen * hk + nq * h)
    f = 4.0 * b * h * d * pairs
    if train:
        n += b * d * size * (asked * h + nq * h + 2 * nk * hk)
        f += 8.0 * b * h * d * pairs
    return {"bytes": float(n), "flops": float(max(f, 0.0))}


# ---- the definitions in 64 bits ----


def _exact_attend(case, seed):
    s = prepare(case, seed)
    b, h, hk, nq, nk = (case[x] for x in ("batch", "heads", "key_heads", "queries", "keys"))
    train = case["op"] == "attend_train"
    results = []
    nql, nkl = _lengths(s)
    step = max(1, min(b, (1 << 28) // (h // hk * nq * nk)))
    kpos, qpos = torch.arange(nk, device="cuda"), torch.arange(nq, device="cuda")
    for r in range(0, b, step):
        end = min(b, r + step)
        lk = nkl[r:end].long() if nkl is not None else torch.full((end - r,), nk, device="cuda")
        lq = nql[r:end].long() if nql is not None else torch.full((end - r,), nq, device="cuda")
        hidden = (kpos >= lk[:, None])[:, None, :] | (qpos >= lq[:, None])[:, :, None]
        if case["causal"]:
            hidden = hidden | (kpos[None, None] - (lk - lq)[:, None, None] > qpos[None, :, None])
        hidden = hidden[:, None]
        per_head = []
        for j in range(hk):
            heads = slice(j * (h // hk), (j + 1) * (h // hk))
            q = s["query"].detach()[r:end, :, heads].double().permute(0, 2, 1, 3).contiguous().requires_grad_(train)
            k = s["key"].detach()[r:end, :, j].double()[:, None].contiguous().requires_grad_(train)
            v = s["value"].detach()[r:end, :, j].double()[:, None].contiguous().requires_grad_(train)
            scores = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(case["dim"])
            # (rows that see nothing: any finite score, and no part in the result)
            nothing = hidden.all(3, keepdim=True)
            p = torch.softmax(scores.masked_fill(hidden & ~nothing, -math.inf), 3)
            o = torch.matmul(p.masked_fill(nothing, 0.0), v)
            found = [o.detach().permute(0, 2, 1, 3)]
            if train:
                do = s["dy"][r:end, :, heads].double().permute(0, 2, 1, 3).contiguous()
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
                found += [dq.permute(0, 2, 1, 3), dk.permute(0, 2, 1, 3), dv.permute(0, 2, 1, 3)]
            per_head.append(found)
            del scores, p, o, q, k, v
        results.append([torch.cat(t, 2) for t in zip(*per_head)])
    return dict(zip(("out", "dq", "dk", "dv"), (torch.cat(t) for t in zip(*results))))


def _exact_rotary(case, seed):
    s = prepare(case, seed)
    pos = s["positions"].double()
    turns = []
    for a, n in enumerate(s["sections"]):
        for j in range(n):
            turns.append(pos[:, a] * math.exp(-math.log(_THETA) * j / n))
    spin = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), torch.stack(turns, 1))[:, None]
    half = case["dim"] // 2
    out = {}
    for i, (name, x, w) in enumerate(zip("qk", (s["query"], s["key"]), s["weights"])):
        parts = []
        dw = 0.0
        for r in range(0, x.shape[0], max(1, (1 << 25) // x[0].numel())):
            at = slice(r, r + max(1, (1 << 25) // x[0].numel()))
            xd = x.detach()[at].double().requires_grad_(True)
            y = xd
            wd = None
            if w is not None:
                wd = w.detach().double().requires_grad_(True)
                y = y * wd / torch.sqrt(y.square().mean(3, keepdim=True) + _EPS)
            z = torch.complex(y[..., :half], y[..., half:]) * spin
            y = torch.cat([z.real, z.imag], 3)
            found = [y.detach()]
            if "dy" in s:
                grads = torch.autograd.grad(y, [xd] if wd is None else [xd, wd], s["dy"][i][at].double())
                found.append(grads[0])
                if wd is not None:
                    dw = dw + grads[1]
            parts.append(found)
        whole = [torch.cat(t) for t in zip(*parts)]
        out[name] = whole[0]
        if "dy" in s:
            if w is not None:
                out["dw" + name] = dw
            out["d" + name] = whole[1]
    return {n: out[n] for n in _ROTARY_OUT if n in out}


def exact(case, seed):
    return _exact_rotary(case, seed) if case["op"].startswith("rotary") else _exact_attend(case, seed)
